"""Adapter directories, on the CPU: what their configuration says beside the tensors."""

import pytest
import torch

from emmy_b200 import loader
from tests.test_adapters_cpu import lora, pair, write_adapter

MODULE = "m.q_proj"


def tensors(r=4):
    return pair(MODULE, r, 16, 24, 1)


@pytest.mark.parametrize("how", ["pissa", "pissa_niter_16", "olora", "corda", "loftq", "lora_ga", "anything_new"])
def test_adapters_that_changed_their_base_are_refused(tmp_path, how):
    write_adapter(tmp_path, tensors(), init_lora_weights=how)
    with pytest.raises(ValueError, match="init_lora_weights"):
        loader.read_adapter(tmp_path)
    m = lora()
    with pytest.raises(ValueError):
        loader.load_adapter(tmp_path, {MODULE: m}, 0)
    assert not m.lora_a.any()


@pytest.mark.parametrize("how", [None, True, False, "gaussian", "eva", "orthogonal"])
def test_adapters_that_left_their_base_alone_are_read(tmp_path, how):
    write_adapter(tmp_path, tensors(), init_lora_weights=how)
    assert loader.read_adapter(tmp_path)[MODULE][2] == 2.0


@pytest.mark.parametrize("config", [dict(alora_invocation_tokens=[5, 7]), dict(use_qalora=True), dict(lora_bias=True)], ids=str)
def test_adapters_that_are_no_plain_product_are_refused(tmp_path, config):
    """Active behind certain tokens only; A on group averages of x; a bias beside B."""
    write_adapter(tmp_path, tensors(), **config)
    with pytest.raises(ValueError, match=next(iter(config))):
        loader.read_adapter(tmp_path)


def test_the_same_keys_at_rest(tmp_path):
    write_adapter(tmp_path, tensors(), alora_invocation_tokens=None, use_qalora=False, lora_bias=False)
    a, b, scaling = loader.read_adapter(tmp_path)[MODULE]
    assert scaling == 2.0 and torch.equal(a, tensors()[f"base_model.model.{MODULE}.lora_A.weight"])


@pytest.mark.parametrize("r", [2, 4, 16])
def test_a_missing_alpha_is_the_formats_default(tmp_path, r):
    write_adapter(tmp_path, tensors(r))
    config = tmp_path / "adapter_config.json"
    config.write_text(config.read_text().replace('"lora_alpha": 8, ', ""))
    assert "lora_alpha" not in config.read_text() and loader.read_adapter(tmp_path)[MODULE][2] == 8 / r


def test_a_directory_without_tensors_is_refused(tmp_path):
    """As of an adapter that was saved in another format: its slot would be cleared and the base served in its place."""
    write_adapter(tmp_path, tensors())
    m = lora()
    loader.load_adapter(tmp_path, {MODULE: m}, 0)
    held = m.lora_a.clone()
    (tmp_path / "adapter_model.safetensors").rename(tmp_path / "adapter_model.bin")
    with pytest.raises(ValueError, match="no adapter tensors"):
        loader.load_adapter(tmp_path, {MODULE: m}, 0)
    assert held.any() and torch.equal(m.lora_a, held)
