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
