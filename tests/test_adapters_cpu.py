"""Adapters around the operators, on the CPU: the module's slots, the adapter directories, the shards, FP8 experts from a checkpoint."""

import json
from types import SimpleNamespace

import pytest
import torch
from safetensors.torch import save_file

from emmy_b200 import linear, loader, ops, shard
from tests.test_loader_cpu import write_checkpoint


def write_adapter(path, tensors, **config):
    path.mkdir(parents=True, exist_ok=True)
    (path / "adapter_config.json").write_text(json.dumps({"peft_type": "LORA", "r": 4, "lora_alpha": 8, "bias": "none", **config}))
    save_file({k: v.clone().contiguous() for k, v in tensors.items()}, str(path / "adapter_model.safetensors"))


def pair(module, r, k, n, seed, prefix="base_model.model."):
    g = torch.Generator().manual_seed(seed)
    return {f"{prefix}{module}.lora_A.weight": torch.randn(r, k, generator=g), f"{prefix}{module}.lora_B.weight": torch.randn(n, r, generator=g)}


def lora(k=16, n=24, slots=2, rank=6, sections=None, dtype=torch.bfloat16):
    return linear.LoRALinear(torch.nn.Linear(k, n, bias=False), slots, rank, dtype, sections)


def test_slots_hold_padded_adapters_and_are_cleared():
    m = lora(sections=(8, 16))
    assert m.rank == 8 and tuple(m.lora_a.shape) == (2, 2, 8, 16) and tuple(m.lora_b.shape) == (2, 24, 8) and not set(m.state_dict()) - {"base.weight"}
    buffers = m.lora_a.data_ptr(), m.lora_b.data_ptr(), m.scaling.data_ptr()
    a, b = torch.randn(3, 16), torch.randn(16, 3)
    m.load_adapter(1, [None, a], [None, b], 0.3)
    assert buffers == (m.lora_a.data_ptr(), m.lora_b.data_ptr(), m.scaling.data_ptr())
    assert m.scaling.tolist() == [0.0, torch.tensor(0.3).item()]
    assert torch.equal(m.lora_a[1, 1, :3], a.bfloat16()) and torch.equal(m.lora_b[1, 8:, :3], b.bfloat16())
    rest = m.lora_a.clone(), m.lora_b.clone()
    rest[0][1, 1, :3], rest[1][1, 8:, :3] = 0, 0
    assert not rest[0].any() and not rest[1].any()
    m.load_adapter(1, [torch.randn(6, 16), None], [torch.randn(8, 6), None], 1.0)  # nothing of the one before stays
    assert not m.lora_a[1, 1].any() and not m.lora_b[1, 8:].any()
    m.clear_adapter(1)
    assert not m.lora_a.any() and not m.lora_b.any() and not m.scaling.any()


def test_slots_refuse_what_does_not_fit():
    m = lora(sections=(8, 16))
    ok = dict(slot=0, a=[torch.zeros(3, 16), None], b=[torch.zeros(8, 3), None])
    m.check_adapter(**ok)
    for bad in (dict(slot=2), dict(slot=-1), dict(a=[torch.zeros(3, 16)]), dict(b=[None, None]), dict(a=[torch.zeros(9, 16), None], b=[torch.zeros(8, 9), None]),
                dict(a=[torch.zeros(3, 8), None]), dict(b=[torch.zeros(16, 3), None]), dict(b=[torch.zeros(8, 4), None])):
        with pytest.raises(ValueError):
            m.check_adapter(**{**ok, **bad})
    for bad in (dict(slots=0), dict(rank=0), dict(sections=(8, 8)), dict(dtype=torch.float32), dict(slots=4097), dict(rank=1025), dict(rank=505, sections=(8, 8, 8)), dict(k=12),
                dict(n=20), dict(sections=(12, 12)), dict(n=72, sections=(8,) * 9), dict(sections=(24, 8, -8))):
        with pytest.raises(ValueError):
            lora(**bad)


def test_scales_stay_f32_when_the_module_changes_type():
    m = lora(dtype=torch.float16)
    m.scaling[0] = 0.3
    m.to(torch.bfloat16)
    assert m.scaling.dtype == torch.float32 and m.scaling[0] == torch.tensor(0.3) and m.lora_a.dtype == torch.bfloat16
    z = torch.zeros(2, 256, 128, dtype=torch.uint8)
    q = linear.QuantMoE(1).load_fp8_experts(z, torch.full((2, 256), 0.3), z[:, :128].contiguous(), torch.full((2, 128), 0.7))
    q.half()
    assert q.gate_up_scale.dtype == q.down_scale.dtype == torch.float32 and q.gate_up_scale[0, 0] == torch.tensor(0.3) and q.packed_gate_up.dtype == torch.uint8


def test_fp8_experts_refuse_what_does_not_fit():
    z = torch.zeros(2, 256, 128, dtype=torch.uint8)
    d, s = z[:, :128].contiguous(), (torch.ones(2, 256), torch.ones(2, 128))
    for bad in ((z, s[0], z, s[1]), (z[:, :192], s[0], d, s[1]), (z, s[1], d, s[1]), (z, torch.ones(2, 2, 1), d, s[1]), (z, torch.ones(2, 1, 1), d, torch.ones(2, 1, 1)),
                (z.view(torch.float8_e5m2), s[0], d, s[1]), (z, s[0], d.view(torch.int8), s[1])):
        with pytest.raises(ValueError):
            linear.QuantMoE(1).load_fp8_experts(*bad)
    linear.QuantMoE(1).load_fp8_experts(z, torch.ones(2, 2, 1), d, torch.ones(2, 1, 1))


def test_adapter_directories(tmp_path):
    t = {**pair("model.layers.0.self_attn.q_proj", 4, 16, 8, 1), **pair("model.layers.0.self_attn.v_proj", 4, 16, 8, 2), **pair("model.layers.0.mlp.down_proj", 2, 24, 16, 3)}
    write_adapter(tmp_path / "a", t, alpha_pattern={"down_proj": 3})
    got = loader.read_adapter(tmp_path / "a")
    assert {k: v[2] for k, v in got.items()} == {"model.layers.0.self_attn.q_proj": 2.0, "model.layers.0.self_attn.v_proj": 2.0, "model.layers.0.mlp.down_proj": 1.5}
    assert torch.equal(got["model.layers.0.mlp.down_proj"][0], t["base_model.model.model.layers.0.mlp.down_proj.lora_A.weight"])
    write_adapter(tmp_path / "rs", t, use_rslora=True)
    assert loader.read_adapter(tmp_path / "rs")["model.layers.0.self_attn.q_proj"][2] == 4.0
    # a fused projection: the k section is left alone; a module that the adapter does not touch loses the slot's adapter
    qkv, down, other = lora(16, 24, sections=(8, 8, 8)), lora(24, 16), lora()
    other.load_adapter(1, torch.ones(2, 16), torch.ones(24, 2), 1.0)
    at = "model.layers.0.self_attn."
    modules = {(at + "q_proj", at + "k_proj", at + "v_proj"): qkv, "model.layers.0.mlp.down_proj": down, "model.layers.1.mlp.down_proj": other}
    loader.load_adapter(tmp_path / "a", modules, 1)
    assert qkv.scaling[1] == 2.0 and down.scaling[1] == 1.5 and not other.lora_a.any() and not other.scaling.any() and not qkv.lora_b[1, 8:16].any()
    assert torch.equal(qkv.lora_b[1, 16:, :4], t[f"base_model.model.{at}v_proj.lora_B.weight"].bfloat16())
    # sections of different scalings: the product stays what it is
    write_adapter(tmp_path / "mixed", t, alpha_pattern={"v_proj": 16})
    loader.load_adapter(tmp_path / "mixed", modules, 0)
    assert qkv.scaling[0] == 2.0 and torch.equal(qkv.lora_b[0, 16:, :4], (2 * t[f"base_model.model.{at}v_proj.lora_B.weight"]).bfloat16())


def test_adapter_directories_that_are_refused(tmp_path):
    t = pair("m.q_proj", 4, 16, 24, 1)
    for i, bad in enumerate((dict(bias="all"), dict(use_dora=True), dict(fan_in_fan_out=True), dict(modules_to_save=["lm_head"]), dict(layer_replication=[[0, 2]]), dict(peft_type="IA3"))):
        write_adapter(tmp_path / f"c{i}", t, **bad)
        with pytest.raises(ValueError):
            loader.read_adapter(tmp_path / f"c{i}")
    a, b = t.values()
    for i, bad in enumerate(({"base_model.model.m.q_proj.lora_A.weight": a}, {**t, "base_model.model.m.lora_embedding_A": a}, {**t, "base_model.model.m.q_proj.lora_magnitude_vector": a[0]},
                             {"m.q_proj.lora_A.weight": a, "m.q_proj.lora_B.weight": b[:, :3]})):
        write_adapter(tmp_path / f"t{i}", bad)
        with pytest.raises(ValueError):
            loader.read_adapter(tmp_path / f"t{i}")
    write_adapter(tmp_path / "ok", t)
    m, before = lora(), lora().lora_a
    for modules, slot in (({"m.k_proj": m}, 0), ({"m.q_proj": m}, 2), ({"m.q_proj": lora(rank=8, n=32)}, 0), ({("m.q_proj", "m.k_proj"): m}, 0)):
        with pytest.raises(ValueError):
            loader.load_adapter(tmp_path / "ok", modules, slot)
    assert torch.equal(m.lora_a, before)


def fp8(n, k, seed, scale):
    bits = torch.randint(0, 120, (n, k), generator=torch.Generator().manual_seed(seed), dtype=torch.uint8)
    return bits.view(torch.float8_e4m3fn), scale


def expert_tensors(e, h, i, kind):
    """per-expert modules of a layer; scales per tensor, per channel or per block"""
    t = {}
    for x in range(e):
        for j, (name, n, k) in enumerate((("gate_proj", i, h), ("up_proj", i, h), ("down_proj", h, i))):
            g = torch.Generator().manual_seed(100 * x + j)
            shape = {"tensor": (), "channel": (n, 1), "block": (n // 128, k // 128)}[kind]
            w, s = fp8(n, k, 7 * x + j, torch.rand(shape, generator=g) + 0.5)
            t[f"m.experts.{x}.{name}.weight"], t[f"m.experts.{x}.{name}.weight_scale"] = w, s
    return t


@pytest.mark.parametrize("kind", ["tensor", "channel", "block"])
def test_fp8_experts_are_stacked(tmp_path, kind):
    e, h, i = 3, 256, 128
    t = expert_tensors(e, h, i, kind)
    write_checkpoint(tmp_path, t, {"quant_method": "fp8"})
    index = loader.CheckpointIndex(tmp_path)
    gate_up, gate_up_scale, down, down_scale = loader.stack_fp8_experts(index, loader.scan_experts(loader.scan(tmp_path, index))["m.experts"])
    assert tuple(gate_up.shape) == (e, 2 * i, h) and tuple(down.shape) == (e, h, i)
    assert tuple(gate_up_scale.shape) == ((e, 2 * i // 128, h // 128) if kind == "block" else (e, 2 * i)) and gate_up_scale.dtype == torch.float32
    for x in range(e):
        for name, bits, scale in (("gate_proj", gate_up[x, :i], gate_up_scale[x][: i // (128 if kind == "block" else 1)]),
                                  ("up_proj", gate_up[x, i:], gate_up_scale[x][i // (128 if kind == "block" else 1) :]), ("down_proj", down[x], down_scale[x])):
            assert torch.equal(bits, t[f"m.experts.{x}.{name}.weight"].view(torch.uint8))
            want = t[f"m.experts.{x}.{name}.weight_scale"]
            assert torch.equal(scale, want if kind == "block" else want.reshape(-1).expand(bits.shape[0]))
    linear.QuantMoE(1).load_fp8_experts(gate_up, gate_up_scale, down, down_scale)


def test_fp8_experts_fused_and_refused(tmp_path):
    e, h, i = 2, 128, 128
    t = {}
    for x in range(e):
        t[f"m.experts.{x}.gate_up_proj.weight"], t[f"m.experts.{x}.gate_up_proj.weight_scale"] = fp8(2 * i, h, x, torch.rand(2 * i))
        t[f"m.experts.{x}.down_proj.weight"], t[f"m.experts.{x}.down_proj.weight_scale"] = fp8(h, i, 9 + x, torch.rand(h))
    write_checkpoint(tmp_path / "fused", t, {"quant_method": "fp8"})
    index = loader.CheckpointIndex(tmp_path / "fused")
    experts = loader.scan_experts(loader.scan(tmp_path / "fused", index))["m.experts"]
    plain, apart = loader.stack_fp8_experts(index, experts), loader.stack_fp8_experts(index, experts, interleaved_gate_up=True)
    for x in range(e):
        w, s = t[f"m.experts.{x}.gate_up_proj.weight"].view(torch.uint8), t[f"m.experts.{x}.gate_up_proj.weight_scale"]
        assert torch.equal(plain[0][x], w) and torch.equal(apart[0][x, :i], w[0::2]) and torch.equal(apart[1][x, i:], s[1::2])
    # interleaved rows of block scales, other blocks, a missing projection, a gap
    block = {}
    for x in range(e):
        block[f"m.experts.{x}.gate_up_proj.weight"], block[f"m.experts.{x}.gate_up_proj.weight_scale"] = fp8(2 * i, h, x, torch.rand(2, 1))
        block[f"m.experts.{x}.down_proj.weight"], block[f"m.experts.{x}.down_proj.weight_scale"] = fp8(h, i, 9 + x, torch.rand(1, 1))
    write_checkpoint(tmp_path / "block", block, {"quant_method": "fp8"})
    index = loader.CheckpointIndex(tmp_path / "block")
    groups = loader.scan_experts(loader.scan(tmp_path / "block", index))["m.experts"]
    with pytest.raises(ValueError, match="alternate"):
        loader.stack_fp8_experts(index, groups, interleaved_gate_up=True)
    with pytest.raises(ValueError, match="no down"):
        loader.stack_fp8_experts(index, {0: {"gate_up": groups[0]["gate_up"]}})
    with pytest.raises(ValueError, match="not 0"):
        loader.stack_fp8_experts(index, {1: groups[1]})
    groups[0]["gate_up"].block = (64, 128)
    with pytest.raises(ValueError, match="128 x 128"):
        loader.stack_fp8_experts(index, groups)


@pytest.mark.parametrize("world", [1, 2, 4])
def test_shards_add_up(world):
    g = torch.Generator().manual_seed(5)
    l, s, r, k, sections = 2, 3, 4, 64, (64, 32, 32)
    a, b, x = torch.randn(l, s, r, k, generator=g), torch.randn(l, sum(sections), r, generator=g), torch.randn(k, generator=g)

    def apply(a, b, widths, x):
        y = [bb @ (a[1, i] @ x) for i, bb in enumerate(b[1].split(list(widths)))]
        return y

    want = apply(a, b, sections, x)
    parts = [shard.column_slice_lora(a, b, rank, world, sections) for rank in range(world)]
    got = [apply(pa, pb, w, x) for pa, pb, w in parts]
    assert all(w == tuple(v // world for v in sections) for _, _, w in parts)
    for i in range(s):
        torch.testing.assert_close(torch.cat([y[i] for y in got]), want[i])
    total = sum(torch.cat(apply(*shard.row_slice_lora(a, b, rank, world), sections, x[rank * k // world : (rank + 1) * k // world])) for rank in range(world))
    torch.testing.assert_close(total, torch.cat(want), atol=1e-4, rtol=1e-4)
    with pytest.raises(ValueError):
        shard.column_slice_lora(a, b, 0, 8, sections)


def test_tensors_of_another_device_are_refused(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    tensor = lambda device: SimpleNamespace(is_cuda=True, is_contiguous=lambda: True, get_device=lambda: device)
    ops._need_here(tensor(1), None, tensor(1))
    with pytest.raises(ValueError, match="cuda:0"):
        ops._need_here(tensor(1), tensor(0))
