"""LoRALinear and QuantMoE as modules, on the CPU: what loading and moving do to their buffers."""

import torch

from emmy_b200 import linear
from tests.test_adapters_cpu import lora


def test_slots_take_trained_parameters_and_stay_buffers():
    """Adapters straight from a model in training: the slots hold their values and no part of their graph."""
    m = lora(sections=(8, 16))
    a, b = torch.nn.Parameter(torch.randn(4, 16)), torch.nn.Parameter(torch.randn(16, 4))
    scaling = torch.nn.Parameter(torch.tensor(0.5))
    for _ in range(2):
        m.load_adapter(1, [None, a * 2], [None, b], scaling)
        assert not any(t.requires_grad or t.grad_fn for t in (m.lora_a, m.lora_b, m.scaling))
        assert torch.equal(m.lora_a[1, 1, :4], (a * 2).bfloat16()) and torch.equal(m.lora_b[1, 8:, :4], b.bfloat16()) and m.scaling[1] == 0.5
    m.clear_adapter(1)
    assert not m.lora_a.any() and not m.scaling.any()


def test_modules_built_without_storage():
    """On the meta device, then given memory: f32 stays f32, the slots are empty; and to the meta device and back to types."""
    with torch.device("meta"):
        m = lora(sections=(8, 16))
        z = torch.empty(2, 256, 128, dtype=torch.uint8)
        q = linear.QuantMoE(1).load_fp8_experts(z, torch.empty(2, 256), torch.empty(2, 128, 128, dtype=torch.uint8), torch.empty(2, 128))
    assert m.lora_a.is_meta and q.gate_up_scale.is_meta
    m.half(), q.half()
    assert m.scaling.dtype == q.down_scale.dtype == torch.float32
    m.to_empty(device="cpu"), q.to_empty(device="cpu")
    for t in (m.lora_a, m.lora_b, m.scaling):
        assert t.device.type == "cpu" and not t.any()
    assert m.scaling.dtype == torch.float32 and m.lora_a.dtype == torch.float16
    assert q.gate_up_scale.dtype == q.down_scale.dtype == torch.float32 and q.gate_up_scale.device.type == "cpu" and q.packed_down.dtype == torch.uint8
    m.load_adapter(0, [torch.ones(2, 16), None], [torch.ones(8, 2), None], 0.3)
    m.to(torch.bfloat16)
    assert m.scaling[0] == torch.tensor(0.3) and m.lora_a[0, 0, :2].all()
    m.to("meta")
    assert m.scaling.is_meta and m.scaling.dtype == torch.float32
