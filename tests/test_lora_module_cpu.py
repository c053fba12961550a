"""LoRALinear and QuantMoE as modules, on the CPU: what loading and moving do to their buffers."""

import torch

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
