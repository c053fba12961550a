"""The FP8 expert layer on prompts: against the formula in 64 bits, and the memory that a call takes."""

import pytest
import torch

from tests import test_gpu_moe_w8 as tm

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("t,e,topk,h,i,block", [(2048, 8, 2, 256, 256, True), (2049, 8, 2, 256, 256, False), (5000, 20, 3, 384, 128, True)])
def test_prompts_match_the_formula(t, e, topk, h, i, block, dtype):
    w, values = tm.experts(e, h, i, block, seed=t)
    x, logits = tm.inputs(t, e, h, dtype, seed=t)
    got = tm.call(x, logits, w, topk)
    tm.close(got, x, logits, values, topk)
    again = x.clone()
    assert tm.call(again, logits, w, topk, out=again) is again and torch.equal(again, got)


def test_scratch_does_not_grow_with_the_prompt():
    from emmy_b200 import lib as L
    from emmy_b200 import linear

    e, topk, h, i = 8, 4, 256, 512
    w, _ = tm.experts(e, h, i, True, seed=1)
    moe = linear.QuantMoE(topk).load_fp8_experts(*w)
    need = [L.load().eq_moe_w8a16_workspace_bytes(t, e, topk, h, i) for t in (2048, 4096)]
    assert need[1] > 1.9 * need[0]
    for t in (2048, 4096, 10000):
        x, logits = tm.inputs(t, e, h, BF16, seed=t)
        with torch.no_grad():
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            y = moe(x, logits)
            took = torch.cuda.max_memory_allocated() - before - y.numel() * 2
        assert took <= need[0] + (1 << 21), t  # (the allocator hands out whole 2 MiB: 43180544 bytes are 21 of them)
    # a workspace of the caller's is for all tokens at once
    ws = torch.empty(need[1], dtype=torch.uint8, device="cuda")
    x, logits = tm.inputs(4096, e, h, BF16, seed=4096)
    whole = tm.call(x, logits, w, topk, workspace=ws)
    assert (whole.double() - moe(x, logits).double()).abs().max() <= 2.0**-7 * whole.abs().max()
    with pytest.raises(RuntimeError, match="EQ_ERR_WORKSPACE"):
        tm.call(x, logits, w, topk, workspace=ws[: need[0]])


def test_a_prompt_in_pieces_captured():
    e, topk, h, i, t = 8, 2, 256, 256, 4500
    w, _ = tm.experts(e, h, i, True, seed=2)
    first, second = tm.inputs(t, e, h, BF16, seed=1), tm.inputs(t, e, h, BF16, seed=2)
    want = [tm.call(*v, w, topk) for v in (first, second)]
    held = [v.clone() for v in first]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tm.call(*held, w, topk)
    for args, ref in ((second, want[1]), (first, want[0])):
        for v, a in zip(held, args):
            v.copy_(a)
        graph.replay()
        assert torch.equal(y, ref)


def test_a_result_that_overlaps_its_input():
    """As it was before prompts came in pieces: rows of the result on other rows of x."""
    e, topk, h, i, t = 8, 2, 256, 256, 5000
    w, _ = tm.experts(e, h, i, True, seed=3)
    x, logits = tm.inputs(t, e, h, BF16, seed=3)
    ws = torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    want = tm.call(x, logits, w, topk, workspace=ws)
    for shift in (-1000, 1000):
        both = torch.zeros(t + 2000, h, dtype=BF16, device="cuda")
        held, out = both[1000 : 1000 + t], both[1000 + shift : 1000 + shift + t]
        held.copy_(x)
        assert torch.equal(tm.call(held, logits, w, topk, out=out), want)
