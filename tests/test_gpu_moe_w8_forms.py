"""What one form of the FP8 expert layer has been shown for, shown for each of them (test_moe_w8_forms_cpu.py holds the cases to their forms)."""

import pytest
import torch

from tests import test_gpu_moe_w8 as tm

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
OWN, DOWN, WIDE = "moe_w8_down_kernel, own", "moe_w8_down_kernel", "moe_w8_down_kernel, wide"
EIGHT, SIXTEEN = "moe_w8_tiles_kernel, eight rows", "moe_w8_tiles_kernel, sixteen rows"
FORM_OF = {"own": OWN, "own, some tokens": OWN, "down": DOWN, "wide": WIDE, "eight rows": EIGHT, "many experts": EIGHT, "sixteen rows": SIXTEEN}
# form -> tokens, experts, top k, hidden, intermediate
CASES = {
    "own": (1, 16, 8, 512, 384),
    "own, some tokens": (5, 16, 3, 512, 384),
    "down": (20, 16, 4, 512, 384),
    "wide": (30, 16, 4, 512, 384),
    "eight rows": (40, 32, 4, 512, 384),
    "many experts": (6, 300, 4, 256, 128),
    "sixteen rows": (90, 16, 4, 512, 384),
}
forms = pytest.mark.parametrize("form", list(CASES))


@forms
@pytest.mark.parametrize("block", [True, False], ids=["block", "channel"])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_rows_of_every_size(form, block, dtype):
    """Rows of zeros, of one value, of very large and very small ones, of outliers beside small values; h beyond f16's range."""
    t, e, topk, h, i = CASES[form]
    w, values = tm.experts(e, h, i, block, seed=13)
    if dtype == F16:  # h is large, its result has to fit
        w, values = (w[0], w[1], w[2], w[3] * 2.0**-30), (values[0], values[1] * 2.0**-30)
    for seed in range(3):
        x, logits = tm.inputs(t, e, h, dtype, seed=seed)
        for r in range(t):
            kind = (r + seed) % 6
            if kind == 0:
                x[r] = 0
            elif kind == 1:
                x[r, 1:] = 0
            elif kind == 2:
                x[r] = (x[r].float() * (2.0**9 if dtype == F16 else 2.0**20)).to(dtype)
            elif kind == 3:
                x[r] = (x[r].float() * 2.0**-14).to(dtype)
            elif kind == 4:
                x[r, ::100] *= 2.0**8
            else:
                x[r, 7] = 2.0**12
        tm.close(tm.call(x, logits, w, topk), x, logits, values, topk)


@forms
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_tokens_do_not_reach_one_another(form, dtype):
    """NaN and infinities in tokens, in logits, in the weights of an expert that nobody picked."""
    t, e, topk, h, i = CASES[form]
    w, values = tm.experts(e, h, i, True, seed=7)
    x, logits = tm.inputs(t, e, h, dtype, seed=t)
    logits[:, -1] = -50.0
    want = tm.call(x, logits, w, topk)
    tm.close(want, x, logits, values, topk)
    w[0][-1] = 0x7F
    w[3][-1] = float("inf")
    assert torch.equal(tm.call(x, logits, w, topk), want)
    if t == 1:
        return
    x[0], x[t // 2, 9] = float("nan"), float("inf")
    got = tm.call(x, logits, w, topk)
    rest = torch.ones(t, dtype=torch.bool, device="cuda")
    rest[[0, t // 2]] = False
    assert torch.equal(got[rest], want[rest]) and got[0].isnan().all() and not torch.isfinite(got[t // 2]).any()
    logits[t - 1, 3] = float("nan")  # its picks change, and with them how the others' sums are cut
    got = tm.call(x, logits, w, topk)
    rest[t - 1] = False
    tm.close(got[rest], x[rest], logits[rest], values, topk)
    assert got[0].isnan().all() and got[t - 1].isnan().all()


@forms
def test_the_same_bits_eager_replayed_and_on_two_streams(form):
    t, e, topk, h, i = CASES[form]
    w, _ = tm.experts(e, h, i, True, seed=10)
    first, second = tm.inputs(t, e, h, BF16, seed=1), tm.inputs(t, e, h, BF16, seed=2)
    want = [tm.call(*first, w, topk), tm.call(*second, w, topk)]
    for _ in range(5):
        assert torch.equal(tm.call(*first, w, topk), want[0])
    held = [v.clone() for v in first]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tm.call(*held, w, topk)
        again = tm.call(out, held[1], w, topk)
    for args, ref in ((second, want[1]), (first, want[0])):
        for v, a in zip(held, args):
            v.copy_(a)
        for _ in range(3):
            graph.replay()
        assert torch.equal(out, ref) and torch.equal(again, tm.call(ref, args[1], w, topk))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        one = [tm.call(*first, w, topk) for _ in range(20)]
    two = [tm.call(*second, w, topk) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[0]) for o in one) and all(torch.equal(o, want[1]) for o in two)


@forms
@pytest.mark.parametrize("kind", ["one", "ties", "few", "far"])
def test_routing_at_its_borders(form, kind):
    """All tokens to the same experts; equal logits; minus infinity beside fewer experts than picks; logits far apart."""
    t, e, topk, h, i = CASES[form]
    w, values = tm.experts(e, h, i, False, seed=5)
    x, logits = tm.inputs(t, e, h, BF16, seed=t)
    if kind == "one":
        logits[:] = torch.arange(e, device="cuda").flip(0) * 0.5
    elif kind == "ties":
        logits = (logits > 0.5).float() * 0.0 - (logits < -0.5).float() + 0.0
        logits[:, ::3] *= -0.0
    elif kind == "few":
        logits[:, topk - 1 :] = float("-inf")
    else:
        logits *= 1e30
    tm.close(tm.call(x, logits, w, topk), x, logits, values, topk)
