"""The routed layer of a few tokens on FP8 experts, on the GPU against the formula in 64 bits.

Tolerance of one value, from the arithmetic.  A chain of MMA steps of sixteen products is off by at most a step of the largest partial sum each
(2^-23 of the sum of magnitudes), the scales and the joins of the warps' sums add a few steps of the same size: c = (K / 16 + K / 128 + 32) 2^-23.
A row whose largest value is V enters a product in f16 after a power of two has taken V to 2^14 or more: its 8 or 11 bits are exact unless they reach below
f16's smallest step, 2^-24, half of which is 2^-39 V; h enters as value + remainder, off by 2^-22 of itself or that.  With G = sum |w x| of gate and U of up, and W
the sums of |w|, gate is off by dg = c G + 2^-39 X W and up by du alike; silu has a slope below 1.1, so h = silu(gate) up is off by 1.1 dg |up| + |silu(gate)| du,
by the exponential, the division and the product (8 x 2^-24 of it) and by its two parts.  y adds p |W_down| of that, its own chains, 16 x 2^-24 for the shares, and
half a step of its dtype for the one rounding.  (A row of f16 is read as it is: its own subnormals are its own.)"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def experts(e, h, i, block, seed):
    """e4m3 weights with scales that differ by expert, row and block, and their values in f64."""
    g = torch.Generator("cuda").manual_seed(seed)

    def one(n, k):
        w = torch.randn(e, n, k, generator=g, device="cuda") * k**-0.5
        if block:
            w = w * (torch.rand(e, n // 128, 1, k // 128, 1, generator=g, device="cuda") + 0.25).expand(e, n // 128, 128, k // 128, 128).reshape(e, n, k)
            s = w.view(e, n // 128, 128, k // 128, 128).abs().amax(dim=(2, 4)) / 448
            wide = s.repeat_interleave(128, 1).repeat_interleave(128, 2)
        else:
            w = w * (torch.rand(e, n, 1, generator=g, device="cuda") + 0.25)
            s = w.abs().amax(dim=2) / 448
            wide = s[:, :, None]
        bits = (w / wide).to(torch.float8_e4m3fn)
        return bits.view(torch.uint8), s.contiguous(), bits.double() * wide.double()

    gu, gus, guv = one(2 * i, h)
    dn, dns, dnv = one(h, i)
    return (gu, gus, dn, dns), (guv, dnv)


def routed(logits, topk):
    """ids and shares [T, topk] in f64, from the definition."""
    lg = logits.double().cpu()
    order = torch.sort(lg, dim=1, descending=True, stable=True).indices[:, :topk]
    v = lg.gather(1, order)
    p = (v - v[:, :1]).exp()
    return order.cuda(), (p / p.sum(1, keepdim=True)).cuda()


def formula(x, logits, values, topk):
    """(y, limit without the last rounding) in f64."""
    guv, dnv = values
    ids, shares = routed(logits, topk)
    xd, (t, h), i = x.double(), x.shape, dnv.shape[2]
    ch, ci = (h / 16 + h / 128 + 32) * 2.0**-23, (i / 16 + i / 128 + topk + 32) * 2.0**-23
    y, limit = torch.zeros(t, h, dtype=torch.float64, device="cuda"), torch.zeros(t, h, dtype=torch.float64, device="cuda")
    for e in ids.unique().tolist():
        rows, slot = (ids == e).nonzero(as_tuple=True)
        gate, up = (xd[rows] @ guv[e].T).chunk(2, 1)
        sg, su = (xd[rows].abs() @ guv[e].abs().T).chunk(2, 1)
        wg, wu = (xd[rows].abs().amax(1, keepdim=True) * guv[e].abs().sum(1)).chunk(2, 1)
        dg, du = ch * sg + 2.0**-39 * wg, ch * su + 2.0**-39 * wu
        silu = gate * torch.sigmoid(gate)
        act = silu * up
        off = 1.1 * dg * up.abs() + silu.abs() * du + act.abs() * (2.0**-22 + 8 * 2.0**-24) + 2.0**-39 * act.abs().amax(1, keepdim=True)
        p = shares[rows, slot][:, None]
        y[rows] += p * (act @ dnv[e].T)
        limit[rows] += p * (off @ dnv[e].abs().T + (ci + 16 * 2.0**-24) * (act.abs() @ dnv[e].abs().T))
    return y, limit


def close(got, x, logits, values, topk):
    ref, limit = formula(x, logits, values, topk)
    limit = limit + (torch.finfo(got.dtype).eps / 2) * (ref.abs() + limit) + (2.0**-25 if got.dtype == F16 else 0)
    assert torch.isfinite(got).all()
    off = (got.double() - ref).abs()
    assert (off <= limit).all(), f"{(off - limit).max().item():.3g} over a limit of {limit.max().item():.3g}"


def inputs(t, e, h, dtype, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(t, h, generator=g, device="cuda").to(dtype), torch.randn(t, e, generator=g, device="cuda").bfloat16().float()


def call(x, logits, w, topk, **kw):
    from emmy_b200 import ops_moe

    return ops_moe.moe_w8a16(x, logits, *w, topk, **kw)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("block", [True, False], ids=["block", "channel"])
@pytest.mark.parametrize(
    "t,e,topk,h,i",
    [
        (1, 1, 1, 128, 128),
        (1, 8, 2, 256, 128),
        (1, 128, 8, 2048, 768),
        (2, 60, 4, 640, 1408),
        (5, 8, 2, 1024, 1792),
        (9, 2, 1, 384, 256),   # blocks of eight rows and of one
        (16, 128, 8, 512, 384),
        (17, 3, 3, 128, 640),  # every expert on every token
        (32, 256, 16, 256, 256),
        (33, 64, 6, 512, 256),
        (32, 257, 2, 256, 128),  # more experts than a CTA routes by itself
        (100, 16, 4, 384, 512),
        (257, 8, 3, 256, 384),
        (700, 1000, 16, 128, 128),
    ],
)
def test_matches_the_formula(t, e, topk, h, i, block, dtype):
    w, values = experts(e, h, i, block, seed=t + e)
    x, logits = inputs(t, e, h, dtype, seed=t)
    got = call(x, logits, w, topk)
    close(got, x, logits, values, topk)
    again = x.clone()
    assert call(again, logits, w, topk, out=again) is again and torch.equal(again, got)  # in place of x


@pytest.mark.parametrize("t", [1, 8, 9, 31, 33, 90])
@pytest.mark.parametrize("kind", ["one", "ties", "infinite", "nan", "far"])
def test_routing_at_its_borders(t, kind):
    """All tokens to the same experts; equal logits; minus infinity beside few picks; tokens with a NaN; logits far apart."""
    e, topk, h, i = 24, 4, 256, 128
    w, values = experts(e, h, i, True, seed=5)
    x, logits = inputs(t, e, h, BF16, seed=t)
    if kind == "one":
        logits[:] = torch.arange(e, device="cuda").flip(0) * 0.5
    elif kind == "ties":
        logits = (logits > 0.5).float() * 0.0 - (logits < -0.5).float() + 0.0
        logits[:, ::3] *= -0.0
    elif kind == "infinite":
        logits[:, 4:] = float("-inf")
    elif kind == "nan":
        logits[::3, 7] = float("nan")  # exp(NaN) is a term of the softmax's sum
        got = call(x, logits, w, topk)
        assert got[::3].isnan().all()
        rest = torch.arange(t, device="cuda") % 3 != 0
        if rest.any():
            close(got[rest], x[rest], logits[rest], values, topk)
        return
    elif kind == "far":
        logits *= 1e30
    close(call(x, logits, w, topk), x, logits, values, topk)


def test_logits_that_leave_too_few_experts():
    """Fewer experts above minus infinity than picks: the others have a share of zero.  Nothing but NaN: the token is NaN, no other one is."""
    e, topk, h, i = 16, 4, 256, 128
    w, values = experts(e, h, i, False, seed=6)
    for t in (6, 40):
        x, logits = inputs(t, e, h, BF16, seed=t)
        logits[2, 1:] = float("-inf")
        close(call(x, logits, w, topk), x, logits, values, topk)
        logits[4] = float("nan")
        got = call(x, logits, w, topk)
        rest = torch.arange(t, device="cuda") != 4
        assert got[4].isnan().all()
        close(got[rest], x[rest], logits[rest], values, topk)


def test_tokens_do_not_reach_one_another():
    e, topk, h, i = 8, 2, 256, 256
    w, _ = experts(e, h, i, True, seed=7)
    for t in (20, 50):
        x, logits = inputs(t, e, h, BF16, seed=t)
        want = call(x, logits, w, topk)
        x[3], x[7, 9] = float("nan"), float("inf")
        got = call(x, logits, w, topk)
        rest = torch.ones(t, dtype=torch.bool, device="cuda")
        rest[[3, 7]] = False
        assert torch.equal(got[rest], want[rest]) and got[3].isnan().all() and not torch.isfinite(got[7]).any()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("t", [1, 3, 20, 40])
def test_rows_of_every_size(t, dtype):
    """Rows of zeros, of one value, of very large and very small ones, of a few outliers beside small values; h beyond f16's range."""
    e, topk, h, i = 16, 4, 512, 256
    w, values = experts(e, h, i, True, seed=13)
    for seed in range(3):
        x, logits = inputs(t, e, h, dtype, seed=seed)
        top = 2.0**14 if dtype == F16 else 2.0**60
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
        w_small = (w[0], w[1], w[2], w[3] * 2.0**-30) if dtype == F16 else w
        v_small = (values[0], values[1] * 2.0**-30) if dtype == F16 else values
        assert x.abs().max() <= top
        close(call(x, logits, w_small, topk), x, logits, v_small, topk)


def test_every_weight_code_and_wide_scales():
    """All finite e4m3 codes, subnormal ones too, with scales from 2^-40 to 2^10."""
    e, h, i = 2, 128, 128
    codes = torch.tensor([c for c in range(256) if c & 127 != 127], dtype=torch.uint8, device="cuda")
    g = torch.Generator("cuda").manual_seed(8)
    gu = codes[torch.randint(0, len(codes), (e, 2 * i, h), generator=g, device="cuda")]
    dn = codes[torch.randint(0, len(codes), (e, h, i), generator=g, device="cuda")]
    gus = torch.full((e, 2 * i), 2.0**-9, device="cuda")
    gus[:, i:] = 2.0**-40
    gus[1, i:] = 2.0**-16
    dns = torch.full((e, h), 2.0**10, device="cuda")
    dns[1] = 2.0**-12
    value = lambda b: b.view(torch.float8_e4m3fn).double()
    values = (value(gu) * gus.double()[:, :, None], value(dn) * dns.double()[:, :, None])
    for t in (7, 40):
        x, logits = inputs(t, e, h, BF16, seed=t)
        close(call(x, logits, (gu, gus, dn, dns), 1), x, logits, values, 1)


def test_far_experts():
    """Weights and scales behind 2^31 elements."""
    e, h, i = 300, 2048, 2048
    g = torch.Generator("cuda").manual_seed(9)
    gu = torch.zeros(e, 2 * i, h, dtype=torch.uint8, device="cuda")
    dn = torch.zeros(e, h, i, dtype=torch.uint8, device="cuda")
    assert gu.numel() > 2**31
    small = torch.randn(2 * i, h, generator=g, device="cuda").to(torch.float8_e4m3fn)
    gu[-1], dn[-1] = small.view(torch.uint8), torch.randn(h, i, generator=g, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
    gus, dns = torch.full((e, 2 * i // 128, h // 128), 0.02, device="cuda"), torch.full((e, h // 128, i // 128), 0.02, device="cuda")
    x, logits = inputs(3, e, h, BF16, seed=1)
    logits[:, -1] = 50.0
    want = call(x, logits[:, -1:].contiguous(), (gu[-1:], gus[-1:], dn[-1:], dns[-1:]), 1)
    assert torch.isfinite(want).all() and want.abs().max() > 0
    assert torch.equal(call(x, logits, (gu, gus, dn, dns), 1), want) or (call(x, logits, (gu, gus, dn, dns), 1) - want).abs().max() <= 2.0**-7 * want.abs().max()


def test_another_stream_and_a_replayed_graph():
    e, topk, h, i = 32, 4, 512, 256
    w, _ = experts(e, h, i, True, seed=10)
    for t in (3, 24, 60):
        first, second = inputs(t, e, h, F16, seed=1), inputs(t, e, h, F16, seed=2)
        want = [call(*first, w, topk), call(*second, w, topk)]
        held = [v.clone() for v in first]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = call(*held, w, topk)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(warm, want[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(call(*held, w, topk), held[1], w, topk)  # two layers
        for args, ref in ((second, want[1]), (first, want[0])):
            for v, a in zip(held, args):
                v.copy_(a)
            for _ in range(3):
                graph.replay()
            assert torch.equal(out, call(ref, args[1], w, topk))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            one = [call(*first, w, topk) for _ in range(20)]
        two = [call(*second, w, topk) for _ in range(20)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[0]) for o in one) and all(torch.equal(o, want[1]) for o in two)


def test_the_same_bits_every_time():
    w, _ = experts(16, 512, 384, False, seed=11)
    for t in (13, 32, 77):
        x, logits = inputs(t, 16, 512, BF16, seed=t)
        want = call(x, logits, w, 4)
        for _ in range(10):
            assert torch.equal(call(x, logits, w, 4), want)


def test_an_empty_batch_and_bad_shapes():
    from emmy_b200.lib import EmmyqError

    w, _ = experts(4, 256, 128, True, seed=12)
    x, logits = inputs(3, 4, 256, BF16, seed=1)
    assert call(x[:0], logits[:0], w, 2).shape == (0, 256)
    gu, gus, dn, dns = w
    for args in ((x[:2], logits, w), (x, logits[:, :3].contiguous(), w), (x, logits.double(), w), (x.float(), logits, w), (x, logits, (gu[:3], gus, dn, dns)),
                 (x, logits, (gu, gus[:, :1].contiguous(), dn, dns)), (x, logits, (gu, gus, dn, dns[:, 0].contiguous())), (x, logits, (gu.view(torch.int8), gus, dn, dns)),
                 (x, logits, (gu, gus.half(), dn, dns))):
        with pytest.raises(ValueError):
            call(*args, 2)
    with pytest.raises(ValueError):
        call(x, logits, w, 2, out=torch.empty(3, 256, dtype=F16, device="cuda"))
    for topk, name in ((0, "EQ_ERR_BAD_ARG"), (5, "EQ_ERR_UNSUPPORTED")):
        with pytest.raises(EmmyqError, match=name):
            call(x, logits, w, topk)
