"""Low-rank adapters of many requests beside a shared projection, on the GPU against the formula in 64 bits.

Tolerance of one value, from the arithmetic: the result is rounded once (half a step of its dtype); A x and B h are summed in f32, in
chains of MMA steps of sixteen products, each step off by at most a step of the largest partial sum (2^-23 of the sum of magnitudes
|scaling| |B| |A| |x|), the joins of the warps' and CTAs' sums included; h enters the second product as value + remainder, off by 2^-18
(bf16) or 2^-22 (f16) of it."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def make(t, k, sections, r, adapters, dtype, seed=0, ids=None):
    g = torch.Generator().manual_seed(seed)
    n = sum(sections)
    x, y = torch.randn(t, k, generator=g).to(dtype), torch.randn(t, n, generator=g).to(dtype)
    a = (torch.randn(adapters, len(sections), r, k, generator=g) * k**-0.5).to(dtype)
    b = (torch.randn(adapters, n, r, generator=g) * r**-0.5).to(dtype)
    scaling = torch.rand(adapters, generator=g) + 0.5
    if ids is None:
        ids = torch.randint(-1, adapters, (t,), generator=g)
    return [v.cuda() for v in (y, x, a, b, scaling, torch.as_tensor(ids, dtype=torch.int32))]


def formula(y, x, a, b, scaling, ids, sections):
    """(result, sum of magnitudes) in f64."""
    out, size = y.double(), torch.zeros_like(y, dtype=torch.float64)
    edges = [0]
    for w in sections:
        edges.append(edges[-1] + w)
    for l in sorted(set(ids.tolist())):
        if not 0 <= l < len(a):
            continue
        rows = (ids == l).nonzero()[:, 0]
        for s in range(len(sections)):
            cols = slice(edges[s], edges[s + 1])
            al, bl, xs, sc = a[l, s].double(), b[l, cols].double(), x[rows].double(), float(scaling[l])
            out[rows, cols] += sc * (xs @ al.T) @ bl.T
            size[rows, cols] = abs(sc) * (xs.abs() @ al.abs().T) @ bl.abs().T
    return out, size


def close(got, y, x, a, b, scaling, ids, sections):
    ref, size = formula(y, x, a, b, scaling, ids, sections)
    dtype, k, r = got.dtype, x.shape[1], a.shape[2]
    chain = (2.0**-18 if dtype == BF16 else 2.0**-22) + (k / 16 + r / 16 + 80) * 2.0**-23
    tiny = 2.0**-25 if dtype == F16 else 0.0  # half a step of f16's subnormals
    limit = (torch.finfo(dtype).eps / 2) * (ref.abs() + chain * size) + chain * size + tiny
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (off <= limit).all(), f"{(off - limit).max().item():.3g} over a limit of {limit.max().item():.3g}"
    none = ~((ids >= 0) & (ids < len(a)))
    assert torch.equal(got[none], y[none])


def call(args, sections, **kw):
    from emmy_b200 import ops_lora

    return ops_lora.lora_add(*args, sections=sections, **kw)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize(
    "t,k,sections,r,adapters",
    [
        (1, 4096, [4096], 16, 8),
        (1, 8, [8], 8, 1),
        (2, 40, [24], 8, 2),
        (3, 264, [1000], 24, 5),
        (7, 5120, [64, 8, 24], 16, 3),
        (16, 512, [512], 64, 1),
        (17, 1792, [1024, 256, 256], 32, 1),
        (48, 4096, [4096, 1024, 1024], 8, 32),
        (255, 256, [40], 128, 64),
        (256, 1024, [2048, 2048], 64, 3),
        (257, 1024, [520], 16, 2),
        (300, 136, [96, 40], 24, 300),
        (321, 512, [256, 256], 256, 7),  # 512 ranks in all: blocks of 16 rows above 256 rows too
        (1000, 2048, [1032], 32, 4),
        (64, 256, [128] * 8, 128, 3),  # eight sections, 1024 ranks
        # prompts: ranks around the steps of 64, columns around the tiles of 128, more tiles than CTAs
        (700, 256, [8200], 128, 5),
        (600, 72, [9000, 3000, 64], 72, 2),
        (900, 640, [4096, 136], 128, 3),
        (513, 4096, [2048], 40, 1),
        (3000, 128, [1000, 24, 5000], 64, 2),
        (2048, 128, [136], 16, 40),  # every CTA's own list of blocks, and one row more than it takes
        (2049, 128, [136], 16, 40),
        (5000, 2048, [6000], 16, 3),
        (4500, 1024, [3000, 4096], 8, 2),
    ],
)
def test_matches_the_formula(t, k, sections, r, adapters, dtype):
    args = make(t, k, sections, r, adapters, dtype, seed=t + k)
    got = call(args, sections)
    close(got, *args, sections)
    # in place: the same bits
    y = args[0].clone()
    same = call([y, *args[1:]], sections, out=y)
    assert same is y and torch.equal(y, got)


@pytest.mark.parametrize("t", [5, 256, 700])
@pytest.mark.parametrize("kind", ["none", "outside", "one", "last", "own", "runs"])
def test_every_kind_of_ids(t, kind):
    adapters = 4096 if kind == "own" else 6
    ids = {
        "none": torch.full((t,), -1),
        "outside": torch.tensor([-1, 6, 2**31 - 1, -(2**31), 2])[torch.arange(t) % 5],
        "one": torch.full((t,), 3),
        "last": torch.where(torch.arange(t) == t - 1, 5, -1),
        "own": torch.arange(t).flip(0) * 5,
        "runs": (torch.arange(t) * 4 // t) % 3 * 2,
    }[kind]
    args = make(t, 64, [72], 8, adapters, BF16, seed=t, ids=ids)
    close(call(args, [72]), *args, [72])


def test_rows_do_not_reach_one_another():
    """What a row holds stays in it: infinities and NaN in one request's activations, in an adapter that nobody asked for, in a
    neighbour's output."""
    for t in (30, 400):
        args = make(t, 128, [136], 16, 4, BF16, seed=3, ids=torch.arange(t) % 3)
        want = call(args, [136])
        y, x, a, b, scaling, ids = [v.clone() for v in args]
        a[3], b[3], scaling[3] = float("nan"), float("inf"), float("nan")
        x[4], y[5] = float("nan"), float("inf")
        x[7, 11] = float("inf")
        got = call([y, x, a, b, scaling, ids], [136])
        rest = torch.ones(t, dtype=torch.bool, device="cuda")
        rest[[4, 5, 7]] = False
        assert torch.equal(got[rest], want[rest])
        assert got[4].isnan().all() and (got[5] == float("inf")).all() and not torch.isfinite(got[7]).any()


def test_f16_rows_of_very_large_and_very_small_values():
    """A x beyond f16's range and far below its smallest step: only the result has to fit."""
    args = make(40, 256, [64], 16, 2, F16, seed=5, ids=torch.arange(40) % 2)
    y, x, a, b, scaling, ids = args
    x[::4] *= 2.0**12
    a[0] *= 2.0**9  # rows of adapter 0 with large x: A x to 2^22
    b[0] *= 2.0**-12
    a[1] *= 2.0**-12
    x[1::4] *= 2.0**-6  # rows of adapter 1: A x near 2^-18
    b[1] *= 2.0**8
    scaling[1] = 2.0**10
    ref, _ = formula(y, x, a, b, scaling, ids, [64])
    assert ref.abs().max() < 65504
    # what a, b and x themselves hold after the scaling is the inputs' affair: they are read as they are
    close(call(args, [64]), *args, [64])


def test_scaling_of_zero_and_below():
    args = make(20, 64, [64], 8, 3, BF16, seed=6)
    args[4][:] = torch.tensor([0.0, -1.5, 1.0])
    close(call(args, [64]), *args, [64])


@pytest.mark.parametrize("t,n,r", [(1111, 4104, 8), (1111, 4104, 64), (1111, 4104, 72), (1111, 4104, 128), (1500, 24584, 16), (1500, 24584, 64)])
@pytest.mark.parametrize("order", ["prompts", "decode and prompts", "interleaved", "reversed"])
def test_where_the_rows_of_a_block_lie(order, t, n, r):
    """Neighbouring rows, few and many rows apart, ragged last quarters, blocks without an adapter; in place and not; the waits' word stays clear."""
    from emmy_b200 import lib as L

    adapters = 7
    i = torch.arange(t)
    ids = {
        "prompts": i * 5 // t - 1,
        "decode and prompts": torch.where(i < 60, i * 5 % 8 - 1, (i - 60) * 3 // t * 2),
        "interleaved": i % 3 - 1,
        "reversed": 6 - i * 7 // t,
    }[order]
    args = make(t, 264, [n], r, adapters, BF16, seed=r, ids=ids)
    ws = torch.full((L.load().eq_lora_workspace_bytes(t, adapters, 1, r),), 255, dtype=torch.uint8, device="cuda")
    got = call(args, [n], workspace=ws)
    L.check(L.load().eq_lora_status(ws.data_ptr(), None))
    close(got, *args, [n])
    y = args[0].clone()
    call([y, *args[1:]], [n], out=y)
    assert torch.equal(y, got)


def test_empty_calls():
    for t in (0,):
        args = make(t, 64, [64], 8, 3, BF16)
        assert call(args, [64]).shape == (0, 64)


def test_far_rows_and_columns():
    """Offsets of y, b and a that pass 2^31 elements."""
    n, r, adapters = 1 << 17, 64, 300
    y = torch.zeros(17000, n, dtype=BF16, device="cuda")
    x = torch.randn(17000, 16, device="cuda").to(BF16)
    a = torch.randn(adapters, 1, r, 16, device="cuda").to(BF16)
    b = torch.zeros(adapters, n, r, dtype=BF16, device="cuda")
    b[adapters - 1, n - 8 :] = 1.0
    b[adapters - 1, :8] = -1.0
    scaling = torch.ones(adapters, device="cuda")
    ids = torch.full((17000,), -1, dtype=torch.int32, device="cuda")
    ids[16990:] = adapters - 1
    assert y.numel() > 2**31 and b.numel() > 2**31
    call([y, x, a, b, scaling, ids], [n], out=y)
    sub = [y[16990:, -8:].clone() * 0, x[16990:], a[-1:], b[-1:, n - 8 :].contiguous(), scaling[-1:], ids[16990:] * 0]
    close(y[16990:, n - 8 :].contiguous(), *sub, [8])
    assert torch.equal(y[16990:, :8], -y[16990:, n - 8 :])
    assert not y[:16990].any() and not y[16990:, 8 : n - 8].any()


def test_another_stream_and_a_replayed_graph():
    """Captured once, replayed on other ids, activations and adapters; two calls at once on two streams with workspaces of their own."""
    for t in (33, 520):
        first, second = make(t, 512, [256], 16, 5, BF16, seed=1), make(t, 512, [256], 16, 5, BF16, seed=2)
        want = [call(first, [256]), call(second, [256])]
        held = [v.clone() for v in first]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = call(held, [256])
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(warm, want[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(held, [256])
        for args, ref in ((second, want[1]), (first, want[0])):
            for h, v in zip(held, args):
                h.copy_(v)
            for _ in range(3):
                graph.replay()
            assert torch.equal(out, ref)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            one = [call(first, [256]) for _ in range(20)]
        two = [call(second, [256]) for _ in range(20)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[0]) for o in one) and all(torch.equal(o, want[1]) for o in two)


def test_the_same_bits_every_time():
    args = make(600, 1024, [512, 128], 32, 9, F16, seed=8)
    want = call(args, [512, 128])
    for _ in range(10):
        assert torch.equal(call(args, [512, 128]), want)


def test_a_row_does_not_depend_on_its_batch_beyond_rounding():
    """The same request alone and in a batch: the sums are cut differently, so equal within the tolerance of each."""
    args = make(256, 1024, [256], 16, 4, BF16, seed=9)
    alone = torch.cat([call([args[0][i : i + 1], args[1][i : i + 1], *args[2:5], args[5][i : i + 1]], [256]) for i in range(0, 256, 37)])
    pick = torch.arange(0, 256, 37)
    close(alone, args[0][pick], args[1][pick], *args[2:5], args[5][pick], [256])


def test_bad_shapes_are_refused():
    from emmy_b200 import ops_lora
    from emmy_b200.lib import EmmyqError

    y, x, a, b, scaling, ids = make(4, 64, [64], 8, 3, BF16)
    ok = lambda **kw: ops_lora.lora_add(**{**dict(y=y, x=x, a=a, b=b, scaling=scaling, adapter_ids=ids), **kw})
    ok()
    for kw in (dict(x=x[:3]), dict(a=a[:2]), dict(b=b[:, :32]), dict(scaling=scaling.double()), dict(adapter_ids=ids.long()), dict(adapter_ids=ids[:2]),
               dict(y=y.half()), dict(a=a.half()), dict(sections=[32, 32]), dict(x=x.float()), dict(out=torch.empty(4, 32, dtype=BF16, device="cuda")),
               dict(a=a[0]), dict(x=x.t().contiguous().t())):
        with pytest.raises(ValueError):
            ok(**kw)
    with pytest.raises(EmmyqError, match="EQ_ERR_UNSUPPORTED"):
        args = make(4, 60, [64], 8, 3, BF16)
        call(args, [64])
    with pytest.raises(EmmyqError, match="EQ_ERR_BAD_ARG"):
        args = make(4, 64, [64], 8, 3, BF16)
        call(args, [56])
