"""What one form of the adapters' kernels has been shown for, shown for each of them: one launch, a list and blocks of 16 rows, tiles of 128 rows.
The cases' sizes lie where each form is taken (test_lora_forms_cpu.py holds them to it)."""

import pytest
import torch

from tests import test_gpu_lora as tl

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
SELF, LIST, TILES = "lora_rows_kernel", "group_rows_kernel + lora_rows_kernel", "lora_expand_kernel"
FORM_OF = {"a thread a row": SELF, "eight rows a thread": SELF, "list": LIST, "many ranks": LIST, "tiles": TILES, "tiles of 128 ranks": TILES}
# form -> purpose -> rows, K, sections, rank, adapters
CASES = {
    "a thread a row": {"plain": (200, 264, [136], 16, 4), "keys": (256, 64, [72], 8, 1400), "extreme": (200, 256, [64], 16, 2)},
    "eight rows a thread": {"plain": (1500, 264, [136, 64], 16, 4), "keys": (1900, 64, [72], 8, 1400), "extreme": (400, 256, [64], 16, 2)},
    "list": {"plain": (2600, 264, [136], 24, 4), "keys": (2500, 64, [72], 8, 1400), "extreme": (2100, 256, [64], 16, 2)},
    "many ranks": {"plain": (2100, 264, [136, 64, 8], 96, 4), "keys": (2100, 64, [72], 136, 1300), "extreme": (2100, 256, [64], 264, 2)},
    "tiles": {"plain": (1111, 264, [6000], 64, 4), "keys": (2500, 64, [2600], 64, 1400), "extreme": (3000, 256, [10440], 16, 2)},
    "tiles of 128 ranks": {"plain": (1111, 264, [4104, 264], 128, 4), "keys": (2500, 64, [1304], 128, 1300), "extreme": (1300, 256, [2400], 128, 2)},
}
forms = pytest.mark.parametrize("form", list(CASES))


def make(case, dtype, seed=0, ids=None):
    """As test_gpu_lora.make, drawn on the GPU."""
    t, k, sections, r, adapters = case
    g = torch.Generator("cuda").manual_seed(seed)
    n = sum(sections)
    draw = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    x, y = draw(t, k).to(dtype), draw(t, n).to(dtype)
    a, b = (draw(adapters, len(sections), r, k) * k**-0.5).to(dtype), (draw(adapters, n, r) * r**-0.5).to(dtype)
    scaling = torch.rand(adapters, generator=g, device="cuda") + 0.5
    if ids is None:
        ids = torch.randint(-1, adapters, (t,), generator=g, device="cuda")
    return [y, x, a, b, scaling, torch.as_tensor(ids, dtype=torch.int32, device="cuda")]


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")], ids=str)
@pytest.mark.parametrize("t,n", [(40, 64), (700, 64), (3000, 4096)])
def test_what_is_not_finite_in_one_section_stays_there(t, n, bad):
    """An adapter whose A overflowed f16 in one section; the other section's sums are far beyond f16's range and its results are not."""
    args = tl.make(t, 256, [n, n], 16, 2, F16, seed=5, ids=torch.zeros(t))
    y, x, a, b, scaling, ids = args
    x *= 2.0**6
    a[:, 1] *= 2.0**12
    b[:, n:] *= 2.0**-14
    a[0, 0, 3, 5] = bad
    got = tl.call(args, [n, n])
    second = [y[:, n:].contiguous(), x, a[:, 1:].contiguous(), b[:, n:].contiguous(), scaling, ids]
    assert (x.double() @ a[0, 1].double().T * scaling[0].item()).abs().amax(1).median() > 65504
    tl.close(got[:, n:].contiguous(), *second, [n])
    assert not torch.isfinite(got[:, :n]).any()


@forms
@pytest.mark.parametrize("order", ["interleaved", "prompts", "decode and prompts", "reversed"])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_rows_do_not_reach_one_another(form, order, dtype):
    """Infinities and NaN in a request's activations, in an adapter that nobody asked for, in a neighbour's output; in place and not; the waits' word."""
    from emmy_b200 import ops_lora

    t, k, sections, r, adapters = case = CASES[form]["plain"]
    i = torch.arange(t)
    ids = {
        "interleaved": i % 3,
        "prompts": i * 4 // t - 1,
        "decode and prompts": torch.where(i < 60, i * 5 % 4 - 1, (i - 60) * 2 // t * 2),
        "reversed": 2 - i * 4 // t,
    }[order]
    args = make(case, dtype, seed=3, ids=ids)
    ws = ops_lora.lora_workspace(t, adapters, len(sections), r, "cuda").fill_(255)
    want = tl.call(args, sections, workspace=ws)
    if t > 256:
        ops_lora.lora_status(ws)
    tl.close(want, *args, sections)
    inplace = args[0].clone()
    tl.call([inplace, *args[1:]], sections, out=inplace)
    assert torch.equal(inplace, want)
    y, x, a, b, scaling, ids = [v.clone() for v in args]
    assert not (ids == 3).any()
    a[3], b[3], scaling[3] = float("nan"), float("inf"), float("nan")
    adapted = (ids >= 0).nonzero()[:, 0]
    nan_x, inf_y, inf_x = adapted[[1, len(adapted) // 2, -1]].tolist()
    x[nan_x], y[inf_y], x[inf_x, 11] = float("nan"), float("inf"), float("inf")
    got = tl.call([y, x, a, b, scaling, ids], sections)
    rest = torch.ones(t, dtype=torch.bool, device="cuda")
    rest[[nan_x, inf_y, inf_x]] = False
    assert torch.equal(got[rest], want[rest])
    assert got[nan_x].isnan().all() and (got[inf_y] == float("inf")).all() and not torch.isfinite(got[inf_x]).any()


@forms
@pytest.mark.parametrize("kind", ["none", "outside", "one", "last", "first", "own", "runs", "few", "any"])
def test_every_kind_of_ids(form, kind):
    """Up to 1400 adapters: both sizes of the list's counters."""
    t, k, sections, r, adapters = case = CASES[form]["keys"]
    i = torch.arange(t)
    g = torch.Generator().manual_seed(t)
    ids = {
        "none": torch.full((t,), -1),
        "outside": torch.tensor([-1, adapters, 2**31 - 1, -(2**31), 2])[i % 5],
        "one": torch.full((t,), adapters - 1),
        "last": torch.where(i == t - 1, adapters - 1, -1),
        "first": torch.where(i == 0, 0, -1),
        "own": i.flip(0),  # those behind the last adapter have none
        "runs": (i * 4 // t) % 3 * (adapters // 3),
        "few": torch.where(torch.rand(t, generator=g) < 0.05, torch.randint(0, adapters, (t,), generator=g), -1),
        "any": torch.randint(-1, adapters + 1, (t,), generator=g),
    }[kind]
    args = make(case, BF16, seed=t, ids=ids)
    got = tl.call(args, sections)
    tl.close(got, *args, sections)
    y = args[0].clone()
    tl.call([y, *args[1:]], sections, out=y)
    assert torch.equal(y, got)


@forms
def test_f16_rows_of_very_large_and_very_small_values(form):
    """A x beyond f16's range and far below its smallest step: only the result has to fit."""
    t, k, sections, r, adapters = case = CASES[form]["extreme"]
    args = make(case, F16, seed=5, ids=torch.arange(t) % 2)
    y, x, a, b, scaling, ids = args
    x[::4] *= 2.0**12
    a[0] *= 2.0**9
    b[0] *= 2.0**-12
    a[1] *= 2.0**-12
    x[1::4] *= 2.0**-6
    b[1] *= 2.0**8
    scaling[1] = 2.0**10
    x[8::16] = 0  # a row of zeros has no largest value
    ref, _ = tl.formula(y, x, a, b, scaling, ids, sections)
    assert ref.abs().max() < 65504
    tl.close(tl.call(args, sections), *args, sections)


@forms
def test_scalings_of_every_sign(form):
    case = CASES[form]["plain"]
    args = make(case, BF16, seed=6)
    args[4][:] = torch.tensor([0.0, -1.5, 1.0, 2.0**-20])
    tl.close(tl.call(args, case[2]), *args, case[2])


@forms
def test_the_same_bits_eager_replayed_and_on_two_streams(form):
    """Captured once, replayed on other ids, activations and adapters; calls at once on two streams."""
    case = CASES[form]["plain"]
    sections = case[2]
    first, second = make(case, F16, seed=1), make(case, F16, seed=2)
    second[5] = second[5].sort().values
    want = [tl.call(first, sections), tl.call(second, sections)]
    for _ in range(5):
        assert torch.equal(tl.call(first, sections), want[0])
    held = [v.clone() for v in first]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tl.call(held, sections)
        again = tl.call([out, *held[1:]], sections)  # the next call on what the last one wrote
    for args, ref in ((second, want[1]), (first, want[0])):
        for h, v in zip(held, args):
            h.copy_(v)
        for _ in range(3):
            graph.replay()
        assert torch.equal(out, ref) and torch.equal(again, tl.call([ref, *args[1:]], sections))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        one = [tl.call(first, sections) for _ in range(20)]
    two = [tl.call(second, sections) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[0]) for o in one) and all(torch.equal(o, want[1]) for o in two)


@pytest.mark.parametrize("n,r", [(28136, 8), (6000, 64), (5200, 72), (4104, 128)])
@pytest.mark.parametrize("order", ["prompts", "decode and prompts", "interleaved", "reversed", "short runs"])
def test_where_the_rows_of_a_tile_lie(order, n, r):
    """Neighbouring rows, few and many rows apart, ragged last quarters, blocks without an adapter; in place and not; the waits' word stays clear."""
    from emmy_b200 import lib as L
    from emmy_b200 import ops_lora

    t, adapters = 1111, 7
    assert L.load().eq_lora_kernel(t, 264, n, r, 1).decode() == TILES
    i = torch.arange(t)
    ids = {
        "prompts": i * 5 // t - 1,
        "decode and prompts": torch.where(i < 60, i * 5 % 8 - 1, (i - 60) * 3 // t * 2),
        "interleaved": i % 3 - 1,
        "reversed": 6 - i * 7 // t,
        "short runs": i // 37 % 5 - 1,
    }[order]
    args = make((t, 264, [n], r, adapters), BF16, seed=r, ids=ids)
    ws = ops_lora.lora_workspace(t, adapters, 1, r, "cuda").fill_(255)
    got = tl.call(args, [n], workspace=ws)
    ops_lora.lora_status(ws)
    tl.close(got, *args, [n])
    y = args[0].clone()
    tl.call([y, *args[1:]], [n], out=y)
    assert torch.equal(y, got)
