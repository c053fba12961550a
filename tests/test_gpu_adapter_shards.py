"""LoRALinear as the local linear of sharded layers: every rank's module on one GPU, one after the other, against the unsharded formula in 64 bits."""

import pytest
import torch

from emmy_b200 import shard
from tests import test_gpu_adapters as ta
from tests import test_gpu_lora as tl

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
SLOTS, RANK = 3, 16


def dense(weight):
    m = torch.nn.Linear(weight.shape[1], weight.shape[0], bias=False, device="cuda", dtype=BF16).requires_grad_(False)
    m.weight.copy_(weight)
    return m


def local(weight, a, b, scaling, sections):
    from emmy_b200 import linear

    m = linear.LoRALinear(dense(weight), SLOTS, RANK, BF16, sections)
    edges = [0]
    for w in sections:
        edges.append(edges[-1] + w)
    for slot in range(SLOTS):
        m.load_adapter(slot, list(a[slot]), [b[slot, i:j] for i, j in zip(edges, edges[1:])], scaling[slot])
    return m


def inputs(t, k, n, sections):
    g = torch.Generator("cuda").manual_seed(t)
    y, x, a, b, scaling, ids = tl.make(t, k, sections, RANK, SLOTS, BF16, seed=t)
    return (torch.randn(n, k, generator=g, device="cuda") * k**-0.5).bfloat16(), x, a, b, scaling, ids


@pytest.mark.parametrize("t", [7, 300])
@pytest.mark.parametrize("world", [2, 4])
def test_column_parallel(t, world):
    """A rank's columns are the unsharded module's, section by section."""
    k, sections = 512, (256, 64, 64)
    weight, x, a, b, scaling, ids = inputs(t, k, sum(sections), sections)
    with torch.no_grad():
        parts = []
        for rank in range(world):
            al, bl, widths = shard.column_slice_lora(a, b, rank, world, sections)
            rows = torch.cat([w.chunk(world)[rank] for w in weight.split(sections)])
            m = local(rows, al, bl, scaling.tolist(), widths)
            y = shard.ColumnParallelLinear(lambda v, m=m: m(v, ids))(x)
            ta.check_lora(m, x, ids, y)
            parts.append((y.split(widths, dim=1), m.base(x).split(widths, dim=1)))
        whole, base = (torch.cat([torch.cat([p[i][s] for p in parts], dim=1) for s in range(len(sections))], dim=1) for i in range(2))
        tl.close(whole, base, x, a, b, scaling, ids, sections)


@pytest.mark.parametrize("t", [7, 300])
@pytest.mark.parametrize("world", [2, 4])
def test_row_parallel(t, world, monkeypatch):
    """The ranks' adapters add up in the linear's own sum.  Every partial is rounded once, the sum once more."""
    k, n = 512, 256
    weight, x, a, b, scaling, ids = inputs(t, k, n, (n,))
    monkeypatch.setattr(shard.dist, "all_reduce", lambda *args, **kw: None)  # one rank at a time: the partials are added below
    total, ref = torch.zeros(t, n, device="cuda"), torch.zeros(t, n, dtype=torch.float64, device="cuda")
    limit = torch.zeros_like(ref)
    eps = torch.finfo(BF16).eps / 2
    with torch.no_grad():
        for rank in range(world):
            rows = slice(rank * k // world, (rank + 1) * k // world)
            al, bl = shard.row_slice_lora(a, b, rank, world)
            m = local(weight[:, rows], al, bl, scaling.tolist(), (n,))
            y = shard.RowParallelLinear(lambda v, m=m: m(v, ids), rows)(x)
            xs = x[:, rows].contiguous()
            ta.check_lora(m, xs, ids, y)
            part, size = tl.formula(m.base(xs), xs, m.lora_a, m.lora_b, m.scaling, ids, (n,))
            chain = 2.0**-18 + (k / 16 + RANK / 16 + 80) * 2.0**-23
            limit += eps * (part.abs() + chain * size) + chain * size + world * 2.0**-23 * part.abs()
            total += y.float()
            ref += part
        whole = m.base.weight.new_zeros(t, n).double()  # the unsharded adapters on the sum of the bases
        for rank in range(world):
            rows = slice(rank * k // world, (rank + 1) * k // world)
            whole += dense(weight[:, rows])(x[:, rows].contiguous()).double()
        whole, _ = tl.formula(whole, x, a, b, scaling, ids, (n,))
    assert (whole - ref).abs().max() <= 2.0**-40 * whole.abs().max()
    off = (total.bfloat16().double() - whole).abs()
    limit = limit + eps * (whole.abs() + limit) + 2.0**-40 * whole.abs().max()
    assert (off <= limit).all()
