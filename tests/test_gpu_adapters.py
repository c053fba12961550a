"""The modules around the adapters and the FP8 experts, on the GPU: every base family, a layer of them as it would be used, captured."""

import pytest
import torch

from oracle import synth
from tests import test_gpu_lora as tl
from tests import test_gpu_moe_w8 as tm
from tests.test_adapters_cpu import expert_tensors, pair, write_adapter
from tests.test_loader_cpu import write_checkpoint

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def base_of(family, k, n, seed=0):
    from emmy_b200 import linear

    if family == "w4a16":
        m = linear.W4A16Linear(k, n, 128, fmt="awq")
        m.load_state_dict({name: torch.from_numpy(v) for name, v in zip(("qweight", "qzeros", "scales"), synth.awq_linear(k, n, seed=seed))})
        return m.cuda().finalize()
    g = torch.Generator("cuda").manual_seed(seed)
    w = torch.randn(n, k, generator=g, device="cuda") * k**-0.5
    if family == "fp8":
        s = w.abs().amax(1) / 448
        return linear.FP8Linear(k, n).cuda().load_float8((w / s[:, None]).to(torch.float8_e4m3fn), s)
    if family == "fp8_block":
        s = w.view(n // 128, 128, k // 128, 128).abs().amax(dim=(1, 3)) / 448
        return linear.FP8BlockLinear(k, n).cuda().load_float8((w / s.repeat_interleave(128, 0).repeat_interleave(128, 1)).to(torch.float8_e4m3fn), s)
    if family == "nvfp4":
        m = linear.NVFP4Linear(k, n).cuda()
        m.weight = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        m.weight_scale = torch.full((n, k // 16), 0.0625, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
        m.input_scale.fill_(0.01)
        return m.finalize()
    return torch.nn.Linear(k, n, bias=False, device="cuda", dtype=BF16).requires_grad_(False)


def filled(base, slots, rank, dtype, sections=None, seed=0):
    """Adapters of differing ranks in all slots but the last."""
    from emmy_b200 import linear

    m = linear.LoRALinear(base, slots, rank, dtype, sections)
    g = torch.Generator().manual_seed(seed)
    for slot in range(slots - 1):
        r = max(1, rank - 3 * slot)
        m.load_adapter(slot, [torch.randn(r, m.in_features, generator=g) * m.in_features**-0.5 for _ in m.sections],
                       [torch.randn(w, r, generator=g) * r**-0.5 for w in m.sections], 0.5 + slot)
    return m


def check_lora(m, x, ids, got):
    y = m.base(x).reshape(-1, m.out_features)
    tl.close(got.reshape(-1, m.out_features), y, x.reshape(-1, m.in_features), m.lora_a, m.lora_b, m.scaling, ids.reshape(-1), m.sections)


@pytest.mark.parametrize("family,dtype", [("w4a16", F16), ("w4a16", BF16), ("fp8", BF16), ("fp8_block", BF16), ("fp8_block", F16), ("nvfp4", BF16), ("dense", BF16)])
@pytest.mark.parametrize("t", [1, 70, 300])
def test_adapters_beside_every_family(family, dtype, t):
    k, n = 512, 384
    m = filled(base_of(family, k, n), 3, 12, dtype, (256, 128))
    g = torch.Generator("cuda").manual_seed(t)
    x = torch.randn(t, 2, k, generator=g, device="cuda").to(dtype)
    ids = torch.randint(-1, 3, (t, 2), generator=g, device="cuda", dtype=torch.int32)
    with torch.no_grad():
        got = m(x, ids)
        assert got.shape == (t, 2, n) and got.dtype == dtype
        check_lora(m, x, ids, got)
        assert torch.equal(m(x), m.base(x))  # no ids: the base alone
        assert torch.equal(got.reshape(-1, n)[ids.reshape(-1) < 0], m.base(x).reshape(-1, n)[ids.reshape(-1) < 0])
        # strides other than the plain ones
        wide = torch.randn(2, t, k, generator=g, device="cuda").to(dtype)
        strided, turned = wide.transpose(0, 1), ids.t().contiguous().t()
        assert torch.equal(m(strided, turned), m(strided.contiguous(), ids))


def test_modules_trace_under_torch_compile():
    from emmy_b200 import linear

    h, i, e = 256, 128, 8
    weights, _ = tm.experts(e, h, i, True, 3)
    m, moe = filled(base_of("fp8_block", h, h), 3, 8, BF16), linear.QuantMoE(2).load_fp8_experts(*weights)
    router = torch.randn(e, h, device="cuda") * h**-0.5

    def layer(x, ids):
        x = m(x, ids)
        return moe(x, x.float() @ router.t())

    x, ids = torch.randn(5, h, device="cuda").bfloat16(), torch.tensor([0, 1, 2, -1, 0], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        assert torch.equal(torch.compile(layer, fullgraph=True, backend="eager")(x, ids), layer(x, ids))
    torch.library.opcheck(torch.ops.emmyq.lora_add, (x, x, m.lora_a, m.lora_b, m.scaling, ids, [h]))
    torch.library.opcheck(torch.ops.emmyq.moe_w8a16, (x, torch.randn(5, e, device="cuda"), *weights, 2))


@pytest.mark.parametrize("kind", ["tensor", "channel", "block"])
def test_fp8_experts_from_a_checkpoint(tmp_path, kind):
    from emmy_b200 import loader

    e, h, i, topk = 4, 256, 128, 2
    t = expert_tensors(e, h, i, kind)
    write_checkpoint(tmp_path, t, {"quant_method": "fp8"})
    index = loader.CheckpointIndex(tmp_path)
    moe = loader.load_experts(index, loader.scan_experts(loader.scan(tmp_path, index))["m.experts"], "cuda", top_k=topk)

    def value(x, name):
        w, s = t[f"m.experts.{x}.{name}.weight"].double(), t[f"m.experts.{x}.{name}.weight_scale"].double()
        return (w * (s.repeat_interleave(128, 0).repeat_interleave(128, 1) if kind == "block" else s)).cuda()

    values = (torch.stack([torch.cat([value(x, "gate_proj"), value(x, "up_proj")]) for x in range(e)]), torch.stack([value(x, "down_proj") for x in range(e)]))
    g = torch.Generator("cuda").manual_seed(2)
    for rows in (1, 6, 40):
        x = (torch.randn(rows, h, generator=g, device="cuda") * 1e-3).bfloat16()
        logits = torch.randn(rows, e, generator=g, device="cuda").bfloat16()
        tm.close(moe(x, logits), x, logits.float(), values, topk)
        assert torch.equal(moe(x[None], logits[None])[0], moe(x, logits))


def test_a_layer_of_them_eager_and_captured(tmp_path):
    """qkv and output projections with adapters read from directories, the router and the FP8 experts: each step against its formula, then
    replayed from one graph while requests and adapters change."""
    from emmy_b200 import linear, loader

    h, i, e, topk, t, slots = 512, 256, 16, 4, 24, 3
    heads = (512, 128, 128)
    qkv = linear.LoRALinear(base_of("fp8_block", h, sum(heads), 1), slots, 16, BF16, heads)
    out = linear.LoRALinear(base_of("w4a16", heads[0], h, 2), slots, 16, BF16)
    names = {("l.q_proj", "l.k_proj", "l.v_proj"): qkv, "l.o_proj": out}
    for n, r in ((0, 16), (1, 5), (2, 8)):
        tensors = {**pair("l.q_proj", r, h, heads[0], 10 + n), **pair("l.v_proj", r, h, heads[2], 20 + n), **pair("l.o_proj", r, heads[0], h, 30 + n)}
        write_adapter(tmp_path / str(n), {key: v * v.shape[1] ** -0.5 for key, v in tensors.items()}, r=r, lora_alpha=r)
    loader.load_adapter(tmp_path / "0", names, 0)
    loader.load_adapter(tmp_path / "1", names, 2)
    weights, values = tm.experts(e, h, i, True, 5)
    moe = linear.QuantMoE(topk).load_fp8_experts(*weights)
    g = torch.Generator("cuda").manual_seed(6)
    router = (torch.randn(e, h, generator=g, device="cuda") * h**-0.5).bfloat16()

    def layer(x, ids, steps=None):
        p = qkv(x, ids)
        q, k, v = p.split(heads, dim=1)
        mixed = q * torch.sigmoid((k * v).float().mean(1, keepdim=True)).to(q.dtype)
        o = out(mixed, ids)
        logits = torch.nn.functional.linear(o, router)
        y = moe(o, logits)
        if steps is not None:
            steps.extend((p, mixed, o, logits))
        return y

    x = torch.randn(t, h, generator=g, device="cuda").bfloat16()
    ids = torch.randint(-1, slots, (t,), generator=g, device="cuda", dtype=torch.int32)

    def checked():
        steps = []
        y = layer(x, ids, steps)
        p, mixed, o, logits = steps
        check_lora(qkv, x, ids, p)
        check_lora(out, mixed, ids, o)
        tm.close(y, o, logits.float(), values, topk)
        return y

    with torch.no_grad():
        first = checked()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x, ids)
        graph.replay()
        assert torch.equal(y, first)
        # other requests, other adapters, in the same buffers
        x.copy_(torch.randn(t, h, generator=g, device="cuda"))
        ids.copy_(torch.randint(-1, slots + 1, (t,), generator=g, device="cuda", dtype=torch.int32))
        loader.load_adapter(tmp_path / "2", names, 1)
        qkv.clear_adapter(0), out.clear_adapter(0)
        graph.replay()
        again = y.clone()
        assert torch.equal(again, checked()) and not torch.equal(again, first)
        # and on a stream of its own
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = layer(x, ids)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, again)


def test_graphs_of_one_pool_replayed_in_turn():
    """Two captures of different sizes whose scratch lies in one pool."""
    from emmy_b200 import linear

    h, e = 256, 8
    weights, _ = tm.experts(e, h, 128, False, 3)
    m, moe = filled(base_of("dense", h, h), 3, 8, BF16), linear.QuantMoE(2).load_fp8_experts(*weights)
    runs, pool = [], torch.cuda.graph_pool_handle()
    with torch.no_grad():
        for t in (3, 40, 300):
            x, ids, logits = torch.randn(t, h, device="cuda").bfloat16(), torch.randint(-1, 3, (t,), device="cuda", dtype=torch.int32), torch.randn(t, e, device="cuda")
            want = moe(m(x, ids), logits)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=pool):
                y = moe(m(x, ids), logits)
            runs.append((graph, y, want, (x, ids, logits)))  # (a graph reads the inputs where they lie)
        for n in (0, 1, 2, 1, 0, 2):
            graph, y, want, _ = runs[n]
            y.zero_()
            graph.replay()
            assert torch.equal(y, want)


def test_calls_on_two_streams_at_once():
    """Every form of both operators beside another call of itself: nothing is shared between calls."""
    from emmy_b200 import ops_moe

    jobs = []
    for t, k, n, r, ids in ((7, 512, 384, 16, None), (300, 512, 384, 16, None), (4000, 1024, 4096, 64, [0] * 1500 + [1] * 2500)):
        args = tl.make(t, k, [n], r, 3, BF16, seed=t, ids=ids)
        jobs.append(lambda args=args: tl.call(args, None))
    for t, e, h, i in ((1, 8, 256, 128), (20, 16, 512, 256), (60, 16, 512, 256)):
        weights, _ = tm.experts(e, h, i, True, t)
        x, logits = tm.inputs(t, e, h, BF16, t)
        jobs.append(lambda x=x, logits=logits, weights=weights: ops_moe.moe_w8a16(x, logits, *weights, 2))
    want = [job() for job in jobs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for turn in range(30):
        for n, job in enumerate(jobs):
            for shift, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    got.append(((n + 3 * shift) % len(jobs), jobs[(n + 3 * shift) % len(jobs)]()))
    torch.cuda.synchronize()
    for n, y in got:
        assert torch.equal(y, want[n]), n
