"""Cases of two serving operators: low-rank adapters of many requests beside a shared projection, and a routed MoE layer of a few
tokens on FP8 experts.

`own` says who computes them: elementary torch operations in 32 bits (False), or the operators of emmy_b200 (True).

    lora   out[t] = y[t] + scaling[l] * B[l] (A[l] x[t])  with l = adapter_ids[t], out[t] = y[t] where l < 0.  A projection that holds
           several linears side by side (q, k and v; gate and up) has an A per linear: columns of linear s read A[l, s].
    moe    out[t] = sum_j p[t, j] W_down[e] (silu(W_gate[e] x[t]) * (W_up[e] x[t]))  over the topk experts e = id[t, j] of the softmax
           of the router's logits (ties to the lowest id), p renormalised to sum to one.  Weights are e4m3 with a multiplier per output
           channel, or per 128 x 128 block.
"""

import math

import torch

own = False

_DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------------------- the cases


def _lora(name, k, sections, rank, adapters, decode, sequences, prompt, dtype):
    """`decode` single tokens of as many requests, then `sequences` prompts of `prompt` tokens in all."""
    case = {"op": "lora", "k": k, "sections": sections, "rank": rank, "adapters": adapters, "decode": decode, "sequences": sequences, "prompt": prompt,
            "dtype": dtype}
    return {"name": name, **case} if name else case


def _moe(name, tokens, experts, topk, hidden, inter, scales, dtype):
    case = {"op": "moe", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "inter": inter, "scales": scales, "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one request that decodes: the output projection of a 4096-wide model
        _lora("lora_t1_r16", 4096, "4096", 16, 8, 1, 0, 0, "bf16"),
        # a few requests of an f16 model, the down projection, an odd count
        _lora("lora_t17_down_r32", 14336, "4096", 32, 4, 17, 0, 0, "f16"),
        # q, k and v of grouped-query attention in one projection, some requests without an adapter
        _lora("lora_t48_qkv_r8", 4096, "4096,1024,1024", 8, 32, 48, 0, 0, "f16"),
        # a full decode batch over many adapters: gate and up of a 5120-wide model
        _lora("lora_t256_gate_up_r64", 5120, "17408,17408", 64, 64, 256, 0, 0, "bf16"),
        # chunked prefill: requests that decode and the prompts of three others in one batch, ragged
        _lora("lora_t1999_mixed_r16", 5120, "5120", 16, 24, 102, 3, 1897, "bf16"),
        # prompts of two adapters, gate and up of a 4096-wide model
        _lora("lora_t8192_gate_up_r64", 4096, "14336,14336", 64, 2, 0, 4, 8192, "bf16"),
        # one token: 128 small experts, eight of them
        _moe("moe_t1_e128", 1, 128, 8, 2048, 768, "block", "bf16"),
        # a few tokens of an f16 model with few and wide experts, scales per channel
        _moe("moe_t5_e8_channel", 5, 8, 2, 4096, 14336, "channel", "f16"),
        # the first batch that touches most of the small experts
        _moe("moe_t16_e128", 16, 128, 8, 2048, 768, "block", "bf16"),
        # an odd batch of mid-sized experts
        _moe("moe_t33_e64_channel", 33, 64, 6, 2048, 1408, "channel", "bf16"),
        # a decode batch: every expert has a few tokens
        _moe("moe_t64_e128_f16", 64, 128, 8, 2048, 768, "block", "f16"),
        # the largest batches that decode together
        _moe("moe_t200_e128", 200, 128, 8, 2048, 768, "block", "bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        dtype = rng.choice(("bf16", "f16"))
        if rng.random() < 0.5:
            k = 8 * _log_int(rng, 64, 1792)
            sections = ",".join(str(8 * _log_int(rng, 64, 1792)) for _ in range(rng.choice((1, 1, 2, 3))))
            rank = rng.choice((8, 16, 24, 32, 64, 128))
            tokens = _log_int(rng, 1, 8192)
            decode = tokens if tokens <= 256 else rng.randint(0, 128)
            sequences = 0 if tokens <= 256 else rng.randint(1, 6)
            case = _lora(None, k, sections, rank, rng.randint(1, 64), decode, sequences, tokens - decode, dtype)
        else:
            experts = rng.choice((8, 16, 60, 64, 128, 256))
            topk = rng.randint(1, 8)
            case = _moe(None, _log_int(rng, 1, 256), experts, topk, 128 * _log_int(rng, 4, 40), 128 * _log_int(rng, 2, 48), rng.choice(("block", "channel")), dtype)
            if 3 * case["experts"] * case["hidden"] * case["inter"] > 3e9:  # weights of one layer that a card holds beside its others
                continue
        if work(case)["bytes"] <= most:
            return case


# ------------------------------------------------------------------------------------------------------------------------- the inputs


def _widths(case):
    return [int(w) for w in case["sections"].split(",")]


def _prepare_lora(case, gen):
    dtype, k, n, rank, adapters = _DTYPE[case["dtype"]], case["k"], sum(_widths(case)), case["rank"], case["adapters"]
    sections, tokens = len(_widths(case)), case["decode"] + case["prompt"]
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    ids = torch.randint(0, adapters, (case["decode"],), generator=gen, device="cuda")
    if case["decode"] > 4:  # one request in eight runs the base model alone
        ids = torch.where(torch.rand(case["decode"], generator=gen, device="cuda") < 0.125, torch.full_like(ids, -1), ids)
    if case["sequences"]:
        cuts = torch.sort(torch.rand(case["sequences"] - 1, generator=gen, device="cuda")).values
        of = torch.searchsorted(cuts, (torch.arange(case["prompt"], device="cuda") + 0.5) / case["prompt"])
        first = torch.randint(0, adapters, (1,), generator=gen, device="cuda")
        ids = torch.cat([ids, (of + first) % adapters])
    return {
        "op": "lora",
        "widths": _widths(case),
        "x": normal(tokens, k).to(dtype),
        "y": normal(tokens, n).to(dtype),
        "a": (normal(adapters, sections, rank, k) / math.sqrt(k)).to(dtype),
        "b": (normal(adapters, n, rank) / math.sqrt(rank)).to(dtype),
        "scaling": torch.rand(adapters, generator=gen, device="cuda") * 1.5 + 0.5,
        "adapter_ids": ids.to(torch.int32),
    }


def _fp8(shape, scales, gen):
    """Normal weights of a linear's usual size and their scales: e4m3 bits [E, N, K], f32 [E, N] or [E, N / 128, K / 128]."""
    e, n, k = shape
    w = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16) * (1 / math.sqrt(k))
    if scales == "block":
        w = w.view(e, n // 128, 128, k // 128, 128)
        s = w.abs().amax(dim=(2, 4), keepdim=True).float() / 448
    else:
        s = w.abs().amax(dim=2, keepdim=True).float() / 448
    bits = (w / s).to(torch.float8_e4m3fn).view(torch.uint8).view(shape)
    return bits, s.reshape(e, n // 128, k // 128) if scales == "block" else s.reshape(e, n)


def _prepare_moe(case, gen):
    e, h, i = case["experts"], case["hidden"], case["inter"]
    gate_up, gate_up_scale = _fp8((e, 2 * i, h), case["scales"], gen)
    down, down_scale = _fp8((e, h, i), case["scales"], gen)
    return {
        "op": "moe",
        "topk": case["topk"],
        "x": torch.randn((case["tokens"], h), generator=gen, device="cuda").to(_DTYPE[case["dtype"]]),
        # a router that computes in 16 bits hands on logits that tie
        "router_logits": torch.randn((case["tokens"], e), generator=gen, device="cuda").bfloat16().float(),
        "gate_up": gate_up,
        "gate_up_scale": gate_up_scale,
        "down": down,
        "down_scale": down_scale,
    }


def prepare(case, seed):
    gen = torch.Generator("cuda")
    gen.manual_seed(int(seed))
    return _prepare_lora(case, gen) if case["op"] == "lora" else _prepare_moe(case, gen)


# ------------------------------------------------------------------------------------------------------------------------- one pass


def _plain_lora(s):
    x, y, ids = s["x"].float(), s["y"].float(), s["adapter_ids"].long()
    adapters, sections, rank, k = s["a"].shape
    n = y.shape[1]
    mine = (ids[:, None] == torch.arange(adapters, device=ids.device)).float() * s["scaling"]  # [T, L], a row of zeros without an adapter
    inner = (x @ s["a"].float().view(-1, k).T).view(-1, adapters, sections, rank) * mine[:, :, None, None]
    # the columns of a linear read that linear's inner products only
    section = torch.bucketize(torch.arange(n, device=x.device), torch.tensor(s["widths"], device=x.device).cumsum(0), right=True)
    reads = (section[:, None] == torch.arange(sections, device=x.device)).float()  # [N, S]
    b = s["b"].float()[:, :, None, :] * reads[None, :, :, None]  # [L, N, S, R]
    delta = inner.reshape(len(x), -1) @ b.permute(1, 0, 2, 3).reshape(n, -1).T
    return (y + delta).to(s["y"].dtype)


def _decoded(bits, scale):
    """f32 values of stacked e4m3 weights [..., N, K] with scales [..., N] or [..., N / 128, K / 128]."""
    w = bits.view(torch.float8_e4m3fn).float()
    if scale.dim() == bits.dim():
        n, k = bits.shape[-2:]
        return (w.view(*bits.shape[:-2], n // 128, 128, k // 128, 128) * scale[..., :, None, :, None]).view(bits.shape)
    return w * scale[..., None]


def _plain_moe(s):
    x, logits, topk = s["x"].float(), s["router_logits"], s["topk"]
    e = logits.shape[1]
    weight = (logits - logits.amax(dim=1, keepdim=True)).exp()
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :topk]  # of equal logits the lowest id first
    picked = weight.gather(1, ids)
    picked = picked / picked.sum(dim=1, keepdim=True)
    if ids.numel() <= e:  # fewer picks than experts: every pick's own weights
        gate_up = _decoded(s["gate_up"][ids], s["gate_up_scale"][ids])
        gate, up = (gate_up @ x[:, None, :, None])[..., 0].chunk(2, dim=2)  # [T, topk, I]
        rows = _decoded(s["down"][ids], s["down_scale"][ids]) @ (gate / (1 + (-gate).exp()) * up)[..., None]
        out = (rows[..., 0] * picked[:, :, None]).sum(dim=1)
    else:  # every expert on every token, those that the router left out with a weight of zero
        p = torch.zeros_like(logits).scatter(1, ids, picked)
        gate_up = _decoded(s["gate_up"], s["gate_up_scale"]) @ x.T  # [E, 2I, T]
        gate, up = gate_up.chunk(2, dim=1)
        act = gate / (1 + (-gate).exp()) * up * p.T[:, None, :]
        out = (_decoded(s["down"], s["down_scale"]) @ act).sum(dim=0).T
    return out.to(s["x"].dtype)


def run(state):
    if state["op"] == "lora":
        if own:
            from emmy_b200 import ops_lora

            return ops_lora.lora_add(state["y"], state["x"], state["a"], state["b"], state["scaling"], state["adapter_ids"], sections=state["widths"])
        return _plain_lora(state)
    if own:
        from emmy_b200 import ops_moe

        return ops_moe.moe_w8a16(state["x"], state["router_logits"], state["gate_up"], state["gate_up_scale"], state["down"], state["down_scale"], state["topk"])
    return _plain_moe(state)


# ------------------------------------------------------------------------------------------------------------- what a pass needs


def _met(kinds, tries):
    """How many of `kinds` equally likely things are met in `tries`, on average."""
    return kinds * (1 - (1 - 1 / kinds) ** tries)


def work(case):
    if case["op"] == "lora":
        k, widths, rank, tokens = case["k"], _widths(case), case["rank"], case["decode"] + case["prompt"]
        n, sections = sum(widths), len(widths)
        with_one = case["decode"] * (0.875 if case["decode"] > 4 else 1) + case["prompt"]
        adapters = max(_met(case["adapters"], with_one - case["prompt"]), min(case["sequences"], case["adapters"]))
        weights = adapters * rank * (sections * k + n) * 2
        rows = (with_one * k + 2 * tokens * n) * 2
        return {"bytes": weights + rows + 4 * tokens, "flops": 2 * with_one * rank * (sections * k + n)}
    h, i, e, tokens = case["hidden"], case["inter"], case["experts"], case["tokens"]
    touched = e * (1 - (1 - case["topk"] / e) ** tokens)  # experts that at least one token picks
    scales = (3 * i * h / 128 / 128 if case["scales"] == "block" else 2 * i + h) * 4
    return {"bytes": touched * (3 * i * h + scales) + tokens * (4 * h + 4 * e), "flops": 6 * tokens * case["topk"] * i * h}


# ------------------------------------------------------------------------------------------------------------- in 64 bits


def _exact_lora(s):
    out = s["y"].double()
    ids = s["adapter_ids"].tolist()
    edges = [0]
    for w in s["widths"]:
        edges.append(edges[-1] + w)
    for adapter in sorted(set(ids)):
        if adapter < 0:
            continue
        rows = torch.tensor([t for t, l in enumerate(ids) if l == adapter], device=out.device)
        xs = s["x"].index_select(0, rows).double()
        parts = []
        for j in range(len(s["widths"])):
            inner = torch.mm(xs, s["a"][adapter, j].double().t())
            parts.append(torch.mm(inner, s["b"][adapter, edges[j] : edges[j + 1]].double().t()))
        out.index_add_(0, rows, torch.cat(parts, dim=1), alpha=float(s["scaling"][adapter]))
    return out


def _e4m3_values():
    """The 256 values of e4m3: sign, four bits of exponent (bias 7), three of fraction, subnormals at exponent zero."""
    values = []
    for code in range(256):
        exponent, fraction = (code >> 3) & 15, code & 7
        size = fraction * 2.0**-9 if exponent == 0 else (8 + fraction) * 2.0 ** (exponent - 10)
        values.append(math.nan if code & 127 == 127 else -size if code & 128 else size)
    return torch.tensor(values, dtype=torch.float64, device="cuda")


def _exact_moe(s):
    table = _e4m3_values()

    def matrix(bits, scale):
        w = table[bits.long()]
        if scale.dim() == 2:
            return w * scale.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
        return w * scale.double().unsqueeze(1)

    logits = s["router_logits"].double()
    tokens, experts = logits.shape
    picks = {}
    for t, row in enumerate(logits.tolist()):
        best = sorted(range(experts), key=lambda e: (-row[e], e))[: s["topk"]]
        total = sum(math.exp(row[e] - row[best[0]]) for e in best)
        for e in best:
            picks.setdefault(e, []).append((t, math.exp(row[e] - row[best[0]]) / total))
    out = torch.zeros(tokens, s["x"].shape[1], dtype=torch.float64, device="cuda")
    for e, of in sorted(picks.items()):
        rows = torch.tensor([t for t, _ in of], device="cuda")
        share = torch.tensor([p for _, p in of], dtype=torch.float64, device="cuda")
        both = torch.mm(s["x"].index_select(0, rows).double(), matrix(s["gate_up"][e], s["gate_up_scale"][e]).t())
        inter = both.shape[1] // 2
        gate, up = both[:, :inter], both[:, inter:]
        act = gate * torch.sigmoid(gate) * up
        out.index_add_(0, rows, torch.mm(act, matrix(s["down"][e], s["down_scale"][e]).t()) * share.unsqueeze(1))
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_lora(state) if state["op"] == "lora" else _exact_moe(state)
