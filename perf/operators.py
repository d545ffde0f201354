"""The operators that close a DeepSeek-V4 attention layer, in their plain form and as this package offers them.

  norm     fused_add_rmsnorm_quant_fp8   residual addition, weighted RMS norm and e4m3 output with scales: the way into the FP8 projections
  paged    paged_latent_attention        a chunk of new tokens (or one per request) over the paged latent cache: causal, optionally with a
                                         sliding window and a few first tokens that stay visible, optionally with a sink logit per head
  sparse   sparse_latent_attention       the same for tokens that each bring a list of cache slots, as the index operators make them

A case is a dict of plain values; `prepare` makes its tensors on the GPU from a seed, `run` is one pass, `work` what a pass cannot do
without and `exact` the result in 64 bits.  `own` says whether `run` calls the package or computes the plain form.
"""
import os
import random
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
HEAD, NOPE, ROPE, GROUP = 512, 448, 64, 64  # a cached token: 448 e4m3 values in groups of 64, 64 bf16 values
RECORD, CODES = NOPE + 2 * ROPE, 8  # bytes of a token's data and of its scale codes
BLOCK = 64  # tokens per cache block
SCALE = HEAD ** -0.5
FP8_MAX, QUANT_EPS = 448.0, 1e-10
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NO_WINDOW = 0


def listed():
    return [
        # one user generating: the shortest call there is
        {"name": "norm, 1 token", "kind": "norm", "tokens": 1, "hidden": 7168, "group": 128, "type": "bf16", "pow2": True, "column_major": False},
        # decode batch of a loaded server, scales laid out as the projection's product takes them
        {"name": "norm, 61 tokens", "kind": "norm", "tokens": 61, "hidden": 7168, "group": 128, "type": "bf16", "pow2": False, "column_major": True},
        # an odd-sized prefill chunk
        {"name": "norm, 4097 tokens", "kind": "norm", "tokens": 4097, "hidden": 7168, "group": 128, "type": "bf16", "pow2": True, "column_major": True},
        # a full prefill chunk of a model with half-precision activations, one scale per token
        {"name": "norm, 8192 tokens, fp16", "kind": "norm", "tokens": 8192, "hidden": 4096, "group": 4096, "type": "fp16", "pow2": False, "column_major": False},
        # one user generating with the sliding-window layer: the least an attention call can have to do
        {"name": "decode, 1 request, window", "kind": "paged", "requests": 1, "heads": 64, "chunk": 1, "context": 1000, "window": 128, "first": 4, "sink": True, "lens_seed": 1},
        # one user with a long context: one row of work to spread over the whole GPU
        {"name": "decode, 1 request, long", "kind": "paged", "requests": 1, "heads": 128, "chunk": 1, "context": 65536, "window": NO_WINDOW, "first": 0, "sink": True, "lens_seed": 2},
        # decode batch of ragged contexts, heads shared out over two GPUs
        {"name": "decode, 61 requests", "kind": "paged", "requests": 61, "heads": 64, "chunk": 1, "context": 16384, "window": NO_WINDOW, "first": 0, "sink": True, "lens_seed": 3},
        # a prefill chunk of three requests behind cached prefixes, heads shared out over eight GPUs
        {"name": "chunk, 3 requests, 16 heads", "kind": "paged", "requests": 3, "heads": 16, "chunk": 1021, "context": 4096, "window": NO_WINDOW, "first": 0, "sink": False, "lens_seed": 4},
        # a prefill chunk in a sliding-window layer
        {"name": "chunk, window", "kind": "paged", "requests": 2, "heads": 64, "chunk": 2048, "context": 8192, "window": 512, "first": 16, "sink": True, "lens_seed": 5},
        # the largest: a prefill chunk with all heads over a cached prefix, every key visible
        {"name": "chunk, 128 heads, causal", "kind": "paged", "requests": 1, "heads": 128, "chunk": 1024, "context": 8192, "window": NO_WINDOW, "first": 0, "sink": True, "lens_seed": 6},
        # decode batch over the indexer's selection
        {"name": "sparse, 61 tokens", "kind": "sparse", "tokens": 61, "heads": 128, "topk": 512, "context": 32768, "ragged": True, "sink": True},
        # a prefill chunk over the indexer's selection
        {"name": "sparse, 509 tokens", "kind": "sparse", "tokens": 509, "heads": 128, "topk": 2048, "context": 16384, "ragged": True, "sink": True},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["norm", "paged", "paged", "sparse"])
    if kind == "norm":
        group = rng.choice([64, 128, 256, 0])
        hidden = 256 * rng.randint(4, 32)
        case = {"kind": kind, "tokens": _log(rng, 1, 8192), "hidden": hidden, "group": group or hidden, "type": rng.choice(["bf16", "fp16"]),
                "pow2": rng.random() < 0.5, "column_major": rng.random() < 0.5}
        case["tokens"] = max(1, min(case["tokens"], 8192 * 4096 // hidden))
        return case
    if kind == "sparse":
        case = {"kind": kind, "tokens": _log(rng, 1, 1024), "heads": rng.choice([8, 16, 32, 64, 96, 128]), "topk": rng.choice([128, 200, 512, 777, 1024, 2048]),
                "context": _log(rng, 2048, 65536), "ragged": rng.random() < 0.7, "sink": rng.random() < 0.7}
        while case["tokens"] * case["heads"] * case["topk"] > 509 * 128 * 2048 or case["tokens"] * max(case["topk"], case["context"] // 8) > 509 * 2048:
            case["tokens"] = case["tokens"] * 2 // 3
        return case
    windowed = rng.random() < 0.5
    case = {"kind": kind, "requests": _log(rng, 1, 64), "heads": rng.choice([8, 16, 24, 32, 64, 96, 128]), "chunk": 1 if rng.random() < 0.5 else _log(rng, 2, 2048),
            "context": _log(rng, 64, 65536), "window": _log(rng, 32, 4096) if windowed else NO_WINDOW, "first": rng.choice([0, 1, 4, 16, 64]) if windowed else 0,
            "sink": rng.random() < 0.7, "lens_seed": rng.randrange(1 << 30)}
    rows = lambda: case["requests"] * case["chunk"] * case["heads"]  # noqa: E731
    keys = lambda: (min(case["context"], case["window"] + case["first"]) if windowed else case["context"]) + case["chunk"]  # noqa: E731
    while rows() * keys() > 1024 * 128 * 9000 or case["requests"] * (case["context"] + case["chunk"]) > 1 << 20:
        name = max(("requests", "chunk", "context"), key=lambda k: case[k] / {"requests": 2, "chunk": 64, "context": 2048}[k])
        case[name] = max(1, case[name] * 2 // 3)
    return case


def _lengths(case):
    """(cached tokens in front of the chunk, new tokens) of each request: ragged, the first request the longest."""
    r = random.Random(case["lens_seed"])
    n = case["requests"]
    context = [case["context"]] + [max(0, round(case["context"] * r.random())) for _ in range(n - 1)]
    new = [case["chunk"]] + [max(1, round(case["chunk"] * r.random())) for _ in range(n - 1)]
    return context, new


def _visible(case):
    """Keys that any new token of a request sees, and the sum over its new tokens of the keys that they see."""
    context, new = _lengths(case)
    window, first = case["window"], case["first"]
    union, pairs = [], []
    for c, n in zip(context, new):
        if window == NO_WINDOW:
            union.append(c + n)
            pairs.append(sum(range(c + 1, c + n + 1)))
        else:
            low = max(0, c - window + 1)
            union.append(c + n - low + min(first, low))
            pairs.append(sum(p + 1 - max(0, p - window + 1) + min(first, max(0, p - window + 1)) for p in range(c, c + n)))
    return union, pairs


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _cache(blocks, g):
    """A cache as the prologue leaves it: normally distributed latent rows of different magnitude, quantised in groups."""
    cache = torch.empty(blocks, BLOCK * (RECORD + CODES), dtype=torch.uint8, device=DEV)
    for at in range(0, blocks, 1024):
        n = min(1024, blocks - at)
        kv = torch.randn(n, BLOCK, HEAD, generator=g, device=DEV) * (0.5 + torch.rand(n, BLOCK, 1, generator=g, device=DEV))
        nope = kv[..., :NOPE].to(torch.bfloat16).float().view(n, BLOCK, NOPE // GROUP, GROUP)
        code = torch.ceil(torch.log2(nope.abs().amax(-1).clamp(min=1e-4) / FP8_MAX)) + 127
        values = (nope / torch.exp2(code - 127).unsqueeze(-1)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
        data = cache[at : at + n, : BLOCK * RECORD].view(n, BLOCK, RECORD)
        data[..., :NOPE] = values.view(n, BLOCK, NOPE).view(torch.uint8)
        data[..., NOPE:] = kv[..., NOPE:].to(torch.bfloat16).view(torch.uint8)
        codes = cache[at : at + n, BLOCK * RECORD :].view(n, BLOCK, CODES)
        codes[..., :7] = code.to(torch.uint8)
        codes[..., 7] = 0
    return cache


def _queries(tokens, heads, g):
    q = torch.randn(tokens, heads, HEAD, generator=g, device=DEV)
    return (q * q.square().mean(-1, keepdim=True).rsqrt()).to(torch.bfloat16)


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "norm":
        t, n, kind = case["tokens"], case["hidden"], TYPES[case["type"]]
        magnitude = torch.exp(0.5 * torch.randn(n, generator=g, device=DEV))  # channels of different size, as hidden states have
        return {
            "case": case,
            "x": (torch.randn(t, n, generator=g, device=DEV) * magnitude).to(kind),
            "residual": (2 * torch.randn(t, n, generator=g, device=DEV) * magnitude).to(kind),
            "weight": (1 + 0.2 * torch.randn(n, generator=g, device=DEV)).to(kind),
            "fp8_max": torch.tensor(FP8_MAX, device=DEV),
        }
    if case["kind"] == "paged":
        context, new = _lengths(case)
        lens = [c + n for c, n in zip(context, new)]
        per_request = [-(-n // BLOCK) for n in lens]
        blocks = sum(per_request) + 3
        order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
        table = torch.zeros(len(lens), max(per_request), dtype=torch.int32, device=DEV)
        at = 0
        for r, n in enumerate(per_request):
            table[r, :n] = order[at : at + n]
            at += n
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV)
        return {
            "case": case, "q": _queries(sum(new), case["heads"], g), "k_cache": _cache(blocks, g), "block_table": table,
            "seq_lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "query_start_loc": starts,
            "attn_sink": torch.randn(case["heads"], generator=g, device=DEV) if case["sink"] else None,
            "out": torch.zeros(sum(new), case["heads"], HEAD, dtype=torch.bfloat16, device=DEV),
            "lse": torch.zeros(sum(new), case["heads"], device=DEV),
            "most_new": max(new), "most_keys": max(_visible(case)[0]),
        }
    t, k, context = case["tokens"], case["topk"], case["context"]
    blocks = -(-context // BLOCK) + 3
    order = torch.randperm(blocks, generator=g, device=DEV)
    chosen = torch.stack([torch.randperm(context, generator=g, device=DEV)[:k] for _ in range(min(t, 32))])  # distinct positions per token
    chosen = ((chosen.repeat(-(-t // 32) if t > 32 else 1, 1)[:t] + torch.randint(0, context, (t, 1), generator=g, device=DEV)) % context)
    indices = torch.full((t, k), -1, dtype=torch.int32, device=DEV)
    indices[:, : chosen.shape[1]] = (order[chosen // BLOCK] * BLOCK + chosen % BLOCK).to(torch.int32)
    lens = torch.full((t,), chosen.shape[1], device=DEV)
    if case["ragged"]:
        lens = torch.minimum(lens, torch.randint(1, 2 * k, (t,), generator=g, device=DEV))
    indices.masked_fill_(torch.arange(k, device=DEV) >= lens[:, None], -1)
    return {
        "case": case, "q": _queries(t, case["heads"], g), "k_cache": _cache(blocks, g), "indices": indices, "lens": lens.to(torch.int32),
        "attn_sink": torch.randn(case["heads"], generator=g, device=DEV) if case["sink"] else None,
        "out": torch.zeros(t, case["heads"], HEAD, dtype=torch.bfloat16, device=DEV),
        "lse": torch.zeros(t, case["heads"], device=DEV),
    }


# ---- plain forms ----------------------------------------------------------------------------------------------------------


def _plain_norm(s):
    case, x, residual = s["case"], s["x"], s["residual"]
    z = x.float() + residual.float()
    residual.copy_(z)
    # the row's statistic in 64 bits: a power-of-two scale lies next to a border that the last bit of 32 would move values across
    r = (z.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float()
    y = (z * r * s["weight"].float()).view(z.shape[0], -1, case["group"])
    scale = y.abs().amax(-1).clamp(min=QUANT_EPS) / s["fp8_max"]
    if case["pow2"]:
        mantissa, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), torch.where(mantissa == 0.5, exponent - 1, exponent))
    x_q = (y / scale.unsqueeze(-1)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(z.shape)
    return {"x_q": x_q, "scales": scale.t().contiguous().t() if case["column_major"] else scale, "residual": residual}


def _plain_keys(cache, slot):
    """Latent rows of cache slots, as fp32: [..., 512]."""
    data = cache[:, : BLOCK * RECORD].view(-1, BLOCK, RECORD)[slot // BLOCK, slot % BLOCK]
    codes = cache[:, BLOCK * RECORD :].view(-1, BLOCK, CODES)[slot // BLOCK, slot % BLOCK]
    nope = data[..., :NOPE].view(torch.float8_e4m3fn).float().view(*slot.shape, NOPE // GROUP, GROUP)
    nope = nope * torch.exp2(codes[..., :7].float() - 127).unsqueeze(-1)
    return torch.cat([nope.view(*slot.shape, NOPE), data[..., NOPE:].contiguous().view(torch.bfloat16).float()], -1)


def _plain_softmax(scores, visible, sink):
    """Weights of the visible keys (all zero in a row without any) and the log of the sum of the keys' exponentials."""
    scores = scores.masked_fill(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    lse = (total.log() + top).squeeze(-1)
    if sink is not None:
        total = total + torch.exp(sink - top)
    return torch.where(total > 0, e / total, torch.zeros_like(e)), lse


def _plain_paged(s):
    case, q, starts = s["case"], s["q"], s["query_start_loc"].long()
    lens, heads = s["seq_lens"].long()[:, None], case["heads"]
    new = (starts[1:] - starts[:-1])[:, None]
    context = lens - new
    # the keys that some new token of a request sees, as one list per request
    k = torch.arange(s["most_keys"], device=q.device)
    low = (context - case["window"] + 1).clamp(min=0) if case["window"] else torch.zeros_like(context)
    first = low.clamp(max=case["first"])
    position = torch.where(k < first, k, k - first + low)
    live = position < lens
    at = position.clamp(max=s["block_table"].shape[1] * BLOCK - 1)
    slot = s["block_table"].long().gather(1, at // BLOCK) * BLOCK + at % BLOCK
    keys = _plain_keys(s["k_cache"], torch.where(live, slot, 0))
    # queries of a request side by side
    i = torch.arange(s["most_new"], device=q.device)
    token = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    queries = q[token].float()  # [requests, most_new, heads, 512]
    scores = torch.matmul(queries.view(len(lens), -1, HEAD), keys.transpose(1, 2)).view(len(lens), -1, heads, k.numel()) * SCALE
    mine = (context + i)[:, :, None]
    visible = live[:, None] & (position[:, None] <= mine)
    if case["window"]:
        visible &= (position[:, None] > mine - case["window"]) | (position[:, None] < case["first"])
    sink = None if s["attn_sink"] is None else s["attn_sink"][:, None]
    weights, lse = _plain_softmax(scores, visible[:, :, None], sink)
    out = torch.matmul(weights.view(len(lens), -1, k.numel()), keys).view(queries.shape)
    t = torch.arange(q.shape[0], device=q.device)
    request = torch.searchsorted(starts[1:], t, right=True)
    s["out"].copy_(out[request, t - starts[request]])
    s["lse"].copy_(lse[request, t - starts[request]])
    return {"out": s["out"], "lse": s["lse"]}


def _plain_sparse(s):
    q, indices = s["q"].float(), s["indices"].long()
    visible = (indices >= 0) & (torch.arange(indices.shape[1], device=q.device) < s["lens"][:, None])
    keys = _plain_keys(s["k_cache"], indices.clamp(min=0))
    scores = torch.matmul(q, keys.transpose(1, 2)) * SCALE
    sink = None if s["attn_sink"] is None else s["attn_sink"][:, None]
    weights, lse = _plain_softmax(scores, visible[:, None], sink)
    s["out"].copy_(torch.matmul(weights, keys))
    s["lse"].copy_(lse)
    return {"out": s["out"], "lse": s["lse"]}


# ---- the package's calls --------------------------------------------------------------------------------------------------


def _package():
    here = os.path.abspath("flaggems-vllm_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import flaggems_vllm

    return flaggems_vllm


def _own(s):
    fg, case = _package(), s["case"]
    if case["kind"] == "norm":
        x_q, scales = fg.fused_add_rmsnorm_quant_fp8(s["x"], s["residual"], s["weight"], EPS, case["group"], case["column_major"], case["pow2"])
        return {"x_q": x_q, "scales": scales, "residual": s["residual"]}
    if case["kind"] == "paged":
        fg.paged_latent_attention(s["q"], s["k_cache"], s["block_table"], s["seq_lens"], s["query_start_loc"], BLOCK, SCALE,
                                  case["window"] or None, case["first"], s["attn_sink"], s["out"], s["lse"])
    else:
        fg.sparse_latent_attention(s["q"], s["k_cache"], s["indices"], s["lens"], BLOCK, SCALE, s["attn_sink"], s["out"], s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def run(s):
    if own:
        return _own(s)
    return {"norm": _plain_norm, "paged": _plain_paged, "sparse": _plain_sparse}[s["case"]["kind"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "norm":
        t, n = case["tokens"], case["hidden"]
        return {"bytes": t * n * (2 + 2 + 2 + 1) + 2 * n + 4 * t * (n // case["group"]), "flops": 8 * t * n}
    heads = case["heads"]
    if case["kind"] == "paged":
        union, pairs = _visible(case)
        context, new = _lengths(case)
        tokens, pairs, table = sum(new), sum(pairs), sum(-(-u // BLOCK) for u in union)
        cached = sum(union) * (RECORD + CODES) + 4 * table + 8 * len(new)
    else:
        tokens, k = case["tokens"], min(case["topk"], case["context"])
        mean = k * (3 * k - 1) / 2 / (2 * k - 1) if case["ragged"] else k  # of min(k, one of 1 .. 2k - 1)
        pairs = tokens * mean
        cached = min(pairs, case["context"]) * (RECORD + CODES) + 4 * pairs + 4 * tokens
    return {"bytes": tokens * heads * (2 * 2 * HEAD + 4) + cached, "flops": 4 * HEAD * heads * pairs}


# ---- in 64 bits, from the definitions -------------------------------------------------------------------------------------


def _e4m3_values():
    """The value of every e4m3 byte: sign, four exponent bits of bias 7, three of mantissa; 0x7f and 0xff are NaN."""
    magnitude = [m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)]
    magnitude[127] = float("nan")
    return torch.tensor(magnitude + [-v for v in magnitude], dtype=torch.float64, device=DEV)


def _exact_keys(cache, slots):
    table, raw = _e4m3_values(), cache.view(cache.shape[0], -1)
    block, offset = slots // BLOCK, slots % BLOCK
    byte = lambda start, n, pitch: raw[block[:, None], start + pitch * offset[:, None] + torch.arange(n, device=DEV)].long()  # noqa: E731
    nope = table[byte(0, NOPE, RECORD)]
    code = byte(BLOCK * RECORD, 7, CODES)
    half = byte(NOPE, 2 * ROPE, RECORD)
    bits = ((half[:, 0::2] + 256 * half[:, 1::2]) << 16).to(torch.int64)
    rope = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32).view(torch.float32).double()
    return torch.cat([nope * torch.exp2(code.double() - 127).repeat_interleave(GROUP, 1), rope], 1)


def _exact_rows(q, keys, hidden, sink):
    """Attention of [n, heads, 512] queries over [k, 512] keys; `hidden` [n, k] marks what a row does not see."""
    score = (q.double().reshape(-1, HEAD) @ keys.t()).view(q.shape[0], q.shape[1], -1) * SCALE
    score.masked_fill_(hidden[:, None], float("-inf"))
    lse = torch.logsumexp(score, -1)
    total = lse if sink is None else torch.logaddexp(lse, sink.double()[None].expand_as(lse))
    weight = torch.exp(score - total[..., None]).nan_to_num(0.0)
    return (weight.view(-1, keys.shape[0]) @ keys).view(q.shape), lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        z = s["x"].double() + s["residual"].double()
        y = z / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS) * s["weight"].double()
        y = y.view(z.shape[0], -1, case["group"])
        scale = y.abs().amax(-1).clamp(min=QUANT_EPS) / FP8_MAX
        if case["pow2"]:
            scale = torch.exp2(torch.ceil(torch.log2(scale)))
        return {"x_q": (y / scale[..., None]).view(z.shape), "scales": scale, "residual": z}
    outs, lses = [], []
    if case["kind"] == "paged":
        context, new = _lengths(case)
        at = 0
        for r, (c, n) in enumerate(zip(context, new)):
            position = torch.arange(c + n, device=DEV)
            keys = _exact_keys(s["k_cache"], s["block_table"][r].long()[position // BLOCK] * BLOCK + position % BLOCK)
            for i in range(0, n, 64):
                mine = torch.arange(c + i, c + min(n, i + 64), device=DEV)[:, None]
                hidden = position > mine
                if case["window"]:
                    hidden |= (position <= mine - case["window"]) & (position >= case["first"])
                o, l = _exact_rows(s["q"][at + i : at + min(n, i + 64)], keys, hidden, s["attn_sink"])
                outs.append(o)
                lses.append(l)
            at += n
    else:
        for t, n in enumerate(s["lens"].tolist()):
            keys = _exact_keys(s["k_cache"], s["indices"][t, :n].long())
            o, l = _exact_rows(s["q"][t : t + 1], keys, torch.zeros(1, n, dtype=torch.bool, device=DEV), s["attn_sink"])
            outs.append(o)
            lses.append(l)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
