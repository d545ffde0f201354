"""A step over a paged latent cache that is held in 4 bits: its block tables, its writer and its readers, in their plain form and as this package
offers them.

  extend    extend_block_tables               block tables, slots, positions and lengths of a step, from the lengths of its requests and a stack of free blocks
  release   release_block_tables              the blocks of finished requests go back onto the stack
  insert    fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert    q norm and rotation in place, latent rows to the cache as MXFP4
  paged     paged_latent_attention_mxfp4      a chunk of new tokens (or one per request) over the cache: causal, optionally with a sliding window and a
                                              few first tokens that stay visible, optionally with a sink logit per head
  sparse    sparse_latent_attention_mxfp4     the same for tokens that each bring a list of cache slots

A cached token is 448 e2m1 values in groups of 32 with a power-of-two scale each and 64 bf16 values.  A case is a dict of plain values; `prepare` makes its
tensors on the GPU from a seed, `run` is one pass, `work` what a pass cannot do without and `exact` the result in 64 bits.  `own` says whether `run` calls the
package or computes the plain form.
"""
import os
import random
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
HEAD, NOPE, ROPE, GROUP = 512, 448, 64, 32  # a cached token: 448 e2m1 values in groups of 32, 64 bf16 values
HALF, RECORD, CODES = NOPE // 2, NOPE // 2 + 2 * ROPE, 16  # bytes of a token's 4-bit values, of its data and of its scale codes (14 and two zeros)
BLOCK = 64  # tokens per cache block of the cases that read or write the cache
SCALE = HEAD ** -0.5
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MAX_POSITION = 65536
NO_WINDOW = 0


def listed():
    return [
        # one user generating: the shortest call there is
        {"name": "extend, 1 request", "kind": "extend", "requests": 1, "chunk": 1, "context": 1000, "block": 64, "pad": 0, "short": False, "lens_seed": 1},
        # decode batch of a loaded server, padded to the size that its graph was captured for
        {"name": "extend, 61 requests", "kind": "extend", "requests": 61, "chunk": 1, "context": 16384, "block": 64, "pad": 3, "short": False, "lens_seed": 2},
        # a step of very many requests, prompts among them, with more demand than the pool has blocks
        {"name": "extend, 1021 requests", "kind": "extend", "requests": 1021, "chunk": 127, "context": 4096, "block": 16, "pad": 0, "short": True, "lens_seed": 3},
        # some requests of a decode batch have ended
        {"name": "release, 61 requests", "kind": "release", "requests": 61, "context": 16384, "block": 64, "share": 0.1, "lens_seed": 4},
        # half of a large batch with long contexts is taken back at once
        {"name": "release, 1021 requests", "kind": "release", "requests": 1021, "context": 16384, "block": 16, "share": 0.5, "lens_seed": 5},
        # decode batch, all heads on this GPU
        {"name": "insert, 61 tokens", "kind": "insert", "tokens": 61, "heads": 128, "padding": 0.0},
        # a full prefill chunk with padded rows
        {"name": "insert, 8192 tokens", "kind": "insert", "tokens": 8192, "heads": 128, "padding": 0.1},
        # one user with a long context: one row of work to spread over the whole GPU
        {"name": "decode, 1 request, long", "kind": "paged", "requests": 1, "heads": 128, "chunk": 1, "context": 65536, "window": NO_WINDOW, "first": 0, "sink": True, "lens_seed": 6},
        # decode batch of ragged contexts, heads shared out over two GPUs
        {"name": "decode, 61 requests", "kind": "paged", "requests": 61, "heads": 64, "chunk": 1, "context": 16384, "window": NO_WINDOW, "first": 0, "sink": True, "lens_seed": 7},
        # the largest: a prefill chunk with all heads over a cached prefix, every key visible
        {"name": "chunk, 128 heads, causal", "kind": "paged", "requests": 1, "heads": 128, "chunk": 1024, "context": 8192, "window": NO_WINDOW, "first": 0, "sink": True, "lens_seed": 8},
        # decode batch over the indexer's selection
        {"name": "sparse, 61 tokens", "kind": "sparse", "tokens": 61, "heads": 128, "topk": 512, "context": 32768, "ragged": True, "sink": True},
        # a prefill chunk over the indexer's selection
        {"name": "sparse, 509 tokens", "kind": "sparse", "tokens": 509, "heads": 128, "topk": 2048, "context": 16384, "ragged": True, "sink": True},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["extend", "extend", "release", "insert", "paged", "paged", "sparse"])
    if kind in ("extend", "release"):
        case = {"kind": kind, "requests": _log(rng, 1, 4096), "context": _log(rng, 64, 65536), "block": rng.choice([16, 32, 64, 128, 256]), "lens_seed": rng.randrange(1 << 30)}
        if kind == "release":
            case["share"] = rng.choice([0.02, 0.1, 0.5, 1.0])
        else:
            case |= {"chunk": 1 if rng.random() < 0.4 else _log(rng, 2, 8192), "pad": rng.choice([0, 0, 1, 3, 17]), "short": rng.random() < 0.2}
            case["chunk"] = max(1, min(case["chunk"], 131072 // case["requests"]))
        case["context"] = max(1, min(case["context"], (1 << 20) // case["requests"] * case["block"]))
        return case
    if kind == "insert":
        case = {"kind": kind, "tokens": _log(rng, 1, 16384), "heads": rng.choice([8, 16, 24, 64, 96, 128]), "padding": rng.choice([0.0, 0.1])}
        case["tokens"] = max(1, min(case["tokens"], 8192 * 128 // case["heads"]))
        return case
    if kind == "sparse":
        case = {"kind": kind, "tokens": _log(rng, 1, 1024), "heads": rng.choice([8, 16, 32, 64, 96, 128]), "topk": rng.choice([128, 200, 512, 777, 1024, 2048]),
                "context": _log(rng, 2048, 65536), "ragged": rng.random() < 0.7, "sink": rng.random() < 0.7}
        while case["tokens"] * case["heads"] * case["topk"] > 509 * 128 * 2048 or case["tokens"] * max(case["topk"], case["context"] // 8) > 509 * 2048:
            case["tokens"] = case["tokens"] * 2 // 3
        return case
    windowed = rng.random() < 0.4
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
    """(cached tokens in front of the step, new tokens) of each request: ragged, the first request the longest."""
    r = random.Random(case["lens_seed"])
    n, chunk = case["requests"], case.get("chunk", 0)
    context = [case["context"]] + [max(0, round(case["context"] * r.random())) for _ in range(n - 1)]
    new = [chunk] + [max(1, round(chunk * r.random())) for _ in range(n - 1)]
    return context, new


def _finished(case):
    r = random.Random(case["lens_seed"] + 1)
    return [r.random() < case["share"] for _ in range(case["requests"])]


def _demand(case):
    """Blocks that the requests of an extending step lack, over all of them, and how many of these the pool has."""
    context, new = _lengths(case)
    b = case["block"]
    need = sum(-(-(c + n) // b) - -(-c // b) for c, n in zip(context, new))
    return need, need * 3 // 4 if case["short"] else need + 7


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


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _latent(*shape, g):
    """Latent rows of different magnitude, some channels larger than the others."""
    kv = torch.randn(*shape, HEAD, generator=g, device=DEV) * (0.5 + torch.rand(*shape, 1, generator=g, device=DEV))
    kv[..., 7::64] *= 4
    return kv


def _cache(blocks, g):
    """A cache as the writer leaves it, made in parts, whose 32-bit copies stay small."""
    cache = torch.empty(blocks, BLOCK * (RECORD + CODES), dtype=torch.uint8, device=DEV)
    for at in range(0, blocks, 1024):
        n = min(1024, blocks - at)
        rows, codes = _plain_rows(_latent(n * BLOCK, g=g).to(torch.bfloat16))
        cache[at : at + n, : BLOCK * RECORD] = rows.view(n, -1)
        cache[at : at + n, BLOCK * RECORD :] = codes.view(n, -1)
    return cache


def _queries(tokens, heads, g):
    q = torch.randn(tokens, heads, HEAD, generator=g, device=DEV)
    return (q * q.square().mean(-1, keepdim=True).rsqrt()).to(torch.bfloat16)


def _paged_lists(lens, block, g, spare):
    """Block table [requests, most blocks of a request] of distinct blocks in random order, and the blocks that are left."""
    per_request = [-(-n // block) for n in lens]
    order = torch.randperm(sum(per_request) + spare, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(lens), max(max(per_request), 1), dtype=torch.int32, device=DEV)
    held = torch.arange(table.shape[1], device=DEV) < _int32(per_request)[:, None]
    table[held] = order[: sum(per_request)]
    return table, order[sum(per_request) :].contiguous()


def _prepare_extend(case, g):
    context, new = _lengths(case)
    need, there = _demand(case)
    table, free = _paged_lists(context, case["block"], g, there + 5)
    wide = torch.full((len(context), max(-(-(c + n) // case["block"]) for c, n in zip(context, new)) + 2), -1, dtype=torch.int32, device=DEV)
    wide[:, : table.shape[1]] = table[:, : wide.shape[1]]
    n, t = len(context), sum(new) + case["pad"]
    empty = lambda *shape, of=torch.int32: torch.zeros(*shape, dtype=of, device=DEV)  # noqa: E731
    return {
        "context_lens": _int32(context), "new_lens": _int32(new), "block_table": wide, "free_blocks": free, "num_free": _int32([there]), "tokens": t,
        # what a serving loop keeps from step to step
        "out": (empty(n + 1), empty(n), empty(t, of=torch.int64), empty(t, of=torch.int64), empty(t), empty(1), empty(1)),
    }


def _prepare_release(case, g):
    lens, _ = _lengths(case)
    table, free = _paged_lists(lens, case["block"], g, 11)
    room = torch.zeros(sum(-(-n // case["block"]) for n in lens), dtype=torch.int32, device=DEV)
    return {"seq_lens": _int32(lens), "finished": torch.tensor(_finished(case), device=DEV), "block_table": table,
            "free_blocks": torch.cat([free, room]), "num_free": _int32([11]), "num_free_out": _int32([0])}


def _prepare_insert(case, g):
    t, h = case["tokens"], case["heads"]
    blocks = 2 * -(-t // BLOCK) + 16
    cache = _cache(blocks, g)
    slots = torch.randperm(blocks * BLOCK, generator=g, device=DEV)[:t]
    slots[torch.randperm(t, generator=g, device=DEV)[: int(t * case["padding"])]] = -1
    inv = 10000.0 ** (-torch.arange(0, ROPE, 2, dtype=torch.float64, device=DEV) / ROPE)
    angle = torch.outer(torch.arange(MAX_POSITION, dtype=torch.float64, device=DEV), inv)
    q = torch.empty(t, h, HEAD, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    return {
        "q": q, "kv": _latent(t, g=g).to(torch.bfloat16), "k_cache": cache, "slot_mapping": slots,
        "position_ids": torch.randint(0, MAX_POSITION, (t,), generator=g, device=DEV), "cos_sin": torch.cat((angle.cos(), angle.sin()), -1).float(),
        # the cache's parts under their own types, as what a pass leaves behind: bytes of two e2m1 values each, rotated values, scale codes
        "parts": {"nope": cache[:, : BLOCK * RECORD].view(blocks, BLOCK, RECORD)[..., :HALF],
                  "rope": cache[:, : BLOCK * RECORD].view(blocks, BLOCK, RECORD)[..., HALF:].view(torch.bfloat16),
                  "codes": cache[:, BLOCK * RECORD :].view(blocks, BLOCK, CODES)},
    }


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind in ("extend", "release", "insert"):
        return {"case": case} | {"extend": _prepare_extend, "release": _prepare_release, "insert": _prepare_insert}[kind](case, g)
    if kind == "paged":
        context, new = _lengths(case)
        lens = [c + n for c, n in zip(context, new)]
        table, _ = _paged_lists(lens, BLOCK, g, 3)
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV)
        return {
            "case": case, "q": _queries(sum(new), case["heads"], g), "k_cache": _cache(sum(-(-n // BLOCK) for n in lens) + 3, g), "block_table": table,
            "seq_lens": _int32(lens), "query_start_loc": starts, "attn_sink": torch.randn(case["heads"], generator=g, device=DEV) if case["sink"] else None,
            "out": torch.zeros(sum(new), case["heads"], HEAD, dtype=torch.bfloat16, device=DEV), "lse": torch.zeros(sum(new), case["heads"], device=DEV),
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
        "out": torch.zeros(t, case["heads"], HEAD, dtype=torch.bfloat16, device=DEV), "lse": torch.zeros(t, case["heads"], device=DEV),
    }


# ---- plain forms ----------------------------------------------------------------------------------------------------------


def _plain_extend(s):
    b, table, free, t = s["case"]["block"], s["block_table"], s["free_blocks"], s["tokens"]
    context, new, width = s["context_lens"].long().clamp(min=0), s["new_lens"].long().clamp(min=0), table.shape[1]
    lens, ends = context + new, new.cumsum(0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    has, needs = ((context + b - 1) // b).clamp(max=width), ((lens + b - 1) // b).clamp(max=width)
    takes = needs - has
    before, total = takes.cumsum(0) - takes, takes.sum()
    there = s["num_free"].long().clamp(0, free.numel())
    # table entries: the i-th block that is taken comes from the i-th place below the stack's top
    page = torch.arange(width, device=table.device)
    taken = before[:, None] + page - has[:, None]
    value = torch.where(taken < there, free[(there - 1 - taken).clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where((page >= has[:, None]) & (page < needs[:, None]), value, table))
    # tokens; those behind the last request are padding
    token = torch.arange(t, device=table.device)
    real = token < ends[-1]
    request = torch.where(real, torch.searchsorted(ends, token, right=True).clamp(max=len(lens) - 1), 0)
    position = torch.where(real, context[request] + token - starts[request], 0)
    entry = table[request, (position // b).clamp(max=width - 1)].long()
    slot = torch.where(real & (position // b < width) & (entry >= 0), entry * b + position % b, -1)
    for to, value in zip(s["out"], (starts, lens, position, slot, request, there - torch.minimum(total, there), total - torch.minimum(total, there))):
        to.copy_(value)
    return {"out": s["out"], "block_table": table}


def _plain_release(s):
    b, table, free = s["case"]["block"], s["block_table"], s["free_blocks"]
    held = (torch.arange(table.shape[1], device=table.device) < ((s["seq_lens"].clamp(min=0) + b - 1) // b)[:, None]) & s["finished"][:, None] & (table >= 0)
    held = held.flatten()
    order = held.cumsum(0)
    there, count = s["num_free"].long().clamp(0, free.numel()), order[-1]
    to = torch.where(held, (there + count - order).clamp(max=free.numel()), free.numel())  # the last one is a place for what goes nowhere
    longer = torch.cat([free, free[:1]])
    longer.scatter_(0, to, table.flatten())
    free.copy_(longer[:-1])
    s["num_free_out"].copy_((there + count).clamp(max=free.numel()))
    return {"free_blocks": free, "num_free": s["num_free_out"]}


def _plain_codes(kv):
    """e2m1 codes and scale codes of latent values, [rows, 448] in 32 bits."""
    x = kv.view(kv.shape[0], NOPE // GROUP, GROUP)
    top = x.abs().amax(-1).clamp(min=6 * 2.0 ** -126)
    mantissa, exponent = torch.frexp(top / 6)
    code = torch.where(mantissa == 0.5, exponent - 1, exponent) + 127
    y = torch.ldexp(x, (127 - code).unsqueeze(-1)).abs()
    # round to nearest, ties to the even code
    at = (y > 0.25).byte() + (y >= 0.75).byte() + (y > 1.25).byte() + (y >= 1.75).byte() + (y > 2.5).byte() + (y >= 3.5).byte() + (y > 5).byte()
    return (at + 8 * torch.signbit(x).byte()).view(kv.shape), code.byte()


def _plain_rows(rows):
    """Records and scale codes of bf16 rows whose last 64 values are in place already."""
    codes, scales = _plain_codes(rows[:, :NOPE].float())
    record = torch.cat([codes[:, 0::2] + 16 * codes[:, 1::2], rows[:, NOPE:].contiguous().view(torch.uint8)], -1)
    return record, torch.cat([scales, torch.zeros_like(scales[:, : CODES - NOPE // GROUP])], -1)


def _plain_rotation(x, cos, sin):
    even, odd = x[..., 0::2], x[..., 1::2]
    left, right = even * cos, odd * sin
    other_left, other_right = even * sin, odd * cos
    return torch.stack([left - right, other_left + other_right], -1).flatten(-2)


def _plain_insert(s):
    q, kv, slots, parts = s["q"], s["kv"], s["slot_mapping"], s["parts"]
    cos, sin = s["cos_sin"][s["position_ids"]].split(ROPE // 2, -1)
    x = q.float()
    x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    q[..., :NOPE] = x[..., :NOPE]
    q[..., NOPE:] = _plain_rotation(x[..., NOPE:], cos[:, None], sin[:, None])
    del x
    rows = kv.clone()
    rows[:, NOPE:] = _plain_rotation(kv[:, NOPE:].float(), cos, sin)
    record, codes = _plain_rows(rows)
    # skipped tokens write slot 0 once more: what the token of that slot brings, or what is there
    slot, skipped, of_zero = slots.clamp(min=0), (slots < 0)[:, None], slots == 0
    block, offset = slot // BLOCK, slot % BLOCK
    zero = of_zero.byte().argmax(0, keepdim=True)
    filled = lambda part, value: torch.where(skipped, torch.where(of_zero.any(), value[zero], part[0, 0]), value)  # noqa: E731
    parts["nope"][block, offset] = filled(parts["nope"], record[:, :HALF])
    parts["rope"][block, offset] = filled(parts["rope"], rows[:, NOPE:])
    parts["codes"][block, offset] = filled(parts["codes"], codes)
    return {"q": q, **parts}


def _plain_keys(cache, slot):
    """Latent rows of cache slots, as fp32: [..., 512]."""
    data = cache[:, : BLOCK * RECORD].view(-1, BLOCK, RECORD)[slot // BLOCK, slot % BLOCK]
    codes = cache[:, BLOCK * RECORD :].view(-1, BLOCK, CODES)[slot // BLOCK, slot % BLOCK]
    values = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=cache.device)
    packed = data[..., :HALF].int()
    nope = values[torch.stack([packed & 15, packed >> 4], -1)].view(*slot.shape, NOPE // GROUP, GROUP)
    nope = nope * torch.exp2(codes[..., : NOPE // GROUP].float() - 127).unsqueeze(-1)
    return torch.cat([nope.view(*slot.shape, NOPE), data[..., HALF:].contiguous().view(torch.bfloat16).float()], -1)


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
    kind = case["kind"]
    if kind == "extend":
        fg.extend_block_tables(s["context_lens"], s["new_lens"], s["block_table"], s["free_blocks"], s["num_free"], case["block"], s["tokens"], s["out"])
        return {"out": s["out"], "block_table": s["block_table"]}
    if kind == "release":
        fg.release_block_tables(s["seq_lens"], s["finished"], s["block_table"], s["free_blocks"], s["num_free"], case["block"], s["num_free_out"])
        return {"free_blocks": s["free_blocks"], "num_free": s["num_free_out"]}
    if kind == "insert":
        fg.fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert(s["q"], s["kv"], s["k_cache"], s["slot_mapping"], s["position_ids"], s["cos_sin"], EPS, BLOCK)
        return {"q": s["q"], **s["parts"]}
    if kind == "paged":
        fg.paged_latent_attention_mxfp4(s["q"], s["k_cache"], s["block_table"], s["seq_lens"], s["query_start_loc"], BLOCK, SCALE,
                                        case["window"] or None, case["first"], s["attn_sink"], s["out"], s["lse"])
    else:
        fg.sparse_latent_attention_mxfp4(s["q"], s["k_cache"], s["indices"], s["lens"], BLOCK, SCALE, s["attn_sink"], s["out"], s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def run(s):
    if own:
        return _own(s)
    return {"extend": _plain_extend, "release": _plain_release, "insert": _plain_insert, "paged": _plain_paged, "sparse": _plain_sparse}[s["case"]["kind"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "extend":
        tokens, taken = sum(_lengths(case)[1]) + case["pad"], _demand(case)
        return {"bytes": 16 * case["requests"] + 20 * tokens + 4 * min(taken) + 4 * taken[0] + 16, "flops": 0}
    if kind == "release":
        blocks = sum(-(-n // case["block"]) for n, done in zip(_lengths(case)[0], _finished(case)) if done)
        return {"bytes": 5 * case["requests"] + 8 * blocks + 8, "flops": 0}
    if kind == "insert":
        t, h = case["tokens"], case["heads"]
        inserted = t - int(t * case["padding"])
        return {"bytes": t * (2 * 2 * HEAD * h + 8 + 4 * ROPE + 8) + inserted * (2 * HEAD + RECORD + CODES), "flops": 4 * t * h * HEAD}
    heads = case["heads"]
    if kind == "paged":
        union, pairs = _visible(case)
        tokens, pairs, table = sum(_lengths(case)[1]), sum(pairs), sum(-(-u // BLOCK) for u in union)
        cached = sum(union) * (RECORD + CODES) + 4 * table + 8 * len(union)
    else:
        tokens, k = case["tokens"], min(case["topk"], case["context"])
        mean = k * (3 * k - 1) / 2 / (2 * k - 1) if case["ragged"] else k  # of min(k, one of 1 .. 2k - 1)
        pairs = tokens * mean
        cached = min(pairs, case["context"]) * (RECORD + CODES) + 4 * pairs + 4 * tokens
    return {"bytes": tokens * heads * (2 * 2 * HEAD + 4) + cached, "flops": 4 * HEAD * heads * pairs}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------------


def _exact_extend(s):
    """The definition as a loop over requests on the host."""
    b, width, table, free = s["case"]["block"], s["block_table"].shape[1], s["block_table"].tolist(), s["free_blocks"].tolist()
    stack, missing, starts, lens, positions, slots, requests = free[: s["num_free"].item()], 0, [0], [], [], [], []
    for r, (c, n) in enumerate(zip(s["context_lens"].tolist(), s["new_lens"].tolist())):
        for page in range(-(-c // b), min(-(-(c + n) // b), width)):
            table[r][page] = stack.pop() if stack else -1
            missing += table[r][page] < 0
        for p in range(c, c + n):
            positions.append(p), requests.append(r)
            slots.append(table[r][p // b] * b + p % b if p // b < width and table[r][p // b] >= 0 else -1)
        starts.append(starts[-1] + n), lens.append(c + n)
    pad = [0] * (s["tokens"] - len(positions))
    lists = (starts, lens, positions + pad, slots + [-1] * len(pad), requests + pad, [len(stack)], [missing])
    return {"out": [torch.tensor(v, dtype=t.dtype, device=DEV) for v, t in zip(lists, s["out"])], "block_table": _int32(table)}


def _exact_release(s):
    b, table, stack = s["case"]["block"], s["block_table"].tolist(), s["free_blocks"].tolist()
    back = [e for r, done in enumerate(s["finished"].tolist()) if done for e in table[r][: -(-s["seq_lens"][r].item() // b)] if e >= 0]
    n = s["num_free"].item()
    stack[n : n + len(back)] = back[::-1]
    return {"free_blocks": _int32(stack), "num_free": _int32([n + len(back)])}


def _exact_rotation(x, position):
    """Pairs (2j, 2j + 1) turned by position / 10000^(2j / 64)."""
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV), position.double()[:, None] / 10000.0 ** (torch.arange(0, ROPE, 2, device=DEV).double() / ROPE))
    pairs = torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous())
    return torch.view_as_real(pairs * turn.view(turn.shape[0], *[1] * (x.dim() - 2), -1)).flatten(-2)


def _exact_insert(s):
    q, kv, slots = s["q"].double(), s["kv"].double(), s["slot_mapping"]
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) / HEAD + EPS)
    q[..., NOPE:] = _exact_rotation(q[..., NOPE:], s["position_ids"])
    nope, rope, codes = s["parts"]["nope"].clone(), s["parts"]["rope"].double(), s["parts"]["codes"].clone()
    there = slots >= 0
    block, offset = slots[there] // BLOCK, slots[there] % BLOCK
    x = kv[there, :NOPE].view(-1, NOPE // GROUP, GROUP)
    power = torch.ceil(torch.log2(x.abs().amax(-1).clamp(min=6 * 2.0 ** -126) / 6))
    code = ((x / torch.exp2(power)[..., None]).abs()[..., None] - torch.tensor(E2M1, dtype=torch.float64, device=DEV)).abs()
    near = code == code.amin(-1, keepdim=True)
    # the nearest value; of two that are as near, the one with an even code
    best = (near.double() * (2 - torch.arange(8, device=DEV) % 2)).argmax(-1) + 8 * torch.signbit(x)
    best = best.view(-1, HALF, 2)
    nope[block, offset] = (best[..., 0] + 16 * best[..., 1]).byte()
    rope[block, offset] = _exact_rotation(kv[there, NOPE:], s["position_ids"][there])
    codes[block, offset] = torch.nn.functional.pad(power + 127, (0, CODES - NOPE // GROUP)).byte()
    return {"q": q, "nope": nope, "rope": rope, "codes": codes}


def _exact_keys(cache, slots):
    values, raw = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=DEV), cache.view(cache.shape[0], -1)
    block, offset = slots // BLOCK, slots % BLOCK
    byte = lambda start, n, pitch: raw[block[:, None], start + pitch * offset[:, None] + torch.arange(n, device=DEV)].long()  # noqa: E731
    packed = byte(0, HALF, RECORD)
    nope = torch.empty(len(slots), NOPE, dtype=torch.float64, device=DEV)
    nope[:, 0::2], nope[:, 1::2] = values[packed % 16], values[packed // 16]
    code = byte(BLOCK * RECORD, NOPE // GROUP, CODES)
    half = byte(HALF, 2 * ROPE, RECORD)
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
    if case["kind"] in ("extend", "release", "insert"):
        return {"extend": _exact_extend, "release": _exact_release, "insert": _exact_insert}[case["kind"]](s)
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
