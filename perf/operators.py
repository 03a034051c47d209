"""What is timed of the operators around a paged KV layer: one layer's share of a serving step.

A paged KV layer is a tensor (2, num_blocks, block_tokens, kv_heads, head_dim), K plane then V
plane; a request's block table lists its blocks in token order. A step gives every request some
new tokens behind those that its blocks hold already. A case's ``kind`` names the operator:

* ``plan``    the step's tables from the requests' lengths: fresh blocks from the free list into
              the block tables, the row ranges of the packed tokens, and each token's slot
              (block * block_tokens + place in the block) and position
* ``write``   the new tokens' K and V rows into the layer, by slot (-1: no slot, no write)
* ``chunk``   attention of the new tokens over the layer, causal: the last of a request's n rows
              sees its whole context, the one before it one token less, and so on
* ``prompt``  causal attention of whole prompts packed one behind the other, over their own K and
              V rows, before any of them is in the layer

Query heads share the KV heads in equal groups (query head h reads KV head h // group). The
softmax scale is head_dim ** -0.5.

A request's lengths are spread log-uniformly by the case's own ``spread`` seed, so that a case
costs the same whatever its inputs are.

Ranges: 1 to 8 KV heads, groups of 1 to 8, head dims 64 and 128, bf16 and fp16, blocks of 8 to 32
tokens, 1 to 256 requests, contexts of 1 to 32768 tokens, chunks of 1 to 2048 tokens, prompts of 1
to 16384; at most 4.5e9 scores of the padded plain form and 2 GiB of keys and values a layer.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_MOST_SCORES = 4.5e9
_MOST_KV = 2 << 30


# ---------------------------------------------------------------------------
# cases

def _plan(name, requests, longs, new, lo, hi, block, spread=1):
    """``longs`` of the requests have up to ``new`` new tokens, the others one."""
    case = {"kind": "plan", "requests": requests, "longs": longs, "new": new, "lo": lo, "hi": hi,
            "block": block, "spread": spread}
    return dict(case, name=name) if name else case


def _write(name, requests, lo, hi, kv_heads, head_dim, block, dtype="bf16", spread=1):
    case = {"kind": "write", "requests": requests, "lo": lo, "hi": hi, "kv_heads": kv_heads,
            "head_dim": head_dim, "block": block, "dtype": dtype, "spread": spread}
    return dict(case, name=name) if name else case


def _chunk(name, requests, longs, new, lo, hi, q_heads, kv_heads, head_dim, block, dtype="bf16",
           spread=1):
    case = {"kind": "chunk", "requests": requests, "longs": longs, "new": new, "lo": lo, "hi": hi,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
            "dtype": dtype, "spread": spread}
    return dict(case, name=name) if name else case


def _prompt(name, requests, lo, hi, q_heads, kv_heads, head_dim, dtype="bf16", spread=1):
    case = {"kind": "prompt", "requests": requests, "lo": lo, "hi": hi, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "spread": spread}
    return dict(case, name=name) if name else case


def listed():
    return [
        # a decode step of a serving batch: one new token a request, few fresh blocks
        _plan("plan_decode", 64, 0, 1, 128, 32768, 16, spread=3),
        # a step that mixes long chunks of prompts with many single tokens
        _plan("plan_mixed", 256, 16, 2048, 16, 32768, 16, spread=2),
        # the tokens of a decode step of an 8B model
        _write("write_decode", 64, 1, 1, 8, 128, 16),
        # a prefill batch of an 8B model
        _write("write_prefill", 8, 4096, 4096, 8, 128, 16),
        # one user of a small model: latency alone
        _chunk("decode_single", 1, 0, 1, 1024, 1024, 32, 8, 64, 16),
        # a full decode batch of an 8B model at one context length
        _chunk("decode_batch", 32, 0, 1, 8192, 8192, 32, 8, 128, 16),
        # one GPU's share of a 70B model under tensor parallelism, mixed contexts
        _chunk("decode_mixed", 64, 0, 1, 128, 32768, 8, 1, 128, 16, spread=3),
        # a few drafted tokens a request, to be verified together
        _chunk("chunk_drafts", 16, 16, 6, 300, 8000, 32, 8, 128, 16, dtype="fp16", spread=4),
        # chunked prefill beside decodes: chunks of prompts behind what their blocks hold
        _chunk("chunk_mixed", 32, 3, 2048, 500, 16000, 32, 8, 128, 16, spread=5),
        # a prefill batch of an 8B model
        _prompt("prompt_batch", 8, 4096, 4096, 32, 8, 128),
        # short and odd prompts of a small model
        _prompt("prompt_ragged", 24, 3, 2050, 32, 8, 64, dtype="fp16", spread=9),
        # one long prompt, one GPU's share of a 70B model
        _prompt("prompt_long", 1, 16384, 16384, 8, 1, 128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above."""
    while True:
        kind = rng.choice(("plan", "write", "chunk", "chunk", "chunk", "prompt", "prompt"))
        requests = _log_int(rng, 1, 256 if kind == "plan" else 64)
        block = rng.choice((8, 16, 16, 32, 24))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        head_dim = rng.choice((64, 128, 128))
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        q_heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 7, 8))
        spread = rng.randrange(1, 1 << 20)
        longs = rng.choice((0, 0, 1, _log_int(rng, 1, 16)))
        longs = min(longs, requests)
        new = _log_int(rng, 2, 2048) if longs else 1
        lo = _log_int(rng, max(new, 16), 16384)
        hi = _log_int(rng, lo, 32768)
        if kind == "plan":
            return _plan(None, requests, longs, new, lo, hi, block, spread)
        if kind == "write":
            lo = _log_int(rng, 1, 4096)
            case = _write(None, requests, lo, _log_int(rng, lo, 4096), kv_heads, head_dim, block,
                          dtype, spread)
            if sum(_lengths(case)[0]) <= 32768:
                return case
            continue
        if kind == "chunk":
            case = _chunk(None, requests, longs, new, lo, hi, q_heads, kv_heads, head_dim, block,
                          dtype, spread)
        else:
            lo = _log_int(rng, 1, 16384)
            case = _prompt(None, min(requests, 32), lo, _log_int(rng, lo, 16384), q_heads,
                           kv_heads, head_dim, dtype, spread)
        if _padded_scores(case) <= _MOST_SCORES and _kv_bytes(case) <= _MOST_KV:
            return case


# ---------------------------------------------------------------------------
# sizes

def _lengths(case):
    """(new tokens, context tokens with the new ones) of every request."""
    rng = random.Random(case["spread"])
    lengths = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["requests"])]
    if case["kind"] in ("write", "prompt"):
        return lengths, list(lengths)
    new = [1] * case["requests"]
    for r in rng.sample(range(case["requests"]), case["longs"]):
        new[r] = rng.randint(max(1, case["new"] // 2), case["new"])
    # a request with a chunk of n tokens has n at least in its context
    return new, [max(n, c) for n, c in zip(new, lengths)]


def _padded_scores(case):
    new, context = _lengths(case)
    longs = [r for r, n in enumerate(new) if n > 1]
    singles = [r for r, n in enumerate(new) if n == 1]
    return case["q_heads"] * sum(
        len(group) * max(new[r] for r in group) * max(context[r] for r in group)
        for group in (longs, singles) if group)


def _kv_bytes(case):
    new, context = _lengths(case)
    longest = max(context)
    # the plain form pads every request to the longest context
    return 4 * len(context) * longest * case["kv_heads"] * case["head_dim"]


def work(case):
    new, context = _lengths(case)
    tokens, requests = sum(new), len(new)
    if case["kind"] == "plan":
        bs = case["block"]
        fresh = sum(-(-c // bs) - -(-(c - n) // bs) for n, c in zip(new, context))
        # lengths in; row ranges, contexts, slots, positions and fresh table entries out, each
        # fresh entry read from the free list; a token's slot needs its block's table entry
        touched = sum((c - 1) // bs - (c - n) // bs + 1 for n, c in zip(new, context))
        return {"bytes": 8 * requests + 8 * requests + 16 * tokens + 8 * fresh + 4 * touched,
                "flops": 0}
    row = case["kv_heads"] * case["head_dim"]
    if case["kind"] == "write":
        return {"bytes": 2 * 2 * 2 * tokens * row + 8 * tokens, "flops": 0}
    # row i of a request's n sees context - n + i + 1 tokens
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, context))
    q_row = case["q_heads"] * case["head_dim"]
    return {"bytes": 2 * 2 * tokens * q_row + 2 * 2 * sum(context) * row,
            "flops": 4 * pairs * q_row}


# ---------------------------------------------------------------------------
# inputs

def _channel_scales(kv_heads, head_dim, gen):
    """K channels of unlike sizes, log-uniform over [0.1, 10], as caches of real models have."""
    u = torch.rand((kv_heads, head_dim), generator=gen, device="cuda")
    return torch.exp(u * math.log(100.0) + math.log(0.1))


def _layer(case, blocks, gen, dtype):
    dims = (blocks, case["block"], case["kv_heads"], case["head_dim"])
    kv = torch.empty((2,) + dims, dtype=dtype, device="cuda")
    kv[0] = torch.randn(dims, generator=gen, device="cuda") * \
        _channel_scales(case["kv_heads"], case["head_dim"], gen)
    kv[1] = torch.randn(dims, generator=gen, device="cuda") * 0.5
    return kv


def _tables(case, lengths, gen, spare=0):
    """(tables, free): block tables (requests, width), int32, -1 behind each request's blocks, of
    a shuffled pool, and the blocks that no table holds."""
    bs = case["block"]
    held = [-(-n // bs) for n in lengths]
    pool = sum(held) + spare
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    counts = torch.tensor(held, device="cuda")
    width = max(1, max(held))
    columns = torch.arange(width, device="cuda")
    first = torch.cumsum(counts, 0) - counts
    at = (first[:, None] + columns).clamp_max(max(pool - 1, 0))
    tables = torch.where(columns < counts[:, None], order[at], -1)
    return tables.to(torch.int32), order[sum(held):].clone()


def _starts(lengths):
    total, starts = 0, [0]
    for n in lengths:
        total += n
        starts.append(total)
    return torch.tensor(starts, dtype=torch.int32, device="cuda")


def _packed_rows(tokens, case, gen, dtype):
    """q, k, v as views of one projection's rows: (tokens, heads, head_dim) each."""
    heads = (case.get("q_heads", 0), case["kv_heads"], case["kv_heads"])
    rows = torch.randn((tokens, sum(heads), case["head_dim"]), generator=gen, device="cuda")
    k = slice(heads[0], heads[0] + heads[1])
    rows[:, k] *= _channel_scales(case["kv_heads"], case["head_dim"], gen)
    rows[:, heads[0] + heads[1]:] *= 0.5
    return rows.to(dtype).split(heads, 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    new, context = _lengths(case)
    kind = case["kind"]
    state = {"kind": kind, "new": new, "context": context, "block": case.get("block")}
    if kind == "plan":
        bs = case["block"]
        cached = [c - n for n, c in zip(new, context)]
        fresh = sum(-(-c // bs) - -(-h // bs) for c, h in zip(context, cached))
        tables, free = _tables(case, cached, gen, spare=fresh + 64)
        wide = torch.full((len(new), -(-max(context) // bs)), -1, dtype=torch.int32, device="cuda")
        wide[:, :tables.shape[1]] = tables
        state.update(
            new_tokens=torch.tensor(new, dtype=torch.int32, device="cuda"),
            cached_tokens=torch.tensor(cached, dtype=torch.int32, device="cuda"), tables=wide,
            free_blocks=free, max_tokens=sum(new) + 16,
            free_start=torch.tensor([seed % 64], dtype=torch.int32, device="cuda"))
        return state
    dtype = _DTYPES[case["dtype"]]
    if kind == "prompt":
        q, k, v = _packed_rows(sum(new), case, gen, dtype)
        state.update(q=q, k=k, v=v, starts=_starts(new), longest=max(new))
        return state
    tables, _ = _tables(case, context, gen)
    blocks = int(sum(-(-c // case["block"]) for c in context))
    if kind == "write":
        bs = case["block"]
        place = torch.cat([torch.arange(n, device="cuda") for n in new])
        of = torch.repeat_interleave(torch.arange(len(new), device="cuda"),
                                     torch.tensor(new, device="cuda"))
        slots = tables[of, place // bs].long() * bs + place % bs
        _, k, v = _packed_rows(sum(new), case, gen, dtype)
        state.update(k=k, v=v, kv=_layer(case, blocks, gen, dtype), slots=slots)
        return state
    q = torch.randn((sum(new), case["q_heads"], case["head_dim"]), generator=gen,
                    device="cuda").to(dtype)
    state.update(q=q, kv=_layer(case, blocks, gen, dtype), tables=tables, starts=_starts(new),
                 contexts=torch.tensor(context, dtype=torch.int32, device="cuda"),
                 longest=max(new))
    return state


# ---------------------------------------------------------------------------
# the plain forms

def _plain_plan(s):
    bs, dev = s["block"], s["tables"].device
    new, cached = s["new_tokens"].long(), s["cached_tokens"].long()
    context = cached + new
    held, need = (cached + bs - 1) // bs, (context + bs - 1) // bs
    fresh = need - held
    base = s["free_start"].long() + torch.cumsum(fresh, 0) - fresh
    columns = torch.arange(s["tables"].shape[1], device=dev)
    at = base[:, None] + columns - held[:, None]
    is_fresh = (columns >= held[:, None]) & (columns < need[:, None])
    there = at < s["free_blocks"].numel()
    ids = s["free_blocks"][at.clamp(0, s["free_blocks"].numel() - 1)]
    s["tables"].copy_(torch.where(is_fresh, torch.where(there, ids, -1), s["tables"]))
    starts = torch.zeros(new.numel() + 1, dtype=torch.int32, device=dev)
    starts[1:] = torch.cumsum(new, 0)
    token = torch.arange(s["max_tokens"], device=dev)
    of = torch.searchsorted(starts[1:].long(), token, right=True)
    used = of < new.numel()
    of = of.clamp_max(new.numel() - 1)
    position = torch.where(used, cached[of] + token - starts[:-1].long()[of], 0)
    block = s["tables"][of, position // bs].long()
    slots = torch.where(used & (block >= 0), block * bs + position % bs, -1)
    taken = s["free_start"].long() + fresh.sum()
    lacking = (taken - s["free_blocks"].numel()).clamp_min(0)
    return {"tables": s["tables"], "query_starts": starts, "context_tokens": context.int(),
            "slots": slots, "positions": position,
            "free_next": taken.clamp_max(s["free_blocks"].numel()).int(), "lacking": lacking.int()}


def _plain_write(s):
    kv, slots = s["kv"], s["slots"]
    keep = slots >= 0
    flat = kv.view(2, -1, kv.shape[3], kv.shape[4])
    flat[0, slots[keep]] = s["k"][keep]
    flat[1, slots[keep]] = s["v"][keep]
    return kv


def _plain_attention(q, k, v, last):
    """q (B, n, q_heads, d), k and v (B, m, kv_heads, d); row (b, i) sees tokens 0 .. last[b, i].
    Float32 throughout; rows that see nothing are zero."""
    b, n, q_heads, d = q.shape
    m, kv_heads = k.shape[1], k.shape[2]
    group = q_heads // kv_heads
    rows = (q.float() * d ** -0.5).view(b, n, kv_heads, group, d).permute(0, 2, 3, 1, 4)
    rows = rows.reshape(b * kv_heads, group * n, d)
    keys = k.float().permute(0, 2, 3, 1).reshape(b * kv_heads, d, m)
    scores = torch.bmm(rows, keys).view(b, kv_heads, group, n, m)
    hidden = torch.arange(m, device=q.device) > last[:, :, None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    values = v.float().permute(0, 2, 1, 3).reshape(b * kv_heads, m, d)
    out = torch.bmm(weights.view(b * kv_heads, group * n, m), values)
    out = out.view(b, kv_heads, group, n, d) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, q_heads, d)


def _padded(rows, starts, counts, longest):
    """The requests' rows as a batch padded to the longest, and where each came from."""
    place = torch.arange(longest, device=rows.device)
    at = starts[:, None] + torch.minimum(place, counts[:, None] - 1)
    return rows[at], at, place < counts[:, None]


def _plain_chunk_of(s, out, requests):
    if not requests:
        return
    q, kv, bs = s["q"], s["kv"], s["block"]
    ids = torch.tensor(requests, device=q.device)
    starts = s["starts"].long()
    counts = (starts[1:] - starts[:-1])[ids]
    contexts = s["contexts"].long()[ids]
    longest = max(s["context"][r] for r in requests)
    rows, at, real = _padded(q, starts[ids], counts, max(s["new"][r] for r in requests))
    blocks = s["tables"][ids, :-(-longest // bs)].long().clamp_min(0)
    k, v = (plane[blocks].flatten(1, 2) for plane in (kv[0], kv[1]))
    place = torch.arange(rows.shape[1], device=q.device)
    last = (contexts - counts)[:, None] + torch.minimum(place, counts[:, None] - 1)
    out[at[real]] = _plain_attention(rows, k, v, last)[real].to(out.dtype)


def _plain_chunk(s):
    out = torch.empty_like(s["q"])
    # (padded to each other, single tokens would cost as much as the chunks beside them)
    _plain_chunk_of(s, out, [r for r, n in enumerate(s["new"]) if n == 1])
    _plain_chunk_of(s, out, [r for r, n in enumerate(s["new"]) if n > 1])
    return out


def _plain_prompt(s):
    starts = s["starts"].long()
    counts = starts[1:] - starts[:-1]
    q, at, real = _padded(s["q"], starts[:-1], counts, s["longest"])
    k, v = s["k"][at], s["v"][at]
    place = torch.arange(s["longest"], device=q.device)
    last = torch.minimum(place, counts[:, None] - 1)
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=q.device)
    out[at[real]] = _plain_attention(q, k, v, last)[real].to(out.dtype)
    return out


# ---------------------------------------------------------------------------
# the framework's calls

def _own(s):
    from unchainkv_amd import splitzip_cuda as sz

    kind = s["kind"]
    if kind == "plan":
        plan = sz.plan_step_paged(s["new_tokens"], s["cached_tokens"], s["tables"],
                                  s["free_blocks"], s["free_start"], s["block"], s["max_tokens"])
        return {"tables": s["tables"], "query_starts": plan.query_starts,
                "context_tokens": plan.context_tokens, "slots": plan.slots,
                "positions": plan.positions, "free_next": plan.free_next,
                "lacking": plan.lacking}
    if kind == "write":
        sz.write_kv_paged(s["k"], s["v"], s["kv"], s["slots"])
        return s["kv"]
    if kind == "chunk":
        return sz.chunk_attention_paged(s["q"], s["kv"], s["tables"], s["starts"], s["contexts"],
                                        max_query=s["longest"])
    return sz.prompt_attention(s["q"], s["k"], s["v"], s["starts"], max_query=s["longest"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plain_plan, "write": _plain_write, "chunk": _plain_chunk,
            "prompt": _plain_prompt}[state["kind"]](state)


# ---------------------------------------------------------------------------
# 64 bits

def _exact_rows(q, k, v, first):
    """One request in float64: q (n, q_heads, d), k and v (m, kv_heads, d); row i sees tokens
    0 .. first + i. A KV head and a piece of the rows at a time."""
    n, q_heads, d = q.shape
    group = q_heads // k.shape[1]
    out = torch.empty((n, q_heads, d), dtype=torch.float64, device=q.device)
    piece = max(1, int(2e8) // max(1, k.shape[0]))
    tokens = torch.arange(k.shape[0], device=q.device)
    for h in range(q_heads):
        keys, values = k[:, h // group].double(), v[:, h // group].double()
        for a in range(0, n, piece):
            rows = q[a:a + piece, h].double()
            scores = rows @ keys.T / math.sqrt(d)
            seen = tokens <= first + a + torch.arange(rows.shape[0], device=q.device)[:, None]
            scores = torch.where(seen, scores, -math.inf)
            out[a:a + piece, h] = torch.softmax(scores, -1) @ values
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "plan":
        return None
    if kind == "write":
        # every value is copied, none is computed
        kv, bs = s["kv"].double(), s["block"]
        kv[0, s["slots"] // bs, s["slots"] % bs] = s["k"].double()
        kv[1, s["slots"] // bs, s["slots"] % bs] = s["v"].double()
        return kv
    out, at = [], 0
    for r, n in enumerate(s["new"]):
        q = s["q"][at:at + n]
        if kind == "prompt":
            k, v = s["k"][at:at + n], s["v"][at:at + n]
        else:
            token = torch.arange(s["context"][r], device=q.device)
            block = s["tables"][r].long()[token // s["block"]]
            k, v = s["kv"][0, block, token % s["block"]], s["kv"][1, block, token % s["block"]]
        out.append(_exact_rows(q, k, v, s["context"][r] - n))
        at += n
    return torch.cat(out)
