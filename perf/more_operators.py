"""What is timed of a beam-searching decode step over paged KV layers, of a decoder alone or of one
that reads an encoder's states.

A paged KV layer is a tensor (2, num_blocks, block_tokens, kv_heads, head_dim), K plane then V
plane; a row of a block table lists a sequence's blocks in token order. A case's ``kind`` names the
operator:

* ``rotate``   the new tokens' K rows, rotated by their positions, and V rows into the layer by slot
               (-1: no slot, no write), and the rotated query rows
* ``cross``    attention of a request's rows (a token of each beam, or a prompt) over all of its
               source's tokens, which lie in a paged layer or in packed rows
* ``select``   the best continuations of a request's beams: of all beams and tokens those with the
               largest score + log softmax, ties to the lowest beam and then the lowest token
* ``reorder``  the block tables follow the chosen parents: full blocks are shared, the last, partly
               filled one is copied in every layer into a block that a dropped beam leaves, and the
               blocks that no beam names any more go back to the free list

Query heads share the KV heads in equal groups (query head h reads KV head h // group). The softmax
scale is head_dim ** -0.5. A rotation's angle is position * base ** (-2 i / rotary) for pair i of
rotary / 2: values i and i + rotary / 2 of a head, or 2 i and 2 i + 1 (interleaved).

Lengths are spread log-uniformly by the case's own ``spread`` seed, and so are the parents, so that
a case costs the same whatever its inputs are.

Ranges: 1 to 20 KV heads, groups of 1 to 8, head dims 64 and 128, bf16 and fp16 (logits f32 too),
blocks of 8 to 32 tokens, 1 to 64 requests, 1 to 16 beams, positions below 131072, 1 to 32768 new
tokens, sources of 0 to 16384 tokens, vocabularies of 500 to 262144, 1 to 32 layers; at most 3e9
scores of the padded plain form and 1.1 GiB of layers.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_POSITIONS = 131072
_BASE = 500000.0
_MOST_SCORES = 3e9
_MOST_PAIRS = 1.8e11  # of a row's and a source's values
_MOST_PLAIN = 250 << 20  # bytes of a plain attention's padded keys, in f32
_MOST_LAYERS = 9 << 27
_MOST_LOGITS = 1 << 26


# ---------------------------------------------------------------------------
# cases

def _named(name, case):
    return dict(case, name=name) if name else case


def _rotate(name, requests, lo, hi, cached, q_heads, kv_heads, head_dim, rotary, interleaved,
            block, dtype="bf16", spread=1):
    """Each request has lo .. hi new tokens behind up to ``cached`` ones."""
    return _named(name, {
        "kind": "rotate", "requests": requests, "lo": lo, "hi": hi, "cached": cached,
        "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "rotary": rotary,
        "interleaved": interleaved, "block": block, "dtype": dtype, "spread": spread})


def _cross(name, requests, rows_lo, rows_hi, lo, hi, q_heads, kv_heads, head_dim, block,
           dtype="bf16", empty=0, spread=1):
    """Rows and source tokens of each request; block 0: packed sources; ``empty`` of them have
    no token."""
    return _named(name, {
        "kind": "cross", "requests": requests, "rows_lo": rows_lo, "rows_hi": rows_hi, "lo": lo,
        "hi": hi, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
        "dtype": dtype, "empty": empty, "spread": spread})


def _select(name, requests, beams, vocab, candidates, dtype="bf16", ended=0, first=False):
    """``ended`` of each request's beams are finished; first: the search's first step, in which
    all beams but one are still empty."""
    return _named(name, {
        "kind": "select", "requests": requests, "beams": beams, "vocab": vocab,
        "candidates": candidates, "dtype": dtype, "ended": ended, "first": first})


def _reorder(name, requests, beams, lo, hi, made, layers, kv_heads, head_dim, block, spread=1):
    """Prompts of lo .. hi tokens and up to ``made`` tokens behind them."""
    return _named(name, {
        "kind": "reorder", "requests": requests, "beams": beams, "lo": lo, "hi": hi, "made": made,
        "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
        "spread": spread})


def listed():
    return [
        # the tokens of a decode step of an 8B model
        _rotate("rotate_decode", 64, 1, 1, 32000, 32, 8, 128, 128, False, 16, spread=3),
        # a prefill batch of an 8B model
        _rotate("rotate_prefill", 8, 4096, 4096, 0, 32, 8, 128, 128, False, 16),
        # chunks of odd lengths far into their contexts, half of each head rotated, pairs side by side
        _rotate("rotate_ragged", 24, 3, 900, 120000, 24, 3, 64, 32, True, 24, dtype="fp16", spread=5),
        # one user of a small model with an encoder: latency alone
        _cross("cross_single", 1, 1, 1, 1000, 1000, 16, 16, 64, 16),
        # a decode batch, five beams a request read their source once
        _cross("cross_beams", 32, 5, 5, 1500, 1500, 20, 20, 64, 16, dtype="fp16"),
        # long documents as sources of prompts, shared KV heads
        _cross("cross_documents", 4, 600, 1500, 4000, 16000, 32, 8, 128, 16, spread=4),
        # prompts over an encoder's output before it is in a layer
        _cross("cross_packed", 16, 100, 450, 300, 2000, 16, 16, 128, 0, empty=1, spread=7),
        # one user, a vocabulary of 32000
        _select("select_single", 1, 4, 32000, 4, dtype="fp32"),
        # a serving batch with a large vocabulary, two candidates a beam, some beams finished
        _select("select_batch", 64, 8, 131072, 16, ended=1),
        # the first step of searches over an odd vocabulary
        _select("select_first", 16, 5, 50001, 5, dtype="fp16", first=True),
        # one user's beams, a small model
        _reorder("reorder_single", 1, 4, 200, 200, 90, 16, 8, 64, 16, spread=2),
        # a serving batch, a share of an 8B model's layers
        _reorder("reorder_batch", 48, 4, 64, 2000, 120, 8, 8, 128, 16, spread=6),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above."""
    while True:
        kind = rng.choice(("rotate", "cross", "cross", "select", "reorder"))
        requests = _log_int(rng, 1, 64)
        block = rng.choice((8, 16, 16, 32, 24))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        head_dim = rng.choice((64, 128))
        kv_heads = rng.choice((1, 2, 3, 4, 8, 8, 12, 20))
        q_heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 4, 7, 8))
        spread = rng.randrange(1, 1 << 20)
        beams = rng.choice((1, 2, 3, 4, 4, 5, 8, 10, 16))
        if kind == "rotate":
            lo = _log_int(rng, 1, 4096)
            rotary = rng.choice((head_dim, head_dim, head_dim // 2, 3 * head_dim // 4, 20))
            case = _rotate(None, requests, lo, _log_int(rng, lo, 4096), rng.choice((0, 4000, 126000)),
                           min(q_heads, 64), kv_heads, head_dim, rotary, rng.random() < 0.4, block,
                           dtype, spread)
            if sum(_rotate_lengths(case)[0]) * (case["q_heads"] + 2 * kv_heads) * head_dim <= 201326592:
                return case
        elif kind == "cross":
            rows = rng.choice((beams, beams, _log_int(rng, 1, 2048)))
            lo = _log_int(rng, 1, 16384)
            case = _cross(None, requests, min(rows, rng.choice((rows, _log_int(rng, 1, 2048)))), rows,
                          lo, _log_int(rng, lo, 16384), q_heads, kv_heads, head_dim,
                          rng.choice((block, block, 0)), dtype, rng.choice((0, 0, 0, 1)), spread)
            if _cross_fits(case):
                return case
        elif kind == "select":
            vocab = _log_int(rng, 500, 262144)
            case = _select(None, requests, beams, vocab, min(2 * beams, beams * rng.choice((1, 2))),
                           rng.choice(("bf16", "fp16", "fp32")), rng.choice((0, 0, min(1, beams - 1))),
                           rng.random() < 0.2)
            if requests * beams * vocab <= _MOST_LOGITS:
                return case
        else:
            lo = _log_int(rng, 1, 2000)
            case = _reorder(None, requests, max(beams, 2), lo, _log_int(rng, lo, 4000),
                            _log_int(rng, 1, 250), _log_int(rng, 1, 32), min(kv_heads, 8), head_dim,
                            block, spread)
            if _reorder_bytes(case) <= _MOST_LAYERS:
                return case


# ---------------------------------------------------------------------------
# sizes

def _rotate_lengths(case):
    """(new tokens, tokens before them) of every request."""
    rng = random.Random(case["spread"])
    new = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["requests"])]
    return new, [rng.randint(0, case["cached"]) if case["cached"] else 0 for _ in new]


def _cross_lengths(case):
    """(rows, source tokens) of every request."""
    rng = random.Random(case["spread"])
    rows = [_log_int(rng, case["rows_lo"], case["rows_hi"]) for _ in range(case["requests"])]
    source = [_log_int(rng, case["lo"], case["hi"]) for _ in rows]
    for r in rng.sample(range(len(rows)), min(case["empty"], len(rows) - 1)):
        source[r] = 0
    return rows, source


def _cross_fits(case):
    rows, source = _cross_lengths(case)
    padded = len(rows) * max(source)
    row = case["kv_heads"] * case["head_dim"]
    return padded * max(rows) * case["q_heads"] <= _MOST_SCORES and 4 * padded * row <= _MOST_PLAIN \
        and sum(n * s for n, s in zip(rows, source)) * case["q_heads"] * case["head_dim"] <= _MOST_PAIRS


def _reorder_lengths(case):
    """(prompt tokens, context tokens) of every request."""
    rng = random.Random(case["spread"])
    prompts = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["requests"])]
    return prompts, [p + rng.randint(0, case["made"]) for p in prompts]


def _reorder_parents(case):
    """Each request's chosen parents: the better beams have more children."""
    rng = random.Random(case["spread"] + 1)
    beams = case["beams"]
    return [[min(rng.randrange(beams), rng.randrange(beams)) for _ in range(beams)]
            for _ in range(case["requests"])]


def _reorder_names(case):
    """For each request, which block of its column every beam names: (beams, columns) numbers that
    count the request's blocks. Columns of the prompt are shared by all; behind it, the further
    back the fewer lines are still apart; the last partly filled block is each beam's own."""
    rng = random.Random(case["spread"] + 2)
    beams, bs, got = case["beams"], case["block"], []
    for prompt, context in zip(*_reorder_lengths(case)):
        full, names, count = context // bs, [], 0
        line = list(range(beams))
        if context % bs:
            names.append(list(range(beams)))
            count = beams
        for column in range(full - 1, -1, -1):
            if column < prompt // bs:
                names.append([count] * beams)
                count += 1
                continue
            merge = sorted(min(rng.randrange(beams), rng.randrange(beams)) for _ in range(beams))
            line = [merge[x] for x in line]
            seen = {x: count + i for i, x in enumerate(sorted(set(line)))}
            names.append([seen[x] for x in line])
            count += len(seen)
        names.reverse()
        got.append(([[column[b] for column in names] for b in range(beams)], count))
    return got


def _reorder_bytes(case):
    blocks = sum(count for _, count in _reorder_names(case))
    return 4 * blocks * case["block"] * case["kv_heads"] * case["head_dim"] * case["layers"]


def work(case):
    kind = case["kind"]
    if kind == "rotate":
        new, cached = _rotate_lengths(case)
        tokens = sum(new)
        used, last = 0, 0  # rows of the table, each once
        for begin, end in sorted((c, c + n) for n, c in zip(new, cached)):
            used += max(0, end - max(begin, last))
            last = max(last, end)
        heads = case["q_heads"] + case["kv_heads"]
        return {"bytes": 4 * tokens * (heads + case["kv_heads"]) * case["head_dim"] + 16 * tokens
                + 4 * used * case["rotary"], "flops": 3 * tokens * heads * case["rotary"]}
    if kind == "cross":
        rows, source = _cross_lengths(case)
        q_row = case["q_heads"] * case["head_dim"]
        return {"bytes": 4 * sum(rows) * q_row
                + 4 * sum(source) * case["kv_heads"] * case["head_dim"],
                "flops": 4 * sum(n * s for n, s in zip(rows, source)) * q_row}
    if kind == "select":
        size = 4 if case["dtype"] == "fp32" else 2
        logits = case["requests"] * case["beams"] * case["vocab"]
        # a finished beam's logits and those of an empty one count for nothing
        read = case["requests"] * (1 if case["first"] else case["beams"] - case["ended"]) * case["vocab"]
        return {"bytes": size * read + 16 * case["requests"] * case["candidates"],
                "flops": 4 * min(read, logits)}
    _, context = _reorder_lengths(case)
    bs, row = case["block"], 2 * case["kv_heads"] * case["head_dim"]
    columns = sum(-(-c // bs) for c in context)
    moved = sum((case["beams"] - len(set(p))) * (c % bs)
                for p, c in zip(_reorder_parents(case), context))
    return {"bytes": 8 * case["beams"] * columns + 4 * moved * row * case["layers"], "flops": 0}


# ---------------------------------------------------------------------------
# inputs

def _channel_scales(kv_heads, head_dim, gen):
    """K channels of unlike sizes, log-uniform over [0.1, 10], as caches of real models have."""
    u = torch.rand((kv_heads, head_dim), generator=gen, device="cuda")
    return torch.exp(u * math.log(100.0) + math.log(0.1))


def _packed_rows(tokens, heads, case, gen):
    """Views of one projection's rows, (tokens, n, head_dim) for each n of ``heads``; the last two
    are K and V."""
    rows = torch.randn((tokens, sum(heads), case["head_dim"]), generator=gen, device="cuda")
    k = sum(heads) - heads[-1] - heads[-2]
    rows[:, k:k + heads[-2]] *= _channel_scales(heads[-2], case["head_dim"], gen)
    rows[:, k + heads[-2]:] *= 0.5
    return rows.to(_DTYPES[case["dtype"]]).split(heads, 1)


def _layer(case, blocks, gen):
    dims = (max(blocks, 1), case["block"], case["kv_heads"], case["head_dim"])
    kv = torch.empty((2,) + dims, dtype=_DTYPES[case["dtype"]], device="cuda")
    kv[0] = torch.randn(dims, generator=gen, device="cuda") * \
        _channel_scales(case["kv_heads"], case["head_dim"], gen)
    kv[1] = torch.randn(dims, generator=gen, device="cuda") * 0.5
    return kv


def _tables(lengths, bs, gen):
    """Block tables (requests, width), int32, -1 behind each request's blocks, of a shuffled pool."""
    held = [-(-n // bs) for n in lengths]
    order = torch.randperm(sum(held), generator=gen, device="cuda").to(torch.int32)
    counts = torch.tensor(held, device="cuda")
    columns = torch.arange(max(1, max(held)), device="cuda")
    at = (torch.cumsum(counts, 0) - counts)[:, None] + columns
    return torch.where(columns < counts[:, None], order[at.clamp_max(max(sum(held) - 1, 0))],
                       -1).to(torch.int32)


def _starts(lengths):
    total, starts = 0, [0]
    for n in lengths:
        total += n
        starts.append(total)
    return torch.tensor(starts, dtype=torch.int32, device="cuda")


def _frequencies(rotary):
    return _BASE ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)


def _prepare_rotate(case, gen):
    new, cached = _rotate_lengths(case)
    bs, tokens = case["block"], sum(new)
    # the blocks that the new tokens lie in, each request's from the block of its first one on
    lead = [c % bs for c in cached]
    tables = _tables([a + n for a, n in zip(lead, new)], bs, gen)
    of = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    place = torch.arange(tokens, device="cuda") - _starts(new)[:-1].long()[of]
    inside = torch.tensor(lead, device="cuda")[of] + place
    slots = tables[of, inside // bs].long() * bs + inside % bs
    q, k, v = _packed_rows(tokens, (case["q_heads"], case["kv_heads"], case["kv_heads"]), case, gen)
    angles = torch.arange(_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * \
        _frequencies(case["rotary"])
    return {"q": q, "k": k, "v": v, "slots": slots,
            "positions": torch.tensor(cached, device="cuda")[of] + place,
            "kv": _layer(case, sum(-(-(a + n) // bs) for a, n in zip(lead, new)), gen),
            "rotation": torch.cat((angles.cos(), angles.sin()), 1).float(),
            "interleaved": case["interleaved"]}


def _prepare_cross(case, gen):
    rows, source = _cross_lengths(case)
    q = torch.randn((sum(rows), case["q_heads"], case["head_dim"]), generator=gen, device="cuda")
    state = {"q": q.to(_DTYPES[case["dtype"]]), "starts": _starts(rows), "most_rows": max(rows),
             "source": torch.tensor(source, dtype=torch.int32, device="cuda"),
             "most_source": max(source), "block": case["block"]}
    if case["block"]:
        blocks = sum(-(-s // case["block"]) for s in source)
        state.update(kv=_layer(case, blocks, gen), tables=_tables(source, case["block"], gen))
    else:
        k, v = _packed_rows(sum(source), (case["kv_heads"], case["kv_heads"]), case, gen)
        state.update(k=k, v=v, source_starts=_starts(source)[:-1])
    return state


def _prepare_select(case, gen):
    r, b, vocab = case["requests"], case["beams"], case["vocab"]
    logits = 2.5 * torch.randn((r, b, vocab), generator=gen, device="cuda")
    # some likely tokens, some that are not allowed
    at = torch.randint(0, vocab, (r, b, 1), generator=gen, device="cuda")
    at = (at + torch.arange(12, device="cuda") * (vocab // 12)) % vocab
    logits.scatter_(2, at, 3 + 8 * torch.rand((r, b, 12), generator=gen, device="cuda"))
    banned = torch.randint(0, vocab, (vocab // 64,), generator=gen, device="cuda")
    logits[:, :, banned] = -math.inf
    scores = -12 * torch.rand((r, b), generator=gen, device="cuda") - 4
    scores = scores.sort(1, descending=True).values
    if case["first"]:
        scores[:, 1:] = -math.inf
    ended = torch.zeros((r, b), dtype=torch.bool, device="cuda")
    ended[:, b // 2:b // 2 + case["ended"]] = True
    return {"logits": logits.to(_DTYPES[case["dtype"]]), "scores": scores, "ended": ended,
            "end_token": vocab // 3, "candidates": case["candidates"]}


def _prepare_reorder(case, gen):
    prompts, context = _reorder_lengths(case)
    r, b, bs = case["requests"], case["beams"], case["block"]
    names = _reorder_names(case)
    width, first, rows = max(-(-c // bs) for c in context) + 2, 0, []
    for table, count in names:
        rows += [[first + x for x in row] + [-1] * (width - len(row)) for row in table]
        first += count
    ids = torch.cat((torch.randperm(first, generator=gen, device="cuda"),
                     torch.tensor([-1], device="cuda"))).to(torch.int32)
    dims = (case["layers"], 2, first, bs, case["kv_heads"], case["head_dim"])
    layers = torch.empty(dims, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    # a list whose first blocks are those in use, the others free
    free = torch.cat((ids[:-1], torch.arange(first, first + 64, dtype=torch.int32, device="cuda")))
    return {"tables": ids[torch.tensor(rows, device="cuda")],
            "parents": torch.tensor(_reorder_parents(case), dtype=torch.int32, device="cuda"),
            "context": torch.tensor(context, dtype=torch.int32, device="cuda").repeat_interleave(b),
            "stack": layers, "layers": list(layers.unbind(0)), "free_blocks": free,
            "free_start": torch.tensor([first], dtype=torch.int32, device="cuda"), "block": bs}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    make = {"rotate": _prepare_rotate, "cross": _prepare_cross, "select": _prepare_select,
            "reorder": _prepare_reorder}[case["kind"]]
    return dict(make(case, gen), kind=case["kind"])


# ---------------------------------------------------------------------------
# the plain forms

def _plain_turned(x, cos, sin, interleaved):
    """x (tokens, heads, head_dim) with its first 2 * pairs values rotated, in f32."""
    pairs = cos.shape[-1]
    y = x.float()
    turned, rest = y[..., :2 * pairs], y[..., 2 * pairs:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        new = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        new = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((new, rest), -1).to(x.dtype)


def _plain_rotate(s):
    table = s["rotation"][s["positions"]][:, None]
    cos, sin = table.chunk(2, -1)
    keep = s["slots"] >= 0
    flat = s["kv"].view(2, -1, s["kv"].shape[3], s["kv"].shape[4])
    flat[0, s["slots"][keep]] = _plain_turned(s["k"], cos, sin, s["interleaved"])[keep]
    flat[1, s["slots"][keep]] = s["v"][keep]
    return {"q": _plain_turned(s["q"], cos, sin, s["interleaved"]), "kv": s["kv"]}


def _plain_cross(s):
    """A batch padded to the most rows and the longest source; f32 throughout."""
    q, starts, source = s["q"], s["starts"].long(), s["source"].long()
    counts = starts[1:] - starts[:-1]
    place = torch.arange(s["most_rows"], device=q.device)
    at = starts[:-1, None] + torch.minimum(place, counts[:, None] - 1)
    real = place < counts[:, None]
    m = s["most_source"]
    token = torch.arange(m, device=q.device)
    if s["block"]:
        blocks = s["tables"][:, :-(-m // s["block"])].long().clamp_min(0)
        k, v = (plane[blocks].flatten(1, 2)[:, :m] for plane in (s["kv"][0], s["kv"][1]))
    else:
        rows = s["source_starts"].long()[:, None] + token
        rows = rows.clamp_max(s["k"].shape[0] - 1)
        k, v = s["k"][rows], s["v"][rows]
    b, n, d = counts.numel(), s["most_rows"], q.shape[2]
    q_heads, kv_heads = q.shape[1], k.shape[2]
    group = q_heads // kv_heads
    rows = (q[at].float() * d ** -0.5).view(b, n, kv_heads, group, d).permute(0, 2, 3, 1, 4)
    rows = rows.reshape(b * kv_heads, group * n, d)
    keys = k.float().permute(0, 2, 3, 1).reshape(b * kv_heads, d, m)
    scores = torch.bmm(rows, keys).view(b, kv_heads, group * n, m)
    scores.masked_fill_((token >= source[:, None])[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    values = v.float().permute(0, 2, 1, 3).reshape(b * kv_heads, m, d)
    out = torch.bmm(weights.view(b * kv_heads, group * n, m), values)
    out = out.view(b, kv_heads, group * n, d) / torch.where(total > 0, total, 1.0)
    out = out.view(b, kv_heads, group, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, q_heads, d)
    result = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    result[at[real]] = out[real].to(q.dtype)
    return result


def _plain_select(s):
    """In 64 bits, so that near candidates of two beams come in the order of their values."""
    logits, scores = s["logits"].double(), s["scores"].double()
    r, b, vocab = logits.shape
    top = logits.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float64).min)
    whole = (logits - top).exp_().sum(-1, keepdim=True).log_() + top
    # an empty or finished beam has nothing to offer, whatever its logits are
    open_beams = ~s["ended"] & (scores > -math.inf)
    values = torch.where(open_beams[..., None] & (logits > -math.inf),
                         logits - whole + scores[..., None], -math.inf)
    end = s["end_token"]
    values[..., end] = torch.where(s["ended"], scores, values[..., end])
    values = values.view(r, b * vocab)
    size, k = b * vocab, s["candidates"]
    last = values.topk(k, -1).values[:, -1:]
    # the k best: what is above the k-th value, and the first that are equal to it
    order = size - torch.arange(size, device=values.device)
    keys = torch.where(values > last, order + size, torch.where(values == last, order, -1))
    places = keys.topk(k, -1).indices.sort(-1).values
    best, by = values.gather(1, places).sort(dim=-1, descending=True, stable=True)
    places = places.gather(1, by)
    return {"scores": best.float(), "parents": (places // vocab).int(), "tokens": places % vocab}


def _plain_reorder(s):
    b = s["parents"].shape[1]
    r, width, bs = s["parents"].shape[0], s["tables"].shape[1], s["block"]
    old, parents = s["tables"].view(r, b, width), s["parents"].long()
    context = s["context"].view(r, b)[:, 0].long()
    full, rest = context // bs, context % bs
    columns = torch.arange(width, device=old.device)
    new = old.gather(1, parents[..., None].expand(r, b, width))
    shared = columns < full[:, None]
    tables = torch.where(shared[:, None], new, old)
    # blocks of full columns that no beam names any more, each at the first beam that named it
    earlier = torch.ones((b, b), dtype=torch.bool, device=old.device).tril(-1)
    kept = (old[:, :, None] == new[:, None]).any(2)
    again = ((old[:, :, None] == old[:, None]) & earlier[..., None]).any(2)
    released = ~kept & ~again & (old >= 0) & shared[:, None]
    # the last blocks: the first child of a parent keeps its block, the others take those that
    # no parent left
    column = full.clamp_max(width - 1)[:, None, None].expand(r, b, 1)
    partly = (rest > 0) & (full < width)
    tail = old.gather(2, column)[..., 0]
    source = tail.gather(1, parents)
    moves = ((source[:, :, None] == source[:, None]) & earlier).any(2) & partly[:, None]
    spare = ~(tail[:, :, None] == source[:, None]).any(2) & (tail >= 0) & partly[:, None]
    spare &= ~((tail[:, :, None] == tail[:, None]) & earlier).any(2)
    spares = tail.gather(1, torch.sort((~spare).int(), dim=1, stable=True).indices)
    turn = torch.cumsum(moves, 1) - 1
    there = turn < spare.sum(1, keepdim=True)
    to = torch.where(moves, torch.where(there, spares.gather(1, turn.clamp_min(0)), -1), source)
    tables = torch.where(partly[:, None, None] & (columns == full[:, None])[:, None], to[..., None],
                         tables)
    left = spare & (torch.cumsum(spare, 1) > moves.sum(1, keepdim=True))
    released |= left[..., None] & (columns == full[:, None])[:, None]
    # behind each other, below the first free one
    flat = released.transpose(1, 2).reshape(-1)
    count = flat.sum()
    first = s["free_start"].long() - count
    places = torch.where(flat, first + torch.cumsum(flat, 0) - 1, s["free_blocks"].numel())
    listed_blocks = torch.cat((s["free_blocks"], s["free_blocks"].new_zeros(1)))
    listed_blocks.scatter_(0, places.clamp_min(0), old.transpose(1, 2).reshape(-1))
    s["free_blocks"].copy_(listed_blocks[:-1])
    # the copies, in all layers at once
    copy = moves & there
    src, dst = source[copy].long(), to[copy].long()
    token = torch.arange(bs, device=old.device)
    used = (token < rest[:, None])[:, None].expand(r, b, bs)[copy][None, None, :, :, None, None]
    stack = s["stack"]
    stack[:, :, dst] = torch.where(used, stack[:, :, src], stack[:, :, dst])
    return {"tables": tables.view(r * b, width), "free_blocks": s["free_blocks"],
            "free_next": first.int(), "layers": s["layers"]}


# ---------------------------------------------------------------------------
# the framework's calls

def _own(s):
    from unchainkv_amd import splitzip_cuda as sz

    kind = s["kind"]
    if kind == "rotate":
        q = sz.rotate_write_kv_paged(s["q"], s["k"], s["v"], s["kv"], s["slots"], s["positions"],
                                     s["rotation"], interleaved=s["interleaved"])
        return {"q": q, "kv": s["kv"]}
    if kind == "cross":
        if s["block"]:
            return sz.cross_attention_paged(s["q"], s["kv"], s["tables"], s["starts"], s["source"],
                                            max_query=s["most_rows"])
        return sz.cross_attention(s["q"], s["k"], s["v"], s["starts"], s["source_starts"],
                                  s["source"], max_query=s["most_rows"],
                                  max_source=s["most_source"])
    if kind == "select":
        choice = sz.beam_select(s["logits"], s["scores"], candidates=s["candidates"],
                                ended=s["ended"], end_token=s["end_token"])
        return {"scores": choice.scores, "parents": choice.parents, "tokens": choice.tokens}
    order = sz.reorder_beams_paged(s["layers"], s["tables"], s["parents"], s["context"],
                                   s["free_blocks"], s["free_start"], s["block"])
    return {"tables": order.tables, "free_blocks": s["free_blocks"], "free_next": order.free_next,
            "layers": s["layers"]}


def run(state):
    if own:
        return _own(state)
    return {"rotate": _plain_rotate, "cross": _plain_cross, "select": _plain_select,
            "reorder": _plain_reorder}[state["kind"]](state)


# ---------------------------------------------------------------------------
# 64 bits

def _exact_turned(x, positions, rotary, interleaved):
    """As complex numbers: a pair times e^(i angle)."""
    angle = positions.double()[:, None] * _frequencies(rotary)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.double().clone()
    if interleaved:
        pair = torch.view_as_complex(y[..., :rotary].unflatten(-1, (-1, 2)).contiguous()) * turn
        y[..., 0:rotary:2], y[..., 1:rotary:2] = pair.real, pair.imag
    else:
        pair = torch.complex(y[..., :rotary // 2].clone(), y[..., rotary // 2:rotary].clone()) * turn
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = pair.real, pair.imag
    return y


def _exact_cross(case, s):
    """A request, a head and a piece of the rows at a time."""
    out, at, first = [], 0, 0
    for r, (n, m) in enumerate(zip(*_cross_lengths(case))):
        if case["block"]:
            token = torch.arange(m, device="cuda")
            block = s["tables"][r].long()[token // case["block"]]
            k, v = s["kv"][0, block, token % case["block"]], s["kv"][1, block, token % case["block"]]
        else:
            k, v = s["k"][first:first + m], s["v"][first:first + m]
        first += m
        rows = torch.zeros((n, case["q_heads"], case["head_dim"]), dtype=torch.float64, device="cuda")
        group = case["q_heads"] // case["kv_heads"]
        for h in range(case["q_heads"] if m else 0):
            keys, values = k[:, h // group].double(), v[:, h // group].double()
            scores = s["q"][at:at + n, h].double() @ keys.T / math.sqrt(case["head_dim"])
            rows[:, h] = torch.softmax(scores, -1) @ values
        out.append(rows)
        at += n
    return torch.cat(out)


def _exact_select(case, s):
    """Every request's candidates, sorted whole."""
    best = []
    for logits, scores, ended in zip(s["logits"], s["scores"], s["ended"]):
        values = torch.log_softmax(logits.double(), -1) + scores.double()[:, None]
        values[ended] = -math.inf
        values[ended, s["end_token"]] = scores.double()[ended]
        values = torch.where(scores[:, None] > -math.inf, values, -math.inf)
        best.append(values.flatten().sort(descending=True).values[:s["candidates"]])
    return {"scores": torch.stack(best), "parents": None, "tokens": None}


def _exact_reorder(case, s):
    """The copies as a host program makes them, request by request."""
    b, bs = case["beams"], case["block"]
    tables = s["tables"].tolist()
    layers = s["stack"].double()
    for r, (parents, context) in enumerate(zip(_reorder_parents(case), _reorder_lengths(case)[1])):
        column, used = context // bs, context % bs
        if not used:
            continue
        tails = [tables[r * b + j][column] for j in range(b)]
        unused = [tails[j] for j in range(b) if j not in parents]
        for j, p in enumerate(parents):
            if p in parents[:j]:
                to = unused.pop(0)
                layers[:, :, to, :used] = layers[:, :, tails[p], :used]
    return {"tables": None, "free_blocks": None, "free_next": None, "layers": list(layers.unbind(0))}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "cross":
        return _exact_cross(case, s)
    if case["kind"] == "select":
        return _exact_select(case, s)
    if case["kind"] == "reorder":
        return _exact_reorder(case, s)
    kv, bs, slots = s["kv"].double(), case["block"], s["slots"]
    kv[0, slots // bs, slots % bs] = _exact_turned(s["k"], s["positions"], case["rotary"],
                                                   case["interleaved"])
    kv[1, slots // bs, slots % bs] = s["v"].double()
    return {"q": _exact_turned(s["q"], s["positions"], case["rotary"], case["interleaved"]), "kv": kv}
