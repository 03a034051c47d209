"""Rounding of the weights of attention over sources, where a request is streamed (at most 16 rows of a
KV head): what the rounding to the type leaves has a product of its own, so that the output's rounding is the
only one of its size.

Bound of an output value, u = half a step of the type (terms as in paged_attention_ref.py): the output's
rounding u |o|; a weight's remainder, at most u of it, is itself rounded, u^2 A; fp16 remainders below
2^-14 lose up to 2^-25 each beside a largest weight of 2^7 at least, n 2^-32 max |v|; the terms of 32-bit scores,
exponentials and sums, 2 d A. Queries are small here, so that d is far below u. A lane adds up the weights of at
most every 16th token, and joins at most 64 sums: its share of d is (n / 16 + 64) 2^-24 where that is less than n 2^-24."""

import numpy as np
import pytest

from paged_attention_ref import HALF_STEP, attend

torch = pytest.importorskip("torch")

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SHAPES = [
    # rows, source tokens, query and KV heads, head dim: whole sources, splits, beside a request of tiles
    ([1], [2], 1, 1, 64), ([5, 1], [33, 7], 4, 4, 64), ([4, 2], [65, 40], 8, 2, 128),
    ([1], [900], 2, 2, 64), ([2], [600], 3, 3, 128), ([3, 40], [50, 60], 2, 2, 64), ([1, 70], [20, 90], 4, 1, 128)]


def make(rows, source, q_heads, kv_heads, dim, dtype, seed=0):
    """Rows of q, and of each request's K and V, in the type. Five tokens of a long source have values, all others
    zeros: the bound's share of sums over many tokens goes by all values, a weight's rounding by its own."""
    rng = np.random.default_rng(seed)

    def draw(size, by=1.0):
        return torch.from_numpy((rng.standard_normal(size) * by).astype(np.float32)).to(DTYPES[dtype])

    q, keys = draw((sum(rows), q_heads, dim), 0.05), [draw((m, kv_heads, dim)) for m in source]
    values = [draw((m, kv_heads, dim)) for m in source]
    for v in values:
        if len(v) > 100:
            v[torch.arange(len(v)) % (len(v) // 5) != 7] = 0
    return q, keys, values


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def worst(got, q, k, v, dtype, scale):
    """The largest error of a request's rows, by its bound."""
    u, tokens = HALF_STEP[dtype], k.shape[0]
    out, _, mean, off = attend(q, k, v, tokens, scale)
    off = off - max(0.0, tokens - tokens / 16 - 64) * 2.0 ** -24
    bound = u * np.abs(out) * 1.01 + (u * u + 2 * off[..., None]) * mean + 1e-30
    if dtype == "fp16":
        bound = bound + tokens * 2.0 ** -32 * np.abs(v).max() + 2.0 ** -25
    return (np.abs(got - out) / bound).max()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,source,q_heads,kv_heads,dim", SHAPES, ids=range(len(SHAPES)))
def test_rounded_weights_pass_the_bound(rows, source, q_heads, kv_heads, dim, dtype):
    """On the CPU: sums of weights rounded to the type alone are outside the bound somewhere in every case of more
    tokens than two, and with their remainders inside."""
    t = DTYPES[dtype]
    q, keys, values = make(rows, source, q_heads, kv_heads, dim, dtype)
    scale, at, alone, both = dim ** -0.5, 0, 0.0, 0.0
    for n, k, v in zip(rows, map(f64, keys), map(f64, values)):
        mine = f64(q[at:at + n])
        at += n
        group = q_heads // kv_heads
        if n * group > 16:
            continue
        got = {False: np.zeros_like(mine), True: np.zeros_like(mine)}
        for i in range(n):
            for h in range(q_heads):
                s = k[:, h // group] @ mine[i, h] * scale
                p = torch.from_numpy(np.exp(s - s.max()) * 128).float()
                w = p.to(t).float()
                rest = (p - w).to(t).float()
                for kept, x in ((False, w), (True, w + rest)):
                    sums = x.double().numpy() @ v[:, h // group] / p.double().sum().item()
                    got[kept][i, h] = torch.from_numpy(sums).to(t).double().numpy()
        alone = max(alone, worst(got[False], mine, k, v, dtype, scale))
        both = max(both, worst(got[True], mine, k, v, dtype, scale))
    assert both <= 1.0
    assert alone > 1.0 or max(source) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,source,q_heads,kv_heads,dim", SHAPES, ids=range(len(SHAPES)))
def test_streamed_rows_lose_only_the_outputs_rounding(rows, source, q_heads, kv_heads, dim, dtype):
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")
    from unchainkv_amd import splitzip_cuda as sz

    assert sz.available(), sz.load_error()
    print("[case]", rows, source, q_heads, kv_heads, dim, dtype, flush=True)
    q, keys, values = make(rows, source, q_heads, kv_heads, dim, dtype)
    block = 16
    held = [-(-m // block) for m in source]
    kv = torch.zeros((2, sum(held), block, kv_heads, dim), dtype=DTYPES[dtype])
    tables = torch.zeros((len(rows), max(held)), dtype=torch.int32)
    at = 0
    for r, (n, k, v) in enumerate(zip(held, keys, values)):
        tables[r, :n] = torch.arange(at, at + n)
        for plane, x in ((0, k), (1, v)):
            kv[plane, at:at + n].view(-1, kv_heads, dim)[:len(x)] = x
        at += n

    def i32(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    starts = i32(np.concatenate([[0], np.cumsum(rows)]).tolist())
    first, count = i32((np.cumsum(source) - source).tolist()), i32(source)
    results = [sz.cross_attention_paged(q.cuda(), kv.cuda(), tables.cuda(), starts, count, max_query=max(rows))]
    if max(rows) * (q_heads // kv_heads) <= 16:  # (packed rows beside tiles are in tiles too)
        results.append(sz.cross_attention(q.cuda(), torch.cat(keys).cuda(), torch.cat(values).cuda(), starts, first,
                                          count, max_query=max(rows), max_source=max(source)))
    for got in results:
        assert got is not None
        at = 0
        for r, n in enumerate(rows):
            if n * (q_heads // kv_heads) <= 16:
                mine = slice(at, at + n)
                assert worst(f64(got[mine]), f64(q[mine]), f64(keys[r]), f64(values[r]), dtype, dim ** -0.5) <= 1.0
            at += n
