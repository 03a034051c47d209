"""Attention over paged layers and of prompts at the edges of its contract: what joined splits keep,
how small a weight counts, which buffers and ranges of rows a call takes. Against float64 (the
bound is derived in paged_attention_ref.py) unless a test says otherwise."""

import numpy as np
import pytest

from paged_attention_ref import HALF_STEP
from test_gpu_paged_attention import DTYPES, Case, f64, i32, say, starts_of, sz  # noqa: F401 (sz)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (64, "fp16")])
@pytest.mark.parametrize("key", [0.0, float("-inf")])
@pytest.mark.parametrize("new,contexts", [([1], [4000]), ([1, 2], [90, 4000]),
                                          ([40, 1], [4000, 50]), ([300], [4000])])
def test_values_of_a_split_without_weight(sz, dim, dtype, key, new, contexts):  # noqa: F811
    """A NaN V value that rows see reaches them where every weight of its split underflows beside
    another split's: the keys of the first half of a context score 0 (or -inf), those of the second
    20 sqrt(dim) (230 powers of two at 64 dims)."""
    say("no weight", dim, dtype, key, new, contexts)
    case = Case(new, contexts, 4, 2, dim, 16, dtype, seed=dim)
    r = int(np.argmax(contexts))
    case.q[:] = 1.0
    for first, last, value in ((0, 2000, key), (2000, 4000, 20.0)):
        case.k[r][first:last] = value
        case.kv[0, case.tables[r, first // 16:last // 16].long()] = value
    case.kv[1, int(case.tables[r, 6]), 4, 0, 5] = float("nan")  # token 100
    case.v[r][100, 0, 5] = float("nan")
    out, lse = case.run(sz)
    at = sum(new[:r])
    rows = out[at:at + new[r]]
    assert torch.isnan(rows[:, :2, 5]).all()
    assert torch.isfinite(rows[:, 2:]).all() and torch.isfinite(rows[:, :2, :5]).all()
    if key == 0.0:  # (a score of -inf has no bound)
        case.verify(out, lse)


@pytest.mark.parametrize("dim,dtype", [(64, "fp16"), (128, "fp16"), (128, "bf16")])
@pytest.mark.parametrize("new", [1, 40])
def test_many_small_weights(sz, dim, dtype, new):  # noqa: F811
    """32768 tokens of weight 2^-26.3 beside one of 1, which is in no value: their sum counts. Enough
    requests (of one table) that no context is cut, so that one reference serves all tokens.

    The bound is paged_attention_ref's, but for what fp16 weights lose: with 2^7 to spare a weight
    below 2^-21 of the largest is off by 2^-32 of it at most."""
    say("small weights", dim, dtype, new)
    requests, heads, block, tail, score = 64, 8, 16, 32768, -18.25
    context = 1 + tail + new - 1
    blocks = -(-context // block)
    kv = torch.empty((2, blocks, block, heads, dim), dtype=DTYPES[dtype], device="cuda")
    kv[0], kv[1] = score / (dim / 8), 1.0
    kv[:, 0, 0] = 0.0
    q = torch.ones((requests * new, heads, dim), dtype=DTYPES[dtype], device="cuda")
    tables = torch.arange(blocks, dtype=torch.int32, device="cuda").expand(requests, -1).contiguous()
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    out = sz.chunk_attention_paged(q, kv, tables, starts_of([new] * requests),
                                   i32([context] * requests), scale=0.125, max_query=new, lse=lse)
    torch.cuda.synchronize()
    seen = tail + np.arange(new)
    share = seen * np.exp(score) / (1 + seen * np.exp(score))
    expect = np.tile(share, requests)[:, None, None]
    off = 2 * (dim + 8) * 2.0 ** -24 * -score + 2.0 ** -20 + context * 2.0 ** -24
    bound = 2 * HALF_STEP[dtype] * expect * 1.01 + 2 * off * expect
    if dtype == "fp16":
        bound = bound + context * 2.0 ** -32 + 2.0 ** -25
    assert (np.abs(f64(out) - expect) <= bound).all()
    expect = np.log1p(np.tile(seen, requests) * np.exp(score))[:, None]
    assert (np.abs(f64(lse) - expect) <= 2 * off + 2.0 ** -22).all()
