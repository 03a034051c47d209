"""Attention over paged layers and of prompts at the edges of its contract: what joined splits keep,
how small a weight counts, which buffers and ranges of rows a call takes. Against float64 (the
bound is derived in paged_attention_ref.py) unless a test says otherwise."""

import numpy as np
import pytest

from paged_attention_ref import HALF_STEP, attend
from test_gpu_paged_attention import (  # noqa: F401 (sz: a fixture)
    DTYPES, MARK, Case, f64, i32, say, starts_of, sz)

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


def test_ranges_that_overlap_leave_whole_rows_or_none(sz):  # noqa: F811
    """Starts that run backwards ask for more items than a call launches: 1024 rows named three times
    and 1280 more, in tiles of 256 rows (32 tokens), each cut into two splits. 3 * 32 + 40 tiles make
    272 items; launched are 72 for the tiles of the rows, 6 for the requests and 193 for splits, so
    that the second split of the last tile is none of them. Each row is right or as it was, and
    nothing outside out, lse and the workspace's size is written."""
    dim, heads, block, context = 128, 8, 16, 3000
    gen = torch.Generator("cuda").manual_seed(31)
    blocks = -(-context // block)
    kv = torch.randn((2, 2 * blocks, block, 1, dim), generator=gen, device="cuda").bfloat16()
    order = torch.randperm(2 * blocks, generator=gen, device="cuda").int().view(2, blocks)
    tables = order[[0, 0, 0, 0, 0, 1]].contiguous()
    starts, rows = i32([0, 1024, 0, 1024, 0, 1024, 2304]), 2304 + 3
    q = torch.randn((rows, heads, dim), generator=gen, device="cuda").bfloat16()
    out = torch.full(q.shape, MARK, dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], MARK, dtype=torch.float32, device="cuda")
    need = sz.chunk_attention_workspace_bytes(rows, 6, heads, 1, dim, blocks * block)
    space = torch.full((need + (1 << 20),), 255, dtype=torch.uint8, device="cuda")  # (NaN partials)
    assert sz.chunk_attention_paged(q, kv, tables, starts, i32([context] * 6), out=out, lse=lse,
                                    workspace=space[:need]) is out
    torch.cuda.synchronize()
    assert (space[need:] == 255).all()
    assert (out[2304:] == MARK).all() and (lse[2304:] == MARK).all()
    left = (out == MARK).flatten(1).all(1)
    assert torch.equal(left, (lse == MARK).all(1))
    say("rows left", int(left.sum()))
    for table, first, n in ((order[0], 0, 1024), (order[1], 1024, 1280)):
        k, v = (plane[table.long()].view(-1, dim)[:context].double() for plane in (kv[0], kv[1]))
        keys, part = k.abs().T, slice(first, first + n)
        x = q[part].double()
        last = context - n + torch.arange(n, device="cuda")
        seen = torch.arange(context, device="cuda") <= last[:, None]
        score = torch.where(seen[:, None], x @ k.T * dim ** -0.5, -torch.inf)
        weight = torch.softmax(score, -1)
        expect, mean = weight @ v, weight @ v.abs()
        off = 2 * (dim + 8) * 2.0 ** -24 * (x.abs() @ keys).amax(-1) * dim ** -0.5 + 2.0 ** -20 + \
            context * 2.0 ** -24
        bound = HALF_STEP["bf16"] * (mean + expect.abs()) * 1.01 + 2 * off[..., None] * mean
        ok = ((out[part] - expect).abs() <= bound).flatten(1).all(1)
        assert (ok | left[part]).all()
        near = (lse[part] - torch.logsumexp(score, -1)).abs() <= 2 * off + 2.0 ** -20
        assert (near.all(1) | left[part]).all()


def test_workspace_of_the_largest_step_serves_smaller_ones(sz):  # noqa: F811
    """One workspace for prompts that are cut and prompts that are not: nothing else is allocated."""
    packed = torch.randn((4096, 48, 128), device="cuda").bfloat16()
    space = torch.empty(sz.prompt_attention_workspace_bytes(32768, 8, 32, 8, 128, 4096),
                        dtype=torch.uint8, device="cuda")
    for new in ([4096], [1024] * 4, [1443], [5, 900]):
        q, k, v = packed[:sum(new)].split((32, 8, 8), 1)
        starts, out = starts_of(new), torch.empty((sum(new), 32, 128), dtype=q.dtype, device="cuda")
        expect = sz.prompt_attention(q, k, v, starts, max_query=max(new))
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        assert sz.prompt_attention(q, k, v, starts, max_query=max(new), out=out, workspace=space) is out
        assert torch.cuda.max_memory_allocated() == held
        assert torch.equal(out, expect)


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (64, "fp16")])
def test_results_joined_by_their_log_sum_exps(sz, dim, dtype):  # noqa: F811
    """Attention over the first tokens and over the others, joined by lse, is attention over all (each
    part is within its bound, so the whole is, as the weights of the parts add up to 1; the parts'
    own rounding adds another half step of the mean)."""
    contexts, firsts = [70, 3000, 40], [32, 2000, 0]
    case = Case([1] * 3, contexts, 4, 2, dim, 16, dtype, seed=dim, spare_rows=0)
    parts = []
    for first, count in ((False, firsts), (True, [c - f for c, f in zip(contexts, firsts)])):
        tables = torch.full_like(case.tables, -1)
        for r, f in enumerate(firsts):
            own = case.tables[r, f // 16:] if first else case.tables[r, :f // 16]
            tables[r, :len(own)] = own
        lse = torch.empty(case.q.shape[:2], dtype=torch.float32, device="cuda")
        parts.append((sz.chunk_attention_paged(case.q, case.kv, tables, case.starts, i32(count),
                                               lse=lse).float(), lse))
    (o1, l1), (o2, l2) = parts
    lse = torch.logaddexp(l1, l2)
    out = f64(o1 * (l1 - lse).exp()[..., None] + o2 * (l2 - lse).exp()[..., None])
    for r, c in enumerate(contexts):
        ref, ref_lse, mean, off = attend(f64(case.q[r:r + 1]), case.k[r], case.v[r], c - 1, case.scale)
        bound = HALF_STEP[dtype] * (2 * mean + np.abs(ref)) * 1.01 + 4 * off[..., None] * mean + 2.0 ** -22
        assert (np.abs(out[r:r + 1] - ref) <= bound + (2.0 ** -24 if dtype == "fp16" else 0)).all()
        assert (np.abs(f64(lse[r:r + 1]) - ref_lse) <= 4 * off + 2.0 ** -20).all()
