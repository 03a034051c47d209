"""Chunk attention over a paged layer and prompt attention against float64 (the bound is derived
in paged_attention_ref.py), at the sizes, masks and layouts where they can go wrong."""

import numpy as np
import pytest

from paged_attention_ref import attend, check, check_lse

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MARK = 7.0  # what rows of no request hold before and after


@pytest.fixture(scope="module")
def sz():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")
    from unchainkv_amd import splitzip_cuda

    assert splitzip_cuda.available(), splitzip_cuda.load_error()
    return splitzip_cuda


def say(*parts):
    print("[case]", *parts, flush=True)


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def starts_of(new):
    return torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Case:
    """A layer, tables and queries; tokens past a request's context and unused blocks are NaN."""

    def __init__(self, new, contexts, q_heads, kv_heads, dim, block, dtype, seed=0, spare_rows=3,
                 big=1.0):
        rng = np.random.default_rng(seed)
        self.new, self.contexts, self.block, self.dtype = new, contexts, block, dtype
        t = DTYPES[dtype]
        held = [-(-c // block) for c in contexts]
        pool = sum(held) + 3
        order = rng.permutation(pool)
        width = max(max(held), 1) + 1
        tables = np.full((len(new), width), -1, np.int32)
        at = 0
        for r, h in enumerate(held):
            tables[r, :h] = order[at:at + h]
            at += h
        kv = torch.full((2, pool, block, kv_heads, dim), float("nan"), dtype=t)
        self.k, self.v = [], []
        for r, c in enumerate(contexts):
            rows = torch.from_numpy(rng.standard_normal((2, c, kv_heads, dim)).astype(np.float32))
            rows[0] *= big
            rows = rows.to(t)
            for p in range(2):
                for j in range(held[r]):
                    part = rows[p, j * block:(j + 1) * block]
                    kv[p, tables[r, j], :part.shape[0]] = part
            self.k.append(f64(rows[0]))
            self.v.append(f64(rows[1]))
        self.q = torch.from_numpy(rng.standard_normal(
            (sum(new) + spare_rows, q_heads, dim)).astype(np.float32)).to(t).cuda()
        self.kv, self.tables = kv.cuda(), torch.from_numpy(tables).cuda()
        self.starts, self.ctx = starts_of(new), i32(contexts)
        self.scale = dim ** -0.5

    def run(self, sz, q=None, **more):
        out = torch.full(self.q.shape, MARK, dtype=self.q.dtype, device="cuda")
        lse = torch.full(self.q.shape[:2], MARK, dtype=torch.float32, device="cuda")
        got = sz.chunk_attention_paged(self.q if q is None else q, self.kv, self.tables,
                                       self.starts, self.ctx, out=out, lse=lse, **more)
        torch.cuda.synchronize()
        assert got is out
        return out, lse

    def verify(self, out, lse, skip=()):
        out, lse, q = f64(out), f64(lse), f64(self.q)
        at, worst = 0, 0.0
        for r, n in enumerate(self.new):
            if r not in skip and n:
                ref, ref_lse, mean, off = attend(q[at:at + n], self.k[r], self.v[r],
                                                 self.contexts[r] - n, self.scale)
                vmax = np.abs(self.v[r][np.isfinite(self.v[r])]).max() if self.contexts[r] else 0.0
                worst = max(worst, check(out[at:at + n], ref, mean, off, self.dtype,
                                         self.contexts[r], vmax))
                check_lse(lse[at:at + n], ref_lse, off)
            at += n
        assert np.all(out[at:] == MARK) and np.all(lse[at:] == MARK)
        say("worst", f"{worst:.3g}", "of the bound")


CHUNKS = [
    # (new tokens, contexts): one token each, short and long
    ([1], [1]),
    ([1, 1, 1], [1, 2, 700]),
    ([1] * 5, [31, 32, 33, 127, 129]),
    # drafted tokens, a request without new tokens between them
    ([3, 0, 4, 2], [40, 17, 4, 300]),
    # chunks around the tile sizes
    ([16, 17, 5], [16, 90, 64]),
    ([64, 1, 33], [200, 260, 33]),
    ([130], [130]),
    # rows that see nothing: contexts shorter than the chunk, and none at all
    ([5, 2, 40], [3, 0, 11]),
]


@pytest.mark.parametrize("new,contexts", CHUNKS)
@pytest.mark.parametrize("q_heads,kv_heads,dim,block,dtype", [
    (8, 2, 128, 16, "bf16"), (4, 4, 64, 8, "fp16"), (7, 1, 64, 24, "bf16"), (6, 2, 128, 5, "fp16")])
def test_chunk_attention(sz, new, contexts, q_heads, kv_heads, dim, block, dtype):
    say("chunk", new, contexts, q_heads, kv_heads, dim, block, dtype)
    case = Case(new, contexts, q_heads, kv_heads, dim, block, dtype, seed=len(new) + dim)
    case.verify(*case.run(sz))


@pytest.mark.parametrize("new", [[1], [1, 1, 5], [16, 33, 64, 65], [127, 3, 0, 129], [300]])
@pytest.mark.parametrize("q_heads,kv_heads,dim,dtype", [
    (8, 2, 128, "bf16"), (4, 4, 64, "fp16"), (3, 1, 64, "bf16"), (10, 2, 128, "fp16")])
def test_prompt_attention(sz, new, q_heads, kv_heads, dim, dtype):
    say("prompt", new, q_heads, kv_heads, dim, dtype)
    rng = np.random.default_rng(sum(new) + dim)
    heads, rows = q_heads + 2 * kv_heads, sum(new) + 2
    packed = torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32))
    packed = packed.to(DTYPES[dtype]).cuda()
    packed[sum(new):] = float("nan")
    q, k, v = packed.split((q_heads, kv_heads, kv_heads), 1)
    out = torch.full((rows, q_heads, dim), MARK, dtype=DTYPES[dtype], device="cuda")
    lse = torch.full((rows, q_heads), MARK, dtype=torch.float32, device="cuda")
    assert sz.prompt_attention(q, k, v, starts_of(new), out=out, lse=lse) is out
    torch.cuda.synchronize()
    got, got_lse, at = f64(out), f64(lse), 0
    for n in new:
        if n:
            part = slice(at, at + n)
            ref, ref_lse, mean, off = attend(f64(q[part]), f64(k[part]), f64(v[part]), 0, dim ** -0.5)
            check(got[part], ref, mean, off, dtype, n, np.abs(f64(v[part])).max())
            check_lse(got_lse[part], ref_lse, off)
        at += n
    assert np.all(got[at:] == MARK) and np.all(got_lse[at:] == MARK)


@pytest.mark.parametrize("q_heads,kv_heads,dim,block,dtype,new,contexts", [
    (32, 8, 128, 16, "bf16", [1] * 6, [8191, 1, 4096, 300, 77, 2048]),
    (8, 1, 128, 16, "fp16", [1, 2, 1], [20001, 9000, 131]),
    (8, 8, 64, 32, "bf16", [2, 40, 9, 1], [3000, 2500, 5001, 999]),
    (4, 1, 64, 16, "fp16", [200], [9000])])
def test_long_contexts_in_splits(sz, q_heads, kv_heads, dim, block, dtype, new, contexts):
    say("splits", q_heads, kv_heads, dim, block, dtype, new, contexts)
    case = Case(new, contexts, q_heads, kv_heads, dim, block, dtype, seed=dim)
    case.verify(*case.run(sz))


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (64, "fp16")])
def test_scores_that_leave_one_weight(sz, dim, dtype):
    """Large scores: the running reference moves often, and most weights vanish."""
    case = Case([1, 3, 70], [900, 500, 333], 4, 2, dim, 16, dtype, seed=3, big=40.0)
    case.verify(*case.run(sz))


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (64, "fp16")])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("new,contexts,where", [
    # (request, token): seen by the last rows of the chunk only
    ([40, 1], [60, 90], (0, 55)), ([3, 1], [300, 90], (0, 298)), ([200, 1], [700, 9], (0, 650))])
def test_values_that_rows_do_not_see(sz, dim, dtype, value, new, contexts, where):
    """A NaN or infinite V row reaches the rows that see it, and no others."""
    case = Case(new, contexts, 4, 2, dim, 16, dtype, seed=dim)
    r, t = where
    block = int(case.tables[r, t // 16])
    case.kv[1, block, t % 16, 0, 5] = value
    case.v[r][t, 0, 5] = value
    case.verify(*case.run(sz))


@pytest.mark.parametrize("new,contexts", [([2, 1], [50, 40]), ([64, 1], [150, 40])])
def test_keys_that_are_not_finite(sz, new, contexts):
    """A NaN key makes the rows that see it NaN (softmax of a NaN score) and no others; a key
    that makes every score -inf leaves no weight: 0 / 0."""
    case = Case(new, contexts, 2, 1, 128, 16, "bf16", seed=1)
    t = contexts[0] - 1
    case.kv[0, int(case.tables[0, t // 16]), t % 16, 0, 3] = float("nan")
    out, _ = case.run(sz)
    n = new[0]
    assert torch.isnan(out[n - 1]).all() and torch.isfinite(out[:n - 1]).all()
    assert torch.isfinite(out[n:sum(new)]).all()
    case.kv[0] = float("-inf")
    case.q[:] = 1.0
    out, _ = case.run(sz)
    assert torch.isnan(out[:sum(new)]).all()


def test_tables_that_name_no_block(sz):
    """Entries outside the layer and contexts past the table: NaN rows there, others untouched."""
    for new in ([1, 1, 2, 1], [40, 30, 64, 33]):
        case = Case(new, [100, 90, 200, 64], 4, 2, 128, 16, "bf16", seed=9)
        case.tables[1, 2] = case.kv.shape[1]
        case.tables[2, 0] = -5
        case.ctx[3] = case.tables.shape[1] * 16 + 1
        out, lse = case.run(sz)
        case.verify(out, lse, skip=(1, 2, 3))
        assert torch.isnan(out[new[0]:sum(new)]).all() and torch.isnan(lse[new[0]:sum(new)]).all()


def test_row_ranges_that_do_not_hold(sz):
    """Ranges outside q, backwards ones and requests past max_query: their rows stay."""
    case = Case([2, 3, 40], [50, 60, 70], 4, 2, 128, 16, "bf16", seed=2)
    out, lse = case.run(sz, max_query=3)
    assert (out[5:] == MARK).all() and (lse[5:] == MARK).all()
    case.verify(out, lse, skip=(2,))
    whole, _ = case.run(sz)
    case.starts = i32([0, 2, 5, 1 << 20])
    out, _ = case.run(sz)
    assert torch.equal(out[:5], whole[:5]) and (out[5:] == MARK).all()
    case.starts = i32([0, 2, 1, 41])  # (row 1 is in two ranges: either's)
    out, _ = case.run(sz)
    assert torch.equal(out[:1], whole[:1]) and (out[41:] == MARK).all()
    case.starts = i32([-1, -1, -1, -1])
    out, _ = case.run(sz)
    assert (out == MARK).all()


def test_strides_and_orders(sz):
    """q as a view of a projection, heads first, and one row for all; the same values."""
    case = Case([3, 30, 1], [40, 95, 200], 8, 2, 128, 16, "bf16", seed=6)
    whole, lse = case.run(sz)
    packed = torch.cat([case.q, torch.full_like(case.q[:, :4], float("nan"))], 1)[:, :8]
    first = case.q.transpose(0, 1).contiguous().transpose(0, 1)
    for q in (packed, first):
        assert not q.is_contiguous()
        out, other = case.run(sz, q=q)
        assert torch.equal(out, whole) and torch.equal(other, lse)
    case.tables = torch.cat([case.tables, case.tables], 1)[:, :case.tables.shape[1]]
    assert not case.tables.is_contiguous()
    out, _ = case.run(sz)
    assert torch.equal(out, whole)
    one = case.q[:1].expand(case.q.shape)
    out, _ = case.run(sz, q=one)
    same, _ = case.run(sz, q=one.contiguous())
    assert torch.equal(out, same)


def test_offsets_past_32_bits(sz):
    """Blocks whose element offsets pass 2^32 (a plane of 9 GB)."""
    kv = torch.empty((2, 280_000, 16, 8, 128), dtype=torch.bfloat16, device="cuda")
    case = Case([1, 40], [70, 120], 8, 8, 128, 16, "bf16", seed=8)
    far = [279_999 - 3 * j for j in range(case.kv.shape[1])]
    kv[:, far] = case.kv
    case.kv = kv
    case.tables = torch.where(case.tables >= 0, i32(far)[case.tables.clamp_min(0).long()], -1).int()
    case.verify(*case.run(sz))
    slots = torch.tensor([far[0] * 16 + 3], device="cuda")
    k = torch.randn((1, 8, 128), device="cuda").bfloat16()
    assert sz.write_kv_paged(k, 2 * k, kv, slots)
    assert torch.equal(kv[0, far[0], 3], k[0]) and torch.equal(kv[1, far[0], 3], 2 * k[0])


def test_same_results_every_time(sz):
    """No order of arrival decides a result: runs of one call are equal, on any stream and
    beside another call."""
    a = Case([1, 5, 60, 1], [3000, 800, 900, 70], 8, 2, 128, 16, "bf16", seed=12)
    b = Case([1] * 8, [500] * 8, 8, 2, 128, 16, "bf16", seed=13)
    first_a, first_b = a.run(sz)[0], b.run(sz)[0]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        got = []
        for case, stream in ((a, streams[0]), (b, streams[1])):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(sz.chunk_attention_paged(case.q, case.kv, case.tables, case.starts, case.ctx))
        torch.cuda.synchronize()
        assert torch.equal(got[0][:67], first_a[:67]) and torch.equal(got[1][:8], first_b[:8])


def test_captured_prompt_follows_new_lengths(sz):
    rows, heads = 300, (8, 2, 2)
    packed = torch.zeros((rows, sum(heads), 64), dtype=torch.bfloat16, device="cuda")
    q, k, v = packed.split(heads, 1)
    starts = i32([0, 0, 0, 0])
    out = torch.full((rows, 8, 64), MARK, dtype=torch.bfloat16, device="cuda")
    assert sz.prompt_attention(q, k, v, starts, out=out) is out  # (loads the kernels)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sz.prompt_attention(q, k, v, starts, out=out)
    for new in ([300, 0, 0], [10, 100, 50], [1, 1, 1], [64, 64, 64]):
        say("replay", new)
        packed.copy_(torch.randn(packed.shape, device="cuda"))
        starts.copy_(starts_of(new))
        out.fill_(MARK)
        graph.replay()
        torch.cuda.synchronize()
        got, at = f64(out), 0
        for n in new:
            if n:
                part = slice(at, at + n)
                ref, _, mean, off = attend(f64(q[part]), f64(k[part]), f64(v[part]), 0, 64 ** -0.5)
                check(got[part], ref, mean, off, "bf16", n, np.abs(f64(v[part])).max())
            at += n
        assert np.all(got[at:] == MARK)
        torch.randn(1 << 16, device="cuda").sum()


def test_attention_refuses(sz):
    case = Case([2, 1], [40, 30], 4, 2, 64, 16, "bf16", seed=1)

    def call(q=case.q, kv=case.kv, tables=case.tables, starts=case.starts, ctx=case.ctx, **more):
        return sz.chunk_attention_paged(q, kv, tables, starts, ctx, **more)

    assert call() is not None
    assert call(q=case.q.float()) is None and call(q=case.q.half()) is None
    assert call(q=case.q[:, :3]) is None  # 3 query heads for 2 KV heads
    assert call(q=case.q[..., :32]) is None
    assert call(q=case.q[0]) is None
    assert call(q=case.q.transpose(1, 2).contiguous().transpose(1, 2)) is None
    odd = torch.zeros(case.q.numel() + 1, dtype=case.q.dtype, device="cuda")[1:].view(case.q.shape)
    assert call(q=odd) is None  # not 16-byte aligned
    assert call(kv=case.kv[:, ::2]) is None and call(kv=case.kv[0]) is None
    assert call(tables=case.tables.long()) is None and call(tables=case.tables[0]) is None
    assert call(starts=case.starts[:2]) is None and call(ctx=case.ctx.long()) is None
    assert call(ctx=case.ctx[:1]) is None and call(max_query=0) is None
    assert call(scale=-1.0) is None and call(scale=float("nan")) is None
    assert call(out=case.q) is None and call(out=torch.empty_like(case.q).half()) is None
    assert call(lse=torch.empty(case.q.shape[:2], device="cuda", dtype=torch.float64)) is None
    assert call(q=case.q.clone().requires_grad_()) is None
    with torch.no_grad():
        assert call(q=case.q.clone().requires_grad_()) is not None
    assert call(q=case.q[:0]).shape == (0, 4, 64)
    k = torch.zeros((5, 2, 64), dtype=torch.bfloat16, device="cuda")
    starts = i32([0, 5])
    q = torch.zeros((5, 4, 64), dtype=torch.bfloat16, device="cuda")
    assert sz.prompt_attention(q, k, k, starts) is not None
    assert sz.prompt_attention(q, k, k[:4], starts) is None
    assert sz.prompt_attention(q, k.half(), k, starts) is None
    assert sz.prompt_attention(q, k, k, starts.long()) is None
    assert sz.prompt_attention(q, k, k, starts, out=q) is None
    assert sz.prompt_attention(q.clone().requires_grad_(), k, k, starts) is None
    assert sz.prompt_attention(q, k, k, starts[:1]) is not None  # no prompts


@pytest.mark.parametrize("q_heads,kv_heads,dim,block,dtype", [
    (8, 2, 128, 16, "bf16"), (8, 2, 64, 8, "fp16"), (4, 4, 64, 24, "bf16"), (3, 1, 128, 7, "fp16")])
def test_single_tokens_beside_chunks(sz, q_heads, kv_heads, dim, block, dtype):
    """Streamed requests, short and cut into splits, in one call with tiles, cut ones too."""
    new, contexts = [1, 70, 2, 1, 0, 33, 1, 3], [5000, 4100, 2600, 1, 900, 33, 129, 0]
    say("beside", q_heads, kv_heads, dim, block, dtype)
    case = Case(new, contexts, q_heads, kv_heads, dim, block, dtype, seed=dim + block)
    case.verify(*case.run(sz))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_streamed_values_and_blocks_beside_chunks(sz, dim, value):
    """What a streamed request's rows do not see does not reach them, nor another request; a table
    entry that is no block makes its rows NaN, in whichever split it is read."""
    case = Case([3, 90, 1], [2600, 300, 2500], 4, 2, dim, 16, "bf16", seed=dim)
    t = 2598  # the second new token
    case.kv[1, int(case.tables[0, t // 16]), t % 16, 1, 9] = value
    case.v[0][t, 1, 9] = value
    case.tables[2, 3] = case.kv.shape[1] + 4
    out, lse = case.run(sz)
    case.verify(out, lse, skip=(2,))
    assert torch.isnan(out[93]).all() and torch.isnan(lse[93]).all()


@pytest.mark.parametrize("longest,context", [(1, 700), (1, 3000), (40, 1500)])
def test_more_requests_than_lanes(sz, longest, context):
    """150 requests: three loads of lengths, in order and with empty ones between."""
    rng = np.random.default_rng(longest + context)
    new = [int(n) for n in rng.integers(0, 2, 150)]
    new[77], new[149] = longest, 1
    contexts = [int(c) for c in rng.integers(1, 90, 150)]
    contexts[3], contexts[77], contexts[149] = context, context, 1200
    new[3] = 1
    say("requests", longest, context)
    case = Case(new, contexts, 4, 2, 64, 16, "bf16", seed=longest)
    case.verify(*case.run(sz))


@pytest.mark.parametrize("heads,dim,dtype,new", [
    ((4, 1), 128, "bf16", [1100, 3, 900]), ((2, 2), 64, "fp16", [1700])])
def test_long_prompts_in_splits(sz, heads, dim, dtype, new):
    say("long prompts", heads, dim, dtype, new)
    q_heads, kv_heads = heads
    rng = np.random.default_rng(dim)
    rows = sum(new) + 1
    packed = torch.from_numpy(rng.standard_normal((rows, q_heads + 2 * kv_heads, dim)).astype(
        np.float32)).to(DTYPES[dtype]).cuda()
    q, k, v = packed.split((q_heads, kv_heads, kv_heads), 1)
    out = torch.full((rows, q_heads, dim), MARK, dtype=DTYPES[dtype], device="cuda")
    assert sz.prompt_attention(q, k, v, starts_of(new), out=out) is out
    torch.cuda.synchronize()
    got, at = f64(out), 0
    for n in new:
        part = slice(at, at + n)
        ref, _, mean, off = attend(f64(q[part]), f64(k[part]), f64(v[part]), 0, dim ** -0.5)
        check(got[part], ref, mean, off, dtype, n, np.abs(f64(v[part])).max())
        at += n
    assert np.all(got[at:] == MARK)


def test_one_workspace_for_steps_of_any_lengths(sz):
    """A captured call and eager ones of other sizes take turns with one workspace: what one left in
    it (slots of splits that the next does not have) changes nothing."""
    long = Case([1, 40, 1], [3000, 2900, 2000], 8, 2, 128, 16, "bf16", seed=20)
    short = Case([40, 1, 1], [50, 60, 900], 8, 2, 128, 16, "bf16", seed=21)
    few = Case([1] * 5, [2000, 300, 4000, 1, 90], 8, 2, 128, 16, "bf16", seed=22)
    size = max(sz.chunk_attention_workspace_bytes(c.q.shape[0], len(c.new), 8, 2, 128,
                                                  c.tables.shape[1] * 16, most)
               for c, most in ((long, 40), (short, 40), (few, 1)))
    space = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    runs = [(long, 40), (short, 40), (few, 1)]
    for case, most in runs:
        case.verify(*case.run(sz, workspace=space, max_query=most))
    out = torch.full(long.q.shape, MARK, dtype=long.q.dtype, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sz.chunk_attention_paged(long.q, long.kv, long.tables, long.starts, long.ctx, out=out,
                                 workspace=space, max_query=40)
    whole, _ = long.run(sz)
    lengths = [3000, 2900, 2000]
    for turn in range(4):
        say("turn", turn)
        case, most = runs[1 + turn % 2]
        case.verify(*case.run(sz, workspace=space, max_query=most))
        out.fill_(MARK)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, whole)
        # the same graph with short contexts, which it does not cut
        long.ctx.copy_(i32([50, 60, 70]))
        short_run, _ = long.run(sz)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, short_run)
        long.ctx.copy_(i32(lengths))


def test_ranges_that_overlap_stay_inside_the_call(sz):
    """Starts that run backwards name more rows than q has: more tiles than the call launches. Rows
    may be left, every other one is right, and nothing outside is written."""
    case = Case([40, 40, 40], [3000, 3000, 3000], 4, 1, 64, 16, "bf16", seed=30)
    case.starts = i32([0, 120, 0, 120])
    case.ctx = i32([3000, 3000, 3000])
    out, _ = case.run(sz)
    assert (out[120:] == MARK).all()
    fresh = Case([40, 40, 40], [3000, 3000, 3000], 4, 1, 64, 16, "bf16", seed=30)
    fresh.verify(*fresh.run(sz))
