"""Attention over sources of other lengths, in paged layers and in packed rows, against float64 (the
bound is derived in paged_attention_ref.py)."""

import numpy as np
import pytest

from paged_attention_ref import attend, check, check_lse

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MARK = 7.0


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


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(counts):
    return i32(np.concatenate([[0], np.cumsum(counts)]).tolist())


class Case:
    """Sources both in a layer and in packed rows, NaN around them; three rows of q are nobody's."""

    def __init__(self, rows, source, q_heads, kv_heads, dim, block, dtype, seed=0):
        rng = np.random.default_rng(seed)
        t = DTYPES[dtype]
        self.rows, self.source, self.dtype, self.scale = rows, source, dtype, dim ** -0.5
        held = [-(-c // block) for c in source]
        order, width = rng.permutation(sum(held) + 2), max(held) + 1
        tables = np.full((len(rows), width), -1, np.int32)
        kv = torch.full((2, sum(held) + 2, block, kv_heads, dim), float("nan"), dtype=t)
        self.k, self.v, at, packed, first = [], [], 0, [[], []], []
        gap = torch.full((3, kv_heads, dim), float("nan"), dtype=t)
        for r, c in enumerate(source):
            kv_rows = torch.from_numpy(rng.standard_normal((2, c, kv_heads, dim)).astype(np.float32)).to(t)
            tables[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
            for p in range(2):
                for j in range(held[r]):
                    part = kv_rows[p, j * block:(j + 1) * block]
                    kv[p, tables[r, j], :part.shape[0]] = part
                packed[p] += [gap, kv_rows[p]]
            first.append(3 * (r + 1) + sum(source[:r]))
            self.k.append(f64(kv_rows[0]))
            self.v.append(f64(kv_rows[1]))
        q = rng.standard_normal((sum(rows) + 3, q_heads, dim)).astype(np.float32)
        self.q, self.kv, self.tables = torch.from_numpy(q).to(t).cuda(), kv.cuda(), i32(tables.tolist())
        self.pk, self.pv = (torch.cat(p + [gap]).cuda() for p in packed)
        self.starts, self.count, self.first = starts_of(rows), i32(source), i32(first)

    def buffers(self):
        return {"out": torch.full(self.q.shape, MARK, dtype=self.q.dtype, device="cuda"),
                "lse": torch.full(self.q.shape[:2], MARK, dtype=torch.float32, device="cuda")}

    def paged(self, sz, **more):
        b = self.buffers()
        assert sz.cross_attention_paged(self.q, self.kv, self.tables, self.starts, self.count, **b,
                                        **more) is b["out"]
        return b["out"], b["lse"]

    def packed(self, sz, k=None, v=None, **more):
        b = self.buffers()
        assert sz.cross_attention(self.q, self.pk if k is None else k, self.pv if v is None else v,
                                  self.starts, self.first, self.count, **b, **more) is b["out"]
        return b["out"], b["lse"]

    def verify(self, out, lse, skip=()):
        out, lse, q, at = f64(out), f64(lse), f64(self.q), 0
        for r, (n, m) in enumerate(zip(self.rows, self.source)):
            if r in skip:
                assert (out[at:at + n] == MARK).all() and (lse[at:at + n] == MARK).all()
            elif n:
                want, want_lse, mean, off = attend(q[at:at + n], self.k[r], self.v[r], m, self.scale)
                v_max = np.abs(self.v[r]).max() if m else 0.0
                check(out[at:at + n], want, mean, off, self.dtype, m, v_max)
                check_lse(lse[at:at + n], want_lse, off)
            at += n
        assert (out[at:] == MARK).all() and (lse[at:] == MARK).all()


SHAPES = [
    # single tokens and beams, one token of source, block boundaries, none at all
    ([1], [1], 2, 2, 64, 16, "bf16"), ([1, 1, 1], [16, 17, 0], 4, 4, 64, 16, "fp16"),
    ([5, 5, 3, 1], [1500, 0, 33, 1031], 4, 4, 64, 16, "fp16"),
    ([4, 2], [1300, 7], 8, 2, 128, 16, "bf16"), ([1, 0, 2], [2500, 9, 64], 8, 1, 128, 24, "fp16"),
    # rows past the streamed ones, tiles' ends, splits
    ([17, 200, 1], [70, 129, 2100], 2, 2, 64, 16, "bf16"), ([300, 3], [65, 640], 4, 1, 128, 8, "fp16"),
    ([40, 257], [1700, 64], 3, 1, 128, 12, "bf16"), ([130, 0, 20], [0, 50, 900], 2, 1, 64, 20, "fp16"),
    ([64] * 3, [3000, 1, 500], 2, 2, 128, 32, "bf16")]


@pytest.mark.parametrize("rows,source,q_heads,kv_heads,dim,block,dtype", SHAPES)
def test_matches_float64(sz, rows, source, q_heads, kv_heads, dim, block, dtype):
    say("cross", rows, source, q_heads, kv_heads, dim, block, dtype)
    case = Case(rows, source, q_heads, kv_heads, dim, block, dtype, seed=sum(rows))
    case.verify(*case.paged(sz, max_query=max(rows)))
    case.verify(*case.paged(sz))
    case.verify(*case.packed(sz, max_query=max(rows), max_source=max(max(source), 1)))
    case.verify(*case.packed(sz))


SPLITS = [
    # short splits of few sources, ends in each of them; as many sources as are taken whole, and one less
    ([1], [769], 2, 2, 64, 16, "bf16"), ([3, 1], [1025, 130], 4, 2, 64, 16, "fp16"),
    ([5], [2049], 3, 3, 128, 16, "bf16"),
    ([2, 1, 0, 4], [513, 9000, 700, 0], 8, 8, 128, 32, "fp16"), ([1], [16385], 4, 1, 64, 64, "bf16"),
    # and of tiles
    ([30], [513], 2, 2, 64, 16, "bf16"), ([70, 3], [1100, 2], 2, 1, 128, 16, "fp16"),
    ([300, 40], [600, 2049], 4, 1, 128, 24, "bf16"),
    ([1] * 192, [1025] + [3, 700] * 95 + [1600], 1, 1, 64, 16, "bf16"),
    ([2] * 191, [1025] + [3, 700] * 95, 2, 1, 128, 16, "fp16")]


@pytest.mark.parametrize("rows,source,q_heads,kv_heads,dim,block,dtype", SPLITS, ids=range(len(SPLITS)))
def test_splits_match_float64(sz, rows, source, q_heads, kv_heads, dim, block, dtype):
    say("splits", rows[:4], source[:4], q_heads, kv_heads, dim, block, dtype)
    case = Case(rows, source, q_heads, kv_heads, dim, block, dtype, seed=max(source))
    case.verify(*case.paged(sz, max_query=max(rows)))
    case.verify(*case.packed(sz, max_query=max(rows), max_source=max(source)))


@pytest.mark.parametrize("seed", range(6))
def test_drawn_shapes(sz, seed):
    rng = np.random.default_rng(100 + seed)
    requests = int(rng.integers(1, 90 if seed == 5 else 9))
    rows = [int(n) for n in 2 ** rng.uniform(0, 3 if seed % 2 else 8, requests) - 1 + (seed != 4)]
    source = [int(n) for n in 2 ** rng.uniform(0, 8 if seed == 5 else 11, requests) - 1]
    kv_heads, dtype = int(rng.integers(1, 4)), ("bf16", "fp16")[seed % 2]
    shape = (rows, source, kv_heads * int(rng.integers(1, 6)), kv_heads, (64, 128)[seed // 2 % 2],
             int(rng.integers(1, 34)), dtype)
    say("drawn", *shape)
    case = Case(*shape, seed=seed)
    if sum(rows) == 0:
        return
    case.verify(*case.paged(sz, max_query=max(rows)))
    case.verify(*case.packed(sz, max_query=max(rows), max_source=max(max(source), 1)))


def test_rows_left_as_they_are(sz):
    """More rows than max_query, a longer source than max_source."""
    say("left")
    case = Case([2, 6, 1], [40, 50, 900], 2, 2, 64, 16, "bf16")
    case.verify(*case.paged(sz, max_query=5), skip=(1,))
    case.verify(*case.packed(sz, max_query=5, max_source=50), skip=(1, 2))
    case.verify(*case.packed(sz, max_source=49), skip=(1, 2))


def test_bad_sources(sz):
    """Rows of a source that is not inside k, or of blocks that are none, are NaN; others keep theirs."""
    say("bad")
    for rows in ([2, 3, 1], [20, 40, 30]):
        case = Case(rows, [40, 50, 30], 2, 2, 64, 16, "bf16")
        good = case.packed(sz)[0]
        most = case.pk.shape[0]
        for first in (-1, most - 49, most, 2 ** 31 - 1):
            case.first[1] = first
            out, lse = case.packed(sz)
            a, b = rows[0], rows[0] + rows[1]
            assert out[a:b].isnan().all() and lse[a:b].isnan().all()
            assert torch.equal(out[:a], good[:a]) and torch.equal(out[b:], good[b:])
        case.tables[1, 1] = 10 ** 6
        out, _ = case.paged(sz)
        assert out[a:b].isnan().all() and not out[:a].isnan().any() and not out[b:].isnan().any()


def test_strided_and_shared_sources(sz):
    """K and V as views of one projection; padded batches; two requests of one source."""
    say("strided")
    case = Case([3, 40], [70, 200], 4, 2, 64, 16, "fp16")
    both = torch.stack((case.pk, case.pv), 1).flatten(1, 2)  # (rows, 2 * heads, dim)
    case.verify(*case.packed(sz, k=both[:, :2], v=both[:, 2:]))
    padded = torch.full((2, 200, 4, 64), float("nan"), dtype=torch.float16, device="cuda")
    for r, (m, f) in enumerate(zip(case.source, case.first.tolist())):
        padded[r, :m] = both[f:f + m]
    rows = padded.flatten(0, 1)
    case.first = i32([0, 200])
    case.verify(*case.packed(sz, k=rows[:, :2], v=rows[:, 2:], max_source=200))
    case.k[0], case.v[0], case.source[0] = case.k[1], case.v[1], 200
    case.first, case.count = i32([200, 200]), i32([200, 200])
    case.verify(*case.packed(sz, k=rows[:, :2], v=rows[:, 2:]))


@pytest.mark.parametrize("rows", ([2, 1], [30, 200]))
def test_infinite_and_nan_values(sz, rows):
    """They reach the rows of their own request, and no other."""
    say("values", rows)
    case = Case(rows, [90, 1100], 2, 2, 128, 16, "bf16")
    good = case.packed(sz)[0].clone()
    f = case.first.tolist()
    case.pv[f[1] + 1090, 0, 5] = float("inf")
    case.pk[f[1] + 3, 1] = float("nan")
    out, lse = case.packed(sz)
    a, b = rows[0], sum(rows)
    assert torch.equal(out[:a], good[:a])
    # (such rows are formed again with weights in 32 bits, so they need not have the bits of `good`: both
    # are within the bound)
    want, _, mean, off = attend(f64(case.q)[a:b], case.k[1], case.v[1], 1100, case.scale)
    check(f64(out)[a:b, 0, :5], want[:, 0, :5], mean[:, 0, :5], off[:, 0], "bf16", 1100, 1.0)
    assert (out[a:b, 0, 5] == float("inf")).all() and out[a:b, 1].isnan().all()
    assert lse[a:b, 1].isnan().all() and lse[a:b, 0].isfinite().all()


def test_beams_and_single_rows_agree(sz):
    """Beams as the rows of one request, and as requests that share its source."""
    say("beams")
    case = Case([4], [777], 8, 2, 128, 16, "bf16")
    out, lse = case.paged(sz, max_query=4)
    case.verify(out, lse)
    apart = Case([1] * 4, [777] * 4, 8, 2, 128, 16, "bf16")
    apart.q, apart.kv, apart.tables = case.q, case.kv, case.tables.repeat(4, 1)
    apart.k, apart.v = case.k * 4, case.v * 4
    apart.verify(*apart.paged(sz, max_query=1))


def test_captured_calls_follow_lengths(sz):
    """A captured call, replayed with other lengths, tables and rows, with its own workspace."""
    say("captured")
    case = Case([4, 4, 4], [900, 1500, 1800], 4, 2, 64, 16, "bf16")
    rows, source = list(case.rows), list(case.source)
    b, b2 = case.buffers(), case.buffers()
    ws = [torch.empty(max(sz.cross_attention_workspace_bytes(15, 3, 4, 2, 64, n, 4), 1), dtype=torch.uint8,
                      device="cuda") for n in (case.tables.shape[1] * 16, 1800)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sz.cross_attention_paged(case.q, case.kv, case.tables, case.starts, case.count, max_query=4,
                                 workspace=ws[0], **b)
        sz.cross_attention(case.q, case.pk, case.pv, case.starts, case.first, case.count, max_query=4,
                           max_source=1800, workspace=ws[1], **b2)
    for new_rows, new_source in ((rows, source), ([1, 4, 2], [900, 3, 0]), ([0, 2, 1], [1, 1500, 1024])):
        case.rows, case.source = new_rows, new_source
        full = case.k, case.v
        case.k = [k[:m] for k, m in zip(case.k, new_source)]
        case.v = [v[:m] for v, m in zip(case.v, new_source)]
        case.starts.copy_(starts_of(new_rows))
        case.count.copy_(i32(new_source))
        for x in (*b.values(), *b2.values()):
            x.fill_(MARK)
        graph.replay()
        torch.cuda.synchronize()
        case.verify(b["out"], b["lse"])
        case.verify(b2["out"], b2["lse"])
        case.k, case.v = full


def test_refuses(sz):
    case = Case([2, 2], [40, 50], 4, 2, 64, 16, "bf16")

    def packed(q=case.q, k=case.pk, v=case.pv, starts=case.starts, first=case.first, count=case.count,
               **more):
        return sz.cross_attention(q, k, v, starts, first, count, **more)

    def paged(q=case.q, kv=case.kv, tables=case.tables, starts=case.starts, count=case.count, **more):
        return sz.cross_attention_paged(q, kv, tables, starts, count, **more)

    assert packed() is not None and paged() is not None
    assert packed(q=case.q.float()) is None and packed(k=case.pk.half()) is None
    assert packed(v=case.pv[:-1]) is None and packed(q=case.q[:, :3]) is None
    assert packed(k=case.pk[..., :32], v=case.pv[..., :32], q=case.q[..., :32]) is None
    assert packed(first=case.first[:1]) is None and packed(count=case.count.long()) is None
    assert packed(starts=case.starts[:2]) is None and packed(first=case.first.cpu()) is None
    assert packed(max_query=0) is None and packed(max_source=-1) is None and packed(scale=-1.0) is None
    assert packed(out=case.pk[:7].view(7, -1, 64)) is None
    assert packed(k=case.pk[:0], v=case.pv[:0]) is None
    assert paged(starts=case.starts[:2]) is None and paged(tables=case.tables.long()) is None
    assert paged(count=case.count[:1]) is None and paged(kv=case.kv[0]) is None
    assert paged(out=case.q) is None
    empty = packed(first=case.first[:0], count=case.count[:0], starts=case.starts[:1])
    assert empty.shape == case.q.shape
