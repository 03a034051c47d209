"""Step plans (block tables, row ranges, slots, positions from request lengths) and the K/V
write, against plain Python; a step's calls run together, eagerly and captured."""

import numpy as np
import pytest

from paged_attention_ref import attend, check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sz():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")
    from unchainkv_amd import splitzip_cuda

    assert splitzip_cuda.available(), splitzip_cuda.load_error()
    return splitzip_cuda


def say(*parts):
    print("[case]", *parts, flush=True)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def plain_plan(new, cached, tables, free, start, block, rows):
    """The plan by plain loops over Python integers."""
    tables = [list(t) for t in tables]
    width = len(tables[0])
    slots, positions, starts, lacking = [-1] * rows, [0] * rows, [0], 0
    begin = start
    for r, (n, c) in enumerate(zip(new, cached)):
        n, c = max(n, 0), max(c, 0)
        for j in range(-(-c // block), -(-(c + n) // block)):
            if j >= width:
                lacking += 1
                continue
            tables[r][j] = free[start] if start < len(free) else -1
            lacking += start >= len(free)
            start += 1
        for i in range(n):
            t, p = starts[-1] + i, c + i
            if t < rows:
                positions[t] = p
                if p // block < width and tables[r][p // block] >= 0:
                    slots[t] = tables[r][p // block] * block + p % block
        starts.append(starts[-1] + n)
    contexts = [max(n, 0) + max(c, 0) for n, c in zip(new, cached)]
    return tables, starts, contexts, slots, positions, min(start, max(begin, len(free))), lacking


def random_step(rng, requests, longest, block, width, free_count):
    cached = rng.integers(0, width * block // 2 + 1, requests).tolist()
    new = [int(rng.integers(0, min(longest, width * block - c) + 1)) for c in cached]
    pool = rng.permutation(requests * width + free_count)
    tables = np.full((requests, width), -1, np.int64)
    at = 0
    for r, c in enumerate(cached):
        held = -(-c // block)
        tables[r, :held] = pool[at:at + held]
        at += held
    return new, cached, tables.tolist(), pool[at:at + free_count].tolist()


def check_plan(sz, new, cached, tables, free, start, block, rows, plan=None, strided=False):
    wide = torch.full((len(new), len(tables[0]) + 3), 77, dtype=torch.int32, device="cuda")
    dev = wide[:, :-3] if strided else torch.empty_like(wide[:, :-3]).contiguous()
    dev.copy_(torch.tensor(tables))
    got = sz.plan_step_paged(i32(new), i32(cached), dev, i32(free), i32([start]), block, rows,
                             plan=plan)
    torch.cuda.synchronize()
    assert got is not None
    ref = plain_plan(new, cached, tables, free, start, block, rows)
    for name, a, b in zip(("tables", "starts", "contexts", "slots", "positions", "next", "lacking"),
                          (dev, got.query_starts, got.context_tokens, got.slots, got.positions,
                           got.free_next[0], got.lacking[0]), ref):
        assert np.array_equal(a.cpu().numpy(), np.array(b)), name
    assert (wide[:, -3:] == 77).all()
    return got


@pytest.mark.parametrize("requests,longest,block,width,rows_spare", [
    (1, 1, 16, 4, 0), (3, 40, 16, 9, 5), (64, 1, 16, 40, 0), (65, 3, 8, 20, 2), (256, 30, 24, 6, 17),
    (1025, 2, 16, 4, 0), (2500, 3, 1, 9, 3), (7, 900, 5, 400, 300)])
def test_plan_matches_plain_loops(sz, requests, longest, block, width, rows_spare):
    say("plan", requests, longest, block, width)
    rng = np.random.default_rng(requests + longest)
    new, cached, tables, free = random_step(rng, requests, longest, block, width, requests * width)
    check_plan(sz, new, cached, tables, free, requests % 5, block, sum(new) + rows_spare,
               strided=requests % 2 == 1)


def test_plan_edges(sz):
    # nothing new, negative lengths, a block boundary on either side
    check_plan(sz, [0, 0], [5, 16], [[3, -1], [4, -1]], [9, 8], 0, 16, 0)
    check_plan(sz, [-3, 4, 1], [4, -2, 15], [[1, -1], [-1, -1], [2, -1]], [9, 8], 0, 16, 9)
    check_plan(sz, [1, 1, 17], [16, 15, 15], [[1, -1, -1], [2, -1, -1], [3, -1, -1]],
               [11, 12, 13, 14], 1, 16, 19)
    # an empty free list, one that ends inside the step, a start past its end
    check_plan(sz, [20], [0], [[-1, -1]], [], 0, 16, 20)
    check_plan(sz, [20, 40], [0, 3], [[-1] * 4, [5, -1, -1, -1]], [10, 11, 12], 0, 16, 60)
    check_plan(sz, [20], [0], [[-1, -1]], [1, 2], 7, 16, 20)
    # a table narrower than the context, fewer rows than tokens
    check_plan(sz, [40, 2], [10, 0], [[6, -1], [-1, -1]], [1, 2, 3, 4], 0, 16, 42)
    check_plan(sz, [40, 2], [10, 0], [[6, -1, -1, -1], [-1] * 4], list(range(20, 30)), 0, 16, 11)


def test_plan_buffers_are_used_again(sz):
    rng = np.random.default_rng(5)
    plan = sz.new_step_plan(20, 700, "cuda")
    for _ in range(3):
        new, cached, tables, free = random_step(rng, 20, 30, 16, 10, 200)
        assert check_plan(sz, new, cached, tables, free, 3, 16, 700, plan=plan) is plan


def test_plan_refuses(sz):
    new, cached, tables, free, start = i32([1, 2]), i32([3, 4]), i32([[0, -1], [1, -1]]), i32([5, 6]), i32([0])
    plan = sz.new_step_plan(2, 8, "cuda")

    def call(new=new, cached=cached, tables=tables, free=free, start=start, block=16, rows=8, plan=plan):
        return sz.plan_step_paged(new, cached, tables, free, start, block, rows, plan=plan)

    assert call() is plan
    assert call(block=0) is None and call(rows=-1) is None
    assert call(new=new.long()) is None and call(cached=cached[:1]) is None
    assert call(tables=tables.t()) is None or tables.shape[1] == 1
    assert call(tables=tables[:1]) is None and call(free=free.cpu()) is None
    assert call(plan=sz.new_step_plan(1, 8, "cuda")) is None
    assert call(rows=9) is None  # more rows than the plan holds
    # results that overlap what is read, or each other
    assert call(cached=plan.context_tokens) is None
    assert call(start=plan.free_next) is None
    assert call(plan=plan._replace(positions=plan.slots)) is None
    assert call(new=new.cpu()) is None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,dim,block,layout", [
    (1, 8, 128, 16, "packed"), (64, 8, 128, 16, "rows"), (37, 3, 80, 5, "packed"),
    (300, 1, 64, 8, "heads"), (9, 2, 7, 3, "odd"), (5, 2, 12, 4, "odd"), (2049, 2, 128, 16, "packed")])
def test_write_kv(sz, tokens, heads, dim, block, layout, dtype):
    say("write", tokens, heads, dim, block, layout, dtype)
    rng = np.random.default_rng(tokens + dim)
    blocks = tokens // block + 4
    kv = torch.from_numpy(rng.standard_normal((2, blocks, block, heads, dim))).to(dtype).cuda()
    if layout == "packed":     # views of one projection
        _, k, v = torch.randn((tokens, 3 * heads, dim), device="cuda").to(dtype).split(heads, 1)
    elif layout == "heads":    # heads first in memory
        k, v = (torch.randn((heads, tokens, dim), device="cuda").to(dtype).transpose(0, 1)
                for _ in range(2))
    elif layout == "odd":      # rows at odd element offsets
        k, v = (torch.randn(tokens * (heads * dim + 1) + 1, device="cuda").to(dtype)[1:]
                .view(tokens, heads * dim + 1)[:, :-1].unflatten(1, (heads, dim)) for _ in range(2))
    else:
        k, v = torch.randn((2, tokens, heads, dim), device="cuda").to(dtype)
    slots = torch.from_numpy(rng.permutation(blocks * block)[:tokens]).cuda()
    slots[::7] = -1
    if tokens > 8:
        slots[3], slots[8] = blocks * block, 1 << 40  # past the layer
    expect = kv.clone()
    flat = expect.view(2, blocks * block, heads, dim)
    keep = (slots >= 0) & (slots < blocks * block)
    flat[0, slots[keep]], flat[1, slots[keep]] = k[keep], v[keep]
    got = sz.write_kv_paged(k, v, kv, slots)
    torch.cuda.synchronize()
    assert got == 4 * tokens * heads * dim
    assert torch.equal(kv, expect)


def test_write_refuses(sz):
    kv = torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    k = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.tensor([0, 1, 2], device="cuda")
    assert sz.write_kv_paged(k, k, kv, slots) == 4 * k.numel()
    assert sz.write_kv_paged(k[:0], k[:0], kv, slots) == 0
    assert sz.write_kv_paged(k.float(), k.float(), kv, slots) is None
    assert sz.write_kv_paged(k.half(), k.half(), kv, slots) is None
    assert sz.write_kv_paged(k, k[:2], kv, slots) is None
    assert sz.write_kv_paged(k, k, kv[:, :, :, :1], slots) is None
    assert sz.write_kv_paged(k, k, kv.transpose(1, 2), slots) is None
    assert sz.write_kv_paged(k, k, kv, slots.int()) is None
    assert sz.write_kv_paged(k, k, kv, slots[:2]) is None
    assert sz.write_kv_paged(k.transpose(1, 2).contiguous().transpose(1, 2), k, kv, slots) is None
    assert sz.write_kv_paged(k.cpu(), k.cpu(), kv, slots) is None
    # rows of the layer itself
    assert sz.write_kv_paged(kv[0, 0, :3], k, kv, slots) is None


class Engine:
    """A few requests served step by step: plan, write, attention, on persistent buffers."""

    def __init__(self, sz, requests, q_heads, kv_heads, dim, block, blocks, rows, seed):
        self.sz, self.block, self.rows = sz, block, rows
        self.rng = np.random.default_rng(seed)
        self.kv = torch.full((2, blocks, block, kv_heads, dim), float("nan"), dtype=torch.bfloat16,
                             device="cuda")
        self.tables = torch.full((requests, blocks), -1, dtype=torch.int32, device="cuda")
        self.free = i32(self.rng.permutation(blocks).tolist())
        self.free_start, self.cached = i32([0]), i32([0] * requests)
        self.new = i32([0] * requests)
        self.heads = (q_heads, kv_heads, kv_heads)
        self.qkv = torch.zeros((rows, sum(self.heads), dim), dtype=torch.bfloat16, device="cuda")
        self.plan = sz.new_step_plan(requests, rows, "cuda")
        self.out = torch.zeros((rows, q_heads, dim), dtype=torch.bfloat16, device="cuda")
        self.workspace = torch.empty(
            sz.chunk_attention_workspace_bytes(rows, requests, q_heads, kv_heads, dim,
                                               blocks * block), dtype=torch.uint8, device="cuda")
        self.history = [[] for _ in range(requests)]

    def feed(self, new):
        rows = self.rng.standard_normal((self.rows,) + tuple(self.qkv.shape[1:])).astype(np.float32)
        self.qkv.copy_(torch.from_numpy(rows).to(torch.bfloat16))
        self.new.copy_(i32(new))

    def calls(self):
        q, k, v = self.qkv.split(self.heads, 1)
        assert self.sz.plan_step_paged(self.new, self.cached, self.tables, self.free,
                                       self.free_start, self.block, self.rows, plan=self.plan)
        assert self.sz.write_kv_paged(k, v, self.kv, self.plan.slots) is not None
        assert self.sz.chunk_attention_paged(q, self.kv, self.tables, self.plan.query_starts,
                                             self.plan.context_tokens, out=self.out,
                                             workspace=self.workspace) is not None
        self.cached.copy_(self.plan.context_tokens)
        self.free_start.copy_(self.plan.free_next)

    def verify(self, new):
        torch.cuda.synchronize()
        assert int(self.plan.lacking[0]) == 0
        qkv = self.qkv.float().cpu().numpy().astype(np.float64)
        out, at = self.out.float().cpu().numpy().astype(np.float64), 0
        for r, n in enumerate(new):
            self.history[r].append(qkv[at:at + n, self.heads[0]:])
            if n:
                seen = np.concatenate(self.history[r])
                k, v = seen[:, :self.heads[1]], seen[:, self.heads[1]:]
                ref, _, mean, off = attend(qkv[at:at + n, :self.heads[0]], k, v, len(seen) - n,
                                           qkv.shape[2] ** -0.5)
                check(out[at:at + n], ref, mean, off, "bf16", len(seen), np.abs(v).max())
            at += n


STEPS = [[30, 5, 0, 1], [1, 1, 17, 1], [1, 1, 1, 1], [0, 40, 1, 0], [1, 1, 1, 3], [2, 0, 2, 60]]


def test_steps_together(sz):
    """Plan, write and attention of a step, as they are used together, over several steps."""
    engine = Engine(sz, 4, 8, 2, 128, 16, 40, 64, seed=3)
    for new in STEPS:
        say("step", new)
        engine.feed(new)
        engine.calls()
        engine.verify(new)


def test_captured_step_follows_new_lengths(sz):
    """One captured step replayed with other lengths, with eager work between the replays."""
    engine = Engine(sz, 4, 8, 2, 64, 16, 40, 64, seed=4)
    engine.feed([0, 0, 0, 0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        engine.calls()  # nothing new: loads the kernels, changes nothing
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine.calls()
    for new in STEPS:
        say("replay", new)
        engine.feed(new)
        graph.replay()
        engine.verify(new)
        torch.randn(1 << 16, device="cuda").sum()
