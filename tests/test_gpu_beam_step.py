"""A beam search over two layers, step after step with the calls that a serving loop makes, eagerly and as
one captured graph, against dense caches that follow the chosen parents by plain copies."""

import numpy as np
import pytest

from paged_attention_ref import attend, check
from test_gpu_beam_select import check as check_choice

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BEAMS, LAYERS, Q_HEADS, KV_HEADS, DIM, BLOCK, VOCAB, WIDTH = 4, 2, 4, 2, 64, 4, 300, 8
PROMPTS, SOURCES, STEPS = [5, 8, 3], [20, 0, 37], 13
ROWS = BEAMS * len(PROMPTS)


@pytest.fixture(scope="module")
def sz():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")
    from unchainkv_amd import splitzip_cuda

    assert splitzip_cuda.available(), splitzip_cuda.load_error()
    return splitzip_cuda


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Search:
    """The state of a search on the device, and one step of it."""

    def __init__(self, sz):
        self.sz = sz
        gen = torch.Generator("cuda").manual_seed(3)

        def rows(*shape):
            return torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16)

        self.embed = rows(LAYERS, VOCAB, Q_HEADS + 2 * KV_HEADS, DIM)
        self.head = torch.randn((Q_HEADS * DIM, VOCAB), generator=gen, device="cuda")
        self.rotation = sz.rotation_table(64, DIM)
        # each request's whole prompt blocks are shared, its beams' last ones their own
        tables, at = np.full((ROWS, WIDTH), -1, np.int32), 0
        for r, n in enumerate(PROMPTS):
            tables[BEAMS * r:BEAMS * (r + 1), :n // BLOCK] = np.arange(at, at + n // BLOCK)
            at += n // BLOCK
            if n % BLOCK:
                tables[BEAMS * r:BEAMS * (r + 1), n // BLOCK] = np.arange(at, at + BEAMS)
                at += BEAMS
        self.blocks = at + ROWS * WIDTH
        self.used = at
        self.tables = torch.from_numpy(tables).cuda()
        self.layers = [torch.full((2, self.blocks, BLOCK, KV_HEADS, DIM), float("nan"), dtype=torch.bfloat16,
                                  device="cuda") for _ in range(LAYERS)]
        self.free = torch.arange(self.blocks, dtype=torch.int32, device="cuda")
        self.free_start = i32([at])
        self.cached = i32(np.repeat(PROMPTS, BEAMS).tolist())
        self.one = torch.ones(ROWS, dtype=torch.int32, device="cuda")
        # the prompts' rows, in the first beam's blocks
        self.prompt = [[rows(n, 2, KV_HEADS, DIM) for n in PROMPTS] for _ in range(LAYERS)]
        for layer, prompts in zip(self.layers, self.prompt):
            for r, n in enumerate(PROMPTS):
                t = torch.arange(n, device="cuda")
                slots = self.tables[BEAMS * r].long()[t // BLOCK] * BLOCK + t % BLOCK
                assert sz.write_kv_paged(prompts[r][:, 0], prompts[r][:, 1], layer, slots)
        # the sources: packed rows, which a layer then holds
        width = -(-max(SOURCES) // BLOCK)
        self.source_tables = torch.arange(len(SOURCES) * width, dtype=torch.int32, device="cuda").view(-1, width)
        self.source_tokens, self.source_starts = i32(SOURCES), i32(np.cumsum([0] + SOURCES)[:-1].tolist())
        self.source_rows = rows(sum(SOURCES), 2, KV_HEADS, DIM)
        self.source = torch.full((2, len(SOURCES) * width, BLOCK, KV_HEADS, DIM), float("nan"),
                                 dtype=torch.bfloat16, device="cuda")
        slots = torch.cat([r * width * BLOCK + torch.arange(n, device="cuda") for r, n in enumerate(SOURCES)])
        assert sz.write_kv_paged(self.source_rows[:, 0], self.source_rows[:, 1], self.source, slots)
        self.starts = i32(list(range(0, ROWS + 1, BEAMS)))
        self.tokens = torch.zeros((len(PROMPTS), BEAMS), dtype=torch.int64, device="cuda")
        self.scores = torch.full((len(PROMPTS), BEAMS), float("-inf"), device="cuda")
        self.scores[:, 0] = 0.0
        # the first reordering gives every beam the first one's tokens
        self.parents = torch.zeros((len(PROMPTS), BEAMS), dtype=torch.int32, device="cuda")
        self.plan = sz.new_step_plan(ROWS, ROWS, "cuda")
        self.choice = sz.new_beam_choice(len(PROMPTS), BEAMS, "cuda")
        self.order = sz.new_beam_order(len(PROMPTS), BEAMS, WIDTH, "cuda")._replace(tables=self.tables)
        self.seen = {}
        self.reorder(self.cached)

    def reorder(self, contexts):
        got = self.sz.reorder_beams_paged(self.layers, self.tables, self.parents, contexts, self.free,
                                          self.free_start, BLOCK, order=self.order)
        assert got is self.order
        self.free_start.copy_(self.order.free_next)

    def step(self):
        sz, seen = self.sz, self.seen
        plan = sz.plan_step_paged(self.one, self.cached, self.tables, self.free, self.free_start, BLOCK, ROWS,
                                  plan=self.plan)
        seen["in"], seen["selfs"], seen["crosses"] = self.tokens.clone(), [], []
        seen["before"] = self.scores.clone()
        self.free_start.copy_(plan.free_next)
        hidden = 0
        for n, layer in enumerate(self.layers):
            row = self.embed[n][self.tokens.view(-1)]
            q, k, v = row.split((Q_HEADS, KV_HEADS, KV_HEADS), 1)
            q = sz.rotate_write_kv_paged(q, k, v, layer, plan.slots, plan.positions, self.rotation)
            seen["selfs"].append(sz.chunk_attention_paged(q, layer, self.tables, plan.query_starts,
                                                          plan.context_tokens, max_query=1))
            if n == 0:
                seen["crosses"].append(sz.cross_attention_paged(
                    q, self.source, self.source_tables, self.starts, self.source_tokens, max_query=BEAMS))
            else:
                seen["crosses"].append(sz.cross_attention(
                    q, self.source_rows[:, 0], self.source_rows[:, 1], self.starts, self.source_starts,
                    self.source_tokens, max_query=BEAMS))
            hidden = hidden + seen["selfs"][-1].float() + seen["crosses"][-1].float()
            seen["q%d" % n] = q
        seen["logits"] = (hidden.flatten(1) @ self.head * 0.2).view(len(PROMPTS), BEAMS, VOCAB)
        sz.beam_select(seen["logits"], self.scores, choice=self.choice)
        self.scores.copy_(self.choice.scores)
        self.tokens.copy_(self.choice.tokens)
        self.parents.copy_(self.choice.parents)
        self.cached.copy_(plan.context_tokens)
        self.reorder(self.cached)


class Dense:
    """Every beam's rows of every layer, copied whole at each choice."""

    def __init__(self, s):
        self.kv = [[f64(s.prompt[n][r // BEAMS]) for r in range(ROWS)] for n in range(LAYERS)]
        self.s, self.source, self.at = s, f64(s.source_rows), np.cumsum([0] + SOURCES)

    def follow(self):
        s, seen = self.s, self.s.seen
        token = seen["in"].view(-1).cpu().numpy()
        for n in range(LAYERS):
            rows, q = f64(s.embed[n]), f64(seen["q%d" % n])
            selfs, crosses = f64(seen["selfs"][n]), f64(seen["crosses"][n])
            for r in range(ROWS):
                k = rows[token[r], Q_HEADS:Q_HEADS + KV_HEADS]
                place = len(self.kv[n][r])
                angle = place * 10000.0 ** (-np.arange(0, DIM, 2) / DIM)
                a, b = k[:, :DIM // 2], k[:, DIM // 2:]
                c, sn = np.cos(angle), np.sin(angle)
                turned = torch.from_numpy(np.concatenate((a * c - b * sn, b * c + a * sn), 1))
                new = np.stack((f64(turned.to(torch.bfloat16)), rows[token[r], Q_HEADS + KV_HEADS:]))
                self.kv[n][r] = np.concatenate((self.kv[n][r], new[None]))
                keys, values = self.kv[n][r][:, 0], self.kv[n][r][:, 1]
                want, _, mean, off = attend(q[r:r + 1], keys, values, place, DIM ** -0.5)
                # (a key value on the border between two of the type's may be rounded either way: one step, 2^-7
                # of it, of one key of 64 dims moves a score by at most 2^-7 |q k| / 8 and an output by twice that)
                near = 2 * 2.0 ** -7 * np.abs(q[r]).max() * np.abs(keys).max() / 8
                check(selfs[r:r + 1], want, mean, off + near / 2, "bf16", place + 1, np.abs(values).max())
                m0, m1 = self.at[r // BEAMS], self.at[r // BEAMS + 1]
                want, _, mean, off = attend(q[r:r + 1], self.source[m0:m1, 0], self.source[m0:m1, 1], m1 - m0,
                                            DIM ** -0.5)
                check(crosses[r:r + 1], want, mean, off, "bf16", m1 - m0, 5.0)
        check_choice(s.choice, seen["logits"], seen["before"], BEAMS)
        parents = s.choice.parents.cpu().numpy()
        for n in range(LAYERS):
            self.kv[n] = [self.kv[n][r // BEAMS * BEAMS + parents[r // BEAMS, r % BEAMS]] for r in range(ROWS)]
        # every block is in a table or in the list's free part, and in one of them alone
        s_tables, first = s.tables.cpu().numpy(), int(s.free_start.item())
        held = {int(s_tables[r, c]) for r in range(ROWS) for c in range(-(-len(self.kv[0][r]) // BLOCK))}
        free = s.free.tolist()[first:]
        assert len(free) == len(set(free)) and not held & set(free)
        assert held | set(free) == set(range(s.blocks))
        assert s.order.lacking.item() == 0 and s.order.unlisted.item() == 0 and s.plan.lacking.item() == 0


def test_a_search_step_by_step(sz):
    s = Search(sz)
    dense = Dense(s)
    for _ in range(STEPS):
        s.step()
        torch.cuda.synchronize()
        dense.follow()


def test_a_captured_search(sz):
    """One graph of a whole step, replayed."""
    s, warm = Search(sz), Search(sz)
    warm.step()
    torch.cuda.synchronize()
    dense, graph = Dense(s), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.step()
    for _ in range(STEPS):
        graph.replay()
        torch.cuda.synchronize()
        dense.follow()


def test_results_are_ordinary_tensors(sz):
    """What the calls allocate for themselves can be used as any other tensor, in either mode."""
    q = torch.randn((3, 4, 64), device="cuda").bfloat16()
    k, v = q[:, :2], q[:, 2:]
    kv = torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    at = torch.arange(3, device="cuda")
    tables, starts, count = i32([[0, 1]]), i32([0, 3]), i32([3])

    def calls():
        choice = sz.beam_select(torch.randn((2, 3, 50), device="cuda"), torch.zeros((2, 3), device="cuda"))
        order = sz.reorder_beams_paged([kv], i32([[0], [1]]), i32([[0, 0]]), i32([3, 3]), i32([3, 2]), i32([0]), 16)
        return [sz.rotate_write_kv_paged(q, k, v, kv, at, at, sz.rotation_table(9, 64)),
                sz.cross_attention_paged(q, kv, tables, starts, count),
                sz.cross_attention(q, k, v, starts, i32([0]), count), *choice, *order]

    for got in calls():
        assert type(got) is torch.Tensor and got.device == q.device and got.is_contiguous()
        assert not got.is_inference() and not got.requires_grad and got._version == 0
        assert torch.equal(got.clone(), got.cpu().cuda()) and torch.empty_like(got).shape == got.shape
        leaf = got.float().clone().requires_grad_()
        (leaf * leaf).sum().backward()
        assert torch.equal(leaf.grad, 2 * leaf)
        got.add_(1)
        assert got._version == 1
    with torch.inference_mode():
        results = calls()
        assert all(got.is_inference() for got in results)
    assert all(torch.isfinite(got.float()).all() for got in results)
