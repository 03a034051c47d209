"""Reordering of beams' tables and layers against plain loops (beam_order_ref.py)."""

import numpy as np
import pytest

from beam_order_ref import reorder

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


def search(rng, requests, beams, longest, block, width):
    """Tables as a search leaves them: a shared prompt, lines that part and end, last blocks of each
    beam's own. (tables, parents, contexts, blocks)"""
    contexts = [int(rng.integers(0, min(longest, width * block) + 1)) for _ in range(requests)]
    tables, at = [], 0
    pool = rng.permutation(requests * beams * (width + 1)).tolist()
    for context in contexts:
        prompt, line = int(rng.integers(0, context + 1)), list(range(beams))
        rows = [[-1] * width for _ in range(beams)]
        for c in range(min(width - 1, context // block), -1, -1):
            if c == context // block:
                names = list(range(beams))
            elif c < prompt // block:
                names = [0] * beams
            else:
                line = [int(rng.integers(0, x + 1)) for x in line]
                names = line
            for b in range(beams):
                rows[b][c] = pool[at + names[b]]
            at += beams
        tables += rows
    parents = [rng.integers(0, beams, beams).tolist() for _ in range(requests)]
    return tables, parents, contexts, requests * beams * (width + 1)


def check(sz, tables, parents, contexts, free, start, block, layers=(), in_place=False, order=None,
          wide=0, **more):
    beams, rows, width = len(parents[0]), len(tables), len(tables[0])
    room = torch.full((rows, width + wide), 77, dtype=torch.int32, device="cuda")
    dev = room[:, :width]
    dev.copy_(torch.tensor(tables))
    want = reorder(tables, parents, contexts, free, start, block)
    copies = want[6]
    kept = [layer.clone() for layer in layers]
    listed = i32(free)
    counts = i32([c for c in contexts for _ in range(beams)])
    if in_place:
        order = sz.new_beam_order(len(parents), beams, width, "cuda")._replace(tables=dev)
    got = sz.reorder_beams_paged(layers, dev, i32(parents), counts, listed, i32([start]), block,
                                 order=order, **more)
    torch.cuda.synchronize()
    assert got is not None and (order is None or got is order)
    for name, a, b in zip(("tables", "copied", "free", "next", "lacking", "unlisted"),
                          (got.tables, got.copied_from, listed, got.free_next[0], got.lacking[0],
                           got.unlisted[0]), want):
        assert np.array_equal(a.cpu().numpy(), np.array(b, dtype=np.int32).reshape(a.shape)), name
    assert (room[:, width:] == 77).all() and (in_place or (dev.cpu() == torch.tensor(tables)).all())
    for layer, old in zip(layers, kept):
        for source, to, tokens in copies:
            old[:, to, :tokens] = old[:, source, :tokens]
        assert torch.equal(layer.view(torch.int16), old.view(torch.int16))
    return got


def layers_of(count, blocks, block, heads, dim, dtype=torch.bfloat16):
    return [torch.randn((2, blocks, block, heads, dim), device="cuda").to(dtype) for _ in range(count)]


@pytest.mark.parametrize("requests,beams,longest,block,width,heads,dim", [
    (1, 1, 40, 16, 4, 2, 64), (1, 4, 200, 16, 14, 8, 64), (5, 3, 90, 8, 20, 1, 128), (20, 5, 60, 24, 7, 3, 5),
    (2, 32, 100, 16, 9, 1, 64), (3, 2, 5000, 8, 700, 1, 8), (70, 4, 33, 32, 3, 1, 64), (2, 7, 30, 1, 30, 2, 4),
    (300, 2, 20, 4, 6, 1, 1)])
def test_matches_plain_loops(sz, requests, beams, longest, block, width, heads, dim):
    say("order", requests, beams, longest, block, width)
    rng = np.random.default_rng(requests + beams)
    for n in range(3):
        tables, parents, contexts, blocks = search(rng, requests, beams, longest, block, width)
        check(sz, tables, parents, contexts, list(range(10 ** 6, 10 ** 6 + blocks + 9)), blocks, block,
              layers_of(n + 1, blocks, block, heads, dim), in_place=n == 1, wide=3 * n)


def test_many_layers(sz):
    say("layers")
    rng = np.random.default_rng(8)
    tables, parents, contexts, blocks = search(rng, 2, 4, 60, 16, 5)
    for count in (0, 64, 65, 130):
        check(sz, tables, parents, contexts, list(range(500)), 400, 16,
              layers_of(count, blocks, 16, 1, 8, torch.float16))


def test_edges(sz):
    say("edges")
    free = list(range(100, 110))
    # nothing held, whole blocks only, every beam on, one parent for all, a context past the table
    check(sz, [[-1, -1], [-1, -1]], [[1, 0]], [0], free, 5, 16)
    check(sz, [[1, 2, -1], [1, 3, -1]], [[1, 1]], [32], free, 5, 16)
    check(sz, [[1, 2], [1, 3], [1, 4]], [[0, 1, 2]], [20], free, 5, 16, layers_of(1, 5, 16, 1, 8))
    check(sz, [[1, 2], [1, 3], [1, 4]], [[2, 2, 2]], [20], free, 5, 16, layers_of(1, 5, 16, 1, 8))
    check(sz, [[1, 2], [3, 4]], [[1, 1]], [40], free, 5, 16, layers_of(1, 5, 16, 1, 8))
    check(sz, [[1, 2], [3, 4]], [[1, 1]], [-7], free, 5, 16)
    # last blocks that are shared or missing, parents that are none
    check(sz, [[1, 2], [1, 2], [1, 2]], [[0, 0, 1]], [20], free, 5, 16, layers_of(1, 3, 16, 1, 8))
    check(sz, [[1, 2], [1, -1], [1, 3]], [[0, 1, 0]], [20], free, 5, 16, layers_of(1, 4, 16, 1, 8))
    check(sz, [[1, 2], [1, 3], [4, 5]], [[-1, 3, 1]], [20], free, 5, 16, layers_of(1, 6, 16, 1, 8))
    check(sz, [[1, 2], [4, 5]], [[9, -2]], [20], free, 5, 16)
    # a free list without room, without entries, a start outside it
    lost = [[1, 2, 3], [1, 4, 5], [6, 7, 8]]
    for listed, start in ((free, 1), (free, 0), (free, -3), (free, 99), ([], 0), ([], 4)):
        check(sz, lost, [[0, 0, 0]], [40], listed, start, 16, layers_of(1, 9, 16, 1, 8))


def test_blocks_outside_the_layer_are_not_copied(sz):
    say("outside")
    layer = layers_of(1, 4, 16, 1, 8)
    kept = layer[0].clone()
    for bad in (4, 10 ** 9):
        got = sz.reorder_beams_paged(layer, i32([[0, 2], [0, bad]]), i32([[0, 0]]), i32([20, 20]),
                                     i32([7] * 9), i32([5]), 16)
        assert got.tables.tolist() == [[0, 2], [0, bad]] and got.copied_from.tolist() == [-1, 2]
        got = sz.reorder_beams_paged(layer, i32([[0, bad], [0, 2]]), i32([[0, 0]]), i32([20, 20]),
                                     i32([7] * 9), i32([5]), 16)
        assert got.copied_from.tolist() == [-1, bad]
    assert torch.equal(layer[0], kept)


def test_captured_calls_follow_the_choice(sz):
    """In place, with other parents and contexts at each replay; then the released blocks are planned."""
    say("captured")
    rng = np.random.default_rng(4)
    tables, parents, _, blocks = search(rng, 3, 4, 70, 8, 12)
    contexts = [70, 33, 64]
    dev, p, c = i32(tables), i32(parents), i32([c for c in contexts for _ in range(4)])
    layers = layers_of(3, blocks, 8, 2, 16)
    free, start = i32(list(range(blocks))), i32([blocks])
    order = sz.new_beam_order(3, 4, 12, "cuda")._replace(tables=dev)
    ws = torch.empty(sz.reorder_beams_workspace_bytes(3, 4, 12), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        assert sz.reorder_beams_paged(layers, dev, p, c, free, start, 8, order=order, workspace=ws) is order
    for _ in range(4):
        tables, parents, contexts, _ = search(rng, 3, 4, 70, 8, 12)
        dev.copy_(i32(tables))
        p.copy_(i32(parents))
        c.copy_(i32([c for c in contexts for _ in range(4)]))
        want = reorder(tables, parents, contexts, free.tolist(), blocks, 8)
        kept = [layer.clone() for layer in layers]
        graph.replay()
        torch.cuda.synchronize()
        assert dev.tolist() == want[0] and order.copied_from.tolist() == want[1]
        assert free.tolist() == want[2] and order.free_next.tolist() == [want[3]]
        for layer, old in zip(layers, kept):
            for source, to, tokens in want[6]:
                old[:, to, :tokens] = old[:, source, :tokens]
            assert torch.equal(layer, old)
    plan = sz.plan_step_paged(i32([1] * 12), c, dev, free, order.free_next, 8, 12)
    fresh = sum(x % 8 == 0 for x in c.tolist())
    assert plan.free_next.item() == order.free_next.item() + fresh


def test_refuses(sz):
    tables, parents, counts = i32([[0, 1], [0, 2]]), i32([[0, 1]]), i32([20, 20])
    free, start, layers = i32([5, 6, 7]), i32([2]), layers_of(2, 4, 16, 1, 8)

    def call(layers=layers, tables=tables, parents=parents, counts=counts, free=free, start=start, block=16,
             **more):
        return sz.reorder_beams_paged(layers, tables, parents, counts, free, start, block, **more)

    assert call() is not None
    assert call(tables=tables.long()) is None and call(tables=tables[:1]) is None
    assert call(parents=parents[0]) is None and call(parents=parents.cpu()) is None
    assert call(counts=counts[:1]) is None and call(free=free.long()) is None
    assert call(start=start[:0]) is None and call(block=0) is None and call(block=8) is None
    assert call(layers=[layers[0], layers[1].half()]) is None
    assert call(layers=[layers[0], layers[1][:, :3].contiguous()]) is None
    assert call(layers=[layers[0].float()]) is None and call(layers=[layers[0][0]]) is None
    order = sz.new_beam_order(1, 2, 2, "cuda")
    assert call(order=order) is order
    assert call(order=sz.new_beam_order(1, 2, 3, "cuda")) is None
    assert call(order=order._replace(copied_from=counts)) is None
    assert call(order=order._replace(free_next=start)) is None
    assert call(order=order._replace(tables=order.tables.t())) is None
    assert call(free=start) is None and call(counts=tables.view(-1)[:2], order=order._replace(
        tables=tables)) is None
    many = i32([[0, 1]] * 33)
    assert call(tables=many, parents=i32([list(range(33))]), counts=i32([20] * 33)) is None
    none = call(tables=tables[:0], parents=parents[:0], counts=counts[:0])
    assert none.tables.shape == (0, 2) and none.free_next.item() == 2
    with pytest.raises(ValueError):
        sz.reorder_beams_workspace_bytes(1, 33, 5)
