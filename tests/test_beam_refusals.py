"""What the C entries of a beam-searching step decline before anything is launched, and what its Python
calls make of gradients: no GPU needed (addresses are made up, and none is read)."""

import ctypes
import random
from types import SimpleNamespace

import pytest

from beam_order_ref import reorder
from test_step_refusals import A, CHUNK, SCALE, lib, no_workspace, refused  # noqa: F401 (lib: a fixture)
from unchainkv_amd import _build
from unchainkv_amd import splitzip_cuda as sz

MiB = 1 << 20

ROTATE = dict(q=A[0], q_row=4096, q_head=256, q_heads=8, k=A[1], k_row=1024, k_head=256, v=A[2], v_row=1024,
              v_head=256, tokens=4, kv_heads=2, dim=128, dtype=0, kv=A[3], plane=MiB, slots=2048, slot=A[4],
              position=A[5], table=A[6], table_rows=100, rotary=64, adjacent=0, out=A[7], stream=0)


def test_rotate_declines(lib):  # noqa: F811
    refused(lib.kvq_splitzip_rotate_write_kv_paged, ROTATE, [
        {name: 0} for name in ("q", "q_heads", "k", "v", "tokens", "kv_heads", "dim", "kv", "slot", "position",
                               "table", "table_rows", "rotary", "out")] + [
        {"rotary": 63}, {"rotary": 130}, {"dtype": 2}, {"slots": 2049}, {"tokens": 1 << 31}, {"dim": 1 << 13},
        {"q": A[0] + 1}, {"k_row": 1023}, {"out": A[7] + 1}, {"table": A[6] + 2}, {"q_heads": 1 << 17},
        # results over what is read, or over each other
        {"out": A[0]}, {"out": A[0] + 3 * 4096 + 7 * 256}, {"out": A[1]}, {"out": A[2] + 512}, {"out": A[4]},
        {"out": A[5] + 16}, {"out": A[6] + 4 * 64 * 100 - 4}, {"out": A[3] + 2 * MiB - 2}, {"kv": A[0]},
        {"kv": A[1] - 2 * MiB + 8}, {"kv": A[2]}, {"kv": A[4]}, {"kv": A[5]}, {"kv": A[6]}])


def test_cross_over_a_layer_declines(lib):  # noqa: F811
    refused(lib.kvq_splitzip_cross_attention_paged, CHUNK, [
        {name: 0} for name in ("q", "tokens", "q_heads", "kv_heads", "dim", "kv", "blocks", "block",
                               "tables", "width", "starts", "contexts", "requests", "max_query",
                               "out")] + [
        {"dim": 96}, {"dtype": 2}, {"kv_heads": 3}, {"max_query": 5}, {"stride": 7}, {"q": A[0] + 2},
        {"kv": A[1] + 8}, {"scale": ctypes.c_float(0.0)}, {"out": A[0] + 2048}, {"out": A[4]},
        {"lse": A[2]}])
    refused(lib.kvq_splitzip_cross_attention_paged, dict(CHUNK, stride=256, width=256),
            no_workspace(lib.kvq_splitzip_cross_attention_least_workspace_bytes(4, 2, 8, 2, 128, 4096, 4)))


CROSS = dict(q=A[0], q_row=2048, q_head=256, k=A[1], k_row=512, k_head=256, v=A[2], v_row=512, v_head=256,
             rows=5000, tokens=4, q_heads=8, kv_heads=2, dim=128, dtype=1, starts=A[3], first=A[4], count=A[5],
             requests=2, max_query=4, max_source=5000, out=A[7], lse=0, workspace=A[6],
             workspace_bytes=1 << 30, scale=SCALE, stream=0)


def test_cross_over_rows_declines(lib):  # noqa: F811
    refused(lib.kvq_splitzip_cross_attention, CROSS, [
        {name: 0} for name in ("q", "k", "v", "rows", "tokens", "q_heads", "kv_heads", "dim", "starts", "first",
                               "count", "requests", "max_query", "out")] + [
        {"dim": 80}, {"dtype": 2}, {"q_heads": 9}, {"max_query": 5}, {"max_source": 5001}, {"rows": 1 << 31},
        {"k": A[1] + 4}, {"k_row": 500}, {"v_head": 8}, {"out": A[7] + 4}, {"k_row": 1 << 28},
        {"scale": ctypes.c_float(float("nan"))}, {"out": A[0]}, {"out": A[1] + 4999 * 512}, {"out": A[2]},
        {"out": A[4]}, {"lse": A[5] + 4}, {"lse": A[7]}])
    for max_query in (2, 4):  # streamed, and in tiles
        size = lib.kvq_splitzip_cross_attention_least_workspace_bytes(4, 2, 16, 2, 128, 5000, max_query)
        refused(lib.kvq_splitzip_cross_attention, dict(CROSS, q_heads=16, max_query=max_query),
                no_workspace(size) + [{"workspace": a - size + 16} for a in A[:6] + A[7:8]])


def test_cross_workspace_serves_smaller_calls(lib):  # noqa: F811
    """No call of smaller sizes asks for more; fewer sources are cut sooner, and a layer's and rows' alike."""
    rng = random.Random(19)
    least, bound = lib.kvq_splitzip_cross_attention_least_workspace_bytes, sz.cross_attention_workspace_bytes

    def up_to(most):
        return min(most, int(2 ** rng.uniform(0, most.bit_length())))

    for q_heads, kv_heads, dim in ((8, 2, 128), (32, 8, 64), (16, 16, 64), (64, 1, 128), (1, 1, 64), (128, 8, 128)):
        for _ in range(400):
            most = [up_to(1 << 20), up_to(4096), up_to(1 << 14), up_to(1 << 10)]
            tokens, requests, source, query = (up_to(n) for n in most)
            query = min(query, tokens)
            small = bound(tokens, requests, q_heads, kv_heads, dim, source, query)
            assert least(tokens, requests, q_heads, kv_heads, dim, source, query) <= small
            assert small <= bound(most[0], most[1], q_heads, kv_heads, dim, most[2], most[3])
    # taken whole: sources of 192 workgroups; cut: of fewer
    assert least(192, 192, 1, 1, 64, 2048, 1) == 0 < least(191, 191, 1, 1, 64, 2048, 1)
    assert least(191, 191, 1, 1, 64, 2048, 1) <= bound(192, 192, 1, 1, 64, 2048, 1)
    assert least(64, 4, 1, 1, 64, 600, 60) > 0 == least(1000, 999, 1, 1, 64, 600, 60)
    assert least(64, 4, 1, 1, 64, 600, 60) <= bound(1000, 999, 1, 1, 64, 600, 60)
    assert least(1, 1, 16, 16, 64, 768, 1) == 0 < least(1, 1, 16, 16, 64, 769, 1)
    for sizes in ((8, 2, 8, 3, 128, 4096), (8, 2, 8, 2, 96, 4096), (-1, 2, 8, 2, 128, 4096), (8, 2, 8, 2, 128, -1)):
        with pytest.raises(ValueError):
            bound(*sizes)
    assert bound(0, 2, 8, 2, 128, 4096) == 0


SELECT = dict(logits=A[0], dtype=2, request=3000, beam=1000, scores=A[1], ended=A[2], requests=2, beams=3,
              vocab=1000, candidates=6, end=999, out_scores=A[3], parents=A[4], tokens=A[5], workspace=A[6],
              workspace_bytes=1 << 30, stream=0)


def test_select_declines(lib):  # noqa: F811
    size = lib.kvq_splitzip_beam_select_workspace_bytes(2, 3, 1000)
    assert size > 0
    refused(lib.kvq_splitzip_beam_select, SELECT, [
        {name: 0} for name in ("logits", "scores", "requests", "beams", "vocab", "candidates", "out_scores",
                               "parents", "tokens", "workspace", "workspace_bytes")] + [
        {"dtype": 3}, {"beams": 33}, {"candidates": 65}, {"vocab": 1, "candidates": 4}, {"end": 1000},
        {"vocab": (1 << 20) + 1}, {"requests": (1 << 20) + 1}, {"logits": A[0] + 2}, {"workspace": A[6] + 8},
        {"workspace_bytes": size - 1},
        {"out_scores": A[0]}, {"parents": A[0] + 4 * 5999}, {"tokens": A[1] + 16}, {"tokens": A[2]},
        {"parents": A[3] + 40}, {"workspace": A[1] - size + 16}, {"workspace": A[5]}])
    for sizes in ((0, 3, 1000), (2, 0, 1000), (2, 33, 1000), (2, 3, 0), (2, 3, 1 << 21)):
        assert lib.kvq_splitzip_beam_select_workspace_bytes(*sizes) == 0


ORDER = dict(layers=(ctypes.c_ulonglong * 2)(A[0], A[1]), count=2, blocks=64, block=16, row=1024, tables=A[2],
             stride=8, width=8, out=A[3], out_stride=8, parents=A[4], contexts=A[5], requests=2, beams=3,
             free=A[6], free_count=50, start=A[7], copied=A[8], next=A[9], lacking=A[10], unlisted=A[11],
             workspace=A[12], workspace_bytes=1 << 30, stream=0)


def test_order_declines(lib):  # noqa: F811
    size = lib.kvq_splitzip_reorder_beams_workspace_bytes(2, 3, 8)
    assert size > 0
    pair = ctypes.c_ulonglong * 2
    refused(lib.kvq_splitzip_reorder_beams_paged, ORDER, [
        {name: 0} for name in ("blocks", "block", "row", "tables", "width", "out", "parents", "contexts",
                               "requests", "beams", "free", "start", "copied", "next", "lacking", "unlisted",
                               "workspace", "workspace_bytes")] + [
        {"layers": None}, {"layers": pair(A[0], 0)}, {"layers": pair(A[0], A[1] + 1)}, {"row": 1023},
        {"stride": 7}, {"out_stride": 7}, {"beams": 33}, {"requests": 1 << 16}, {"blocks": 1 << 28},
        {"free_count": 1 << 31}, {"workspace": A[12] + 8}, {"workspace_bytes": size - 1},
        {"layers": pair(A[0], A[2])}, {"layers": pair(A[0], A[3] - MiB)}, {"layers": pair(A[6], A[1])},
        {"out": A[2] + 4}, {"out": A[2], "out_stride": 9}, {"out": A[4]}, {"out": A[5] - 160}, {"free": A[2]},
        {"free": A[7] - 196}, {"copied": A[5]}, {"copied": A[4] + 20}, {"next": A[7]}, {"lacking": A[9]},
        {"unlisted": A[8] + 20}, {"workspace": A[0] + 2 * MiB - 16}, {"workspace": A[3] - size + 16}])
    for sizes in ((0, 3, 8), (2, 0, 8), (2, 33, 8), (2, 3, 0)):
        assert lib.kvq_splitzip_reorder_beams_workspace_bytes(*sizes) == 0


def test_plain_reordering():
    """The loops that the GPU results are held to, on a case worked out by hand: blocks of 4 tokens, 10
    held. Beam 0 has both children, so beam 1's second and last blocks are left; the last one takes the
    copy of beam 0's, the second is released."""
    got = reorder([[5, 6, 7, -1], [5, 8, 9, -1]], [[0, 0]], [10], [1, 2, 3, 4], 2, 4)
    assert got == ([[5, 6, 7, -1], [5, 6, 9, -1]], [-1, 7], [1, 8, 3, 4], 1, 0, 0, [(7, 9, 2)])


torch = pytest.importorskip("torch")


def test_tensors_off_the_gpu_are_declined():
    q, k = torch.zeros((2, 8, 64)), torch.zeros((2, 2, 64))
    kv = torch.zeros((2, 4, 16, 2, 64))
    ints, longs = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    tables = torch.zeros((2, 4), dtype=torch.int32)
    assert sz.rotate_write_kv_paged(q, k, k, kv, longs, longs, sz.rotation_table(9, 64, device="cpu")) is None
    assert sz.cross_attention_paged(q, kv, tables, ints, ints[:2]) is None
    assert sz.cross_attention(q, k, k, ints, ints[:2], ints[:2]) is None
    assert sz.beam_select(torch.zeros((1, 2, 9)), torch.zeros((1, 2))) is None
    assert sz.reorder_beams_paged([], tables, tables[:1, :2], ints[:2], ints, ints[:1], 16) is None


@pytest.fixture
def entered(monkeypatch):
    """The names of the entries that were called."""
    if not _build.BINDING_PATH.exists():
        _build.build_binding()
    names, u64 = [], ctypes.c_ulonglong

    def entry(name, *types):
        def call(*args):
            names.append(name)
            return 1
        return ctypes.CFUNCTYPE(ctypes.c_longlong, *types)(call)

    calls = {f"kvq_splitzip_{n}": entry(n, *[u64] * count) for n, count in (
        ("rotate_write_kv_paged", 25), ("beam_select", 17), ("reorder_beams_paged", 24))}
    for n, count in (("cross_attention_paged", 22), ("cross_attention", 25)):
        calls[f"kvq_splitzip_{n}"] = entry(n, *[u64] * count, ctypes.c_float, u64)
    sizes = {f"kvq_splitzip_{n}_workspace_bytes": ctypes.CFUNCTYPE(u64, *[u64] * count)(lambda *a: 16)
             for n, count in (("beam_select", 3), ("reorder_beams", 3), ("cross_attention_least", 7))}
    lib = SimpleNamespace(**calls, **sizes)
    monkeypatch.setattr(sz, "_load", lambda: lib)
    monkeypatch.setattr(sz, "_is_cuda", lambda t: True)
    monkeypatch.setattr(sz, "_call_on", lambda device, torch, fn, *args: fn(*args, 0))
    return names


def rows(heads):
    return torch.zeros((3, heads, 64), dtype=torch.bfloat16)


def layer():
    return torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16)


def i32(values):
    return torch.tensor(values, dtype=torch.int32)


def rotate(q=None, k=None, v=None, kv=None, table=None, **more):
    q, k, v = (rows(n) if t is None else t for n, t in ((4, q), (2, k), (2, v)))
    return sz.rotate_write_kv_paged(q, k, v, layer() if kv is None else kv, torch.arange(3), torch.arange(3),
                                    torch.zeros((9, 64)) if table is None else table, **more)


def paged(q=None, kv=None, **more):
    return sz.cross_attention_paged(rows(4) if q is None else q, layer() if kv is None else kv, i32([[0, 1]]),
                                    i32([0, 3]), i32([9]), **more)


def packed(q=None, k=None, v=None, **more):
    q, k, v = (rows(n) if t is None else t for n, t in ((4, q), (2, k), (2, v)))
    return sz.cross_attention(q, k, v, i32([0, 3]), i32([0]), i32([3]), **more)


def select(logits=None, scores=None, **more):
    return sz.beam_select(torch.zeros((1, 2, 9)) if logits is None else logits,
                          torch.zeros((1, 2)) if scores is None else scores, **more)


def order(kv=None, **more):
    return sz.reorder_beams_paged([layer() if kv is None else kv], i32([[0], [1]]), i32([[0, 0]]), i32([3, 3]),
                                  i32([7]), i32([0]), 16, **more)


CALLS = [(rotate, "q", rows(4)), (rotate, "k", rows(2)), (rotate, "v", rows(2)), (rotate, "kv", layer()),
         (rotate, "table", torch.zeros((9, 64))), (rotate, "out", rows(4)),
         (paged, "q", rows(4)), (paged, "kv", layer()), (paged, "out", rows(4)), (paged, "lse", torch.zeros(3, 4)),
         (packed, "q", rows(4)), (packed, "k", rows(2)), (packed, "v", rows(2)), (packed, "out", rows(4)),
         (packed, "lse", torch.zeros((3, 4))), (select, "logits", torch.zeros((1, 2, 9))),
         (select, "scores", torch.zeros((1, 2))), (order, "kv", layer())]


@pytest.mark.parametrize("call,name,tensor", CALLS, ids=[f"{c.__name__}-{n}" for c, n, _ in CALLS])
def test_gradients_that_a_call_would_lose(entered, call, name, tensor):
    """Tensors that require a gradient, while gradients are recorded, and tangents are declined."""
    leaf = tensor.clone().requires_grad_()
    assert call(**{name: leaf}) is None and call(**{name: leaf * 2}) is None
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        assert call(**{name: fw.make_dual(tensor.clone(), torch.ones_like(tensor))}) is None
    assert not entered
    with torch.no_grad():
        assert call(**{name: leaf}) is not None
    assert call(**{name: tensor.clone()}) is not None and len(entered) == 2


def test_writes_count_as_in_place_operations(entered):
    kv, out, lse, choice = layer(), rows(4), torch.zeros((3, 4)), sz.new_beam_choice(1, 2, "cpu")
    into = sz.new_beam_order(1, 2, 1, "cpu")
    for written, call in (((kv, out), lambda: rotate(kv=kv, out=out)), ((kv,), lambda: rotate(kv=kv)),
                          ((out, lse), lambda: paged(out=out, lse=lse)), ((out,), lambda: packed(out=out)),
                          (choice, lambda: select(choice=choice)), ((kv, *into), lambda: order(kv=kv, order=into))):
        before = [t._version for t in written]
        assert call() is not None
        assert all(t._version > b for t, b in zip(written, before))
    with torch.inference_mode():
        assert rotate(kv=layer()) is not None and order(kv=layer()) is not None
        kv, out, choice, into = layer(), rows(4), sz.new_beam_choice(1, 2, "cpu"), sz.new_beam_order(1, 2, 1, "cpu")
    # (such tensors count no writes, used outside that mode neither)
    assert rotate(kv=kv, out=out) is not None and paged(kv=kv, out=out) is not None
    assert packed(out=out) is not None and select(choice=choice) is not None and order(kv=kv, order=into) is not None


def test_arguments_that_are_no_tensors(entered):
    for call in (lambda: rotate(k=[1.0]), lambda: rotate(table=3), lambda: select(scores=2.0),
                 lambda: order(kv="layer"), lambda: paged(kv=1), lambda: packed(v=(2,)), lambda: paged(out=0)):
        with pytest.raises(TypeError, match="a tensor is wanted"):
            call()
    assert not entered


def test_failures_of_the_entries_are_raised(entered):
    lib = sz._load()
    failing = ctypes.CFUNCTYPE(ctypes.c_longlong, *[ctypes.c_ulonglong] * 25)(lambda *a: -1)
    lib.kvq_splitzip_rotate_write_kv_paged, lib.kvq_splitzip_last_error = failing, lambda: b"no such device"
    kv = layer()
    with pytest.raises(RuntimeError, match="no such device"):
        rotate(kv=kv)
    assert kv._version == 0


def test_bounds_and_scales(entered):
    """max_query and max_source count as at most the rows there are; a scale is any number."""
    assert paged(max_query=99, scale=1) is not None and packed(max_query=2, max_source=10 ** 9, scale=0.5) is not None
    assert paged(max_query=0) is None and paged(max_query=-3) is None and packed(max_source=-1) is None
    with pytest.raises(TypeError):
        paged(scale="half")
    with pytest.raises(TypeError):
        packed(max_query=1.5)
    assert len(entered) == 2


def test_calls_that_do_nothing(entered):
    none = i32([])
    got = sz.reorder_beams_paged([layer()], torch.zeros((0, 5), dtype=torch.int32),
                                 torch.zeros((0, 4), dtype=torch.int32), none, i32([7, 8]), i32([9]), 16)
    assert got.free_next.tolist() == [2] and got.lacking.tolist() == [0] and got.unlisted.tolist() == [0]
    assert sz.beam_select(torch.zeros((0, 2, 9)), torch.zeros((0, 2))).tokens.shape == (0, 2)
    out = torch.full((3, 4, 64), 7.0, dtype=torch.bfloat16)
    assert sz.cross_attention(rows(4), rows(2), rows(2), i32([0]), none, none, out=out) is out
    assert (out == 7).all() and not entered


def test_results_given_in_part_are_declined(entered):
    """Not left as they were, beside results that nobody gets."""
    choice, into = sz.new_beam_choice(1, 2, "cpu"), sz.new_beam_order(1, 2, 1, "cpu")
    for name in choice._fields:
        assert select(choice=choice._replace(**{name: None})) is None
    for name in into._fields:
        assert order(order=into._replace(**{name: None})) is None
    assert not entered and select(choice=choice) is choice and order(order=into) is into
