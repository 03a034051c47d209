"""What the step's Python calls make of their arguments, with the C entries replaced: no GPU needed."""

from types import SimpleNamespace

import pytest

from unchainkv_amd import splitzip_cuda as sz

torch = pytest.importorskip("torch")
fw = torch.autograd.forward_ad


@pytest.fixture
def entered(monkeypatch):
    """The names of the entries that were called; each takes its arguments."""
    names = []

    def entry(name):
        def call(*args):
            names.append(name)
            return 1
        return call

    lib = SimpleNamespace(**{n: entry(n) for n in (
        "kvq_splitzip_plan_step_paged", "kvq_splitzip_write_kv_paged",
        "kvq_splitzip_chunk_attention_paged", "kvq_splitzip_prompt_attention")})
    monkeypatch.setattr(sz, "_load", lambda: lib)
    monkeypatch.setattr(sz, "_is_cuda", lambda t: True)
    monkeypatch.setattr(sz, "_call_on", lambda device, torch, fn, *args: fn(*args, 0))
    monkeypatch.setattr(sz, "_attention_workspace", lambda name, device, sizes: 0)
    return names


def rows(heads, count=3):
    return torch.zeros((count, heads, 64), dtype=torch.bfloat16)


def i32(values):
    return torch.tensor(values, dtype=torch.int32)


def write(k=None, v=None, kv=None):
    k, v = (rows(2) if t is None else t for t in (k, v))
    return sz.write_kv_paged(k, v, layer() if kv is None else kv, torch.arange(3))


def layer():
    return torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16)


def chunk(q=None, kv=None, **more):
    return sz.chunk_attention_paged(rows(4) if q is None else q, layer() if kv is None else kv,
                                    i32([[0, 1]]), i32([0, 3]), i32([9]), **more)


def prompt(q=None, k=None, v=None, **more):
    q, k, v = (rows(n) if t is None else t for n, t in ((4, q), (2, k), (2, v)))
    return sz.prompt_attention(q, k, v, i32([0, 3]), **more)


CALLS = [(write, "k", rows(2)), (write, "v", rows(2)), (write, "kv", layer()),
         (chunk, "q", rows(4)), (chunk, "kv", layer()), (chunk, "out", rows(4)),
         (chunk, "lse", torch.zeros((3, 4))),
         (prompt, "q", rows(4)), (prompt, "k", rows(2)), (prompt, "v", rows(2)),
         (prompt, "out", rows(4)), (prompt, "lse", torch.zeros((3, 4)))]


@pytest.mark.parametrize("call,name,tensor", CALLS, ids=[f"{c.__name__}-{n}" for c, n, _ in CALLS])
def test_gradients_that_a_call_would_lose(entered, call, name, tensor):
    """Tensors that require a gradient, while gradients are recorded, and forward-mode tangents are
    declined before anything is launched; without either the call is made."""
    leaf = tensor.clone().requires_grad_()
    assert call(**{name: leaf}) is None and call(**{name: leaf * 2}) is None
    with fw.dual_level():
        dual = fw.make_dual(tensor.clone(), torch.ones_like(tensor))
        assert call(**{name: dual}) is None
        with torch.no_grad():  # (tangents go on without gradients)
            assert call(**{name: dual}) is None
        assert not entered
        assert call(**{name: tensor.clone()}) is not None
    with torch.no_grad():
        assert call(**{name: leaf}) is not None
    assert call(**{name: tensor.clone()}) is not None
    assert len(entered) == 3


def test_writes_count_as_in_place_operations(entered):
    """A backward pass that saved what a call then writes into refuses to run."""
    kv, out, lse = layer(), rows(4), torch.zeros((3, 4))
    tables, plan = i32([[0, -1]]), sz.new_step_plan(1, 4, "cpu")

    def saved(t):
        return (torch.ones(t.shape, dtype=t.dtype, requires_grad=True) * t).sum()

    calls = [
        ((kv,), lambda: write(kv=kv)), ((kv,), lambda: write(kv=kv[:])),
        ((out, lse), lambda: chunk(out=out, lse=lse)), ((out, lse), lambda: prompt(out=out, lse=lse)),
        ((tables, *plan), lambda: sz.plan_step_paged(i32([3]), i32([4]), tables, i32([5]), i32([0]),
                                                     16, 4, plan=plan))]
    for written, call in calls:
        before = [t._version for t in written]
        losses = [saved(t) for t in written if t.is_floating_point()]
        assert call() is not None
        assert all(t._version > b for t, b in zip(written, before))
        for loss in losses:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
    with torch.inference_mode():
        assert write(kv=layer()) and chunk(out=rows(4)) is not None
    # a call that is declined has written nothing
    before = kv._version
    assert write(k=rows(2).float(), kv=kv) is None and kv._version == before


def test_heads_without_values(entered):
    """No default scale is formed of a head_dim of 0."""
    q, k = rows(4)[..., :0], rows(2)[..., :0]
    assert prompt(q, k, k) is None and prompt(q, k, k, scale=1.0) is None
    assert chunk(q) is None and not entered


@pytest.mark.parametrize("width", (0, 3))
def test_a_step_of_no_requests(entered, width):
    """Every row is nobody's, nothing is taken from the free list, and the rows of q stay."""
    none, tables = i32([]), torch.zeros((0, width), dtype=torch.int32)
    for start in (4, -2):
        for plan in (None, sz.new_step_plan(0, 5, "cpu")):
            got = sz.plan_step_paged(none, none, tables, i32([7, 8]), i32([start]), 16, 5, plan=plan)
            assert plan is None or got is plan
            assert got.query_starts.tolist() == [0] and got.context_tokens.tolist() == []
            assert got.slots.tolist() == [-1] * 5 and got.positions.tolist() == [0] * 5
            assert got.free_next.tolist() == [max(start, 0)] and got.lacking.tolist() == [0]
    out = torch.full((3, 4, 64), 7.0, dtype=torch.bfloat16)
    assert sz.chunk_attention_paged(rows(4), layer(), tables, got.query_starts, got.context_tokens,
                                    out=out) is out
    assert (out == 7).all() and not entered
    assert sz.plan_step_paged(none, none, tables, i32([7]), i32([0]), 0, 5) is None
    assert sz.plan_step_paged(none, i32([1]), tables, i32([7]), i32([0]), 16, 5) is None
