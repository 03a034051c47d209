"""Attention over paged layers and of prompts at the edges of its contract: what joined splits keep,
how small a weight counts, which buffers and ranges of rows a call takes. Against float64 (the
bound is derived in paged_attention_ref.py) unless a test says otherwise."""

import numpy as np
import pytest

from test_gpu_paged_attention import Case, f64, say, sz  # noqa: F401 (a fixture)

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
