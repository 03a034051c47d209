"""The search that the beam selection's results are held to tells values apart that 32 bits do not (no GPU)."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_beam_select import order_of, values_of  # noqa: E402


def test_planted_orders_are_seen():
    logits = torch.full((1, 2, 9), float("-inf"))
    logits[0, 0, :2], logits[0, 1, 3:6] = 0.0, 0.0
    near = float(np.float32(-0.5 - np.log(2) + np.log(3)))
    v = values_of(logits, torch.tensor([[-0.5, near]]))[0]
    assert 0 < abs(v[0] - v[12]) < 2.0 ** -24 and order_of(v)[0] == (0 if v[0] > v[12] else 12)
