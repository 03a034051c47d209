"""Float64 causal attention used as the reference for the paged chunk and prompt kernels: a
request's rows over its own tokens, with the bound that the kernels' roundings obey.

Bound of an output value, u = half a step of the type (2^-8 bf16, 2^-11 fp16):
* the weights are rounded to the type before the second product: u * A, A = sum p |v| / sum p;
  (fp16 weights below 2^-14 lose up to 2^-25 each: n * 2^-25 * max |v|, as the largest weight
  is 1 at least);
* the output is rounded: u * |o|;
* scores are f32 sums of D products (at most (D + 8) roundings of 2^-24 of sum |q k|, scaling
  included) and weights f32 exponentials and sums (2^-20 is ample for exp2 and the division, and
  n * 2^-24 for sums of n terms): each weight is off by d = 2 (D + 8) 2^-24 S + 2^-20 + n 2^-24
  relative, S = the largest scale * sum |q k|, and a quotient of two such sums by 2 d A.
lse is off by d and the rounding of its own f32 value."""

import numpy as np

HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def attend(q, k, v, first, scale):
    """q (n, q_heads, d), k, v (m, kv_heads, d), float64; row i sees tokens 0 .. first + i.
    Returns (out, lse, A, d): A and d per row as above (A per value)."""
    n, q_heads, dim = q.shape
    group = q_heads // k.shape[1]
    out, mean = np.zeros((n, q_heads, dim)), np.zeros((n, q_heads, dim))
    lse, off = np.full((n, q_heads), -np.inf), np.zeros((n, q_heads))
    for i in range(n):
        seen = min(first + i + 1, k.shape[0])
        if seen <= 0:
            continue
        for h in range(q_heads):
            keys, values = k[:seen, h // group], v[:seen, h // group]
            s = keys @ q[i, h] * scale
            top = s.max()
            with np.errstate(invalid="ignore"):
                p = np.exp(s - top)
                out[i, h] = p @ values / p.sum()
                mean[i, h] = p @ np.abs(values) / p.sum()
            lse[i, h] = top + np.log(p.sum())
            reach = (np.abs(keys) @ np.abs(q[i, h])).max() * scale
            off[i, h] = 2 * (dim + 8) * 2.0 ** -24 * reach + 2.0 ** -20 + seen * 2.0 ** -24
    return out, lse, mean, off


def check(got, out, mean, off, dtype, tokens, v_max):
    """got within the bound of out; NaN and infinite values at the same places."""
    u = HALF_STEP[dtype]
    bound = u * (mean + np.abs(out)) * 1.01 + 2 * off[..., None] * mean + 1e-30
    if dtype == "fp16":
        bound = bound + tokens * 2.0 ** -25 * v_max + 2.0 ** -25
    finite = np.isfinite(out)
    assert np.array_equal(np.isnan(got), np.isnan(out))
    assert np.array_equal(got[np.isinf(out)], out[np.isinf(out)])
    err = np.abs(got - out)[finite]
    worst = (err / bound[finite]).max() if err.size else 0.0
    assert worst <= 1.0, f"off by {worst:.3g} of the bound, {err.max():.3g}"
    return worst


def check_lse(got, lse, off):
    none = np.isneginf(lse)
    assert np.all(np.isneginf(got[none]))
    ok = ~none & np.isfinite(lse)
    err = np.abs(got[ok] - lse[ok])
    assert np.all(err <= 2 * off[ok] + 2.0 ** -22 * np.abs(lse[ok]) + 2.0 ** -22)
