"""The rotated K/V write against the rotation in 64 bits, at the types, head layouts, strides and slots
where it can go wrong.

Bound of a rotated value x c - y s: cosine, sine, both products and their sum are rounded to 32 bits
(each by at most 2^-24 of what it is, so all by less than 2^-22 (|x| + |y|)), then the result to the
rows' type (half a step: 2^-8 of it, or 2^-11 and 2^-25 for fp16 values below its normal range)."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
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
    return t.detach().double().cpu().numpy()


def turned(x, positions, rotary, base, adjacent):
    """(result, bound without the last rounding) of rows (tokens, heads, dim)."""
    angle = positions[:, None].astype(np.float64) * base ** (-np.arange(0, rotary, 2) / rotary)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a = slice(0, rotary, 2) if adjacent else slice(0, rotary // 2)
    b = slice(1, rotary, 2) if adjacent else slice(rotary // 2, rotary)
    out, reach = x.copy(), np.zeros_like(x)
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    reach[..., a] = reach[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return out, reach * 2.0 ** -22


def near(got, want, off, dtype):
    u = HALF_STEP[dtype]
    bound = off * (1 + u) + np.where(off > 0, u * np.abs(want) + (2.0 ** -25 if dtype == "fp16" else 0), 0)
    assert np.all(np.abs(got - want) <= bound * 1.001 + 1e-37)


def make(tokens, q_heads, kv_heads, dim, dtype, seed, spread=0, shift=0):
    """q, k, v as views of rows with ``spread`` values between the heads' and ``shift`` before them."""
    heads = q_heads + 2 * kv_heads
    gen = torch.Generator().manual_seed(seed)
    flat = torch.randn(tokens * heads * (dim + spread) + shift, generator=gen) * 3
    rows = flat.to(DTYPES[dtype]).cuda()[shift:].view(tokens, heads, dim + spread)[..., :dim]
    return rows.split((q_heads, kv_heads, kv_heads), 1)


def check(sz, tokens, q_heads, kv_heads, dim, rotary, adjacent, dtype, spread=0, shift=0, block=16,
          base=10000.0, far=5000, drop=(), seed=0):
    q, k, v = make(tokens, q_heads, kv_heads, dim, dtype, seed, spread, shift)
    rng = np.random.default_rng(seed)
    blocks = -(-tokens // block) + 2
    slots = rng.permutation(blocks * block)[:tokens].astype(np.int64)
    for t, s in drop:
        slots[t] = s
    positions = rng.integers(0, far, tokens)
    positions[0] = far - 1
    kv = torch.full((2, blocks, block, kv_heads, dim), MARK, dtype=DTYPES[dtype], device="cuda")
    table = sz.rotation_table(far, rotary, base)
    got = sz.rotate_write_kv_paged(q, k, v, kv, torch.from_numpy(slots).cuda(),
                                   torch.from_numpy(positions).cuda(), table, interleaved=adjacent)
    torch.cuda.synchronize()
    assert got is not None and got.is_contiguous() and got.shape == q.shape
    near(f64(got), *turned(f64(q), positions, rotary, base, adjacent), dtype)
    want = np.full((2, blocks * block, kv_heads, dim), MARK)
    off = np.zeros_like(want)
    there = (slots >= 0) & (slots < blocks * block)
    rotated, reach = turned(f64(k), positions, rotary, base, adjacent)
    want[0, slots[there]], off[0, slots[there]] = rotated[there], reach[there]
    want[1, slots[there]] = f64(v)[there]
    near(f64(kv).reshape(want.shape), want, off, dtype)


@pytest.mark.parametrize("adjacent", (False, True))
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary,dtype", [
    (1, 32, 8, 128, 128, "bf16"), (7, 8, 8, 64, 64, "fp16"), (129, 3, 1, 128, 64, "bf16"),
    (33, 5, 5, 80, 32, "fp16"), (18, 2, 1, 64, 20, "bf16"), (5, 1, 1, 2, 2, "fp16"),
    (9, 4, 2, 96, 96, "bf16"), (6, 71, 1, 64, 48, "bf16"), (11, 3, 3, 7, 6, "bf16"),
    (4, 2, 2, 256, 256, "fp16"), (3, 2, 1, 1040, 1040, "bf16"), (4, 1, 1, 200, 190, "fp16")])
def test_matches_the_rotation(sz, tokens, q_heads, kv_heads, dim, rotary, dtype, adjacent):
    say("rotate", tokens, q_heads, kv_heads, dim, rotary, dtype, adjacent)
    check(sz, tokens, q_heads, kv_heads, dim, rotary, adjacent, dtype, seed=tokens)


@pytest.mark.parametrize("adjacent", (False, True))
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary,spread,shift", [
    (5, 64, 20, 128, 20, 0, 0), (3, 64, 20, 128, 128, 0, 0), (4, 71, 9, 64, 64, 0, 1), (6, 200, 4, 64, 48, 4, 0),
    (3, 128, 128, 68, 20, 0, 4), (2, 300, 1, 128, 126, 0, 0), (1, 1, 400, 64, 4, 0, 0)])
def test_many_heads(sz, tokens, q_heads, kv_heads, dim, rotary, spread, shift, adjacent):
    """Heads shared by several waves, in units of 16, 8 and 2 bytes; one token without a slot."""
    say("heads", tokens, q_heads, kv_heads, dim, rotary, spread, shift, adjacent)
    check(sz, tokens, q_heads, kv_heads, dim, rotary, adjacent, "bf16", spread, shift, seed=q_heads,
          drop=[(tokens - 1, -1)] if tokens > 2 else ())


@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary,shift", [
    (257, 32, 8, 128, 128, 0), (256, 32, 8, 128, 128, 0), (700, 2, 1, 64, 32, 0), (85, 1, 1, 2, 2, 0),
    (33, 16, 2, 128, 64, 0), (9, 2, 2, 128, 128, 1), (300, 3, 1, 64, 20, 4), (31, 8, 8, 64, 64, 0)])
def test_tokens_that_share_a_workgroup(sz, tokens, q_heads, kv_heads, dim, rotary, shift):
    """As many tokens as a workgroup's threads hold units of, ends of them, and one more unit than threads."""
    say("shared", tokens, q_heads, kv_heads, dim, rotary, shift)
    for adjacent in (False, True):
        check(sz, tokens, q_heads, kv_heads, dim, rotary, adjacent, "fp16", shift=shift, seed=tokens,
              drop=[(0, -1), (tokens // 2, -1), (tokens - 1, 1 << 40)])


def test_more_tokens_than_a_launch_takes(sz):
    say("many tokens")
    tokens = (1 << 24) + 5
    at = torch.arange(tokens, device="cuda")
    q = (at % 251).to(torch.bfloat16).view(-1, 1, 1).expand(-1, 1, 2).contiguous()
    k, v = q + 1, q + 2
    kv = torch.full((2, tokens + 3, 1, 1, 2), MARK, dtype=torch.bfloat16, device="cuda")
    # quarters of a turn: (x, y) -> (x, y), (-y, x), (-x, -y), (y, -x)
    table = torch.tensor([[1.0, 0.0], [0.0, 1.0], [-1.0, 0.0], [0.0, -1.0]], device="cuda")
    got = sz.rotate_write_kv_paged(q, k, v, kv, at.flip(0), at % 4, table)
    for turned, x in ((got, q), (kv[0, :tokens].flip(0)[:, 0], k)):
        x, y = x[..., 0], x[..., 1]
        for turn, pair in enumerate(((x, y), (-y, x), (-x, -y), (y, -x))):
            assert torch.equal(turned[turn::4], torch.stack(pair, -1)[turn::4])
    assert torch.equal(kv[1, :tokens].flip(0)[:, 0], v) and (kv[:, tokens:] == MARK).all()


@pytest.mark.parametrize("spread,shift", [(8, 0), (0, 1), (3, 5), (16, 8)])
def test_strides_and_addresses(sz, spread, shift):
    say("strides", spread, shift)
    check(sz, 21, 4, 2, 64, 32, False, "bf16", spread=spread, shift=shift)
    check(sz, 21, 4, 2, 64, 64, True, "fp16", spread=spread, shift=shift)


def test_far_positions(sz):
    say("far")
    check(sz, 64, 4, 2, 128, 128, False, "fp16", base=500000.0, far=1 << 20)


def test_rows_without_a_slot(sz):
    say("slots")
    check(sz, 40, 4, 2, 128, 64, False, "bf16", drop=[(0, -1), (7, -1), (8, 10 ** 12), (39, 80)])
    check(sz, 10, 4, 2, 64, 20, True, "bf16", drop=[(t, -1) for t in range(10)])


def test_positions_outside_the_table(sz):
    say("positions")
    q, k, v = make(4, 2, 1, 64, "bf16", 3)
    kv = torch.full((2, 2, 8, 1, 64), MARK, dtype=torch.bfloat16, device="cuda")
    got = sz.rotate_write_kv_paged(q, k, v, kv, torch.arange(4, device="cuda"),
                                   torch.tensor([0, 50, -1, 49], device="cuda"),
                                   sz.rotation_table(50, 32))
    assert got[:, :, :32].isnan().any(-1).any(-1).tolist() == [False, True, True, False]
    assert got[1:3, :, :32].isnan().all() and torch.equal(got[:, :, 32:], q[:, :, 32:])
    row = kv[0, 0, :, 0]
    assert row[1:3, :32].isnan().all() and not row[[0, 3]].isnan().any() and (row[4:] == MARK).all()
    assert torch.equal(row[:4, 32:], k[:, 0, 32:]) and torch.equal(kv[1, 0, :4], v)


def test_values_pass_through(sz):
    """Infinite and NaN values stay in their own pairs; what is not rotated keeps its bits."""
    say("values")
    q, k, v = (t.clone() for t in make(3, 2, 1, 64, "bf16", 4))
    q[0, 0, 3], k[1, 0, 40], v[2, 0, 0] = float("inf"), float("nan"), float("-inf")
    kv = torch.zeros((2, 1, 8, 1, 64), dtype=torch.bfloat16, device="cuda")
    got = sz.rotate_write_kv_paged(q, k, v, kv, torch.arange(3, device="cuda"),
                                   torch.tensor([5, 6, 7], device="cuda"), sz.rotation_table(9, 64))
    bad = ~got.isfinite()
    assert bad.nonzero().tolist() == [[0, 0, 3], [0, 0, 35]]
    assert (~kv[0].isfinite()).nonzero()[:, 1:].tolist() == [[1, 0, 8], [1, 0, 40]]
    assert torch.equal(kv[1, 0, :3].view(torch.int16), v.view(torch.int16))


def test_table(sz):
    table = sz.rotation_table(300, 10, 100.0, device="cpu")
    angle = np.arange(300)[:, None] * 100.0 ** (-np.arange(0, 10, 2) / 10)
    assert table.dtype == torch.float32
    assert np.abs(f64(table) - np.concatenate((np.cos(angle), np.sin(angle)), 1)).max() <= 2.0 ** -24
    scaled = sz.rotation_table(300, 10, frequencies=100.0 ** (-np.arange(0, 10, 2) / 10), device="cpu")
    # (torch's powers and numpy's may differ in their last bit, and angles by 300 times as much)
    assert (scaled - table).abs().max() <= 2.0 ** -23


def test_out_longer_vectors_and_streams(sz):
    say("out")
    q, k, v = make(6, 4, 2, 64, "bf16", 5)
    table, slots = sz.rotation_table(40, 64), torch.arange(9, device="cuda")
    kv, kv2 = (torch.zeros((2, 2, 8, 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    first = sz.rotate_write_kv_paged(q, k, v, kv, slots, slots + 20, table)
    out = torch.full_like(first, MARK)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        assert sz.rotate_write_kv_paged(q, k, v, kv2, slots, slots + 20, table, out=out) is out
    torch.cuda.synchronize()
    assert torch.equal(out, first) and torch.equal(kv, kv2)
    empty = sz.rotate_write_kv_paged(q[:0], k[:0], v[:0], kv, slots, slots, table)
    assert empty.shape == (0, 4, 64)


def test_refuses(sz):
    q, k, v = make(6, 4, 2, 64, "bf16", 6)
    kv = torch.zeros((2, 2, 8, 2, 64), dtype=torch.bfloat16, device="cuda")
    at, table = torch.arange(6, device="cuda"), sz.rotation_table(40, 64)

    def call(q=q, k=k, v=v, kv=kv, slots=at, positions=at, table=table, **more):
        return sz.rotate_write_kv_paged(q, k, v, kv, slots, positions, table, **more)

    assert call() is not None
    assert call(q=q.float()) is None and call(k=k[:5]) is None and call(v=v[:, :1]) is None
    assert call(q=q[..., :32]) is None and call(kv=kv[..., :1, :]) is None
    assert call(slots=at[:5]) is None and call(positions=at.int()) is None
    assert call(positions=at.cpu()) is None and call(table=table.half()) is None
    assert call(table=table[:, :63]) is None and call(table=table[:0].contiguous()) is None
    assert call(table=sz.rotation_table(40, 66)) is None
    assert call(out=torch.empty_like(q)[:, :3]) is None
    whole = torch.zeros((6, 4, 64), dtype=torch.bfloat16, device="cuda")
    assert call(q=whole, out=whole) is None
    assert call(k=kv[0, 0, :6], v=kv[0, 0, :6]) is None
    with pytest.raises(ValueError):
        sz.rotation_table(4, 7)
    with pytest.raises(ValueError):
        sz.rotation_table(4, 8, frequencies=[1.0])
