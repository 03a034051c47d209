"""Shapes of the rotated K/V write that no thread-for-a-unit launch takes (more than 256 units of a token and more
than 256 tokens), by the heads that a lane takes together, with more pairs than a wave has lanes; and more tokens than
a launch of either kernel takes. The bound is that of test_gpu_rotate_write.py."""

import pytest

from test_gpu_rotate_write import MARK, check, say, sz  # noqa: F401 (sz: a fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("adjacent", (False, True))
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary,dtype", [
    # a head for each lane, up to three and up to five
    (300, 24, 3, 128, 32, "bf16"), (257, 62, 2, 64, 16, "fp16"), (300, 16, 4, 128, 64, "bf16"),
    (301, 40, 8, 128, 64, "fp16"), (290, 32, 8, 128, 128, "bf16"),
    # the same in units of 8 and of 2 bytes
    (270, 30, 2, 68, 4, "fp16"), (270, 14, 2, 128, 20, "bf16"),
    (260, 30, 6, 68, 36, "fp16"), (259, 9, 1, 27, 6, "bf16"), (261, 7, 3, 41, 22, "fp16"),
    # more units of a head than lanes, each a pass of its own: in units of 16, 8 and 2 bytes
    (300, 2, 1, 1040, 1040, "bf16"), (300, 4, 2, 1040, 1040, "fp16"), (280, 2, 1, 2064, 2064, "bf16"),
    (300, 2, 1, 300, 260, "bf16"), (300, 5, 2, 540, 520, "fp16"), (300, 2, 1, 131, 130, "bf16"),
    (258, 4, 3, 270, 262, "fp16")])
def test_rows_by_waves(sz, tokens, q_heads, kv_heads, dim, rotary, dtype, adjacent):  # noqa: F811
    say("waves", tokens, q_heads, kv_heads, dim, rotary, dtype, adjacent)
    check(sz, tokens, q_heads, kv_heads, dim, rotary, adjacent, dtype, seed=tokens + dim,
          drop=[(0, -1), (tokens // 2, 1 << 40), (tokens - 1, -1)])


@pytest.mark.parametrize("dim,rotary", [(66, 66), (258, 2)])
def test_later_launches(sz, dim, rotary):  # noqa: F811
    """One token more than a workgroup's share in 2^22 workgroups (132 units of a token, one token to a
    workgroup), and than 8 waves of each token in 2^25 waves (772 units)."""
    tokens = (1 << 22) + 5
    say("launches", tokens, dim, rotary)
    at = torch.arange(tokens, device="cuda")
    q = ((at % 247).to(torch.bfloat16)[:, None] + (torch.arange(dim, device="cuda") % 5).to(torch.bfloat16))[:, None]
    k, v = q + 2, q + 4  # (whole numbers up to 256 are exact)
    kv = torch.full((2, tokens + 3, 1, 1, dim), MARK, dtype=torch.bfloat16, device="cuda")
    # quarters of a turn: (x, y) -> (x, y), (-y, x), (-x, -y), (y, -x)
    table = torch.tensor([[1.0, 0.0], [0.0, 1.0], [-1.0, 0.0], [0.0, -1.0]], device="cuda")
    table = table.repeat_interleave(rotary // 2, 1).contiguous()
    got = sz.rotate_write_kv_paged(q, k, v, kv, at.flip(0), at % 4, table)
    torch.cuda.synchronize()
    half = rotary // 2
    # (place p of the layer has token tokens - 1 - p)
    for turned, rows, first, step in ((got[:, 0], q[:, 0], 0, 1),
                                      (kv[0, :tokens, 0, 0], k.flip(0)[:, 0], tokens - 1, -1)):
        for n in range(4):
            x, y = rows[n::4, :half], rows[n::4, half:rotary]
            pair = ((x, y), (-y, x), (-x, -y), (y, -x))[(first + step * n) % 4]
            assert torch.equal(turned[n::4, :rotary], torch.cat(pair, 1))
        assert torch.equal(turned[:, rotary:], rows[:, rotary:])
    assert torch.equal(kv[1, :tokens, 0, 0], v.flip(0)[:, 0]) and (kv[:, tokens:] == MARK).all()
    del q, k, v, kv, got
    torch.cuda.empty_cache()
