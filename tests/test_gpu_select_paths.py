"""Shapes of the beam selection's kernels: many rows of several pieces, groups of segments to a lane, several waves to a
beam, with finished beams whose end token lies in any of them; and values of two beams that only 64 bits tell
apart. Bounds are those of test_gpu_beam_select.py."""

import numpy as np
import pytest

from test_gpu_beam_select import DTYPES, OFF, check, make, say, sz  # noqa: F401 (sz: a fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def check_large(choice, logits, scores, candidates, ended=None, end_token=0):
    """``check`` with its 64-bit values and orders formed on the GPU (no NaN or infinity but -inf)."""
    requests, beams, vocab = logits.shape
    for r in range(requests):
        x = logits[r].double()
        v = x - torch.logsumexp(x, 1, keepdim=True) + scores[r, :, None].double()
        v[x == -float("inf")] = -float("inf")
        if ended is not None:
            v[ended[r]] = -float("inf")
            v[ended[r], end_token] = scores[r, ended[r]].double()
        place = choice.parents[r].long() * vocab + choice.tokens[r]
        assert place.unique().numel() == candidates and 0 <= place.min() and place.max() < beams * vocab
        want, taken = v.flatten().topk(candidates).values, v.flatten()[place]
        for got, slack in ((taken, 2 * OFF), (choice.scores[r].double(), 2 * OFF + 2.0 ** -24 * want.abs())):
            assert torch.equal(got == -float("inf"), want == -float("inf"))
            assert ((got - want).abs() <= slack)[want > -float("inf")].all()
        for beam in choice.parents[r].unique().tolist():
            # within a beam, and among equal values, the order is exact
            mine = choice.tokens[r][(choice.parents[r] == beam) & (want > -float("inf"))]
            assert torch.equal(mine, v[beam].sort(descending=True, stable=True).indices[:mine.numel()])


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("requests,beams,vocab", [(1024, 8, 2500), (700, 8, 5001), (1400, 4, 4100)])
def test_pieces_of_a_wave(sz, requests, beams, vocab, dtype):  # noqa: F811
    """Rows of several pieces of 4 KB, 16384 and more in all. Maxima that rise and fall between them, a first or a
    second piece without a token, NaN and infinity in one of them."""
    piece = 4096 // torch.empty((), dtype=DTYPES[dtype]).element_size()
    assert requests * beams * -(-vocab // piece) >= 16384 and vocab > piece
    say("pieces", requests, beams, vocab, dtype)
    gen = torch.Generator("cuda").manual_seed(vocab)
    logits = torch.randn((requests, beams, vocab), device="cuda", generator=gen).mul_(3).to(DTYPES[dtype])
    scores = -20 * torch.rand((requests, beams), device="cuda", generator=gen)
    inf = float("inf")
    logits[1, :, :piece] += 40      # the maximum in the first piece,
    logits[2, :, piece:] += 40      # and in the second
    logits[3, 0, :piece] = -inf
    logits[3, 1, piece:] = -inf
    logits[4] = -inf                # nothing but one token, in the last piece
    logits[4, :, vocab - 1] = 1.0
    logits[5, 0, 7], logits[5, 1, vocab - 1] = float("nan"), float("nan")
    logits[6, 2, piece - 1], logits[6, 3, piece] = inf, inf
    logits[7, :, :piece], logits[7, 1, vocab - 2] = -inf, float("nan")
    logits[8, :, :piece] = torch.finfo(DTYPES[dtype]).min
    scores[9, 1:] = -inf
    got = sz.beam_select(logits, scores, candidates=12)
    torch.cuda.synchronize()
    some = list(range(24)) + list(range(requests - 24, requests))
    check([t[some] for t in got], logits[some], scores[some], 12)
    # the others: by a search in 64 bits on the GPU, which values come out
    v = torch.log_softmax(logits[10:].double(), -1) + scores[10:, :, None]
    want = v.flatten(1).topk(12, 1).values
    taken = v.flatten(1).gather(1, got.parents[10:].long() * vocab + got.tokens[10:])
    assert ((taken - want).abs() <= 2 * OFF).all() and ((got.scores[10:] - want).abs() <= 2 * OFF + 2.0 ** -19).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("requests,beams,vocab,candidates", [
    (1, 9, 262145, 18), (2, 9, 300001, 64), (1, 6, 600001, 12), (1, 32, 1 << 20, 64), (1, 17, (1 << 20) - 3, 17),
    (2, 20, 140000, 40), (3, 3, 300001, 6), (1, 1, 1 << 20, 5), (1, 2, 700000, 9), (1, 5, 1 << 20, 10)])
def test_groups_of_segments(sz, requests, beams, vocab, candidates, dtype):  # noqa: F811
    """Finished beams, with the end token in the first, a middle and the last segment; rows that allow few tokens,
    none, or all alike."""
    say("groups", requests, beams, vocab, candidates, dtype)
    logits, scores = make(requests, beams, 1000, dtype, seed=vocab % 1000)
    gen = torch.Generator("cuda").manual_seed(vocab)
    logits = torch.randn((requests, beams, vocab), device="cuda", generator=gen).mul_(3).to(DTYPES[dtype])
    check_large(sz.beam_select(logits, scores, candidates=candidates), logits, scores, candidates)
    ended = torch.zeros((requests, beams), dtype=torch.bool, device="cuda")
    ended[:, beams // 2] = True
    scores[:, beams // 2] = 1.0
    for token in (0, vocab // 2, vocab - 257, vocab - 1):
        got = sz.beam_select(logits, scores, candidates=candidates, ended=ended, end_token=token)
        check_large(got, logits, scores, candidates, ended, token)
        assert (got.parents[:, 0] == beams // 2).all() and (got.tokens[:, 0] == token).all()
    logits[0, 0, :vocab - 300] = float("-inf")
    if beams > 2:
        logits[0, 1] = float("-inf")
        logits[0, 2] = 0.5
    check_large(sz.beam_select(logits, scores, candidates=candidates), logits, scores, candidates)


def near_offers(tops):
    """Pairs of beams that allow m and n equal tokens, logits ``tops``, and so offer score - log m and score - log n:
    (m, n, logits, scores, the two offers). The second score is the 32-bit number that brings the offers closest,
    or one beside it: they differ by at most two steps of it."""
    for m, n in ((2, 3), (3, 5), (7, 300), (1000, 9), (513, 4097)):
        for base in (-0.5, -3.0, -17.25):
            first = np.float32(base)
            second = np.float32(np.float64(first) - np.log(m) + np.log(n))
            for near in (second, np.nextafter(second, np.float32(9)), np.nextafter(second, np.float32(-99))):
                a, b = np.float64(first) - np.log(m), np.float64(near) - np.log(n)
                if abs(a - b) < 1e-12:
                    continue
                logits = torch.full((1, 2, 6000), float("-inf"), device="cuda")
                logits[0, 0, 11:11 + m], logits[0, 1, 1:1 + n] = tops
                yield m, n, logits, torch.tensor([[float(first), float(near)]], device="cuda"), a, b


@pytest.mark.parametrize("tops", [(0.25, -8.0), (-4.0, 0.0), (0.25, -7.5)])
def test_values_that_64_bits_tell_apart(sz, tops):  # noqa: F811
    """Offers that differ by less than 32 bits hold of them come in the order of 64 bits, where the sums
    are exact: of m times 2^0.

    A weight is 2^(x log2 e - r) times 2^-(top log2 e - r), r = top log2 e rounded: exactly one for a maximum of 0 or
    a power of two, whose r is not rounded. For others, as -7.5, both exponentials and their product are rounded, and
    up to 16 + 6 additions in a wave: by at most 2^-24 each, 25 * 2^-24 in all, which offers may be apart by in
    either order."""
    say("near", tops)
    exact = all(np.frexp(abs(t))[0] in (0.0, 0.5) for t in tops)
    cases = 0
    for m, n, logits, scores, a, b in near_offers(tops):
        got = sz.beam_select(logits, scores, candidates=2)
        worse = 0 if exact else 25 * 2.0 ** -24
        if abs(a - b) > worse:
            # (the better beam's first two tokens)
            assert got.parents.tolist() == [[int(b > a)] * 2], (m, n)
            assert got.tokens.tolist() == [[1, 2] if b > a else [11, 12]]
        assert (got.scores.double() - max(a, b)).abs().max() <= worse + abs(a) * 2.0 ** -24
        cases += 1
    assert cases >= 40
