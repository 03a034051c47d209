"""Beam selection against 64-bit values on the host.

Bound of a value: the sum of exponentials is off by the roundings of its 32-bit terms, each of
(3 |d| + 2) 2^-24 of it (the difference d to the maximum, its product, the exponential), of at most
ln(vocab) + 1 <= 15 on the terms' average, and of at most 64 additions and 32 changes of reference in a
lane, 8 joins: (47 + 104) 2^-24 < 2^-16.7 of it, and so is its logarithm. Scores are rounded once more,
2^-24 of them. Values of one beam have one and the same logarithm: their order is exact."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

OFF = 2.0 ** -16.7
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def sz():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")
    from unchainkv_amd import splitzip_cuda

    assert splitzip_cuda.available(), splitzip_cuda.load_error()
    return splitzip_cuda


def say(*parts):
    print("[case]", *parts, flush=True)


def values_of(logits, scores, ended=None, end_token=0):
    """(requests, beams * vocab) float64."""
    x, s = logits.double().cpu().numpy(), scores.double().cpu().numpy()
    with np.errstate(all="ignore"):
        top = x.max(-1, keepdims=True)
        top = np.where(np.isneginf(top), 0.0, top)
        # (the largest logit first: beside one of 3e38 the logarithm would be lost)
        v = x - top - np.log(np.exp(x - top).sum(-1, keepdims=True)) + s[..., None]
    v[np.isneginf(x)] = -np.inf
    v[np.isneginf(s)] = -np.inf
    if ended is not None:
        e = ended.cpu().numpy()
        v[e] = -np.inf
        v[e, end_token] = s[e]
    return v.reshape(len(v), -1)


def order_of(v):
    """Places by value, NaN first, then by place."""
    return np.argsort(np.where(np.isnan(v), -np.inf, -v), kind="stable")


def check(choice, logits, scores, candidates, ended=None, end_token=0, exact=False):
    vocab = logits.shape[2]
    values = values_of(logits, scores, ended, end_token)
    got = [t.cpu().numpy() for t in choice]
    for r, v in enumerate(values):
        want = order_of(v)[:candidates]
        place = got[1][r].astype(np.int64) * vocab + got[2][r]
        assert len(set(place.tolist())) == candidates and (place >= 0).all() and (place < v.size).all()
        if exact:
            assert place.tolist() == want.tolist()
        a, b = v[place], v[want]
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isinf(a), np.isinf(b))
        fine = np.isfinite(b)
        # near values of two beams may come in either order
        assert (np.abs(a - b)[fine] <= 2 * OFF).all()
        assert (np.abs(got[0][r] - b)[fine] <= 2 * OFF + 2.0 ** -24 * np.abs(b[fine])).all()
        assert np.array_equal(np.isnan(got[0][r]), np.isnan(b)) and (got[0][r][np.isneginf(b)] == -np.inf).all()
        for beam in set(got[1][r].tolist()):
            mine = got[1][r] == beam
            there = place[mine & fine]
            assert there.tolist() == [p for p in order_of(v).tolist() if p // vocab == beam][:len(there)]


def make(requests, beams, vocab, dtype, seed=0, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn((requests, beams, vocab), generator=gen) * spread).to(DTYPES[dtype]).cuda()
    return logits, (-20 * torch.rand((requests, beams), generator=gen)).cuda()


@pytest.mark.parametrize("dtype", ("bf16", "fp16", "fp32"))
@pytest.mark.parametrize("requests,beams,vocab,candidates", [
    (1, 1, 1, 1), (2, 3, 5, 15), (1, 4, 32000, 4), (3, 2, 255, 7), (2, 5, 257, 10), (5, 1, 2049, 64),
    (1, 32, 700, 64), (2, 8, 50257, 16), (70, 2, 1000, 2), (1, 3, 300001, 6), (1, 1, 1 << 20, 3),
    (2, 20, 140000, 5)])
def test_matches_64_bits(sz, requests, beams, vocab, candidates, dtype):
    say("select", requests, beams, vocab, candidates, dtype)
    logits, scores = make(requests, beams, vocab, dtype, seed=vocab)
    choice = sz.beam_select(logits, scores, candidates=candidates)
    torch.cuda.synchronize()
    check(choice, logits, scores, candidates, exact=beams == 1)


@pytest.mark.parametrize("vocab", (5, 513, 9001))
def test_equal_values_come_in_order(sz, vocab):
    """Ties: the lowest beam, then the lowest token, at any address; also of equal rows."""
    say("ties", vocab)
    logits = torch.zeros((2, 3, vocab), device="cuda", dtype=torch.bfloat16)
    logits[1] = torch.randint(0, 2, (vocab,), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    scores = torch.full((2, 3), -1.5, device="cuda")
    check(sz.beam_select(logits, scores, candidates=14), logits, scores, 14, exact=True)
    rows, scores = make(1, 1, vocab, "fp16", seed=2)
    logits, scores = rows.repeat(2, 4, 1), scores.repeat(2, 4)
    check(sz.beam_select(logits, scores, candidates=12), logits, scores, 12, exact=True)
    # values that only their logits tell apart, and by less than 64 bits hold
    logits = torch.zeros((1, 1, vocab), device="cuda")
    logits[0, 0, vocab // 2], logits[0, 0, -1] = 1e-30, 1e-20
    check(sz.beam_select(logits, scores[:1, :1].contiguous(), candidates=5), logits, scores[:1, :1], 5,
          exact=True)


def test_sorted_and_crowded_rows(sz):
    """All of the best in one place, and in as many as there can be."""
    say("sorted")
    for vocab in (4096, 70000):
        rising = torch.arange(vocab, device="cuda", dtype=torch.float32) / 500
        logits = torch.stack((rising, rising.flip(0), rising.roll(300)))[None]
        scores = torch.tensor([[-3.0, -3.25, -3.375]], device="cuda")
        for candidates in (3, 64):
            check(sz.beam_select(logits, scores, candidates=candidates), logits, scores, candidates)


@pytest.mark.parametrize("dtype", ("bf16", "fp32"))
@pytest.mark.parametrize("requests,beams,vocab,candidates", [
    (2, 1, 300, 64), (1, 16, 2989, 32), (3, 8, 689, 16), (20, 10, 1572, 20), (1, 1, 7, 5), (2, 3, 8, 20),
    (1, 2, 1029, 64), (3, 4, 3, 12)])
def test_more_candidates_than_segments(sz, requests, beams, vocab, candidates, dtype):
    """Rows that are short for what is asked of them, whole and with one beam or one value in use; rows that end
    inside a load, or are shorter than one."""
    say("short", requests, beams, vocab, candidates, dtype)
    logits, scores = make(requests, beams, vocab, dtype, seed=candidates)
    check(sz.beam_select(logits, scores, candidates=candidates), logits, scores, candidates)
    one = scores.clone()
    one[:, 1:] = -float("inf")
    check(sz.beam_select(logits, one, candidates=candidates), logits, one, candidates)
    ended = torch.zeros((requests, beams), dtype=torch.bool, device="cuda")
    ended[:, 0] = True
    choice = sz.beam_select(logits, scores, candidates=candidates, ended=ended, end_token=vocab - 1)
    check(choice, logits, scores, candidates, ended, vocab - 1)
    logits[:] = 1.5
    check(sz.beam_select(logits, one, candidates=candidates), logits, one, candidates, exact=True)
    logits[..., 1:] = -float("inf")
    check(sz.beam_select(logits, one, candidates=candidates), logits, one, candidates, exact=True)


def test_masks(sz):
    """Tokens that are not allowed, by -inf and by the lowest value; rows that allow none; beams not in
    use; too little to offer."""
    say("masks")
    logits, scores = make(4, 3, 3001, "fp32", seed=3)
    logits[0, :, 5:] = float("-inf")
    logits[1, 1] = float("-inf")
    logits[1, 2, 7:] = torch.finfo(torch.float32).min
    scores[2, 1:] = float("-inf")
    logits[2, 2, 4] = float("nan")  # (of a beam that offers nothing)
    scores[3] = float("-inf")
    check(sz.beam_select(logits, scores, candidates=20), logits, scores, 20)
    logits[0, 0] = torch.finfo(torch.float32).min  # all at the lowest value: each has 1 / vocab
    check(sz.beam_select(logits, scores, candidates=20), logits, scores, 20)
    alone = sz.beam_select(logits[:1, :1], scores[:1, :1].contiguous(), candidates=3)
    assert alone.tokens.tolist() == [[0, 1, 2]]
    assert np.allclose(alone.scores.tolist(), scores[0, 0].item() - np.log(3001), atol=1e-5)
    low, s = make(2, 2, 800, "bf16", seed=4)
    low[:, 0, 3:] = torch.finfo(torch.bfloat16).min
    check(sz.beam_select(low, s, candidates=9), low, s, 9)


def test_ended_beams(sz):
    say("ended")
    logits, scores = make(5, 4, 1200, "bf16", seed=5)
    ended = torch.zeros((5, 4), dtype=torch.bool, device="cuda")
    ended[0, 1] = ended[1, :] = ended[2, 0] = ended[3, 3] = True
    scores[2, 0], scores[3, 3] = 0.5, float("-inf")
    logits[0, 1, 9] = float("nan")  # (not looked at)
    for token in (0, 700, 1199):
        got = sz.beam_select(logits, scores, candidates=8, ended=ended, end_token=token)
        check(got, logits, scores, 8, ended, token)
    assert got.tokens[2, 0] == 1199 and got.scores[2, 0] == 0.5 and got.parents[2, 0] == 0


def test_nan_and_infinite_logits(sz):
    say("nan")
    logits, scores = make(3, 3, 900, "fp32", seed=6)
    logits[0, 1, 700], logits[1, 2, 3], logits[1, 2, 4:300] = float("nan"), float("inf"), float("-inf")
    got = sz.beam_select(logits, scores, candidates=6)
    check(got, logits, scores, 6)
    assert got.parents[:2].tolist() == [[1] * 6, [2] * 6]
    assert got.tokens[:2].tolist() == [[0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 300, 301]]
    logits[2], logits[2, :, 511] = float("-inf"), float("nan")  # (nothing else in its segment)
    got = sz.beam_select(logits, scores, candidates=4)
    check(got, logits, scores, 4, exact=True)


@pytest.mark.parametrize("dtype", ("bf16", "fp32"))
def test_strides_and_addresses(sz, dtype):
    """Views of padded vocabularies, of every other beam, at odd addresses."""
    say("strides", dtype)
    wide, scores = make(3, 8, 1111, dtype, seed=7)
    logits = wide[:, 1::2, 3:1104]
    scores = scores[:, 1::2].contiguous()
    check(sz.beam_select(logits, scores, candidates=8), logits, scores, 8)
    one = wide[:1, :1].expand(3, 4, 1111)  # one row for all
    check(sz.beam_select(one, scores, candidates=8), one, scores, 8)


def test_extreme_spreads(sz):
    say("spreads")
    for spread in (0.0, 1e-3, 60.0, 1e4, 1e30):
        logits, scores = make(2, 3, 5000, "fp32", seed=8, spread=spread)
        check(sz.beam_select(logits, scores, candidates=9), logits, scores, 9)


def test_many_rows(sz):
    """More rows than a grid's dimension holds."""
    say("many rows")
    logits, scores = make(33000, 2, 40, "bf16", seed=12)
    got = sz.beam_select(logits, scores, candidates=3)
    values = values_of(logits, scores)
    want = np.argsort(-values, axis=1, kind="stable")[:, :3]
    place = got.parents.long().cpu().numpy() * 40 + got.tokens.cpu().numpy()
    a, b = np.take_along_axis(values, place, 1), np.take_along_axis(values, want, 1)
    assert (np.abs(a - b) <= 2 * OFF).all() and (np.diff(np.sort(place, 1), axis=1) > 0).all()


def test_captured_and_repeated_calls(sz):
    """A captured call follows its inputs; the same inputs give the same bits."""
    say("captured")
    logits, scores = make(6, 4, 20011, "bf16", seed=9)
    choice = sz.new_beam_choice(6, 8, "cuda")
    ws = torch.empty(sz.beam_select_workspace_bytes(6, 4, 20011), dtype=torch.uint8, device="cuda")
    first = sz.beam_select(logits, scores, candidates=8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert sz.beam_select(logits, scores, candidates=8, choice=choice, workspace=ws) is choice
    for n in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check(choice, logits, scores, 8)
        if n == 0:
            assert all(torch.equal(a, b) for a, b in zip(choice, first))
        new, new_scores = make(6, 4, 20011, "bf16", seed=20 + n)
        logits.copy_(new)
        scores.copy_(new_scores)


def test_refuses(sz):
    logits, scores = make(2, 3, 100, "bf16")
    ended = torch.zeros((2, 3), dtype=torch.bool, device="cuda")

    def call(logits=logits, scores=scores, **more):
        return sz.beam_select(logits, scores, **more)

    assert call().scores.shape == (2, 3)
    assert call(logits=logits.double()) is None and call(logits=logits[0]) is None
    assert call(logits=logits[..., ::2]) is None and call(scores=scores[:1]) is None
    assert call(scores=scores.half()) is None and call(scores=scores.cpu()) is None
    assert call(candidates=0) is None and call(candidates=65) is None and call(candidates=301) is None
    assert call(ended=ended) is None and call(ended=ended, end_token=100) is None
    assert call(ended=ended, end_token=-1) is None and call(ended=ended.int(), end_token=1) is None
    assert call(choice=sz.new_beam_choice(2, 4, "cuda")) is None
    good = sz.new_beam_choice(2, 3, "cuda")
    assert call(choice=good._replace(scores=scores)) is None
    assert call(logits=logits.repeat(1, 11, 1), scores=scores.repeat(1, 11)) is None
    assert call(logits=logits.clone().requires_grad_()) is None
    assert sz.beam_select(logits[:0], scores[:0], candidates=2).tokens.shape == (0, 2)
    with pytest.raises(ValueError):
        sz.beam_select_workspace_bytes(1, 33, 100)


@pytest.mark.parametrize("dtype", ("bf16", "fp32"))
@pytest.mark.parametrize("beams", (1, 4, 16, 17, 32))
def test_rows_that_one_workgroup_scans(sz, beams, dtype):
    """As many logits as a request's one workgroup reads by itself, and one more."""
    chunk = 2048 if dtype == "bf16" else 1024
    for vocab in (max(16 // beams, 1) * chunk, max(16 // beams, 1) * chunk + 1):
        say("one launch", beams, vocab, dtype)
        logits, scores = make(3, beams, vocab, dtype, seed=beams)
        logits[1, 0, : vocab // 2] = -float("inf")
        scores[2, beams // 2:] = -float("inf")
        if beams > 1:
            scores[2, 0] = -3.0
        ended = torch.zeros((3, beams), dtype=torch.bool, device="cuda")
        ended[0, beams - 1] = beams > 1
        choice = sz.beam_select(logits, scores, candidates=min(2 * beams, 64), ended=ended, end_token=vocab - 1)
        check(choice, logits, scores, min(2 * beams, 64), ended, vocab - 1)
