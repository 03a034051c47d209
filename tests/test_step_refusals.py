"""What the step's C entries decline before anything is launched: no GPU needed (addresses are
made up, and none is read)."""

import ctypes

import pytest

from unchainkv_amd import splitzip_cuda as sz

A = [(i + 1) << 32 for i in range(16)]  # addresses far from each other
SCALE = ctypes.c_float(0.5)


@pytest.fixture(scope="module")
def lib():
    lib = sz._load()
    if lib is None:
        pytest.skip(f"HIP library not built: {sz.load_error()}")
    return lib


def refused(fn, good, changes):
    """Every change to the good arguments is declined with 0."""
    for change in changes:
        args = dict(good, **change)
        assert fn(*args.values()) == 0, change


PLAN = dict(new=A[0], cached=A[1], requests=3, tables=A[2], stride=8, width=8, free=A[3], count=9,
            start=A[4], block=16, rows=10, starts=A[5], contexts=A[6], slots=A[7], positions=A[8],
            next=A[9], lacking=A[10], stream=0)


def test_plan_declines(lib):
    refused(lib.kvq_splitzip_plan_step_paged, PLAN, [
        {name: 0} for name in ("new", "cached", "requests", "tables", "width", "free", "start",
                               "block", "starts", "contexts", "slots", "positions", "next",
                               "lacking")] + [
        {"stride": 7}, {"requests": 1 << 31}, {"width": 1 << 31, "stride": 1 << 31},
        {"rows": 1 << 31}, {"block": 1 << 31}, {"count": 1 << 31},
        # a result over an input or another result
        {"contexts": A[1]}, {"contexts": A[1] + 8}, {"next": A[4]}, {"lacking": A[9]},
        {"positions": A[7] + 8 * 9}, {"slots": A[2] + 4 * 20}, {"tables": A[0] - 4 * 20}])


WRITE = dict(k=A[0], v=A[1], tokens=4, heads=2, head_bytes=256, k_row=1024, k_head=256, v_row=1024,
             v_head=256, kv=A[2], plane=1 << 20, count=2048, slots=A[3], stream=0)


def test_write_declines(lib):
    refused(lib.kvq_splitzip_write_kv_paged, WRITE, [
        {name: 0} for name in ("k", "v", "tokens", "heads", "head_bytes", "kv", "slots")] + [
        {"tokens": 1 << 31}, {"count": 2049}, {"heads": 1 << 20, "head_bytes": 1 << 20},
        {"k": A[2] + 512}, {"v": A[2] + (1 << 20) + 512}, {"k": A[2] - 4 * 1024 + 600}])


CHUNK = dict(q=A[0], q_row=2048, q_head=256, tokens=4, q_heads=8, kv_heads=2, dim=128, dtype=0,
             kv=A[1], blocks=64, block=16, tables=A[2], stride=8, width=8, starts=A[3],
             contexts=A[4], requests=2, max_query=4, out=A[5], lse=0, workspace=A[6],
             workspace_bytes=1 << 30, scale=SCALE, stream=0)


def test_chunk_declines(lib):
    refused(lib.kvq_splitzip_chunk_attention_paged, CHUNK, [
        {name: 0} for name in ("q", "tokens", "q_heads", "kv_heads", "dim", "kv", "blocks", "block",
                               "tables", "width", "starts", "contexts", "requests", "max_query",
                               "out")] + [
        {"dim": 96}, {"dim": 256}, {"dtype": 2}, {"q_heads": 7}, {"kv_heads": 3}, {"max_query": 5},
        {"stride": 7}, {"q": A[0] + 2}, {"q_row": 2040}, {"q_head": 250}, {"kv": A[1] + 8},
        {"out": A[5] + 8}, {"blocks": 1 << 28}, {"tokens": 1 << 31, "max_query": 1},
        {"scale": ctypes.c_float(0.0)}, {"scale": ctypes.c_float(-1.0)},
        {"scale": ctypes.c_float(float("nan"))}, {"scale": ctypes.c_float(float("inf"))},
        {"scale": ctypes.c_float(3e38)},
        {"out": A[0] + 2048}, {"out": A[1] + (1 << 18)}])


def no_workspace(size):
    return [{"workspace": 0}, {"workspace_bytes": 0}, {"workspace_bytes": 1000}, {"workspace": A[6] + 8},
            {"workspace_bytes": size - 1}]


@pytest.mark.parametrize("max_query", (4, 400))  # streamed, and in tiles
def test_chunk_declines_without_its_workspace(lib, max_query):
    long = dict(CHUNK, tokens=400, stride=256, width=256, max_query=max_query)
    size = lib.kvq_splitzip_chunk_attention_workspace_bytes(400, 2, 8, 2, 128, 4096, max_query)
    assert size > 1000
    refused(lib.kvq_splitzip_chunk_attention_paged, long, no_workspace(size))
    # contexts that are never split need none
    assert lib.kvq_splitzip_chunk_attention_workspace_bytes(400, 2, 8, 2, 128, 128, max_query) == 0


PROMPT = dict(q=A[0], q_row=2048, q_head=256, k=A[1], k_row=512, k_head=256, v=A[2], v_row=512,
              v_head=256, tokens=4, q_heads=8, kv_heads=2, dim=128, dtype=1, starts=A[3], requests=2,
              max_query=4, out=A[4], lse=0, workspace=A[5], workspace_bytes=1 << 30, scale=SCALE,
              stream=0)


def test_prompt_declines(lib):
    refused(lib.kvq_splitzip_prompt_attention, PROMPT, [
        {name: 0} for name in ("q", "k", "v", "tokens", "q_heads", "kv_heads", "dim", "starts",
                               "requests", "max_query", "out")] + [
        {"dim": 80}, {"dtype": 2}, {"q_heads": 9}, {"max_query": 5}, {"k": A[1] + 4},
        {"k_row": 500}, {"v_head": 8}, {"out": A[4] + 4},
        {"scale": ctypes.c_float(-0.5)}, {"out": A[1]}, {"out": A[2] + 512}, {"out": A[0]}])


def test_prompt_declines_without_its_workspace(lib):
    long = dict(PROMPT, tokens=2000, max_query=2000, workspace=A[6])
    size = lib.kvq_splitzip_prompt_attention_workspace_bytes(2000, 2, 8, 2, 128, 2000)
    assert size > 1000
    refused(lib.kvq_splitzip_prompt_attention, long, no_workspace(size))
    assert lib.kvq_splitzip_prompt_attention_workspace_bytes(2000, 2, 8, 2, 128, 400) == 0


def test_workspace_sizes(lib):
    """0 for sizes that are declined; never smaller for more tokens, requests or context."""
    assert lib.kvq_splitzip_chunk_attention_workspace_bytes(4, 2, 8, 3, 128, 128, 4) == 0
    assert lib.kvq_splitzip_prompt_attention_workspace_bytes(4, 2, 8, 2, 96, 4) == 0
    last = 0
    for tokens, requests, context in [(1, 1, 64), (4, 1, 64), (4, 2, 64), (64, 2, 640), (64, 2, 6400),
                                      (512, 64, 6400), (4096, 64, 64000)]:
        size = lib.kvq_splitzip_chunk_attention_workspace_bytes(tokens, requests, 8, 2, 128, context,
                                                                tokens)
        assert size >= last > -1
        last = size


def test_tensors_off_the_gpu_are_declined():
    torch = pytest.importorskip("torch")
    q = torch.zeros((2, 8, 64), dtype=torch.bfloat16)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    kv = torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16)
    ints = torch.zeros(3, dtype=torch.int32)
    tables = torch.zeros((2, 4), dtype=torch.int32)
    assert sz.plan_step_paged(ints, ints, tables, ints, ints, 16, 4) is None
    assert sz.write_kv_paged(k, k, kv, torch.zeros(2, dtype=torch.int64)) is None
    assert sz.chunk_attention_paged(q, kv, tables, ints, ints) is None
    assert sz.prompt_attention(q, k, k, ints) is None
