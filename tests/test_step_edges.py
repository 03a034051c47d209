"""What the step's calls decline and need before anything is launched, beyond
test_step_refusals.py: no GPU needed (addresses are made up, and none is read)."""

import random

import pytest

from test_step_refusals import A, CHUNK, PROMPT, WRITE, lib, refused  # noqa: F401 (lib: a fixture)
from unchainkv_amd import splitzip_cuda as sz

MiB = 1 << 20


def test_lse_over_what_a_call_reads_or_writes(lib):  # noqa: F811
    refused(lib.kvq_splitzip_chunk_attention_paged, CHUNK, [
        {"lse": address} for address in
        # q's last head, V's last block, a table's last row, lengths, the end of out
        (A[0], A[0] + 4 * 2048 - 16, A[1] + 4 * 64 * 16 * 2 * 128 - 16, A[2] + 4 * 15, A[3] + 8,
         A[4] + 4, A[5] + 4 * 8 * 256 - 4)])
    refused(lib.kvq_splitzip_prompt_attention, PROMPT, [
        {"lse": address} for address in (A[0], A[1] + 512, A[2] + 4 * 512 - 8, A[3] + 8, A[4])])


def test_out_over_lengths_and_tables(lib):  # noqa: F811
    refused(lib.kvq_splitzip_chunk_attention_paged, CHUNK,
            [{"out": A[2]}, {"out": A[3] - 4 * 8 * 256 + 16}, {"out": A[4]}])
    refused(lib.kvq_splitzip_prompt_attention, PROMPT, [{"out": A[3]}])


@pytest.mark.parametrize("max_query", (4, 400))  # streamed, and in tiles
def test_workspace_over_anything(lib, max_query):  # noqa: F811
    # tensors 4 GiB apart, the workspace ends behind the first byte of one or begins before its last
    long = dict(CHUNK, tokens=400, stride=256, width=256, max_query=max_query, lse=A[7])
    size = lib.kvq_splitzip_chunk_attention_workspace_bytes(400, 2, 8, 2, 128, 4096, max_query)
    assert size % 16 == 0
    refused(lib.kvq_splitzip_chunk_attention_paged, long, [
        {"workspace": a - size + 16} for a in A[:6] + A[7:8]] + [
        {"workspace": A[0] + 400 * 2048 - 16}, {"workspace": A[1] + 4 * 64 * 16 * 2 * 128 - 16},
        {"workspace": A[2] + 4 * 500}, {"workspace": A[5] + 400 * 8 * 256 - 16},
        {"workspace": A[7] + 400 * 8 * 4 - 16}])
    long = dict(PROMPT, tokens=2000, max_query=2000, workspace=A[6], lse=A[7])
    size = lib.kvq_splitzip_prompt_attention_workspace_bytes(2000, 2, 8, 2, 128, 2000)
    refused(lib.kvq_splitzip_prompt_attention, long,
            [{"workspace": a - size + 16} for a in A[:5] + A[7:8]])


def test_slots_over_the_layer(lib):  # noqa: F811
    refused(lib.kvq_splitzip_write_kv_paged, WRITE,
            [{"slots": A[2]}, {"slots": A[2] + 2 * MiB - 8}, {"slots": A[2] - 24}])


def test_workspace_of_a_bound_past_the_rows(lib):  # noqa: F811
    """max_query above the rows of q counts as the rows, as in the calls."""
    chunk, prompt = sz.chunk_attention_workspace_bytes, sz.prompt_attention_workspace_bytes
    assert chunk(8, 2, 32, 8, 128, 8192, 16) == chunk(8, 2, 32, 8, 128, 8192, 8) > 0
    assert chunk(8, 2, 32, 8, 128, 8192) == chunk(8, 2, 32, 8, 128, 8192, 8)
    assert prompt(1443, 1, 8, 2, 128, 5000) == prompt(1443, 1, 8, 2, 128) > 0
    entry = lib.kvq_splitzip_chunk_attention_workspace_bytes
    assert entry(8, 2, 32, 8, 128, 8192, 1 << 40) == entry(8, 2, 32, 8, 128, 8192, 8) > 0


def test_workspace_serves_smaller_calls(lib):  # noqa: F811
    """No call of smaller sizes has a larger workspace, and none asks for more than it."""
    rng = random.Random(7)
    least = lib.kvq_splitzip_prompt_attention_least_workspace_bytes

    def up_to(most):
        return min(most, int(2 ** rng.uniform(0, most.bit_length())))

    for q_heads, kv_heads, dim in ((8, 2, 128), (32, 8, 128), (32, 8, 64), (64, 1, 128), (7, 7, 64),
                                   (128, 8, 128)):
        for _ in range(400):
            most = [up_to(1 << 20), up_to(4096), up_to(1 << 17), up_to(1 << 15)]
            tokens, requests, context, query = (up_to(n) for n in most)
            query = min(query, tokens)
            big = sz.chunk_attention_workspace_bytes(most[0], most[1], q_heads, kv_heads, dim,
                                                     most[2], most[3])
            assert sz.chunk_attention_workspace_bytes(tokens, requests, q_heads, kv_heads, dim,
                                                      context, query) <= big
            big = sz.prompt_attention_workspace_bytes(most[0], most[1], q_heads, kv_heads, dim, most[3])
            small = sz.prompt_attention_workspace_bytes(tokens, requests, q_heads, kv_heads, dim, query)
            assert least(tokens, requests, q_heads, kv_heads, dim, query) <= small <= big
    # many prompts are not cut, one of the same rows or fewer is
    assert least(4096, 1, 8, 2, 128, 4096) <= least(1443, 1, 8, 2, 128, 1443)
    assert sz.prompt_attention_workspace_bytes(32768, 8, 32, 8, 128, 4096) >= least(1443, 1, 32, 8, 128, 1443) > 0


def test_workspace_of_sizes_that_no_call_takes():
    for sizes in ((8, 2, 8, 3, 128), (8, 2, 8, 2, 96), (8, 2, 0, 2, 128), (8, 2, 8, 0, 128), (-1, 2, 8, 2, 128),
                  (8, -2, 8, 2, 128), (1 << 28, 2, 8, 2, 128)):
        with pytest.raises(ValueError):
            sz.chunk_attention_workspace_bytes(*sizes, 4096)
        with pytest.raises(ValueError):
            sz.prompt_attention_workspace_bytes(*sizes)
    with pytest.raises(ValueError):
        sz.chunk_attention_workspace_bytes(8, 2, 8, 2, 128, -1)
    # calls that do nothing
    assert sz.chunk_attention_workspace_bytes(0, 2, 8, 2, 128, 4096) == 0
    assert sz.prompt_attention_workspace_bytes(8, 0, 8, 2, 128) == 0
