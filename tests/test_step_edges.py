"""What the step's calls decline and need before anything is launched, beyond
test_step_refusals.py: no GPU needed (addresses are made up, and none is read)."""

import pytest

from test_step_refusals import A, CHUNK, PROMPT, WRITE, lib, refused  # noqa: F401 (lib: a fixture)

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
