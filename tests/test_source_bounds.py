"""Up to which length of the longest source a streamed call joins nothing (no GPU: sizes of workspaces, for 256 CUs)."""

import pytest

from test_step_refusals import lib  # noqa: F401 (a fixture)


@pytest.mark.parametrize("requests,kv_heads,dim,most", [
    (1, 1, 64, 768), (1, 32, 64, 768), (4, 8, 128, 512), (33, 1, 64, 1024), (3, 11, 128, 1024), (191, 1, 64, 1024),
    (192, 1, 64, 2048), (24, 8, 128, 2048), (500, 4, 64, 2048)])
def test_sources_that_are_not_cut(lib, requests, kv_heads, dim, most):  # noqa: F811
    least = lib.kvq_splitzip_cross_attention_least_workspace_bytes
    for group in (1, 4):
        sizes = requests, requests, group * kv_heads, kv_heads, dim
        assert least(*sizes, most, 1) == 0 < least(*sizes, most + 1, 1)
