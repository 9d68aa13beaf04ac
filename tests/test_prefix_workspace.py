"""What attention behind shared prefixes asks for as its workspace, on the CPU: each row and head has its sums once for every span, however the
rows are spread over requests and groups."""
import ctypes as C

import pytest

from e2e_browser_voice_agent_b200 import _lib, build, kv8

HEADS, KV_HEADS, DIM = 28, 4, 128


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def need(lib, n_req, rows, max_q, max_kv, groups, max_prefix, prefix_cols=256):
    own = _lib.Kv8AttentionArgs(kv=1 << 20, kv_scale=2 << 20, n_pages=4096, page_size=16, kv_heads=KV_HEADS, head_dim=DIM, heads=HEADS,
                                type=2, table_cols=256, n_req=n_req, rows=rows, max_q=max_q, max_kv=max_kv, scale=0.1)
    a = _lib.Kv8PrefixArgs(own, prefix_cols=prefix_cols, n_groups=groups, max_prefix=max_prefix)
    return lib.h2c_kv8_prefix_attention_workspace(C.byref(a))


@pytest.mark.parametrize("n_req,rows,max_q,max_kv,groups,max_prefix", [
    (256, 511, 256, 2048, 1, 2048),         # single tokens beside a chunk of a prompt
    (1024, 1535, 512, 2048, 1, 2048),
    (1024, 1535, 512, 2048, 12, 600),
    (8192, 8192, 1, 500, 4096, 2048),       # thousands of groups of few rows
    (8192, 8191 + 256, 256, 500, 8192, 4000),
    (64, 64 * 200, 200, 800, 5, 4000), (2, 2, 1, 4000, 1, 4000), (300, 300, 1, 100, 1, 4096), (1, 256, 256, 4000, 1, 4096)])
def test_a_row_and_head_once_a_span(lib, n_req, rows, max_q, max_kv, groups, max_prefix):
    # of the kernel for many rows: spans of 512 keys or more; of the one for few: two tiles of 8 rows for each request (group) and kv head, cut
    # into spans until there are 5,328
    row = DIM * 4 + 8
    most = sum(rows * HEADS * -(-keys // 512) + 8 * (5328 + 2 * n * KV_HEADS) for n, keys in ((n_req, max_kv), (groups, max_prefix)))
    assert 0 < need(lib, n_req, rows, max_q, max_kv, groups, max_prefix) <= row * most


@pytest.mark.parametrize("groups,rows,max_prefix,few", [(8, 32, 640, True), (2, 6, 4096, True), (3, 15, 1280, True), (1, 32, 8000, False)])
def test_few_rows_among_groups_are_the_kernel_for_few(lib, groups, rows, max_prefix, few):
    """Rows of 7 heads a kv head: with the row tiles that the groups can have together the keys visited are below 2^17. The kernel for many rows
    would ask for 25 MB for its sums behind long tables; the one for few asks for less than that in these calls."""
    visits = (rows * 7 // 8 + groups) * KV_HEADS * max_prefix
    assert (visits <= 2**17) == few
    assert (need(lib, rows, rows, 1, 100, groups, max_prefix, 512) < 192 * 256 * DIM * 4) == few
