"""The C entries of the 8-bit serving operators refuse outputs that share memory with what other threads still read, or with one
another, and sizes that counters do not hold, before anything touches a device (so these run without one)."""
import ctypes as C

import pytest

from e2e_browser_voice_agent_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def message(lib):
    return lib.h2c_last_error(None).decode()


def refused(lib, rc, who, *words):
    assert rc == _lib.ERR_INVALID
    text = message(lib)
    assert text.startswith(who + ":") and all(w in text for w in words), text


# Stand for device addresses, 1 MiB apart: never looked at.
A = [(i + 1) << 20 for i in range(16)]
PLAN = dict(n_req=8, page=16, cached=A[0], total=A[1], table=A[2], cols=4, ring=A[3], n_pages=8, state=A[4], out=A[5], kv_len=A[6],
            q_start=A[7], slot=A[8], position=A[9], max_tokens=40, status=A[10], stream=None)
SIZES = dict(cached=32, total=32, table=128, ring=32, state=16, out=16, kv_len=32, q_start=36, slot=160, position=160, status=8)
NAMES = dict(table="block_table", ring="free_ring", state="free_state", out="free_state_out")


@pytest.mark.parametrize("written", ["table", "ring", "out", "kv_len", "q_start", "slot", "position", "status"])
@pytest.mark.parametrize("other", list(SIZES))
def test_plan_refuses_outputs_over_other_arguments(lib, written, other):
    if other == written:
        return
    for at in (PLAN[other], PLAN[other] + SIZES[other] - 4, PLAN[other] - SIZES[written] + 4):
        rc = lib.h2c_kv8_plan(*{**PLAN, written: at}.values())
        if other == "state" and written == "out" and at == PLAN[other]:
            refused(lib, rc, "h2c_kv8_plan", "free_state_out")
        else:
            refused(lib, rc, "h2c_kv8_plan", "share memory", NAMES.get(written, written), NAMES.get(other, other))


MATMUL = dict(x_type=0, x=A[0], x_row=64, x_scale=None, w=A[1], w_row=64, w_scale=A[2], m=5, n=30, k=50, y_type=0, y=A[3], y_row=30,
              bias=A[4], workspace=A[5], workspace_bytes=1 << 16, stream=None)
CODES = {**MATMUL, "x_type": 3, "x_scale": A[6], "workspace": None, "workspace_bytes": 0}


@pytest.mark.parametrize("change,words", [
    (dict(y=A[1] + 29 * 64 + 48), ("y", "w")), (dict(y=A[2] + 116), ("y", "w_scale")), (dict(y=A[4] - 5 * 120 + 4), ("y", "bias")),
    (dict(y=A[5]), ("workspace", "y")), (dict(workspace=A[0]), ("workspace", "x")), (dict(workspace=A[1] + 16), ("workspace", "w")),
    (dict(workspace=A[2]), ("workspace", "w_scale")),
])
def test_matmul_refuses_outputs_over_other_arguments(lib, change, words):
    refused(lib, lib.h2c_i8_matmul(*{**MATMUL, **change}.values()), "h2c_i8_matmul", "share memory", *words)


@pytest.mark.parametrize("change,words", [
    (dict(y=A[0]), ("y", "codes")), (dict(y=A[0] + 4 * 64 + 48), ("y", "codes")), (dict(y=A[6] + 16), ("y", "x_scale")),
    (dict(y=A[0] - 4 * 120 - 4), ("y", "codes")),
])
def test_matmul_of_codes_refuses_outputs_over_them(lib, change, words):
    refused(lib, lib.h2c_i8_matmul(*{**CODES, **change}.values()), "h2c_i8_matmul", "share memory", *words)


@pytest.mark.parametrize("y_row", [0, 29, -29, 1])
def test_matmul_refuses_rows_of_y_that_overlap(lib, y_row):
    refused(lib, lib.h2c_i8_matmul(*{**MATMUL, "y_row": y_row}.values()), "h2c_i8_matmul", "rows of y overlap")


def attention(lib, **change):
    a = dict(q=A[0], q_row=256, q_head=64, out=A[1], out_row=256, out_head=64, lse=A[2], kv=A[3], kv_scale=A[4], n_pages=8,
             page_size=16, kv_heads=2, head_dim=64, heads=4, type=0, block_table=A[5], table_cols=4, n_req=2, q_start=A[6],
             kv_len=A[7], rows=3, max_q=2, max_kv=60, window=0, scale=0.125, workspace=None, workspace_bytes=0)
    assert set(change) <= set(a)
    return lib.h2c_kv8_attention(C.byref(_lib.Kv8AttentionArgs(**{**a, **change})), None)


@pytest.mark.parametrize("change,words", [
    (dict(out=A[0] + 4), ("out", "q itself")), (dict(out=A[0] - 3 * 1024 + 16), ("out", "q itself")),
    (dict(out=A[0], out_row=320), ("out", "q itself")), (dict(out=A[0], out_row=64, out_head=192), ("out", "q itself")),
    (dict(out=A[3]), ("out", "kv")), (dict(out=A[4]), ("out", "kv_scale")), (dict(out=A[5]), ("out", "block_table")),
    (dict(out=A[6]), ("out", "q_start")), (dict(out=A[7]), ("out", "kv_len")), (dict(lse=A[1] + 64), ("lse", "out")),
    (dict(lse=A[0]), ("lse", "q")), (dict(lse=A[7] - 44), ("lse", "kv_len")),
    (dict(max_kv=4000, workspace=A[1], workspace_bytes=1 << 30), ("workspace", "out")),
    (dict(max_kv=4000, workspace=A[0], workspace_bytes=1 << 30), ("workspace", "q")),
])
def test_attention_refuses_outputs_over_other_arguments(lib, change, words):
    # (the workspace lies below the other addresses: its size does not reach them)
    refused(lib, attention(lib, **change), "h2c_kv8_attention", *words)


@pytest.mark.parametrize("row,head", [(0, 64), (256, 0), (63, 1024), (256, 63), (100, 240), (192, 64), (-128, 64), (130, 64)])
def test_attention_refuses_vectors_of_out_that_overlap(lib, row, head):
    refused(lib, attention(lib, out=A[1] + 4096, out_row=row, out_head=head), "h2c_kv8_attention", "vectors of out overlap")


APPEND = dict(kv=A[0], scale=A[1], n_pages=8, page=16, kv_heads=2, head_dim=64, type=0, k=A[2], k_row=128, k_head=64, v=A[3],
              v_row=128, v_head=64, rows=3, slot=A[4], stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(k=A[0] + 32764), ("kv", "k")), (dict(v=A[0] - 1532), ("kv", "v")), (dict(slot=A[0] + 16), ("kv", "slot")),
    (dict(scale=A[2] + 16), ("kv_scale", "k")), (dict(scale=A[4] - 124), ("kv_scale", "slot")), (dict(scale=A[0] + 64), ("kv_scale", "kv")),
    (dict(k=A[0] + 40000, k_row=-4096), ("kv", "k")),
])
def test_append_refuses_a_cache_over_its_rows(lib, change, words):
    refused(lib, lib.h2c_kv8_append(*{**APPEND, **change}.values()), "h2c_kv8_append", "share memory", *words)


@pytest.mark.parametrize("k_out,v_out,words", [(A[0] + 16, A[6], ("k_out", "kv")), (A[6], A[1], ("v_out", "kv_scale")),
                                               (A[6], A[6] + 1520, ("v_out", "k_out")), (A[4] - 1520, A[6], ("k_out", "slot"))])
def test_read_refuses_outputs_over_other_arguments(lib, k_out, v_out, words):
    rc = lib.h2c_kv8_read(A[0], A[1], 8, 16, 2, 64, A[4], 3, 0, k_out, v_out, None)
    refused(lib, rc, "h2c_kv8_read", "share memory", *words)


@pytest.mark.parametrize("change,words", [(dict(q=A[0]), ("q", "x")), (dict(q=A[0] + 2 * 200 - 16), ("q", "x")),
                                          (dict(scale=A[0] + 4), ("scale", "x")), (dict(scale=A[1] + 64), ("scale", "q"))])
def test_quantize_refuses_outputs_over_its_values(lib, change, words):
    a = dict(type=0, x=A[0], x_row=50, rows=3, k=50, q=A[1], q_row=64, scale=A[2], stream=None)
    refused(lib, lib.h2c_i8_quantize(*{**a, **change}.values()), "h2c_i8_quantize", "share memory", *words)


def test_rows_up_to_the_integers_last_are_refused(lib):
    """Counters that step past the last row would wrap around."""
    for rows in (2**31 - 1, 2**31 - 60000):
        refused(lib, lib.h2c_i8_matmul(*{**MATMUL, "m": rows}.values()), "h2c_i8_matmul", "sizes")
        refused(lib, lib.h2c_i8_matmul(*{**MATMUL, "n": rows}.values()), "h2c_i8_matmul", "sizes")
        refused(lib, lib.h2c_i8_quantize(0, A[0], 50, rows, 50, A[1], 64, A[2], None), "h2c_i8_quantize", "rows")
        refused(lib, lib.h2c_kv8_append(*{**APPEND, "rows": rows}.values()), "h2c_kv8_append", "rows")
        refused(lib, lib.h2c_kv8_read(A[0], A[1], 8, 16, 2, 64, A[4], rows, 0, A[5], A[6], None), "h2c_kv8_read", "rows")
        refused(lib, attention(lib, rows=rows), "h2c_kv8_attention", "rows")


def test_arrays_that_are_not_aligned_to_their_elements_are_refused(lib):
    for name in SIZES:
        rc = lib.h2c_kv8_plan(*{**PLAN, name: PLAN[name] + 2}.values())
        refused(lib, rc, "h2c_kv8_plan", NAMES.get(name, name), "aligned")
    refused(lib, lib.h2c_kv8_plan(*{**PLAN, "state": PLAN["state"] + 4}.values()), "h2c_kv8_plan", "free_state", "8 bytes")
    for name in ("lse", "kv_scale", "block_table", "q_start", "kv_len"):
        refused(lib, attention(lib, **{name: A[9] + 1}), "h2c_kv8_attention", name, "aligned")
    for name, word in (("scale", "kv_scale"), ("slot", "slot")):
        refused(lib, lib.h2c_kv8_append(*{**APPEND, name: A[9] + 2}.values()), "h2c_kv8_append", word, "aligned")
    refused(lib, lib.h2c_kv8_read(A[0], A[1] + 2, 8, 16, 2, 64, A[4], 3, 0, A[5], A[6], None), "h2c_kv8_read", "kv_scale", "aligned")
    refused(lib, lib.h2c_kv8_read(A[0], A[1], 8, 16, 2, 64, A[4] + 2, 3, 0, A[5], A[6], None), "h2c_kv8_read", "slot", "aligned")
    for name in ("w_scale", "bias"):
        refused(lib, lib.h2c_i8_matmul(*{**MATMUL, name: A[9] + 2}.values()), "h2c_i8_matmul", name, "aligned")
    refused(lib, lib.h2c_i8_matmul(*{**CODES, "x_scale": A[9] + 2}.values()), "h2c_i8_matmul", "x_scale", "aligned")
    refused(lib, lib.h2c_i8_quantize(0, A[0], 50, 3, 50, A[1], 64, A[2] + 2, None), "h2c_i8_quantize", "scale", "aligned")
