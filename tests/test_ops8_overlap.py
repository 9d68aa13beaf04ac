"""The C entries of the 8-bit serving operators refuse outputs that share memory with what other threads still read, or with one
another, before anything touches a device (so these run without one)."""
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
