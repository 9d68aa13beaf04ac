"""The C entries of the norm, rotary positions, logits and attention behind shared prefixes refuse arguments that do not fit with a status and a message, before anything
touches a device (so these run without one), and so do the Python calls."""
import ctypes as C

import pytest
import torch

from e2e_browser_voice_agent_b200 import _lib, build, int8, kv8, logits, rope


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def refused(lib, rc, who, *words, code=_lib.ERR_INVALID):
    assert rc == code
    text = lib.h2c_last_error(None).decode()
    assert text.startswith(who + ":") and all(w in text for w in words), text


# Stand for device addresses, 1 MiB apart: never looked at.
A = [(i + 1) << 20 for i in range(16)]
NORM = dict(x_type=2, x=A[0], x_row=50, res_type=0, residual=A[1], res_row=50, sum=A[2], sum_row=50, weight=A[3], eps=1e-6, rows=3, k=50,
            q=A[4], q_row=64, scale=A[5], stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(rows=-1), ("rows",)), (dict(rows=2**31 - 1), ("rows",)), (dict(k=0), ("rows of 0",)), (dict(k=131073, q_row=131088), ("rows of",)),
    (dict(eps=-1.0), ("eps",)), (dict(eps=float("nan")), ("eps",)), (dict(x=None), ("null",)), (dict(weight=None), ("null",)),
    (dict(q=None), ("null",)), (dict(scale=None), ("null",)), (dict(sum=None), ("null",)), (dict(residual=None), ("null",)),
    (dict(x=A[0] + 1), ("x must be aligned",)), (dict(residual=A[1] + 2), ("residual", "aligned")), (dict(sum=A[2] + 2), ("sum", "aligned")),
    (dict(weight=A[3] + 2), ("weight", "aligned")), (dict(scale=A[5] + 1), ("scale", "aligned")), (dict(q=A[4] + 8), ("q must",)),
    (dict(q_row=48), ("q must",)), (dict(q_row=56), ("q must",)),
    (dict(sum_row=49), ("rows of sum overlap",)), (dict(sum_row=-49), ("rows of sum overlap",)), (dict(sum_row=0), ("rows of sum overlap",)),
    (dict(sum=A[1], sum_row=51), ("sum must be residual itself",)), (dict(sum=A[1] + 4), ("sum must be residual itself",)),
    (dict(sum=A[0]), ("sum must be x itself",)),                        # float32 sums over bfloat16 values
    (dict(res_type=2, sum=A[0] + 2), ("sum must be x itself",)), (dict(sum=A[3]), ("sum", "weight")), (dict(sum=A[4]), ("sum", "q")),
    (dict(sum=A[5]), ("scale", "sum")), (dict(q=A[0]), ("q", "x")), (dict(q=A[1]), ("q", "residual")), (dict(q=A[3]), ("q", "weight")),
    (dict(q=A[5]), ("q", "scale")), (dict(scale=A[0]), ("scale", "x")), (dict(scale=A[1]), ("scale", "residual")),
    (dict(scale=A[3] + 196), ("scale", "weight")),
])
def test_norm_refuses(lib, change, words):
    refused(lib, lib.h2c_i8_norm(*{**NORM, **change}.values()), "h2c_i8_norm", *words)


def test_norm_types_and_nothing_to_do(lib):
    refused(lib, lib.h2c_i8_norm(*{**NORM, "x_type": 3}.values()), "h2c_i8_norm", "type 3", code=_lib.ERR_BAD_TYPE)
    refused(lib, lib.h2c_i8_norm(*{**NORM, "res_type": 1}.values()), "h2c_i8_norm", "residual", code=_lib.ERR_BAD_TYPE)
    assert lib.h2c_i8_norm(*{**NORM, "rows": 0, "x": None}.values()) == _lib.OK


VALUES = dict(q=A[0], q_row=64, scale=A[1], rows=3, k=50, type=0, y=A[2], stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(rows=-1), ("rows",)), (dict(k=0), ("rows of 0",)), (dict(q=None), ("null",)), (dict(scale=None), ("null",)), (dict(y=None), ("null",)),
    (dict(q=A[0] + 4), ("q must",)), (dict(q_row=48), ("q must",)), (dict(y=A[2] + 2), ("y", "aligned")), (dict(y=A[0] + 60), ("y", "q")),
    (dict(y=A[1] - 596), ("y", "scale")), (dict(scale=A[1] + 2), ("scale", "aligned")),
])
def test_values_refuses(lib, change, words):
    refused(lib, lib.h2c_i8_values(*{**VALUES, **change}.values()), "h2c_i8_values", *words)
    refused(lib, lib.h2c_i8_values(*{**VALUES, "type": 3}.values()), "h2c_i8_values", code=_lib.ERR_BAD_TYPE)
    assert lib.h2c_i8_values(*{**VALUES, "rows": 0, "y": None}.values()) == _lib.OK


ROPE = dict(type=0, q=A[0], q_row=256, q_head=64, q_out=A[1], q_out_row=256, q_out_head=64, q_heads=4, k=A[2], k_row=128, k_head=64,
            k_out=A[3], k_out_row=128, k_out_head=64, k_heads=2, tokens=5, head_dim=64, position=A[4], frequency=A[5], rotary=64,
            interleaved=0, magnitude=1.0, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(tokens=-1), ("tokens",)), (dict(q_heads=-1), ("heads",)), (dict(k_heads=70000), ("heads",)), (dict(head_dim=1026), ("head_dim",)),
    (dict(rotary=63), ("rotary_dim",)), (dict(rotary=66), ("rotary_dim",)), (dict(rotary=0), ("rotary_dim",)), (dict(interleaved=2), ("interleaved",)),
    (dict(q=None), ("null",)), (dict(k_out=None), ("null",)), (dict(position=None), ("null",)), (dict(frequency=None), ("null",)),
    (dict(q=A[0] + 2), ("q", "aligned")), (dict(k_out=A[3] + 1), ("k_out", "aligned")), (dict(position=A[4] + 2), ("position", "aligned")),
    (dict(frequency=A[5] + 4), ("frequency", "aligned")),
    (dict(q_out_row=0), ("vectors of q_out overlap",)), (dict(q_out_head=63), ("vectors of q_out overlap",)),
    (dict(k_out_row=100, k_out_head=64), ("vectors of k_out overlap",)),
    (dict(q_out=A[0], q_out_row=320), ("q_out must be q itself",)), (dict(q_out=A[0] + 4), ("q_out must be q itself",)),
    (dict(k_out=A[0]), ("k_out", "q")), (dict(q_out=A[2]), ("q_out", "k")), (dict(k_out=A[1] + 5 * 1024 - 4), ("share memory",)),
    (dict(q_out=A[4]), ("q_out", "position")), (dict(k_out=A[5]), ("k_out", "frequency")),
])
def test_rope_refuses(lib, change, words):
    refused(lib, lib.h2c_rope(*{**ROPE, **change}.values()), "h2c_rope", *words)


def test_rope_types_and_nothing_to_do(lib):
    refused(lib, lib.h2c_rope(*{**ROPE, "type": 3}.values()), "h2c_rope", code=_lib.ERR_BAD_TYPE)
    assert lib.h2c_rope(*{**ROPE, "tokens": 0, "q": None}.values()) == _lib.OK
    assert lib.h2c_rope(*{**ROPE, "q_heads": 0, "k_heads": 0, "q": None}.values()) == _lib.OK


LOGITS = dict(type=0, logits=A[0], in_row=100, out=A[1], out_row=100, rows=3, vocab=100, tokens=A[2], tokens_row=20, columns=20, length=A[3],
              repetition=A[4], presence=A[5], frequency=A[6], bias_id=A[7], bias=A[8], n_bias=4, allowed=A[9], allowed_row=4, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(rows=-1), ("rows",)), (dict(vocab=0), ("rows of 0",)), (dict(vocab=2**30 + 1), ("rows of",)), (dict(columns=-1), ("columns",)),
    (dict(n_bias=-1), ("n_bias",)), (dict(n_bias=1025), ("n_bias",)), (dict(logits=None), ("null",)), (dict(out=None), ("null",)),
    (dict(bias=None), ("null",)), (dict(bias_id=None), ("null",)), (dict(length=None), ("null",)), (dict(tokens=None), ("null",)),
    (dict(tokens=None, length=None), ("penalties need",)), (dict(logits=A[0] + 2), ("aligned",)), (dict(out=A[1] + 1), ("aligned",)),
    (dict(out_row=99), ("rows of out overlap",)), (dict(out=A[0], out_row=101), ("out must be logits itself",)),
    (dict(out=A[0] + 4), ("out must be logits itself",)), (dict(out=A[0] - 4 * 200), ("out must be logits itself",)),
    *[(dict(out=A[i]), ("out", n)) for i, n in ((2, "tokens"), (3, "length"), (4, "repetition"), (5, "presence"), (6, "frequency"),
                                                (7, "bias_id"), (8, "bias"), (9, "allowed"))],
    (dict(length=A[3] + 2), ("length", "aligned")), (dict(allowed=A[9] + 1), ("allowed", "aligned")),
])
def test_logits_refuses(lib, change, words):
    refused(lib, lib.h2c_logits_adjust(*{**LOGITS, **change}.values()), "h2c_logits_adjust", *words)


def test_logits_types_and_nothing_to_do(lib):
    refused(lib, lib.h2c_logits_adjust(*{**LOGITS, "type": 3}.values()), "h2c_logits_adjust", code=_lib.ERR_BAD_TYPE)
    assert lib.h2c_logits_adjust(*{**LOGITS, "rows": 0, "logits": None}.values()) == _lib.OK
    refused(lib, lib.h2c_logits_adjust(*{**LOGITS, "rows": 2**25, "vocab": 2**22, "in_row": 2**22, "out_row": 2**22, "out": 1 << 50, "tokens": None,
                                         "length": None, "repetition": None, "presence": None, "frequency": None, "n_bias": 0,
                                         "allowed": None}.values()), "h2c_logits_adjust", "too many")


X, W = torch.zeros(3, 50), torch.ones(50)


@pytest.mark.parametrize("call,error,word", [
    (lambda: int8.norm(X, W), ValueError, "CUDA"),
    (lambda: int8.norm(X.long(), W), TypeError, "x:"),
    (lambda: int8.norm(X, W.double()), TypeError, "weight"),
    (lambda: int8.norm(X, W[:9]), ValueError, "weight"),
    (lambda: int8.norm(X[0], W), ValueError, "x:"),
    (lambda: int8.norm(X.t(), torch.ones(3)), ValueError, "dense"),
    (lambda: int8.norm(X, W, out=X), ValueError, "out"),
    (lambda: int8.norm(X, W, residual=X[:2]), ValueError, "residual"),
    (lambda: int8.norm(X, W, residual=X.half()), TypeError, "residual"),
    (lambda: int8.norm(X.half(), W, residual=X, out=X.half()), TypeError, "out"),
    (lambda: int8.norm(X, W, residual=X, out=X[:, :9]), ValueError, "out"),
    (lambda: int8.values(X, W), TypeError, "codes"),
    (lambda: int8.values(X.to(torch.int8), W[:3], k=51), ValueError, "k:"),
    (lambda: int8.values(X.to(torch.int8), W[:3], dtype=torch.int8), TypeError, "dtype"),
    (lambda: int8.values(X.to(torch.int8), W), ValueError, "scale"),
])
def test_norm_calls_refuse(call, error, word):
    with pytest.raises(error, match=word):
        call()


Q, P, F = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32), torch.ones(32, dtype=torch.float64)


@pytest.mark.parametrize("call,error,word", [
    (lambda: rope.rotate(Q, P, F), ValueError, "CUDA"),
    (lambda: rope.rotate(Q.long(), P, F), TypeError, "q:"),
    (lambda: rope.rotate(Q[0], P, F), ValueError, "q:"),
    (lambda: rope.rotate(Q.transpose(1, 2), P, F), ValueError, "dense"),
    (lambda: rope.rotate(Q, P[:2], F), ValueError, "position"),
    (lambda: rope.rotate(Q, P.long(), F), TypeError, "position"),
    (lambda: rope.rotate(Q, P, F.float()), TypeError, "frequency"),
    (lambda: rope.rotate(Q, P, torch.ones(33, dtype=torch.float64)), ValueError, "frequency"),
    (lambda: rope.rotate(Q, P, F[:0]), ValueError, "frequency"),
    (lambda: rope.rotate(Q, P, F, k=Q.half()), TypeError, "k:"),
    (lambda: rope.rotate(Q, P, F, k=Q[:2]), ValueError, "k:"),
    (lambda: rope.rotate(Q, P, F, k_out=Q), ValueError, "k_out"),
    (lambda: rope.rotate(Q, P, F, out=Q[:2]), ValueError, "out"),
    (lambda: rope.rotate(Q, P, F, k=Q, k_out=Q[:2]), ValueError, "k_out"),
    (lambda: rope.frequencies(5), ValueError, "rotary_dim"),
    (lambda: rope.frequencies(6, 1.0), ValueError, "base"),
    (lambda: rope.frequencies(6, factor=0.5), ValueError, "factor"),
    (lambda: rope.frequencies(6, scaling="other"), ValueError, "scaling"),
    (lambda: rope.frequencies(2, scaling="ntk"), ValueError, "ntk"),
    (lambda: rope.frequencies(6, scaling="yarn", factor=2.0), ValueError, "original"),
])
def test_rope_calls_refuse(call, error, word):
    with pytest.raises(error, match=word):
        call()


L, T, N, S = torch.zeros(3, 100), torch.zeros(3, 9, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.ones(3)


@pytest.mark.parametrize("call,error,word", [
    (lambda: logits.adjust(L), ValueError, "CUDA"),
    (lambda: logits.adjust(L.double()), TypeError, "logits"),
    (lambda: logits.adjust(L[0]), ValueError, "logits"),
    (lambda: logits.adjust(L.t()), ValueError, "dense"),
    (lambda: logits.adjust(L, out=L[:2]), ValueError, "out"),
    (lambda: logits.adjust(L, out=L.half()), TypeError, "out"),
    (lambda: logits.adjust(L, tokens=T), ValueError, "belong together"),
    (lambda: logits.adjust(L, tokens=T.long(), length=N), TypeError, "tokens"),
    (lambda: logits.adjust(L, tokens=T[:2], length=N), ValueError, "tokens"),
    (lambda: logits.adjust(L, tokens=T, length=N[:2]), ValueError, "length"),
    (lambda: logits.adjust(L, repetition=S), ValueError, "repetition"),
    (lambda: logits.adjust(L, tokens=T, length=N, presence=S.half()), TypeError, "presence"),
    (lambda: logits.adjust(L, bias_id=T), ValueError, "belong together"),
    (lambda: logits.adjust(L, bias_id=T, bias=torch.zeros(3, 8)), ValueError, "bias"),
    (lambda: logits.adjust(L, bias_id=torch.zeros(3, 1025, dtype=torch.int32), bias=torch.zeros(3, 1025)), ValueError, "bias_id"),
    (lambda: logits.adjust(L, allowed=torch.zeros(3, 3, dtype=torch.int32)), ValueError, "allowed"),
    (lambda: logits.adjust(L, allowed=torch.zeros(3, 4)), TypeError, "allowed"),
])
def test_logits_calls_refuse(call, error, word):
    with pytest.raises(error, match=word):
        call()


def prefix_args(**change):
    a = dict(q=A[0], q_row=256, q_head=64, out=A[1], out_row=256, out_head=64, lse=A[2], kv=A[3], kv_scale=A[4], n_pages=8, page_size=16,
             kv_heads=2, head_dim=64, heads=4, type=0, block_table=A[5], table_cols=4, n_req=2, q_start=A[6], kv_len=A[7], rows=3,
             max_q=2, max_kv=60, window=0, scale=0.125, workspace=A[12], workspace_bytes=1 << 20)
    p = dict(prefix_table=A[8], prefix_len=A[9], group_start=A[10], prefix_cols=4, n_groups=2, max_prefix=60)
    assert set(change) <= {*a, *p}
    own = _lib.Kv8AttentionArgs(**{k: change.get(k, v) for k, v in a.items()})
    return _lib.Kv8PrefixArgs(own, **{k: change.get(k, v) for k, v in p.items()})


@pytest.mark.parametrize("change,words", [
    (dict(page_size=48), ("page_size",)), (dict(head_dim=32), ("head_dim",)), (dict(heads=5), ("multiple",)), (dict(n_req=9000), ("n_req",)),
    (dict(max_kv=-1), ("negative",)), (dict(window=5), ("window",)), (dict(n_groups=-1), ("n_groups",)), (dict(n_groups=9000), ("n_groups",)),
    (dict(prefix_cols=-1), ("negative",)), (dict(max_prefix=-1), ("negative",)), (dict(rows=2**31 - 70000), ("rows",)),
    (dict(q=None), ("null",)), (dict(block_table=None), ("null",)), (dict(prefix_table=None), ("null",)), (dict(prefix_len=None), ("null",)),
    (dict(group_start=None), ("null",)), (dict(kv=A[3] + 4), ("aligned",)), (dict(q=A[0] + 2), ("aligned",)),
    (dict(prefix_table=A[8] + 2), ("prefix_table", "aligned")), (dict(prefix_len=A[9] + 1), ("prefix_len", "aligned")),
    (dict(group_start=A[10] + 2), ("group_start", "aligned")), (dict(workspace=None), ("workspace",)), (dict(workspace=A[12] + 8), ("workspace",)),
    (dict(workspace_bytes=100), ("workspace",)), (dict(out=A[0] + 4), ("out", "q itself")), (dict(out=A[0], out_row=320), ("out", "q itself")),
    (dict(out_row=0), ("vectors of out overlap",)),
    *[(dict(out=A[i]), ("out", n)) for i, n in ((3, "kv"), (4, "kv_scale"), (5, "block_table"), (6, "q_start"), (7, "kv_len"), (8, "prefix_table"),
                                                (9, "prefix_len"), (10, "group_start"))],
    *[(dict(lse=A[i]), ("lse", n)) for i, n in ((0, "q"), (1, "out"), (8, "prefix_table"), (9, "prefix_len"), (10, "group_start"))],
    *[(dict(workspace=A[i]), ("workspace", n)) for i, n in ((0, "q"), (1, "out"), (5, "block_table"), (8, "prefix_table"), (10, "group_start"))],
])
def test_prefix_attention_refuses(lib, change, words):
    refused(lib, lib.h2c_kv8_prefix_attention(C.byref(prefix_args(**change)), None), "h2c_kv8_prefix_attention", *words)


def test_prefix_attention_of_nothing_and_its_workspace(lib):
    assert lib.h2c_kv8_prefix_attention(None, None) == _lib.ERR_INVALID
    refused(lib, lib.h2c_kv8_prefix_attention(C.byref(prefix_args(type=3)), None), "h2c_kv8_prefix_attention", code=_lib.ERR_BAD_TYPE)
    for change in (dict(n_req=0), dict(rows=0), dict(max_q=0)):
        assert lib.h2c_kv8_prefix_attention(C.byref(prefix_args(q=None, **change)), None) == _lib.OK
        assert lib.h2c_kv8_prefix_attention_workspace(C.byref(prefix_args(**change))) == 0
    need = lib.h2c_kv8_prefix_attention_workspace(C.byref(prefix_args()))
    assert 0 < need < 1 << 20
    assert lib.h2c_kv8_prefix_attention_workspace(C.byref(prefix_args(n_groups=0))) < need
    refused(lib, lib.h2c_kv8_prefix_attention(C.byref(prefix_args(workspace_bytes=need - 1)), None), "h2c_kv8_prefix_attention", str(need))


KV, KS, I = torch.zeros(8, 2, 2, 16, 64, dtype=torch.int8), torch.zeros(8, 2, 2), torch.zeros(9, dtype=torch.int32)


@pytest.mark.parametrize("change,error,word", [
    ({}, ValueError, "CUDA"), (dict(ptable=I[:2]), ValueError, "prefix_table"), (dict(ptable=I.view(3, 3)), ValueError, "prefix_table"),
    (dict(ptable=I[:8].view(2, 4).long()), TypeError, "prefix_table"), (dict(plen=I[:2].long()), TypeError, "prefix_len"),
    (dict(gs=I[:2]), ValueError, "group_start"), (dict(q=Q.long()), TypeError, "q:"), (dict(max_prefix=2**31), ValueError, "32 bits"),
    (dict(table=I[:2]), ValueError, "block_table"), (dict(out=Q[:2]), ValueError, "out"),
])
def test_prefix_attention_calls_refuse(change, error, word):
    a = {**dict(q=Q, kv=KV, sc=KS, ptable=I[:8].view(2, 4), plen=I[:2], gs=I[:3], table=I[:8].view(2, 4), q_start=I[:3], kv_len=I[:2], max_q=2,
                max_kv=60, max_prefix=60), **change}
    with pytest.raises(error, match=word):
        kv8.prefix_attention(*[v for k, v in a.items() if k != "out"], out=a.get("out"))
