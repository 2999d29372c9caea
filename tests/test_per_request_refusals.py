"""The adapters' and the sampler's C entry points refuse malformed calls on the host, before any device
work, with the library's error cases (no GPU)."""
import ctypes

import pytest

from splosh_amd import _lib

A, B, R, S, X, OUT, SLOTS, WS = (ctypes.c_void_p(0x10000 * i) for i in range(1, 9))


def adapters(**change):
    base = dict(a=A, b=B, ranks=R, scales=S, count=3, max_rank=16, rows=128, inner=64, a_slot_stride=16 * 64,
                a_row_stride=64, b_slot_stride=128 * 16, b_row_stride=16)
    base.update(change)
    return _lib.Adapters(*[base[name] for name, _ in _lib.Adapters._fields_])


def add(w, x=X, ldx=64, out=OUT, ldc=128, dtype=_lib.BF16, slots=SLOTS, rows=4, ws=WS, ws_bytes=1 << 30):
    st = _lib.lib().splosh_adapters_add(ctypes.byref(w), x, ldx, out, ldc, dtype, slots, rows, ws, ws_bytes, None)
    return _lib.STATUS_NAMES.get(st, st)


@pytest.mark.parametrize("change,case", [
    ({"a": None}, "nullPointer"), ({"b": None}, "nullPointer"), ({"count": 0}, "invalidShape"),
    ({"max_rank": 0}, "invalidShape"), ({"rows": -1}, "invalidShape"), ({"inner": 0}, "invalidShape"),
    ({"max_rank": 257, "b_row_stride": 257}, "unsupported"), ({"a_row_stride": 63}, "invalidRowStride"),
    ({"b_row_stride": 15}, "invalidRowStride"), ({"a_slot_stride": -1}, "invalidRowStride"),
    ({"b_slot_stride": -1}, "invalidRowStride"), ({"count": 1 << 40}, "arithmeticOverflow"),
    ({"a_slot_stride": 1 << 62}, "arithmeticOverflow"), ({"b_row_stride": 1 << 62}, "arithmeticOverflow"),
    ({"a": ctypes.c_void_p(0x10001)}, "unsupported"), ({"ranks": ctypes.c_void_p(0x10002)}, "unsupported"),
])
def test_adapters_weight(change, case):
    assert add(adapters(**change)) == case


@pytest.mark.parametrize("change,case", [
    ({"x": None}, "nullPointer"), ({"out": None}, "nullPointer"), ({"slots": None}, "nullPointer"),
    ({"rows": 0}, "invalidShape"), ({"ldx": 63}, "invalidShape"), ({"ldc": 127}, "invalidShape"),
    ({"dtype": 2}, "unsupported"), ({"ws": None}, "workspaceTooSmall"), ({"ws_bytes": 16384}, "workspaceTooSmall"),
    ({"ws": ctypes.c_void_p(0x80008)}, "workspaceTooSmall"), ({"out": ctypes.c_void_p(0x60001)}, "unsupported"),
    ({"dtype": _lib.F32, "out": ctypes.c_void_p(0x60002)}, "unsupported"), ({"slots": ctypes.c_void_p(0x70002)}, "unsupported"),
    ({"rows": 1 << 40, "ws_bytes": 1 << 62}, "unsupported"), ({"rows": 1 << 62}, "arithmeticOverflow"),
])
def test_adapters_call(change, case):
    assert add(adapters(), **change) == case


def test_adapters_group():
    lib = _lib.lib()

    def group(ws, outs, ldcs, count=None):
        n = len(ws)
        return _lib.STATUS_NAMES.get(lib.splosh_adapters_add_group(
            (_lib.Adapters * n)(*ws), n if count is None else count, X, 128, (ctypes.c_void_p * n)(*outs),
            (ctypes.c_int64 * n)(*ldcs), _lib.F32, SLOTS, 4, WS, 1 << 30, None))

    other = adapters(inner=128, a_row_stride=128)
    assert group([adapters(), other], [0x10000, 0x20000], [128, 128]) == "invalidShape"
    assert group([adapters(), adapters()], [0x10000, 0x10000], [128, 128]) == "layoutMismatch"
    assert group([adapters()], [0x10000], [128], count=0) == "invalidShape"
    assert group([adapters()], [0x10000], [128], count=9) == "invalidShape"
    assert lib.splosh_adapters_add_group(None, 1, X, 64, None, None, 0, SLOTS, 1, WS, 1, None) == 12
    assert lib.splosh_adapters_workspace_bytes(None, 1, 4) == 0
    assert lib.splosh_adapters_workspace_bytes(ctypes.byref(adapters()), 0, 4) == 0
    assert lib.splosh_adapters_workspace_bytes(ctypes.byref(adapters()), 1, 0) == 0
    assert lib.splosh_adapters_workspace_bytes(ctypes.byref(adapters()), 1, 4) >= 16384 + 4 * 16 * 4


LOGITS, U, T, K, P, Q, TOK, LP = (ctypes.c_void_p(0x10000 * i) for i in range(1, 9))


def sample(logits=LOGITS, ld=1000, dtype=_lib.F32, rows=4, vocab=1000, u=U, t=T, k=K, p=P, q=Q, tokens=TOK, logprobs=LP,
           ws=WS, ws_bytes=1 << 40):
    st = _lib.lib().splosh_sample(logits, ld, dtype, rows, vocab, u, t, k, p, q, tokens, logprobs, ws, ws_bytes, None)
    return _lib.STATUS_NAMES.get(st, st)


@pytest.mark.parametrize("change,case", [
    ({"logits": None}, "nullPointer"), ({"tokens": None}, "nullPointer"), ({"rows": 0}, "invalidShape"),
    ({"vocab": 0}, "invalidShape"), ({"ld": 999}, "invalidRowStride"), ({"dtype": 7}, "unsupported"),
    ({"vocab": (1 << 21) + 1, "ld": 1 << 24}, "unsupported"), ({"rows": 1 << 40, "ld": 1 << 40}, "arithmeticOverflow"),
    ({"rows": 1 << 40}, "unsupported"),
    ({"logits": ctypes.c_void_p(0x10002)}, "unsupported"), ({"u": ctypes.c_void_p(0x10002)}, "unsupported"),
    ({"logprobs": ctypes.c_void_p(0x10002)}, "unsupported"), ({"k": ctypes.c_void_p(0x10001)}, "unsupported"),
    ({"ws": None}, "workspaceTooSmall"), ({"ws_bytes": 100}, "workspaceTooSmall"),
    ({"ws": ctypes.c_void_p(0x80008)}, "workspaceTooSmall"),
])
def test_sample_call(change, case):
    assert sample(**change) == case


def test_sample_workspace():
    size = _lib.lib().splosh_sample_workspace_bytes
    assert size(0, 10) == 0 and size(1, 0) == 0 and size(1, (1 << 21) + 1) == 0
    assert size(1, 1) >= 16384 and size(64, 248320) >= size(1, 248320)
