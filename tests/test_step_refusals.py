"""The C entry points of a packed step's attention layers and of its drafted tokens refuse malformed calls on the host,
before any device work, with the library's error cases; and where rows and pages lie that are none (no GPU)."""
import ctypes
import subprocess
from pathlib import Path

import pytest

import test_mma_waitcounts as wc
from splosh_amd import _lib

P = [ctypes.c_void_p(0x10000 * i) for i in range(1, 12)]
ODD = ctypes.c_void_p(0x10001)


def fields(cls, base, change):
    base.update(change)
    return cls(*[base[name] for name, _ in cls._fields_])


def cache(**change):
    return fields(_lib.Cache, dict(data=P[0], pages=10, page_stride=4 * (64 * 128 + 256) * 2, page_tokens=64, heads=4, dim=128), change)


def packed(**change):
    return fields(_lib.Packed, dict(starts=P[1], lengths=P[2], table=P[3], requests=3, table_stride=5, table_pages=5), change)


def heads(**change):
    return fields(_lib.Heads, dict(x=P[4], row_stride=512, head_stride=128, heads=4, weight=None, out=None, ld_out=0), change)


def queries(**change):
    return heads(**{**dict(x=P[5], row_stride=1024, heads=8, out=P[6], ld_out=1024), **change})


def at(x):
    """The address of a struct."""
    return ctypes.addressof(x) if isinstance(x, ctypes.Structure) else x


def name(st):
    return _lib.STATUS_NAMES.get(st, st)


def write(c=None, p=None, k=None, v=None, q=None, dtype=_lib.BF16, rows=7, frequencies=P[7], rotary=64):
    args = (c or cache(), p or packed(), k or heads(), v or heads(), q or queries())
    return name(_lib.lib().splosh_cache_write(*map(at, args), dtype, rows,
                                              frequencies, rotary, 1e-6, None))


def read(c=None, p=None, rows=7, k=P[4], ldk=512, v=P[5], ldv=512):
    args = (c or cache(), p or packed())
    return name(_lib.lib().splosh_cache_read(*map(at, args), rows, k, ldk, v, ldv, None))


def attend(c=None, p=None, q=P[5], row=1024, head=128, heads=8, rows=7, shared=64, scale=0.1, out=P[6], ld=1024, ws=P[8],
           ws_bytes=1 << 40):
    args = (c or cache(), p or packed())
    return name(_lib.lib().splosh_attend(q, row, head, heads, *map(at, args), rows, shared, scale, out, ld, ws, ws_bytes, None))


@pytest.mark.parametrize("change,case", [
    ({"data": None}, "nullPointer"), ({"data": ODD}, "unsupported"), ({"pages": 0}, "invalidShape"), ({"heads": -1}, "invalidShape"),
    ({"dim": 0}, "invalidShape"), ({"dim": 96}, "unsupported"), ({"page_tokens": 48}, "unsupported"), ({"heads": 2000}, "unsupported"),
    ({"page_stride": 4 * (64 * 128 + 256) * 2 - 16}, "invalidRowStride"), ({"page_stride": 4 * (64 * 128 + 256) * 2 + 8}, "invalidRowStride"),
    ({"pages": 1 << 31}, "arithmeticOverflow"), ({"page_stride": 1 << 62}, "arithmeticOverflow")])
def test_caches(change, case):
    for call in (write, read, attend):
        assert call(c=cache(**change)) == case


@pytest.mark.parametrize("change,case", [
    ({"starts": None}, "nullPointer"), ({"lengths": None}, "nullPointer"), ({"table": None}, "nullPointer"), ({"requests": 0}, "invalidShape"),
    ({"table_pages": 0}, "invalidShape"), ({"requests": 65536}, "unsupported"), ({"table_stride": 4}, "invalidRowStride"),
    ({"table_stride": 1 << 62}, "arithmeticOverflow"), ({"table_pages": 1 << 25, "table_stride": 1 << 25}, "unsupported"),
    ({"starts": ODD}, "unsupported"), ({"table": ODD}, "unsupported")])
def test_steps(change, case):
    for call in (write, read, attend):
        assert call(p=packed(**change)) == case


@pytest.mark.parametrize("call,case", [
    (lambda: write(rows=0), "invalidShape"), (lambda: write(rows=1 << 23), "unsupported"), (lambda: write(dtype=5), "unsupported"),
    (lambda: write(rotary=130), "invalidShape"), (lambda: write(rotary=7), "invalidShape"), (lambda: write(rotary=-2), "invalidShape"),
    (lambda: write(frequencies=None), "nullPointer"), (lambda: write(frequencies=ODD), "unsupported"),
    (lambda: write(k=heads(x=None)), "nullPointer"), (lambda: write(v=heads(x=None)), "nullPointer"),
    (lambda: write(k=heads(out=P[9])), "layoutMismatch"), (lambda: write(v=heads(weight=P[9])), "layoutMismatch"),
    (lambda: write(k=heads(heads=3)), "invalidShape"), (lambda: write(v=heads(heads=0)), "invalidShape"),
    (lambda: write(k=heads(row_stride=100)), "invalidRowStride"), (lambda: write(k=heads(head_stride=127)), "invalidRowStride"),
    (lambda: write(k=heads(row_stride=1 << 62)), "arithmeticOverflow"), (lambda: write(k=heads(x=ODD)), "unsupported"),
    (lambda: write(k=heads(x=ctypes.c_void_p(0x10002)), dtype=_lib.F32), "unsupported"),
    (lambda: write(q=queries(out=None)), "nullPointer"), (lambda: write(q=queries(ld_out=1000)), "invalidRowStride"),
    (lambda: write(q=queries(heads=0)), "invalidShape"), (lambda: write(q=queries(weight=ODD)), "unsupported"),
    (lambda: read(rows=0), "invalidShape"), (lambda: read(k=None, v=None), "nullPointer"), (lambda: read(ldk=511), "invalidRowStride"),
    (lambda: read(ldv=1 << 62), "arithmeticOverflow"), (lambda: read(k=P[5]), "layoutMismatch"), (lambda: read(v=ODD), "unsupported"),
    (lambda: attend(q=None), "nullPointer"), (lambda: attend(out=None), "nullPointer"), (lambda: attend(rows=-1), "invalidShape"),
    (lambda: attend(heads=6, ld=1024), "invalidShape"), (lambda: attend(heads=0), "invalidShape"), (lambda: attend(row=100), "invalidRowStride"),
    (lambda: attend(head=64), "invalidRowStride"), (lambda: attend(ld=1000), "invalidRowStride"), (lambda: attend(shared=32), "invalidShape"),
    (lambda: attend(shared=-64), "invalidShape"), (lambda: attend(shared=64 * 6), "invalidShape"), (lambda: attend(scale=0.0), "invalidShape"),
    (lambda: attend(scale=float("nan")), "invalidShape"), (lambda: attend(scale=float("inf")), "invalidShape"),
    (lambda: attend(ws=None), "workspaceTooSmall"), (lambda: attend(ws_bytes=16383), "workspaceTooSmall"),
    (lambda: attend(ws=ctypes.c_void_p(0x10008)), "workspaceTooSmall"), (lambda: attend(q=ODD), "unsupported")])
def test_calls(call, case):
    assert call() == case


@pytest.mark.parametrize("change,case", [
    ({"parts": None}, "nullPointer"), ({"count": 0}, "invalidShape"), ({"count": 9}, "invalidShape"), ({"dim": 192}, "unsupported"),
    ({"rows": 0}, "invalidShape"), ({"positions": None}, "nullPointer"), ({"positions": ODD}, "unsupported"),
    ({"frequencies": None}, "nullPointer"), ({"rotary": 129}, "invalidShape"), ({"same": True}, "layoutMismatch"), ({"dtype": 3}, "unsupported")])
def test_rotation(change, case):
    a = dict(count=2, dtype=_lib.BF16, rows=5, dim=128, positions=P[7], frequencies=P[8], rotary=64)
    same = change.pop("same", False)
    listed = (_lib.Heads * 2)(queries(), queries(x=P[4], out=P[6] if same else P[9]))
    parts = change.pop("parts", ctypes.addressof(listed))
    a.update(change)
    assert name(_lib.lib().splosh_rotate_heads(parts, a["count"], a["dtype"], a["rows"], a["dim"], a["positions"], a["frequencies"],
                                               a["rotary"], 1e-6, None)) == case


@pytest.mark.parametrize("change,case", [
    ({"logits": None}, "nullPointer"), ({"tokens": None}, "nullPointer"), ({"starts": None}, "nullPointer"), ({"u": None}, "nullPointer"),
    ({"out": None}, "nullPointer"), ({"accepted": None}, "nullPointer"), ({"rows": 0}, "invalidShape"), ({"vocab": 0}, "invalidShape"),
    ({"requests": 0}, "invalidShape"), ({"ld": 999}, "invalidRowStride"), ({"ldd": 999}, "invalidRowStride"), ({"dtype": 4}, "unsupported"),
    ({"ddtype": 4}, "unsupported"), ({"vocab": (1 << 21) + 1, "ld": 1 << 22, "ldd": 1 << 22}, "unsupported"), ({"rows": 65536}, "unsupported"),
    ({"requests": 65536}, "unsupported"), ({"ld": 1 << 62}, "arithmeticOverflow"), ({"logits": ODD}, "unsupported"), ({"out": ODD}, "unsupported"),
    ({"out": P[2]}, "layoutMismatch"), ({"accepted": P[5]}, "layoutMismatch"), ({"out": ctypes.c_void_p(0x30000 - 4 * 7)}, "layoutMismatch"),
    ({"out": ctypes.c_void_p(0x30000 + 4 * 7)}, "layoutMismatch"), ({"accepted": ctypes.c_void_p(0x40000 + 4 * 2)}, "layoutMismatch"), ({"ws": None}, "workspaceTooSmall"), ({"ws_bytes": 16400}, "workspaceTooSmall")])
def test_verification(change, case):
    a = dict(logits=P[0], ld=1000, dtype=_lib.F32, rows=8, vocab=1000, tokens=P[2], starts=P[3], requests=2, u=P[4], t=P[7], draft=P[1], ldd=1000,
             ddtype=_lib.F32, out=P[5], accepted=P[6], ws=P[8], ws_bytes=1 << 30)
    a.update(change)
    assert name(_lib.lib().splosh_verify(*a.values(), None)) == case


def test_sizes():
    lib = _lib.lib()
    assert lib.splosh_cache_page_bytes(4, 256, 256) == 4 * 8 * (64 * 256 + 256)
    assert [lib.splosh_cache_page_bytes(*a) for a in ((0, 64, 32), (1, 65, 32), (1, 64, 33), (1, 64, 0))] == [0] * 4
    c, p = cache(), packed()
    assert lib.splosh_attend_workspace_bytes(at(c), at(p), 7, 6, 0) == 0 and lib.splosh_attend_workspace_bytes(at(c), at(p), 0, 8, 0) == 0
    assert lib.splosh_attend_workspace_bytes(None, at(p), 7, 8, 0) == 0 and lib.splosh_verify_workspace_bytes(1, 1 << 22, 1) == 0
    assert lib.splosh_attend_workspace_bytes(at(c), at(p), 7, 8, 0) >= 16384 <= lib.splosh_verify_workspace_bytes(8, 1000, 2)


PLACES = """
#include "cache.hpp"
#include <cstdio>
using namespace splosh;
int main() {
    // 5 pages; three columns a request in rows of four.
    const int32_t table[] = {0, 4, 5, 99, -1, 3, 2147483647, 99};
    const CacheView cache{nullptr, 0, 5, 64, 2, 1};
    const PackedView packed{nullptr, nullptr, table, 4, 3, 2, 0};
    const int positions[] = {-2147483648, -1, 0, 63, 64, 127, 128, 191, 192, 2147483647};
    for (int request = -1; request < 2; ++request)
        for (int p : positions) {
            int page = -7, at = -7;
            const bool found = place_of(cache, packed, request, p, page, at);
            printf("%d %d %d %d %d\\n", request, p, (int)found, found ? page : 0, found ? at : 0);
        }
}
"""


@pytest.mark.skipif(not Path(wc.HIPCC).exists(), reason="needs hipcc")
def test_places(tmp_path):
    """A position's page and place: none for a request or position below 0, past the table, or of a page that is none."""
    source, program = tmp_path / "places.cpp", tmp_path / "places"
    source.write_text(PLACES)
    subprocess.run([wc.HIPCC, "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", f"-I{wc.ROOT / 'include'}", f"-I{wc.ROOT / 'splosh_amd/csrc'}",
                    str(source), "-o", str(program)], check=True, capture_output=True)
    table = {0: [0, 4, 5], 1: [-1, 3, 2147483647]}
    for line in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines():
        request, p, found, page, at = map(int, line.split())
        want = table[request][p // 64] if request >= 0 and 0 <= p < 192 else -1
        assert (found, page, at) == ((1, want, p % 64) if 0 <= want < 5 else (0, 0, 0)), line
