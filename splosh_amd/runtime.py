"""Operator entry points of the q4 / Q5_K path on torch device tensors.

PyTorch-ROCm supplies device memory and streams only; every computation is a call into
libsplosh_q4.so through its C ABI. The names follow the reference's host API:

* ``Q4GemmRuntime.dispatch`` -- Runtime/Q4Runtime.swift:94-145 (gemm_q4, fp32 out, synchronous).
* ``Engine.gemm`` / ``Engine.mlp_in`` -- Runtime/Engine.swift:1652, :1911 (stream-ordered).
* ``dequant``, ``tile128``, ``q5k_repack`` -- DequantOracle.dequantize, Converter.tile,
  GgufPlanes.repack on the device.
* ``add_adapters`` / ``sample`` -- what differs between the requests of a packed step: low-rank
  adapters beside a projection, and the choice of each row's next token.
* ``rotate_heads`` / ``cache_write`` / ``cache_read`` / ``attend`` -- a packed step's attention layers between their
  projections: norms and rotation of the heads, the 8-bit paged cache, attention over it.
* ``verify`` -- the drafted tokens of a verify step against the target's probabilities.

Buffer-size checks (GemmQ4Error.bufferTooSmall) happen here because the C ABI sees raw pointers.
"""
import contextlib
import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import GemmQ4Error, SploshError
from .quant import GROUP_SIZE, TILE_ROWS, GemmQ4Shape, Q4BufferLayout

AUTO = _lib.KERNEL_AUTO
STREAM = _lib.KERNEL_STREAM
DEQUANT = _lib.KERNEL_DEQUANT
TILE = _lib.KERNEL_TILE
SCALAR = _lib.KERNEL_SCALAR
PREFILL = _lib.KERNEL_PREFILL
ROW_MAJOR = _lib.ROW_MAJOR
TILED128 = _lib.TILED128
# The start of a workspace the kernels need zeroed before its first use (their arrival counters).
WORKSPACE_COUNTER_BYTES = 16384


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _stream(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _require(t, nbytes, name):
    # The bytes the pointer may address: to the end of the tensor's storage (a strided view of a
    # larger buffer reaches past its own elements).
    have = t.untyped_storage().nbytes() - t.storage_offset() * t.element_size()
    if have < nbytes:
        raise GemmQ4Error(8, f"bufferTooSmall(name: {name}, expected: {nbytes}, observed: {have})")
    if not t.is_cuda:
        raise SploshError(12, f"{name} is not a device tensor")


def _dtype_code(dtype):
    if dtype == torch.float32:
        return _lib.F32
    if dtype == torch.bfloat16:
        return _lib.BF16
    raise SploshError(13, f"unsupported output dtype {dtype}")


@dataclass
class Q4Weight:
    """A resident MLX affine q4 weight (the reference's Q4Handle): int32 packed words, bf16 scale
    and bias sidecars (as int16 or bfloat16 tensors), `rows` outputs x `inner` inputs."""

    packed: torch.Tensor
    scales: torch.Tensor
    biases: torch.Tensor
    rows: int
    inner: int
    order: int = TILED128
    row_stride_words: int = 0

    def __post_init__(self):
        groups = (self.inner + GROUP_SIZE - 1) // GROUP_SIZE
        if self.order == TILED128:
            words = self.rows * groups * 8
        else:
            if self.row_stride_words == 0:
                self.row_stride_words = ((self.inner + 7) // 8 * 4 + 127) // 128 * 32
            words = self.rows * self.row_stride_words
        _require(self.packed, words * 4, "packed")
        _require(self.scales, self.rows * groups * 2, "scales")
        _require(self.biases, self.rows * groups * 2, "biases")

    def c(self):
        return _lib.Q4Weight(self.packed.data_ptr(), self.scales.data_ptr(), self.biases.data_ptr(), self.rows,
                             self.inner, self.row_stride_words, self.order, 0)

    @property
    def nbytes(self):
        """Algorithmic bytes: N K / 2 codes + N (K / 64) * 4 sidecar bytes."""
        return self.rows * self.inner // 2 + self.rows * (self.inner // GROUP_SIZE) * 4


@dataclass
class Q5KWeight:
    """A GGUF Q5_K weight in plane form (Model/GgufPlanes.swift:8-20)."""

    plane0: torch.Tensor
    plane1: torch.Tensor
    meta: torch.Tensor
    rows: int
    inner: int

    def __post_init__(self):
        groups = self.inner // 32
        _require(self.plane0, self.rows * groups * 16, "plane0")
        _require(self.plane1, self.rows * groups * 4, "plane1")
        _require(self.meta, self.rows * (self.inner // 256) * 16, "meta")

    def c(self):
        return _lib.Q5KWeight(self.plane0.data_ptr(), self.plane1.data_ptr(), self.meta.data_ptr(), self.rows,
                              self.inner)

    @property
    def nbytes(self):
        return self.rows * (self.inner // 256) * 176


@dataclass
class Q4KWeight:
    """A GGUF Q4_K weight in plane form (GgufPlanes.swift:64: plane0 and meta, no plane1)."""

    plane0: torch.Tensor
    meta: torch.Tensor
    rows: int
    inner: int

    def __post_init__(self):
        _require(self.plane0, self.rows * (self.inner // 32) * 16, "plane0")
        _require(self.meta, self.rows * (self.inner // 256) * 16, "meta")

    def c(self):
        return _lib.Q5KWeight(self.plane0.data_ptr(), None, self.meta.data_ptr(), self.rows, self.inner)

    @property
    def nbytes(self):
        return self.rows * (self.inner // 256) * 144


def _on(stream):
    """The stream a call's kernels run on (the caller's, else torch's current one)."""
    return stream if stream is not None else torch.cuda.current_stream()


def _allocating(stream):
    """The context a call's own tensors are allocated in: the stream the kernel uses them from, so
    torch's caching allocator orders any reuse of the block after that kernel. Nothing to enter when
    that is torch's current stream already (entering it costs a small call 4 us)."""
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _out(a, rows, n, out, out_dtype, stream=None):
    if out is None:
        with _allocating(stream):
            out = torch.empty((rows, n), dtype=out_dtype, device=a.device)
    return out


# ggml type id -> (block elements, block bytes) of the formats kept in native blocks
# (GgufQuant.swift:13-48): Q8_0, Q3_K, Q6_K, IQ4_NL, IQ3_S, IQ4_XS.
GGUF_NATIVE = {8: (32, 34), 11: (256, 110), 14: (256, 210), 20: (32, 18), 21: (256, 110), 23: (256, 136)}


# splosh_gguf_gemm's layout flag: the ROWS32 order of the native blocks (splosh_gguf_repack_rows32).
GGUF_ROWS32 = 0x100


@dataclass
class GgufWeight:
    """A GGUF weight in native blocks (rows x inner): in the order its file holds them (rows back to
    back), or with rows32=True in the ROWS32 order of gguf_repack_rows32 (the units of 256
    elements of 32 consecutive rows interleaved, rows padded to a multiple of 32)."""

    native: torch.Tensor
    gguf_type: int
    rows: int
    inner: int
    rows32: bool = False

    def __post_init__(self):
        if self.gguf_type not in GGUF_NATIVE:
            raise SploshError(13, f"ggml type {self.gguf_type} is not kept in native blocks")
        elems, size = GGUF_NATIVE[self.gguf_type]
        stored = (self.rows + 31) // 32 * 32 if self.rows32 else self.rows
        _require(self.native, stored * (self.inner // elems) * size, "native")

    @property
    def type_id(self):
        """The type id the entry points take: the ggml id, with the layout flag for ROWS32."""
        return self.gguf_type | (GGUF_ROWS32 if self.rows32 else 0)


def gguf_repack_rows32(w, stream=None):
    """splosh_gguf_repack_rows32: the same weight in the ROWS32 order (a new device tensor)."""
    if w.rows32:
        raise SploshError(2, "the weight is already in the ROWS32 order")
    nbytes = _lib.lib().splosh_gguf_rows32_bytes(w.gguf_type, w.rows, w.inner)
    if nbytes == 0:
        raise SploshError(2, "no ROWS32 form for this type or shape (inner % 256 != 0)")
    out = torch.empty(nbytes, dtype=torch.uint8, device=w.native.device)
    _lib.check(_lib.lib().splosh_gguf_repack_rows32(w.gguf_type, _ptr(w.native), w.rows, w.inner, _ptr(out),
                                                    _stream(stream)))
    return GgufWeight(out, w.gguf_type, w.rows, w.inner, rows32=True)


def workspace_bytes(rows, columns, inner):
    """splosh_workspace_bytes: the split-K scratch the kernels can use for this shape (0: none)."""
    return _lib.lib().splosh_workspace_bytes(rows, columns, inner)


def heads_workspace_bytes(rows, columns, inner):
    """splosh_heads_workspace_bytes: the workspace a head-ordered GGUF GEMM needs."""
    return _lib.lib().splosh_heads_workspace_bytes(rows, columns, inner)


class _Scratch:
    """The split-K scratch of one call: (pointer, bytes), and the tensor that owns it, held by the
    caller until the kernel has been launched."""

    def __init__(self, ptr, nbytes, owner=None):
        self.ptr, self.nbytes, self.owner = ptr, nbytes, owner

    def __iter__(self):
        return iter((self.ptr, self.nbytes))


def _workspace(workspace, rows, n, inner, device, stream=None, heads=False, q4=None):
    """The split-K scratch of the kernels: the caller's tensor (an empty one: none), or a fresh one
    from torch's stream-ordered allocator sized by splosh_workspace_bytes, or, for a q4 call under
    AUTO (``q4``: the weight, the row stride and the pair flag), by splosh_q4_workspace_bytes: a
    5 MB fill that the one-row kernels never look at, and entering the current stream twice, were
    two thirds of the smallest eager call (K5120 -> N1024, one row 35.4 -> 12.8 us with both gone).
    The counters of a fresh one are zeroed; it is allocated on the stream the kernel runs on, so
    the fill is ordered before the
    kernel; the caller keeps the returned object (and with it the tensor) until the kernel has
    been launched, after which the allocator hands the block out again only to work ordered after
    that kernel on the same stream."""
    if workspace is not None and workspace.numel() == 0:
        return _Scratch(None, 0)
    if workspace is not None:
        return _Scratch(_ptr(workspace), workspace.numel() * workspace.element_size(), workspace)
    if q4 is not None:
        weight, lda, pair = q4
        need = _lib.lib().splosh_q4_workspace_bytes(ctypes.byref(weight), lda, rows, pair)
    else:
        need = (_lib.lib().splosh_heads_workspace_bytes if heads else _lib.lib().splosh_workspace_bytes)(rows, n, inner)
    if need == 0:
        return _Scratch(None, 0)
    with _allocating(stream):
        buf = torch.empty(need, dtype=torch.uint8, device=device)
        buf[:WORKSPACE_COUNTER_BYTES].zero_()
    return _Scratch(_ptr(buf), need, buf)


def gemm(w, a, out=None, residual=None, out_dtype=torch.bfloat16, kernel=AUTO, rows=None, stream=None,
         workspace=None, key_heads=0):
    """Engine.gemm (Runtime/Engine.swift:1652-1806): out = a @ dequant(w)^T (+ residual).

    ``a`` is bf16 [rows, inner] (row stride a.stride(0)); ``out`` [rows, w.rows] in fp32 or bf16;
    ``residual`` may be ``out`` itself. ``key_heads`` > 0 (GGUF weights only): the weight's inner
    columns are in a GGUF file's value-head order and the activations in the engine's (the `heads`
    kernels, engine_gguf.metal:55-72)."""
    rows = a.shape[0] if rows is None else rows
    if a.dtype != torch.bfloat16:
        raise SploshError(13, "activations must be bf16")
    if a.stride(-1) != 1:
        raise SploshError(1, "activation rows must be contiguous")
    out = _out(a, rows, w.rows, out, out_dtype, stream)
    _require(a, ((rows - 1) * a.stride(0) + w.inner) * 2, "a")
    _require(out, ((rows - 1) * out.stride(0) + w.rows) * out.element_size(), "output")
    if residual is not None:
        if residual.dtype != out.dtype or residual.stride(0) != out.stride(0):
            raise SploshError(13, "residual must match the output's dtype and row stride")
    if key_heads and isinstance(w, Q4Weight):
        raise SploshError(13, "the value-head order applies to GGUF weights only")
    is_q4 = isinstance(w, Q4Weight)
    wc = None if isinstance(w, GgufWeight) else w.c()
    scratch = _workspace(workspace, rows, w.rows, w.inner, a.device, stream, heads=bool(key_heads),
                         q4=(wc, a.stride(0), 0) if is_q4 and kernel == AUTO else None)
    ws, ws_bytes = scratch  # (scratch is held until the launch)
    if wc is None:
        if key_heads:
            st = _lib.lib().splosh_gguf_gemm_heads(w.type_id, _ptr(w.native), w.rows, w.inner, key_heads, _ptr(a),
                                                   a.stride(0), _ptr(out), out.stride(0), _dtype_code(out.dtype),
                                                   _ptr(residual), rows, ws, ws_bytes, _stream(stream))
        else:
            st = _lib.lib().splosh_gguf_gemm(w.type_id, _ptr(w.native), w.rows, w.inner, _ptr(a), a.stride(0),
                                             _ptr(out), out.stride(0), _dtype_code(out.dtype), _ptr(residual),
                                             rows, ws, ws_bytes, _stream(stream))
        _lib.check(st)
        return out
    if key_heads:
        fn = _lib.lib().splosh_q4k_gemm_heads if isinstance(w, Q4KWeight) else _lib.lib().splosh_q5k_gemm_heads
        _lib.check(fn(ctypes.byref(wc), key_heads, _ptr(a), a.stride(0), _ptr(out), out.stride(0),
                      _dtype_code(out.dtype), _ptr(residual), rows, kernel, ws, ws_bytes, _stream(stream)))
        return out
    if is_q4:
        st = _lib.lib().splosh_q4_gemm(ctypes.byref(wc), _ptr(a), a.stride(0), _ptr(out), out.stride(0),
                                       _dtype_code(out.dtype), _ptr(residual), rows, kernel, ws, ws_bytes,
                                       _stream(stream))
    else:
        fn = _lib.lib().splosh_q4k_gemm if isinstance(w, Q4KWeight) else _lib.lib().splosh_q5k_gemm
        st = fn(ctypes.byref(wc), _ptr(a), a.stride(0), _ptr(out), out.stride(0), _dtype_code(out.dtype),
                _ptr(residual), rows, kernel, ws, ws_bytes, _stream(stream))
    _lib.check(st)
    return out


def gemm_group(weights, a, outs=None, out_dtype=torch.bfloat16, kernel=AUTO, rows=None, stream=None,
               workspace=None):
    """Several projections of one activation in one launch (the reference's concurrent encoder of a
    layer's independent projections, Engine.swift:1402, 1131-1140): [a @ dequant(w)^T for w in
    weights], each in its own output. Returns the outputs."""
    rows = a.shape[0] if rows is None else rows
    if a.dtype != torch.bfloat16 or a.stride(-1) != 1:
        raise SploshError(13, "activations must be bf16 with contiguous rows")
    weights = list(weights)
    if outs is None:
        outs = [None] * len(weights)
    outs = [_out(a, rows, w.rows, o, out_dtype, stream) for w, o in zip(weights, outs)]
    _require(a, ((rows - 1) * a.stride(0) + weights[0].inner) * 2, "a")
    for w, o in zip(weights, outs):
        _require(o, ((rows - 1) * o.stride(0) + w.rows) * o.element_size(), "output")
        if o.dtype != outs[0].dtype:
            raise SploshError(13, "grouped outputs must share one dtype")
    scratch = _workspace(workspace, rows, sum(w.rows for w in weights), weights[0].inner, a.device, stream)
    ws, ws_bytes = scratch
    wcs = (_lib.Q4Weight * len(weights))(*[w.c() for w in weights])
    out_ptrs = (ctypes.c_void_p * len(outs))(*[_ptr(o) for o in outs])
    ldcs = (ctypes.c_int64 * len(outs))(*[o.stride(0) for o in outs])
    _lib.check(_lib.lib().splosh_q4_gemm_group(wcs, len(weights), _ptr(a), a.stride(0), out_ptrs, ldcs,
                                               _dtype_code(outs[0].dtype), rows, kernel, ws, ws_bytes,
                                               _stream(stream)))
    return outs


def gemm_emit(w, a, norm_weight, out=None, residual=None, kernel=AUTO, rows=None, stream=None, workspace=None):
    """Engine.gemm with emit (engine_na.metal:322-473): out = a @ dequant(w)^T (+ residual), fp32,
    and the next RMSNorm's operand from it: (bf16 out * norm_weight, per-64 sums of those values,
    per-64 sums of out^2). Returns (out, values, sums, squares)."""
    rows = a.shape[0] if rows is None else rows
    if a.dtype != torch.bfloat16 or a.stride(-1) != 1:
        raise SploshError(13, "activations must be contiguous bf16 rows")
    out = _out(a, rows, w.rows, out, torch.float32, stream)
    if out.dtype != torch.float32:
        raise SploshError(13, "the emitting projection writes fp32")
    _require(a, ((rows - 1) * a.stride(0) + w.inner) * 2, "a")
    _require(out, ((rows - 1) * out.stride(0) + w.rows) * 4, "output")
    if norm_weight.dtype != torch.bfloat16 or norm_weight.numel() < w.rows:
        raise SploshError(13, "norm_weight must be bf16 with one value a column")
    with _allocating(stream):
        values = torch.empty((rows, w.rows), dtype=torch.bfloat16, device=a.device)
        sums = torch.empty((rows, w.rows // 64), dtype=torch.float32, device=a.device)
        squares = torch.empty_like(sums)
    wc = w.c()
    scratch = _workspace(workspace, rows, w.rows, w.inner, a.device, stream)  # held until the launch
    ws, ws_bytes = scratch
    _lib.check(_lib.lib().splosh_q4_gemm_emit(ctypes.byref(wc), _ptr(a), a.stride(0), _ptr(out), out.stride(0),
                                              _ptr(residual), rows, _ptr(norm_weight), _ptr(values), values.stride(0),
                                              _ptr(sums), _ptr(squares), kernel, ws, ws_bytes, _stream(stream)))
    return out, values, sums, squares


def mlp_in(gate, up, a, out=None, out_dtype=torch.bfloat16, kernel=AUTO, rows=None, stream=None, workspace=None):
    """Engine.mlpIn (Runtime/Engine.swift:1911-1966): out = silu(a @ gate^T) * (a @ up^T), one
    pass over the activations for both weights."""
    rows = a.shape[0] if rows is None else rows
    if a.dtype != torch.bfloat16 or a.stride(-1) != 1:
        raise SploshError(13, "activations must be contiguous bf16 rows")
    out = _out(a, rows, gate.rows, out, out_dtype, stream)
    _require(a, ((rows - 1) * a.stride(0) + gate.inner) * 2, "a")
    _require(out, ((rows - 1) * out.stride(0) + gate.rows) * out.element_size(), "output")
    gc, uc = gate.c(), up.c()
    scratch = _workspace(workspace, rows, gate.rows, gate.inner, a.device, stream,
                         q4=(gc, a.stride(0), 1) if kernel == AUTO else None)
    ws, ws_bytes = scratch  # (scratch is held until the launch)
    st = _lib.lib().splosh_q4_mlp_in(ctypes.byref(gc), ctypes.byref(uc), _ptr(a), a.stride(0), _ptr(out),
                                     out.stride(0), _dtype_code(out.dtype), rows, kernel, ws, ws_bytes,
                                     _stream(stream))
    _lib.check(st)
    return out


def dequant(w, out=None, stream=None):
    """DequantOracle.dequantize / GgufTensorType.decode on the device: fp32 [rows, inner]."""
    if out is None:
        dev = (w.packed.device if isinstance(w, Q4Weight) else w.native.device if isinstance(w, GgufWeight)
               else w.plane0.device)
        out = torch.empty((w.rows, w.inner), dtype=torch.float32, device=dev)
    _require(out, w.rows * w.inner * 4, "output")
    if isinstance(w, GgufWeight):
        _lib.check(_lib.lib().splosh_gguf_dequant(w.type_id, _ptr(w.native), w.rows, w.inner, _ptr(out),
                                                  _stream(stream)))
        return out
    wc = w.c()
    fn = (_lib.lib().splosh_q4_dequant if isinstance(w, Q4Weight) else
          _lib.lib().splosh_q4k_dequant if isinstance(w, Q4KWeight) else _lib.lib().splosh_q5k_dequant)
    _lib.check(fn(ctypes.byref(wc), _ptr(out), _stream(stream)))
    return out


def tile128(src, rows, groups, element_bytes, inverse=False, out=None, stream=None):
    """Converter.tile (Model/Retile.swift:135-153) on the device (or its inverse)."""
    if out is None:
        out = torch.empty_like(src)
    nbytes = rows * groups * element_bytes
    _require(src, nbytes, "src")
    _require(out, nbytes, "dst")
    fn = _lib.lib().splosh_untile128 if inverse else _lib.lib().splosh_tile128
    _lib.check(fn(_ptr(src), _ptr(out), rows, groups, element_bytes, _stream(stream)))
    return out


def q4_to_tiled(w, stream=None):
    """A row-major (unpadded) q4 weight retiled to the 128-row layout the kernels prefer."""
    if w.order == TILED128:
        return w
    groups = w.inner // GROUP_SIZE
    if w.row_stride_words != w.inner // 8:
        packed = w.packed.view(w.rows, -1)[:, : w.inner // 8].contiguous()
    else:
        packed = w.packed
    tp = tile128(packed, w.rows, groups, 32, stream=stream)
    ts = tile128(w.scales, w.rows, groups, 2, stream=stream)
    tb = tile128(w.biases, w.rows, groups, 2, stream=stream)
    return Q4Weight(tp, ts, tb, w.rows, w.inner, TILED128)


def q5k_repack(native, rows, inner, stream=None):
    """GgufPlanes.repack for Q5_K on the device: native uint8 blocks -> Q5KWeight."""
    groups = inner // 32
    dev = native.device
    p0 = torch.empty(rows * groups * 16, dtype=torch.uint8, device=dev)
    p1 = torch.empty(rows * groups * 4, dtype=torch.uint8, device=dev)
    meta = torch.empty(rows * (inner // 256) * 16, dtype=torch.uint8, device=dev)
    _require(native, rows * (inner // 256) * 176, "native")
    _lib.check(_lib.lib().splosh_q5k_repack(_ptr(native), rows, inner, _ptr(p0), _ptr(p1), _ptr(meta),
                                            _stream(stream)))
    return Q5KWeight(p0, p1, meta, rows, inner)


def q5k_unpack(w, stream=None):
    native = torch.empty(w.rows * (w.inner // 256) * 176, dtype=torch.uint8, device=w.plane0.device)
    _lib.check(_lib.lib().splosh_q5k_unpack(_ptr(w.plane0), _ptr(w.plane1), _ptr(w.meta), w.rows, w.inner,
                                            _ptr(native), _stream(stream)))
    return native


def q4k_repack(native, rows, inner, stream=None):
    """GgufPlanes.repack for Q4_K on the device: native 144-byte blocks -> Q4KWeight."""
    dev = native.device
    p0 = torch.empty(rows * (inner // 32) * 16, dtype=torch.uint8, device=dev)
    meta = torch.empty(rows * (inner // 256) * 16, dtype=torch.uint8, device=dev)
    _require(native, rows * (inner // 256) * 144, "native")
    _lib.check(_lib.lib().splosh_q4k_repack(_ptr(native), rows, inner, _ptr(p0), _ptr(meta), _stream(stream)))
    return Q4KWeight(p0, meta, rows, inner)


def q4k_unpack(w, stream=None):
    native = torch.empty(w.rows * (w.inner // 256) * 144, dtype=torch.uint8, device=w.plane0.device)
    _lib.check(_lib.lib().splosh_q4k_unpack(_ptr(w.plane0), _ptr(w.meta), w.rows, w.inner, _ptr(native),
                                            _stream(stream)))
    return native


class Q4GemmRuntime:
    """Q4GemmRuntime (Runtime/Q4Runtime.swift:29-157): the oracle-grade gemm_q4 submission API."""

    def dispatch(self, shape: GemmQ4Shape, layout: Q4BufferLayout, a, packed, scales, biases, output, stream=None):
        """Validate, encode gemm_q4 (one thread per output), and wait (Q4Runtime.swift:94-145)."""
        shape.validate(layout)
        _require(a, shape.rows * shape.inner * 2, "a")
        _require(packed, layout.packed_word_count * 4, "packed")
        _require(scales, layout.sidecar_count * 2, "scales")
        _require(biases, layout.sidecar_count * 2, "biases")
        _require(output, shape.rows * shape.columns * 4, "output")
        st = _lib.lib().splosh_gemm_q4(_ptr(a), _ptr(packed), _ptr(scales), _ptr(biases), _ptr(output), shape.rows,
                                       shape.columns, shape.inner, ctypes.byref(layout.c), _stream(stream))
        _lib.check(st)
        (stream or torch.cuda.current_stream()).synchronize()


class Engine:
    """The GEMM entry points of the reference's Engine (Runtime/Engine.swift:1652, :1911), stream
    ordered; `kernel` replaces the reference's SPLOSH_* kernel-selection environment variables."""

    def __init__(self, kernel=AUTO, stream=None):
        self.kernel = kernel
        self.stream = stream

    def gemm(self, w, input, output, residual=False, rows=None):
        return gemm(w, input, out=output, residual=output if residual else None, kernel=self.kernel, rows=rows,
                    stream=self.stream)

    def mlp_in(self, gate, up, input, output, rows=None):
        return mlp_in(gate, up, input, out=output, kernel=self.kernel, rows=rows, stream=self.stream)


def version():
    return _lib.lib().splosh_version().decode()


# ---- operand producers (the steps either side of a GEMM) ----------------------------------------


def _f32_rows(t, name):
    if t.dtype != torch.float32 or t.dim() != 2 or t.stride(1) != 1:
        raise SploshError(13, f"{name} must be fp32 [rows, dim] with contiguous rows")
    return t


def _operand_out(x, out, sums):
    rows, dim = x.shape
    if out is None:
        out = torch.empty((rows, dim), dtype=torch.bfloat16, device=x.device)
    if sums is None:
        sums = torch.empty((rows, dim // 64), dtype=torch.float32, device=x.device)
    return out, sums


def prepare_operand(x, out=None, sums=None, stream=None):
    """sp_na_prepare (engine_na.metal:38-56): fp32 [rows, dim] -> (bf16 operand, per-64 sums)."""
    x = _f32_rows(x, "x")
    out, sums = _operand_out(x, out, sums)
    _lib.check(_lib.lib().splosh_prepare_operand(_ptr(x), x.stride(0), x.shape[0], x.shape[1], _ptr(out),
                                                 out.stride(0), _ptr(sums), _stream(stream)))
    return out, sums


def silu_mul_operand(gate, up, row_inv=None, out=None, sums=None, stream=None):
    """sp_silu_mul_na (engine.metal:200-218): bf16(silu(g s) (u s)) and its per-64 sums."""
    gate, up = _f32_rows(gate, "gate"), _f32_rows(up, "up")
    if up.shape != gate.shape or up.stride(0) != gate.stride(0):
        raise SploshError(13, "gate and up must share shape and row stride")
    out, sums = _operand_out(gate, out, sums)
    _lib.check(_lib.lib().splosh_silu_mul_operand(_ptr(gate), _ptr(up), gate.stride(0), _ptr(row_inv), gate.shape[0],
                                                  gate.shape[1], _ptr(out), out.stride(0), _ptr(sums),
                                                  _stream(stream)))
    return out, sums


def emit_operand(hidden, norm_weight, values=None, sums=None, squares=None, stream=None):
    """The next RMSNorm-ed GEMM's operand (engine_na.metal:26-36, 365-411): (bf16 hidden * weight,
    per-64 sums of it, per-64 sums of hidden^2)."""
    hidden = _f32_rows(hidden, "hidden")
    if norm_weight.dtype != torch.bfloat16 or norm_weight.numel() < hidden.shape[1]:
        raise SploshError(13, "norm_weight must be bf16 with dim values")
    values, sums = _operand_out(hidden, values, sums)
    if squares is None:
        squares = torch.empty_like(sums)
    _lib.check(_lib.lib().splosh_emit_operand(_ptr(hidden), hidden.stride(0), _ptr(norm_weight), hidden.shape[0],
                                              hidden.shape[1], _ptr(values), values.stride(0), _ptr(sums),
                                              _ptr(squares), _stream(stream)))
    return values, sums, squares


def row_inv(squares, dim, eps, out=None, stream=None):
    """sp_row_inv (engine.metal:222-233): 1 / sqrt(sum(squares[row]) / dim + eps)."""
    if squares.dtype != torch.float32 or not squares.is_contiguous():
        raise SploshError(13, "squares must be contiguous fp32 [rows, groups]")
    rows, groups = squares.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=squares.device)
    _lib.check(_lib.lib().splosh_row_inv(_ptr(squares), rows, groups, dim, float(eps), _ptr(out), _stream(stream)))
    return out


def embed(w, tokens, out=None, out_dtype=torch.float32, stream=None):
    """sp_embed_q4 (engine.metal:39-57) for a q4 table, sp_gguf_embed (engine_gguf.metal:302-318)
    for a GGUF one (planes or native blocks): rows tokens[i] of the decoded table, [count, inner].
    tokens: uint32 ids on the device (int32 tensors are taken as their bits); an id past the table
    gives zeros."""
    if tokens.dtype not in (torch.int32,) or not tokens.is_contiguous():
        raise SploshError(13, "tokens must be a contiguous int32 tensor of uint32 ids")
    count = tokens.numel()
    if out is None:
        out = torch.empty((count, w.inner), dtype=out_dtype, device=tokens.device)
    _require(out, ((count - 1) * out.stride(0) + w.inner) * out.element_size(), "output")
    if isinstance(w, GgufWeight):
        _lib.check(_lib.lib().splosh_gguf_embed(w.type_id, _ptr(w.native), w.rows, w.inner, _ptr(tokens), count,
                                                _ptr(out), out.stride(0), _dtype_code(out.dtype), _stream(stream)))
        return out
    wc = w.c()
    fn = (_lib.lib().splosh_q4_embed if isinstance(w, Q4Weight) else
          _lib.lib().splosh_q4k_embed if isinstance(w, Q4KWeight) else _lib.lib().splosh_q5k_embed)
    _lib.check(fn(ctypes.byref(wc), _ptr(tokens), count, _ptr(out), out.stride(0), _dtype_code(out.dtype),
                  _stream(stream)))
    return out


# ---- per-request operators of a packed step ------------------------------------------------------
#
# The checks here ask a tensor for little and pass plain addresses: a call on one row takes about as long on
# the host as its kernels on the device.


def _index(t, name):
    """The index of the device that a call's operands are on."""
    if not t.is_cuda:
        raise SploshError(12, f"{name} is not a device tensor")
    return t.get_device()


_HERE = contextlib.nullcontext()


def _launch(index):
    """What a call is launched in: its operands' device made the current one, where it is not."""
    return _HERE if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _raw_stream(stream, index):
    # (What torch.cuda.current_stream(index).cuda_stream is, without the object: 0.1 us for 0.8.)
    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(index)


def _vector(t, rows, dtype, index, name):
    """The address of a per-row array: contiguous, of at least `rows` values, on device `index` (None: none)."""
    if t is None:
        return None
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
        raise SploshError(13, f"{name} must be a contiguous {dtype} vector")
    if t.get_device() != index:
        raise SploshError(13, f"{name} is on {t.device}, the operands on cuda:{index}")
    if t.numel() < rows:
        raise GemmQ4Error(8, f"bufferTooSmall(name: {name}, expected: {rows}, observed: {t.numel()})")
    return t.data_ptr()


def _matrix(t, rows, columns, index, name):
    """The address of a [rows, columns] operand: contiguous rows of at least `columns`, on device `index`."""
    if not t.is_cuda:
        raise SploshError(12, f"{name} is not a device tensor")
    shape, strides = t.shape, t.stride()
    if len(shape) != 2 or (strides[1] != 1 and shape[1] > 1) or t.get_device() != index:
        raise SploshError(13, f"{name} must be [rows, columns] with contiguous rows, on cuda:{index}")
    if shape[1] < columns:
        raise GemmQ4Error(1, f"{name} has {shape[1]} columns, {columns} are needed")
    if shape[0] < rows:
        raise GemmQ4Error(8, f"bufferTooSmall(name: {name}, expected: {rows} rows, observed: {shape[0]})")
    return t.data_ptr()


def _given_workspace(workspace, index):
    """(address, bytes) of a caller's workspace on device `index`; one dense block, all of whose bytes are its own."""
    if workspace.get_device() != index:
        raise SploshError(13, f"workspace is on {workspace.device}, the operands on cuda:{index}")
    if not workspace.is_contiguous():
        raise SploshError(13, "workspace must be contiguous")
    return workspace.data_ptr(), workspace.nbytes


def _row_stride(t):
    """The row stride of a checked operand (a single row's can be anything)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


@dataclass(frozen=True)
class Adapters:
    """The low-rank adapters of one projection (splosh_adapters): ``a`` bf16 [count, max_rank, inner]
    and ``b`` bf16 [count, rows, max_rank] (last dimensions contiguous), ``scales`` fp32 [count]
    (None: 1) and ``ranks`` int32 [count] (None: max_rank for all). Slot s adds
    scales[s] * b[s][:, :r] @ (a[s][:r] @ x), r = ranks[s]. The tensors are taken as they are: adapters
    are exchanged by writing into them, and other tensors need a handle of their own (this one keeps the
    addresses that it was made with, so its fields cannot be assigned)."""

    a: torch.Tensor
    b: torch.Tensor
    scales: torch.Tensor = None
    ranks: torch.Tensor = None

    def __post_init__(self):
        a, b = self.a, self.b
        if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
            raise SploshError(13, "adapter matrices must be bf16")
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or 0 in a.shape + b.shape:
            raise GemmQ4Error(1, "adapters are a [count, max_rank, inner] and b [count, rows, max_rank]")
        if (a.stride(2) != 1 and a.shape[2] > 1) or (b.stride(2) != 1 and b.shape[2] > 1):
            raise SploshError(13, "adapter rows must be contiguous")
        index = _index(a, "a")
        if b.get_device() != index:
            raise SploshError(13, f"b is on {b.device}, a on {a.device}")
        count, max_rank, inner = a.shape
        rows = b.shape[1]
        scales = _vector(self.scales, count, torch.float32, index, "scales")
        ranks = _vector(self.ranks, count, torch.int32, index, "ranks")

        def stride(t, dim, least):  # (of a dimension of one, anything)
            return t.stride(dim) if t.shape[dim] > 1 else max(t.stride(dim), least)

        c = _lib.Adapters(a.data_ptr(), b.data_ptr(), ranks, scales, count, max_rank, rows, inner, stride(a, 0, 0),
                          stride(a, 1, inner), stride(b, 0, 0), stride(b, 1, max_rank))
        for name, value in dict(index=index, count=count, max_rank=max_rank, inner=inner, rows=rows, _c=c).items():
            object.__setattr__(self, name, value)

    def c(self):
        return self._c


def adapters_workspace_bytes(adapters, rows):
    """splosh_adapters_workspace_bytes: the scratch a call on these projections' adapters needs."""
    adapters = [adapters] if isinstance(adapters, Adapters) else list(adapters)
    cs = (_lib.Adapters * len(adapters))(*[w.c() for w in adapters])
    return _lib.lib().splosh_adapters_workspace_bytes(cs, len(adapters), rows)


def _adapted(a, w, rows):
    """(rows, device index, address) of the activation that adapters `w` are for."""
    rows = a.shape[0] if rows is None else rows
    if rows <= 0:
        raise GemmQ4Error(1, "rows must be positive")
    if a.dtype != torch.bfloat16:
        raise SploshError(13, "activations must be bf16")
    index = _index(a, "a")
    return rows, index, _matrix(a, rows, w.inner, index, "a")


def _added(out, w, rows, index):
    """The address of an output that adapters `w` add to."""
    if w.index != index:
        raise SploshError(13, f"adapters are on cuda:{w.index}, the activations on cuda:{index}")
    return _matrix(out, rows, w.rows, index, "output")


def add_adapters_group(outs, a, adapters, slots, rows=None, stream=None, workspace=None):
    """splosh_adapters_add_group: the adapters' part of several projections of one activation,
    outs[i][m] += adapters[i] of slots[m] on a[m], in place. ``a`` is the projections' bf16 activation
    [rows, inner], ``outs`` their outputs (gemm_group's; fp32 or bf16), ``slots`` int32 [rows], the
    adapter of each row (negative or past the count: none). Returns the outputs."""
    outs, adapters = list(outs), list(adapters)
    n = len(outs)
    if n != len(adapters) or n == 0:
        raise GemmQ4Error(1, "one output for each projection's adapters")
    rows, index, x = _adapted(a, adapters[0], rows)
    dtype = outs[0].dtype
    if any(o.dtype != dtype for o in outs):
        raise SploshError(13, "grouped outputs must share one dtype")
    ptrs = [_added(o, w, rows, index) for w, o in zip(adapters, outs)]
    slot_ptr = _vector(slots, rows, torch.int32, index, "slots")
    lib, code = _lib.lib(), _dtype_code(dtype)
    cs = (_lib.Adapters * n)(*[w._c for w in adapters])
    with _launch(index):
        if workspace is None:
            with _allocating(stream):
                workspace = torch.empty(max(1, lib.splosh_adapters_workspace_bytes(cs, n, rows)), dtype=torch.uint8,
                                        device=a.device)
        st = lib.splosh_adapters_add_group(cs, n, x, _row_stride(a), (ctypes.c_void_p * n)(*ptrs),
                                           (ctypes.c_int64 * n)(*[_row_stride(o) for o in outs]), code, slot_ptr, rows,
                                           *_given_workspace(workspace, index), _raw_stream(stream, index))
    if st:
        _lib.check(st)
    return outs


def add_adapters(out, a, adapters, slots, rows=None, stream=None, workspace=None):
    """splosh_adapters_add: add_adapters_group for one projection. Returns ``out``."""
    if workspace is None:
        return add_adapters_group((out,), a, (adapters,), slots, rows, stream)[0]
    rows, index, x = _adapted(a, adapters, rows)
    ptr, slot_ptr = _added(out, adapters, rows, index), _vector(slots, rows, torch.int32, index, "slots")
    with _launch(index):
        st = _lib.lib().splosh_adapters_add(ctypes.byref(adapters._c), x, _row_stride(a), ptr, _row_stride(out),
                                            _dtype_code(out.dtype), slot_ptr, rows, *_given_workspace(workspace, index),
                                            _raw_stream(stream, index))
    if st:
        _lib.check(st)
    return out


def sample_workspace_bytes(rows, vocab):
    """splosh_sample_workspace_bytes: the scratch a sampling call needs (0: not a valid shape)."""
    return _lib.lib().splosh_sample_workspace_bytes(rows, vocab)


def sample(logits, uniforms=None, temperature=None, top_k=None, top_p=None, min_p=None, out=None, logprobs=None,
           stream=None, workspace=None):
    """splosh_sample: the next token of each row of ``logits`` (fp32 or bf16 [rows, vocab]), and the
    natural logarithm of the probability it was drawn with. The parameters are fp32 (top_k: int32)
    device vectors [rows]; None leaves that one off. uniforms None: the largest logit of every row
    (as temperature 0 in one row). Returns (tokens int32, logprobs fp32); a row with nothing to choose
    gets token -1, which embed turns into zeros."""
    index = _index(logits, "logits")
    ptr = _matrix(logits, 0, 0, index, "logits")
    rows, vocab = logits.shape
    if rows == 0 or vocab == 0:
        raise GemmQ4Error(1, "rows and vocab must be positive")
    f32, code = torch.float32, _dtype_code(logits.dtype)
    params = (_vector(uniforms, rows, f32, index, "uniforms"), _vector(temperature, rows, f32, index, "temperature"),
              _vector(top_k, rows, torch.int32, index, "top_k"), _vector(top_p, rows, f32, index, "top_p"),
              _vector(min_p, rows, f32, index, "min_p"))
    lib = _lib.lib()
    with _launch(index):
        if out is None or logprobs is None or workspace is None:
            with _allocating(stream):
                out = torch.empty(rows, dtype=torch.int32, device=logits.device) if out is None else out
                logprobs = torch.empty(rows, dtype=f32, device=logits.device) if logprobs is None else logprobs
                if workspace is None:
                    workspace = torch.empty(max(1, lib.splosh_sample_workspace_bytes(rows, vocab)), dtype=torch.uint8,
                                            device=logits.device)
        st = lib.splosh_sample(ptr, _row_stride(logits), code, rows, vocab, *params,
                               _vector(out, rows, torch.int32, index, "out"), _vector(logprobs, rows, f32, index, "logprobs"),
                               *_given_workspace(workspace, index), _raw_stream(stream, index))
    if st:
        _lib.check(st)
    return out, logprobs


# ---- the attention layers of a packed step, and its drafted tokens ---------------------------------


@dataclass(frozen=True)
class Packed:
    """How a step's rows are packed (splosh_packed): ``starts`` int32 [requests + 1], the first row of each request
    and their end; ``lengths`` int32 [requests], each request's tokens in the cache once the step's own are in it;
    ``table`` int32 [requests, pages], its pages in order (contiguous rows). The tensors are taken as they are:
    the next step's values are written into them, and other tensors need a handle of their own."""

    starts: torch.Tensor
    lengths: torch.Tensor
    table: torch.Tensor

    def __post_init__(self):
        table = self.table
        index = _index(table, "table")
        if table.dtype != torch.int32 or table.dim() != 2 or 0 in table.shape or (table.stride(1) != 1 and table.shape[1] > 1):
            raise SploshError(13, "table must be int32 [requests, pages] with contiguous rows")
        requests, pages = table.shape
        starts = _vector(self.starts, requests + 1, torch.int32, index, "starts")
        lengths = _vector(self.lengths, requests, torch.int32, index, "lengths")
        c = _lib.Packed(starts, lengths, table.data_ptr(), requests, _row_stride(table), pages)
        for name, value in dict(index=index, requests=requests, _c=c, _at=ctypes.addressof(c)).items():
            object.__setattr__(self, name, value)

    def c(self):
        return self._c


def cache_page_bytes(heads, dim, page_tokens):
    """splosh_cache_page_bytes: the bytes of one page (0: not a valid shape)."""
    return _lib.lib().splosh_cache_page_bytes(heads, dim, page_tokens)


@dataclass(frozen=True)
class Cache:
    """Keys and values of one layer in 8 bits (splosh_cache): ``data`` uint8 [pages, bytes], a page a row of
    cache_page_bytes(heads, dim, page_tokens) bytes or more, 16-byte aligned."""

    data: torch.Tensor
    page_tokens: int
    heads: int
    dim: int

    def __post_init__(self):
        data = self.data
        index = _index(data, "data")
        need = cache_page_bytes(self.heads, self.dim, self.page_tokens)
        if not need:
            raise SploshError(13, "a cache has dim 64, 128 or 256 and page_tokens a multiple of 32")
        if data.dtype != torch.uint8 or data.dim() != 2 or 0 in data.shape or (data.stride(1) != 1 and data.shape[1] > 1):
            raise SploshError(13, "data must be uint8 [pages, bytes] with contiguous pages")
        if data.shape[1] < need:
            raise GemmQ4Error(8, f"bufferTooSmall(name: page, expected: {need}, observed: {data.shape[1]})")
        stride = data.stride(0) if data.shape[0] > 1 else (data.shape[1] + 15) // 16 * 16
        c = _lib.Cache(data.data_ptr(), data.shape[0], stride, self.page_tokens, self.heads, self.dim)
        for name, value in dict(index=index, pages=data.shape[0], _c=c, _at=ctypes.addressof(c)).items():
            object.__setattr__(self, name, value)

    def c(self):
        return self._c

    @classmethod
    def empty(cls, pages, page_tokens, heads, dim, device):
        """A cache of `pages` pages that holds nothing yet."""
        data = torch.zeros((pages, cache_page_bytes(heads, dim, page_tokens)), dtype=torch.uint8, device=device)
        return cls(data, page_tokens, heads, dim)


def _head_vectors(t, rows, heads, dim, dtype, index, name):
    """(address, row stride, head stride, heads) of `rows` rows of `heads` (None: its own) vectors of `dim`."""
    shape, strides = t.shape, t.stride()
    if t.get_device() != index:
        raise SploshError(13 if t.is_cuda else 12, f"{name} is on {t.device}, the operands on cuda:{index}")
    if len(shape) != 3 or t.dtype != dtype or (strides[2] != 1 and shape[2] > 1):
        raise SploshError(13, f"{name} must be {dtype} [rows, heads, dim] with contiguous vectors")
    have, count, size = shape
    if size != dim or count == 0 or (heads is not None and count != heads):
        raise GemmQ4Error(1, f"{name} is {tuple(shape)}, [rows, {heads or 'heads'}, {dim}] is needed")
    if have < rows:
        raise GemmQ4Error(8, f"bufferTooSmall(name: {name}, expected: {rows} rows, observed: {have})")
    # (The stride of a dimension of one can be anything.)
    return t.data_ptr(), strides[0] if have > 1 else max(strides[0], dim), strides[1] if count > 1 else max(strides[1], dim), count


def _dense_heads(t, rows, heads, dim, index, name):
    """(address, row stride) of a bf16 output [rows, heads, dim] whose rows are dense."""
    ptr, row, head, _ = _head_vectors(t, rows, heads, dim, torch.bfloat16, index, name)
    if head != dim and heads > 1:
        raise SploshError(13, f"{name} must have dense rows")
    return ptr, row if t.shape[0] > 1 else max(row, heads * dim)


def _address(t, rows, dtype, index, name):
    """_vector with 0 for None."""
    return 0 if t is None else _vector(t, rows, dtype, index, name)


def rotate_heads(xs, positions, frequencies, weights=None, eps=1e-6, outs=None, rows=None, stream=None):
    """splosh_rotate_heads: queries and keys (any number of tensors [rows, heads, dim], fp32 or bf16 alike, strided as
    their projections left them) normed over each head by ``weights`` (bf16 [dim] each; None: no norm) and their
    pairs (i, i + len(frequencies)) turned by positions[m] * frequencies[i] (int32 [rows], fp32; None: not). Returns bf16
    [rows, heads, dim] each."""
    count = len(xs)
    if not 0 < count <= 8:
        raise GemmQ4Error(1, "one to eight tensors")
    if (weights is not None and len(weights) != count) or (outs is not None and len(outs) != count):
        raise GemmQ4Error(1, "a weight and an output for each tensor")
    first = xs[0]
    index = _index(first, "x")
    dtype, dim = first.dtype, first.shape[-1]
    rows = first.shape[0] if rows is None else rows
    if rows <= 0:
        raise GemmQ4Error(1, "rows must be positive")
    code, bf16 = _dtype_code(dtype), torch.bfloat16
    if outs is None:
        with _launch(index), _allocating(stream):
            outs = [torch.empty((rows, x.shape[1], dim), dtype=bf16, device=x.device) for x in xs]
    parts = b""
    for i, x in enumerate(xs):
        part = _head_vectors(x, rows, None, dim, dtype, index, "x")
        weight = 0 if weights is None else _address(weights[i], dim, bf16, index, "weight")
        parts += _lib.HEADS.pack(*part, weight, *_dense_heads(outs[i], rows, part[3], dim, index, "output"))
    at = _address(positions, rows, torch.int32, index, "positions")
    freq, rotary = (0, 0) if frequencies is None else (_vector(frequencies, 0, torch.float32, index, "frequencies"), 2 * frequencies.numel())
    with _launch(index):
        st = _lib.lib().splosh_rotate_heads(parts, count, code, rows, dim, at, freq, rotary, eps, _raw_stream(stream, index))
    if st:
        _lib.check(st)
    return outs


def cache_write(cache, packed, k, v, q=None, frequencies=None, k_weight=None, q_weight=None, eps=1e-6, out=None, rows=None,
                stream=None):
    """splosh_cache_write: a step's keys (normed by ``k_weight``, turned by their rows' positions; neither where that is
    None) and values, [rows, cache.heads, dim] fp32 or bf16, into the cache at the places of ``packed``. With ``q``
    [rows, heads, dim] also the step's queries normed and turned, in the same launch: returned as bf16 (``out``)."""
    index, dim, dtype = cache.index, cache.dim, k.dtype
    if packed.index != index:
        raise SploshError(13, f"the table is on cuda:{packed.index}, the cache on cuda:{index}")
    rows = k.shape[0] if rows is None else rows
    if rows <= 0:
        raise GemmQ4Error(1, "rows must be positive")
    code, bf16, pack = _dtype_code(dtype), torch.bfloat16, _lib.HEADS.pack
    kc = pack(*_head_vectors(k, rows, cache.heads, dim, dtype, index, "k"), _address(k_weight, dim, bf16, index, "k_weight"), 0, 0)
    vc = pack(*_head_vectors(v, rows, cache.heads, dim, dtype, index, "v"), 0, 0, 0)
    freq, rotary = (0, 0) if frequencies is None else (_vector(frequencies, 0, torch.float32, index, "frequencies"), 2 * frequencies.numel())
    qc = None
    if q is not None:
        part = _head_vectors(q, rows, None, dim, dtype, index, "q")
        if out is None:
            with _launch(index), _allocating(stream):
                out = torch.empty((rows, part[3], dim), dtype=bf16, device=q.device)
        qc = pack(*part, _address(q_weight, dim, bf16, index, "q_weight"), *_dense_heads(out, rows, part[3], dim, index, "output"))
    with _launch(index):
        st = _lib.lib().splosh_cache_write(cache._at, packed._at, kc, vc, qc, code, rows, freq, rotary, eps, _raw_stream(stream, index))
    if st:
        _lib.check(st)
    return out if q is not None else None


def cache_read(cache, packed, rows=None, k=None, v=None, stream=None):
    """splosh_cache_read: what the cache holds at the places of ``packed``'s rows, as bf16 (k, v) [rows, heads, dim]. Of a
    request with n rows these are its last n tokens. rows: that of k or v where they are given."""
    index, heads, dim = cache.index, cache.heads, cache.dim
    if packed.index != index:
        raise SploshError(13, f"the table is on cuda:{packed.index}, the cache on cuda:{index}")
    if rows is None:
        if k is None and v is None:
            raise GemmQ4Error(1, "rows or an output is needed")
        rows = (k if k is not None else v).shape[0]
    if rows <= 0:
        raise GemmQ4Error(1, "rows must be positive")
    if k is None and v is None:
        with _launch(index), _allocating(stream):
            k, v = (torch.empty((rows, heads, dim), dtype=torch.bfloat16, device=cache.data.device) for _ in "kv")
    kp = (None, 0) if k is None else _dense_heads(k, rows, heads, dim, index, "k")
    vp = (None, 0) if v is None else _dense_heads(v, rows, heads, dim, index, "v")
    with _launch(index):
        st = _lib.lib().splosh_cache_read(cache._at, packed._at, rows, *kp, *vp, _raw_stream(stream, index))
    if st:
        _lib.check(st)
    return k, v


def attend_workspace_bytes(cache, packed, rows, q_heads, shared=0):
    """splosh_attend_workspace_bytes: the scratch an attention call needs (0: not a valid shape)."""
    with _launch(cache.index):
        return _lib.lib().splosh_attend_workspace_bytes(cache._at, packed._at, rows, q_heads, shared)


def attend(q, cache, packed, shared=0, scale=None, out=None, rows=None, stream=None, workspace=None):
    """splosh_attend: causal attention of a step's queries (bf16 [rows, heads, dim], strided as they are) over the cache,
    which holds the step's own keys and values already. shared: the first tokens (whole pages) that all requests have in
    common, read once for all through request 0's pages. scale None: dim ** -0.5. Returns bf16 [rows, heads, dim] with
    dense rows, the out projection's activation."""
    index, dim = cache.index, cache.dim
    if packed.index != index:
        raise SploshError(13, f"the table is on cuda:{packed.index}, the cache on cuda:{index}")
    rows = q.shape[0] if rows is None else rows
    if rows <= 0:
        raise GemmQ4Error(1, "rows must be positive")
    part = _head_vectors(q, rows, None, dim, torch.bfloat16, index, "q")
    lib = _lib.lib()
    with _launch(index):
        if out is None or workspace is None:
            with _allocating(stream):
                out = torch.empty((rows, part[3], dim), dtype=torch.bfloat16, device=q.device) if out is None else out
                if workspace is None:
                    need = lib.splosh_attend_workspace_bytes(cache._at, packed._at, rows, part[3], shared)
                    workspace = torch.empty(max(1, need), dtype=torch.uint8, device=q.device)
        st = lib.splosh_attend(*part, cache._at, packed._at, rows, shared, dim ** -0.5 if scale is None else scale,
                               *_dense_heads(out, rows, part[3], dim, index, "output"),
                               *_given_workspace(workspace, index), _raw_stream(stream, index))
    if st:
        _lib.check(st)
    return out


def verify_workspace_bytes(rows, vocab, requests):
    """splosh_verify_workspace_bytes: the scratch a verification needs (0: not a valid shape)."""
    return _lib.lib().splosh_verify_workspace_bytes(rows, vocab, requests)


def verify(logits, tokens, starts, uniforms, temperature=None, draft=None, out=None, accepted=None, stream=None,
           workspace=None):
    """splosh_verify: the drafted tokens of a verify step against the target's logits (fp32 or bf16 [rows, vocab]).
    ``tokens`` int32 [rows], the ids that the step embedded; ``starts`` int32 [requests + 1]; ``uniforms`` fp32 [rows];
    ``temperature`` fp32 [requests] (None: 1); ``draft`` the draft's probabilities [rows, vocab] by the row that judges the
    token (fp32 or bf16; None: drafted by a lookup or greedily). Returns (out int32 [rows], accepted int32 [requests]): from starts[r]
    on the accepted tokens of request r and the new one, then -1."""
    index = _index(logits, "logits")
    ptr = _matrix(logits, 0, 0, index, "logits")
    rows, vocab = logits.shape
    requests = starts.numel() - 1
    if rows == 0 or vocab == 0 or requests < 1:
        raise GemmQ4Error(1, "rows, vocab and requests must be positive")
    f32, i32 = torch.float32, torch.int32
    inputs = (_vector(tokens, rows, i32, index, "tokens"), _vector(starts, requests + 1, i32, index, "starts"), requests,
              _vector(uniforms, rows, f32, index, "uniforms"), _vector(temperature, requests, f32, index, "temperature"))
    judged = (None, 0, 0) if draft is None else (_matrix(draft, rows, vocab, index, "draft"), _row_stride(draft), _dtype_code(draft.dtype))
    code, lib = _dtype_code(logits.dtype), _lib.lib()
    with _launch(index):
        if out is None or accepted is None or workspace is None:
            with _allocating(stream):
                out = torch.empty(rows, dtype=i32, device=logits.device) if out is None else out
                accepted = torch.empty(requests, dtype=i32, device=logits.device) if accepted is None else accepted
                if workspace is None:
                    workspace = torch.empty(max(1, lib.splosh_verify_workspace_bytes(rows, vocab, requests)), dtype=torch.uint8,
                                            device=logits.device)
        st = lib.splosh_verify(ptr, _row_stride(logits), code, rows, vocab, *inputs, *judged,
                               _vector(out, rows, i32, index, "out"), _vector(accepted, requests, i32, index, "accepted"),
                               *_given_workspace(workspace, index), _raw_stream(stream, index))
    if st:
        _lib.check(st)
    return out, accepted
