"""Tensor-level entry points over the C ABI: each lifted kernel family on torch CUDA tensors.

torch supplies device memory and the current stream only; every computation runs in libunpopped_sm100.so.
Inputs must already be on a CUDA device; nothing here moves data to the host or computes on it. The one
exception is `scan_host`, whose buffers are in host memory: the library itself streams them through the device.
"""
from __future__ import annotations

import ctypes
import threading

import numpy as np
import torch

from . import _lib
from ._lib import ACCUM, COMBINE, EK, OOB, OP, ROPE_SCALING, check

_OPS = {"sum": OP["SUM"], "max": OP["MAX"], "min": OP["MIN"]}
_OOBS = {"skip": OOB["SKIP"], "clamp": OOB["CLAMP"], "zero_fill": OOB["ZERO_FILL"]}
_IDX = {torch.int32: EK["I32"], torch.int64: EK["I64"], torch.uint32: EK["U32"]}


# the current stream's handle without a Stream object around it: 0.1 us against 2.4 us a call
_raw_stream = torch._C._cuda_getCurrentRawStream


def _stream(t: torch.Tensor):
    return ctypes_ptr(_raw_stream(t.get_device()))


def ctypes_ptr(v):
    return None if v in (0, None) else v


def _cuda(t: torch.Tensor, name: str):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")


# ---- workspaces: zero-filled once per (device, stream, kind); the kernels re-arm them after every launch ----
_ws_lock = threading.Lock()
_ws_cache: dict = {}


def _ws_key(kind: str, device: torch.device):
    """Of the device's current stream; a device without an index is the current one."""
    index = torch.cuda.current_device() if device.index is None else device.index
    return kind, index, _raw_stream(index)


def workspace(kind: str, nbytes: int, device: torch.device) -> torch.Tensor:
    """A zero-filled device workspace for `kind`, reused by later calls on the same stream. While a CUDA graph is being
    captured, a new one for this call alone: its zero fill is then a part of the graph and its memory the graph's own, so
    replays depend neither on another graph nor on a buffer that a later call may outgrow."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
    key = _ws_key(kind, device)
    with _ws_lock:
        ws = _ws_cache.get(key)
        if ws is None or ws.numel() < nbytes:
            ws = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
            _ws_cache[key] = ws
        return ws


def workspace_status(ws: torch.Tensor) -> int:
    """Waits for the stream and returns UP_OK or UP_ERR_DEVICE_TIMEOUT. After a wait that ran out the workspace is zero-filled, as before its
    first use: a launch that gave up leaves counters of unfinished tiles behind, by which later launches would add parts that are not there."""
    status = _lib.load().up_sm100_workspace_status(ws.data_ptr(), _stream(ws))
    if status == _lib.UP_ERR_DEVICE_TIMEOUT:
        ws.zero_()
    return status


def check_workspace(kind: str, device: torch.device):
    """Raises UpError if a device wait of a call on the current stream ran out since the last check; the results of the calls between are not
    to be used. The next call works again."""
    ws = _ws_cache.get(_ws_key(kind, device))
    if ws is not None:
        check(workspace_status(ws), f"{kind} device wait")


_bound = None


def _calls():
    """The calls of csrc/bind.cpp; like the library, there is no substitute for them."""
    global _bound
    if _bound is None:
        try:
            from . import _bind
        except ImportError as e:
            raise ImportError("the serving operators' calls are not built for this torch and Python: "
                              "run python -m unpopped_b200.build") from e
        _bind.init(check, workspace, _ws_cache)
        _bound = _bind
    return _bound


# ---- row sum ----
def row_sum(x: torch.Tensor, accum: str = "f32", block: int = 256, out: torch.Tensor | None = None) -> torch.Tensor:
    """Sum of each row of a 2-D f32 tensor (last axis). accum='f32' (fixed-order f32 tree) or 'auto' (f64 in
    the launched lift's documented order for a block of `block` threads, bit-exact)."""
    _cuda(x, "x")
    if x.dtype != torch.float32 or x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("row_sum takes a 2-D float32 tensor with contiguous rows")
    rows, cols = x.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(_lib.load().up_sm100_row_sum_f32(x.data_ptr(), rows, cols, x.stride(0), out.data_ptr(),
                                           ACCUM[accum.upper()], block, _stream(x)), "row_sum")
    return out


# ---- max + argmax ----
def reduce2d(x: torch.Tensor, op: str, axis: int = 1, accum: str = "auto", block: int | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """Reduction of a [rows, cols] f32 or i32 tensor with contiguous rows over axis 1 (the last; one value per
    row) or axis 0 (the outer; one per column). f32: sum, mean, max, min; i32: sum, prod, max, min, and, or, xor."""
    _cuda(x, "x")
    if x.dim() != 2 or x.stride(1) != 1 or x.dtype not in (torch.float32, torch.int32):
        raise ValueError("reduce2d takes a 2-D float32 or int32 tensor with contiguous rows")
    if axis not in (0, 1):
        raise ValueError("axis is 0 or 1")
    rows, cols = x.shape
    n = rows if axis == 1 else cols
    if out is None:
        out = torch.empty(n, dtype=x.dtype, device=x.device)
    L = _lib.load()
    if x.dtype == torch.float32:
        b = block if block is not None else (256 if axis == 1 else 1)
        check(L.up_sm100_reduce2d_f32(x.data_ptr(), rows, cols, x.stride(0), axis, OP[op.upper()],
                                      ACCUM[accum.upper()], b, out.data_ptr(), _stream(x)), "reduce2d_f32")
    else:
        check(L.up_sm100_reduce2d_i32(x.data_ptr(), rows, cols, x.stride(0), axis, OP[op.upper()], out.data_ptr(),
                                      _stream(x)), "reduce2d_i32")
    return out


def row_reduce(x: torch.Tensor, form: str, block: int = 256, eps: float = 1e-3,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """A RowReduce form over the rows of a [rows, cols] f32 tensor (contiguous rows): "softmax", "rms_norm"
    (x / sqrt(mean(x * x) + eps)) or "centred" ((x - mean) / max(x - mean)), for logical block `block`."""
    _cuda(x, "x")
    if x.dim() != 2 or x.stride(1) != 1 or x.dtype != torch.float32:
        raise ValueError("row_reduce takes a 2-D float32 tensor with contiguous rows")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if out.shape != x.shape or out.stride(1) != 1 or out.dtype != torch.float32:
        raise ValueError("out has x's shape with contiguous rows")
    L = _lib.load()
    check(L.up_sm100_row_reduce_f32(x.data_ptr(), x.shape[0], x.shape[1], x.stride(0),
                                    _lib.ROW_REDUCE_FORM[form.upper()], block, eps, out.data_ptr(), out.stride(0),
                                    _stream(x)), "row_reduce_f32")
    return out


def col_sum_splitk(x: torch.Tensor, n_chunks: int, mean: bool = False,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The split-K variant of the outer-axis f32 Sum (Mean) of a [rows, cols] tensor with contiguous rows: f64
    partials over n_chunks row chunks, added in chunk order. Allocates its workspace."""
    _cuda(x, "x")
    if x.dim() != 2 or x.stride(1) != 1 or x.dtype != torch.float32:
        raise ValueError("col_sum_splitk takes a 2-D float32 tensor with contiguous rows")
    rows, cols = x.shape
    if out is None:
        out = torch.empty(cols, dtype=torch.float32, device=x.device)
    L = _lib.load()
    nb = L.up_sm100_col_sum_splitk_workspace_bytes(rows, cols, n_chunks)
    ws = torch.empty(max(8, nb), dtype=torch.uint8, device=x.device)
    check(L.up_sm100_col_sum_f32_splitk(x.data_ptr(), rows, cols, x.stride(0), n_chunks, int(mean), ws.data_ptr(),
                                        ws.numel(), out.data_ptr(), _stream(x)), "col_sum_f32_splitk")
    return out


def window(x: torch.Tensor, op: str, size: int, stride: int = 1, dilation: int = 1, pad_lo: int = 0,
           pad_hi: int | None = None, count_include_pad: bool = False, axis: int = -1,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """1-D window pooling (sum, mean, max, min) of a dense f32 or i32 tensor along `axis`; the output extent is
    (k_in + pad_lo + pad_hi - dilation*(size-1) - 1) // stride + 1 (pad_hi defaults to pad_lo)."""
    _cuda(x, "x")
    if not x.is_contiguous() or x.dtype not in (torch.float32, torch.int32):
        raise ValueError("window takes a contiguous float32 or int32 tensor")
    axis = axis % x.dim()
    k_in = x.shape[axis]
    ph = pad_lo if pad_hi is None else pad_hi
    k_out = (k_in + pad_lo + ph - dilation * (size - 1) - 1) // stride + 1
    shape = list(x.shape)
    shape[axis] = max(k_out, 0)
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    outer = int(np.prod(x.shape[:axis], dtype=np.int64))
    inner = int(np.prod(x.shape[axis + 1:], dtype=np.int64))
    L = _lib.load()
    check(L.up_sm100_window(x.data_ptr(), EK["F32"] if x.dtype == torch.float32 else EK["I32"], outer, k_in, inner,
                            OP[op.upper()], size, stride, dilation, pad_lo, int(count_include_pad), out.data_ptr(),
                            shape[axis], _stream(x)), "window")
    return out


def im2col(x: torch.Tensor, kernel: tuple, stride: tuple = (1, 1), pad: tuple = (0, 0), dilation: tuple = (1, 1),
           out: torch.Tensor | None = None) -> torch.Tensor:
    """The 2-D unfold of a contiguous NCHW tensor into [N, C*kh*kw, oH*oW], raw bits, zeros outside the input."""
    _cuda(x, "x")
    if x.dim() != 4 or not x.is_contiguous():
        raise ValueError("im2col takes a contiguous NCHW tensor")
    n, c, h, w = x.shape
    (kh, kw), (sh, sw), (ph, pw), (dh, dw) = kernel, stride, pad, dilation
    oh = (h + 2 * ph - dh * (kh - 1) - 1) // sh + 1
    ow = (w + 2 * pw - dw * (kw - 1) - 1) // sw + 1
    if out is None:
        out = torch.empty((n, c * kh * kw, max(oh, 0) * max(ow, 0)), dtype=x.dtype, device=x.device)
    L = _lib.load()
    check(L.up_sm100_im2col(x.data_ptr(), x.element_size(), n, c, h, w, kh, kw, sh, sw, ph, pw, dh, dw,
                            out.data_ptr(), _stream(x)), "im2col")
    return out


def reduce3d(x: torch.Tensor, op: str, accum: str = "auto", block: int = 1,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """Reduction of an [outer, rows, cols] f32 or i32 tensor over its middle axis into [outer, cols]; the rows and
    the output rows are contiguous. Each output cell is the outer-axis fold of reduce2d over its batch."""
    _cuda(x, "x")
    if x.dim() != 3 or x.stride(2) != 1 or x.dtype not in (torch.float32, torch.int32):
        raise ValueError("reduce3d takes a 3-D float32 or int32 tensor with contiguous rows")
    outer, rows, cols = x.shape
    if out is None:
        out = torch.empty((outer, cols), dtype=x.dtype, device=x.device)
    if out.dim() != 2 or tuple(out.shape) != (outer, cols) or out.stride(1) != 1:
        raise ValueError("out is [outer, cols] with contiguous rows")
    L = _lib.load()
    if x.dtype == torch.float32:
        check(L.up_sm100_reduce3d_f32(x.data_ptr(), outer, rows, cols, x.stride(0), x.stride(1), OP[op.upper()],
                                      ACCUM[accum.upper()], block, out.data_ptr(), out.stride(0), _stream(x)),
              "reduce3d_f32")
    else:
        check(L.up_sm100_reduce3d_i32(x.data_ptr(), outer, rows, cols, x.stride(0), x.stride(1), OP[op.upper()],
                                      out.data_ptr(), out.stride(0), _stream(x)), "reduce3d_i32")
    return out


_SC_EK = {torch.int32: EK["I32"], torch.int64: EK["I64"], torch.uint32: EK["U32"], torch.float32: EK["F32"],
          torch.float64: EK["F64"]}


def scatter(updates: torch.Tensor, ids: torch.Tensor, out: torch.Tensor, combine: str = "add") -> torch.Tensor:
    """out[t][j] (combine)= updates[i][j] with t = ids[i][j] (a full-shape index, scatter) or ids[i] (1-D, index_add),
    over axis 0; targets outside [0, out.shape[0]) are skipped. Updates `out` in place and returns it."""
    for t, name in ((updates, "updates"), (ids, "ids"), (out, "out")):
        _cuda(t, name)
    if updates.dim() != 2 or out.dim() != 2 or updates.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("scatter takes rank-2 updates and destination with contiguous rows")
    if updates.dtype != out.dtype or updates.dtype not in _SC_EK or ids.dtype not in _IDX:
        raise ValueError("scatter dtypes: updates/out I32, U32, I64, F32 or F64; ids I32, I64 or U32")
    if ids.dim() == 2:
        if ids.shape != updates.shape or ids.stride(1) != 1:
            raise ValueError("a full-shape index has the updates' shape and contiguous rows")
        ids_stride = ids.stride(0)
    else:
        if ids.dim() != 1 or ids.shape[0] != updates.shape[0] or ids.stride(0) != 1:
            raise ValueError("a row index is 1-D, one per update row, contiguous")
        ids_stride = 0
    check(_lib.load().up_sm100_scatter(updates.data_ptr(), updates.shape[0], updates.shape[1], updates.stride(0),
                                       _SC_EK[updates.dtype], ids.data_ptr(), _IDX[ids.dtype], ids_stride,
                                       COMBINE[combine.upper()], out.data_ptr(), out.shape[0], out.stride(0),
                                       _stream(out)), "scatter")
    return out


def bincount(x: torch.Tensor, counts: torch.Tensor) -> torch.Tensor:
    """counts[x[i]] += 1 for every in-range x[i]; `counts` (int32) keeps its prior contents."""
    _cuda(x, "x")
    _cuda(counts, "counts")
    if counts.dtype != torch.int32 or not counts.is_contiguous() or not x.is_contiguous() or x.dtype not in _IDX:
        raise ValueError("bincount takes contiguous I32/I64/U32 values and contiguous int32 counts")
    check(_lib.load().up_sm100_bincount(x.data_ptr(), x.numel(), _IDX[x.dtype], counts.data_ptr(), counts.numel(),
                                        _stream(counts)), "bincount")
    return counts


def row_max_argmax(x: torch.Tensor, index_dtype=torch.int32, want_max: bool = True, want_argmax: bool = True):
    """(max as f32, argmax) of each row of a 2-D bf16 tensor: NaN-propagating max, first index of the maximum
    with NaN the greatest value."""
    _cuda(x, "x")
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("row_max_argmax takes a 2-D bfloat16 tensor with contiguous rows")
    rows, cols = x.shape
    mx = torch.empty(rows, dtype=torch.float32, device=x.device) if want_max else None
    am = torch.empty(rows, dtype=index_dtype, device=x.device) if want_argmax else None
    p32 = am.data_ptr() if (am is not None and index_dtype == torch.int32) else None
    p64 = am.data_ptr() if (am is not None and index_dtype == torch.int64) else None
    check(_lib.load().up_sm100_row_max_argmax_bf16(x.data_ptr(), rows, cols, x.stride(0),
                                                   mx.data_ptr() if mx is not None else None, p32, p64,
                                                   _stream(x)), "row_max_argmax")
    return mx, am


# ---- scans ----
def scan(x: torch.Tensor, op: str = "sum", exclusive: bool = False, reverse: bool = False,
         carry: torch.Tensor | None = None, out: torch.Tensor | None = None,
         ws: torch.Tensor | None = None) -> torch.Tensor:
    """Scan of int32 rows along the last axis (decoupled look-back, one pass)."""
    _cuda(x, "x")
    if x.dtype != torch.int32 or not x.is_contiguous():
        raise ValueError("scan takes a contiguous int32 tensor")
    k = x.shape[-1] if x.dim() > 0 else 1
    rows = x.numel() // k if k > 0 else 0
    if out is None:
        out = torch.empty_like(x)
    L = _lib.load()
    nbytes = L.up_sm100_scan_workspace_bytes(rows, k)
    if ws is None:
        ws = workspace("scan", nbytes, x.device)
    check(L.up_sm100_scan_i32(x.data_ptr(), out.data_ptr(), rows, k, _OPS[op], int(exclusive), int(reverse),
                              carry.data_ptr() if carry is not None else None, ws.data_ptr(), ws.numel(),
                              _stream(x)), "scan")
    return out


def scan_host(x, op: str = "sum", exclusive: bool = False, reverse: bool = False, carry: int | None = None,
              out=None):
    """Scan of int32 rows held in HOST memory (a numpy array or a CPU tensor, pinned for the full copy rate),
    streamed through the device with the copies overlapped; returns the output in host memory."""
    is_t = isinstance(x, torch.Tensor)
    if is_t:
        if x.device.type != "cpu" or x.dtype != torch.int32 or not x.is_contiguous():
            raise ValueError("scan_host takes a contiguous int32 tensor in host memory")
        if out is None:
            out = torch.empty_like(x, pin_memory=x.is_pinned())
        xp, yp = x.data_ptr(), out.data_ptr()
    else:
        x = np.ascontiguousarray(x)
        if x.dtype != np.int32:
            raise ValueError("scan_host takes an int32 array")
        if out is None:
            out = np.empty_like(x)
        xp, yp = x.ctypes.data, out.ctypes.data
    k = x.shape[-1] if x.ndim > 0 else 1
    rows = (x.size if not is_t else x.numel()) // k if k > 0 else 0
    c = ctypes.c_int32(carry) if carry is not None else None
    check(_lib.load().up_sm100_scan_i32_host(xp, yp, rows, k, _OPS[op], int(exclusive), int(reverse),
                                             ctypes.byref(c) if c is not None else None), "scan_host")
    return out


def reduce_i32(x: torch.Tensor, op: str = "sum", out: torch.Tensor | None = None) -> torch.Tensor:
    """Fold of a whole int32 tensor to one int32 (SUM wraps)."""
    _cuda(x, "x")
    if x.dtype != torch.int32 or not x.is_contiguous():
        raise ValueError("reduce_i32 takes a contiguous int32 tensor")
    if out is None:
        out = torch.empty(1, dtype=torch.int32, device=x.device)
    check(_lib.load().up_sm100_reduce_i32(x.data_ptr(), x.numel(), _OPS[op], out.data_ptr(), _stream(x)),
          "reduce_i32")
    return out


# ---- gather ----
def gather_rows(table: torch.Tensor, ids: torch.Tensor, oob: str = "skip",
                out: torch.Tensor | None = None) -> torch.Tensor:
    """out[n] = table[ids[n]] (rows copied bit for bit); out-of-range ids per `oob`."""
    _cuda(table, "table")
    _cuda(ids, "ids")
    if not table.is_contiguous() or ids.dim() != 1 or not ids.is_contiguous():
        raise ValueError("gather_rows takes a contiguous table and 1-D contiguous ids")
    if ids.dtype not in _IDX:
        raise ValueError("ids must be int32, int64 or uint32")
    V = table.shape[0]
    row_bytes = (table[0].numel() if V > 0 else int(torch.Size(table.shape[1:]).numel())) * table.element_size()
    n = ids.shape[0]
    if out is None:
        out = (torch.zeros if oob == "skip" else torch.empty)((n,) + tuple(table.shape[1:]), dtype=table.dtype,
                                                              device=table.device)
    check(_lib.load().up_sm100_gather_rows(table.data_ptr() if V > 0 else None, V, row_bytes, ids.data_ptr(),
                                           _IDX[ids.dtype], n, _OOBS[oob], out.data_ptr(), _stream(table)),
          "gather_rows")
    return out


# ---- int4 dequant and W4A16 ----
def dequant_i4(w_packed: torch.Tensor, scale: torch.Tensor, group: int, out: torch.Tensor | None = None):
    """bf16 [N, K] from int4 [N, K] packed two per byte ([N, K/2] uint8) and f16 scales [N, K/group]."""
    try:
        call = _calls().dequant_i4
    except ImportError:  # unlike the serving operators it needs the C library only, 3 us a call slower
        call = _dequant_i4
    return call(w_packed, scale, group, out)


def _dequant_i4(w_packed, scale, group, out):
    _cuda(w_packed, "w")
    _cuda(scale, "scale")
    n, kh = w_packed.shape
    if out is None:
        out = torch.empty((n, 2 * kh), dtype=torch.bfloat16, device=w_packed.device)
    check(_lib.load().up_sm100_dequant_i4_bf16(w_packed.data_ptr(), scale.data_ptr(), n, 2 * kh, group, out.data_ptr(),
                                               _stream(w_packed)), "dequant_i4")
    return out


def w4a16(w_packed: torch.Tensor, scale: torch.Tensor, x: torch.Tensor, group: int,
          out: torch.Tensor | None = None, ws: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 [M, N] = x [M, K] (bf16) times the dequantized int4 weights [N, K], f32 accumulation on tcgen05."""
    for t, nm in ((w_packed, "w"), (scale, "scale"), (x, "x")):
        _cuda(t, nm)
    n, kh = w_packed.shape
    k = 2 * kh
    m = x.shape[0]
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    L = _lib.load()
    if ws is None:
        ws = workspace("w4a16", L.up_sm100_w4a16_workspace_bytes(m, n, k, group), x.device)
    check(L.up_sm100_w4a16_gemm(w_packed.data_ptr(), scale.data_ptr(), x.data_ptr(), m, n, k, group, out.data_ptr(),
                                ws.data_ptr(), ws.numel(), _stream(x)), "w4a16")
    return out


# ---- rotary positions, the 4-bit paged cache and its attention ----
def rope_table(n_pos: int, rot: int, base: float = 10000.0, scaling: tuple | None = None, gain: float = 1.0,
               device="cuda") -> torch.Tensor:
    """The f32 [n_pos, rot] table that `rope` and `kv4_append` read: gain * cos(p f_i) in the first rot/2 columns, gain *
    sin(p f_i) in the others, f_i = base^(-2i/rot). `scaling` for contexts longer than a model was trained on:
    ("linear", factor), ("base", factor), ("wavelength", factor, low, high, orig_len) or
    ("ramp", factor, low, high, orig_len); up_sm100.h has their formulas."""
    out = torch.empty((n_pos, rot), dtype=torch.float32, device=device)
    kind, rest = ("none", ()) if scaling is None else (scaling[0], scaling[1:])
    if len(rest) != {"none": 0, "linear": 1, "base": 1, "wavelength": 4, "ramp": 4}.get(kind, -1):
        raise ValueError(f"rope_table: no such scaling {scaling!r}")
    factor, low, high, orig = tuple(float(v) for v in rest) + (1.0, 0.0, 0.0, 0.0)[len(rest):]
    if out.get_device() != torch.cuda.current_device():
        raise ValueError("the table must be on the current CUDA device")
    check(_lib.load().up_sm100_rope_table(out.data_ptr(), n_pos, rot, base, ROPE_SCALING[kind.upper()], factor, low,
                                          high, orig, gain, _stream(out)), "rope_table")
    return out


def rope(x: torch.Tensor, positions: torch.Tensor | None, table: torch.Tensor, layout: str = "half",
         out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions: x [tokens, heads, dim] or [batch, seq, heads, dim] (float32, float16, bfloat16; any strides with
    the dimension contiguous) with the first table.shape[1] dimensions of each head turned by the token's position.
    layout "half" pairs dimensions (i, i + rot/2), "interleaved" (2i, 2i + 1). positions: int32 or int64, one a token
    ([seq] serves every sequence of a batch), None counts from 0; one outside the table gives NaN. out may be x.
    Like every function here it is no part of autograd: the result requires no gradient, `rope_backward` gives it."""
    return _calls().rope(x, positions, table, layout, out, False)


def rope_backward(grad: torch.Tensor, positions: torch.Tensor | None, table: torch.Tensor, layout: str = "half",
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of `rope` with respect to its input, from the gradient of its output (what a torch.autograd.Function
    around `rope` returns from its backward)."""
    return _calls().rope(grad, positions, table, layout, out, True)


def kv4_cache(pages: int, kv_heads: int, dim: int, page: int = 16, group: int = 32, device="cuda") -> tuple:
    """A new paged 4-bit cache, the tuple (k, v, k_scale, v_scale) that `kv4_append` and `kv4_attention` take: k and v
    uint8 [pages, kv_heads, page, dim/2] (int4 two per byte, low nibble = even dimension), the scales float16
    [pages, kv_heads, page, dim/group]. A slot reads as zeros until it is written."""
    rows = (pages, kv_heads, page)
    return tuple(torch.zeros(rows + (n,), dtype=t, device=device)
                 for n, t in ((dim // 2, torch.uint8), (dim // 2, torch.uint8), (dim // group, torch.float16),
                              (dim // group, torch.float16)))


def kv4_append(k: torch.Tensor, v: torch.Tensor, cache: tuple, slots: torch.Tensor,
               positions: torch.Tensor | None = None, table: torch.Tensor | None = None,
               q: torch.Tensor | None = None, layout: str = "half",
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes new tokens into a paged 4-bit cache (`kv4_cache`) in one launch and returns their rotated queries.

    k, v [tokens, kv_heads, dim] and q [tokens, heads, dim] (or None) are bfloat16 or float16, of any strides with the
    dimension contiguous (views of one projection's output, say). With a table (`rope_table`), q and k turn by their
    token's position first, as `rope` does; without one they do not. k and v are quantised to int4 with an f16 scale a
    group. slots (int32 or int64, one a token): the token's place, page * page_size + place in the page; a slot outside the
    cache (-1: padding) leaves the token out. q_out may be q."""
    return _calls().kv4_append(k, v, cache, slots, positions, table, q, layout, q_out)


def kv4_attention(q: torch.Tensor, cache: tuple, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  cu_q: torch.Tensor | None = None, causal: bool = True, window: int = 0,
                  scale: float | None = None, out: torch.Tensor | None = None, want_lse: bool = False,
                  ws: torch.Tensor | None = None):
    """Attention of query tokens over a paged 4-bit cache (`kv4_cache`): out [tokens, heads, dim] of q's type, and with
    want_lse the f32 [tokens, heads] log-sum-exp of each query's logits.

    q [tokens, heads, dim] bfloat16 or float16 (rows 16-byte aligned), heads a multiple of the cache's; query head h reads
    key/value head h // (heads // kv_heads). seq_lens int32 [batch]: a sequence's cached tokens, the new ones included;
    block_table int32 [batch, width]: its pages. cu_q int32 [batch + 1]: where each sequence's query tokens begin in q;
    None: one token a sequence. The query tokens are the last of their sequence: each sees the cached tokens up to its own
    (`causal`), and of these the last `window` where window > 0. A query that sees nothing gives 0 (and -inf).
    ws: a workspace of the caller's, contiguous and zero-filled once; without one the stream's is used, or a captured graph's
    own. A batch of long prompts and single tokens takes less time as two calls."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return _calls().kv4_attention(q, cache, block_table, seq_lens, cu_q, causal, window, scale, out, want_lse, ws)


# ---- 8-bit products with a scale for each block of 128, and experts ----
def f8_quantise(x: torch.Tensor, rows: torch.Tensor | None = None, gate: bool = False):
    """(q, scale): the rows of x [tokens, k] (float32, float16, bfloat16; rows of whole 16 bytes, k a multiple of 16) as
    float8_e4m3fn [n, k] with one f32 scale for each 128 values of a row, [n, ceil(k / 128)] (a block's scales lie beside one
    another in memory, as `f8_matmul` reads them fastest). rows (int32 [n]): row r is x[rows[r]], and zeros where that is no row of
    x (`expert_route`'s rows). gate: x holds 2k values a row, and y = silu(x[:, :k]) * x[:, k:] is quantised, in f32.
    scale = max|y| / 448 over a block's finite values; an infinity or a NaN reads back as NaN. q and scale are parts of one allocation (saving
    one, or keeping it, saves or keeps both; clone it to part them). No part of autograd."""
    return _calls().f8_quantise(x, rows, gate)


def f8_quantise_weight(w: torch.Tensor):
    """(q, scale): weights [n, k] or [experts, n, k] as float8_e4m3fn with one f32 scale for each block of 128 x 128,
    [(experts,) ceil(n / 128), ceil(k / 128)]: what `f8_matmul` and `f8_expert_matmul` take. Types and sizes as `f8_quantise`."""
    return _calls().f8_quantise_weight(w)


def f8_matmul(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, dtype=torch.bfloat16,
              out: torch.Tensor | None = None, ws: torch.Tensor | None = None) -> torch.Tensor:
    """[rows, n] = x [rows, k] times w [n, k], both float8_e4m3fn with their scales (`f8_quantise`, `f8_quantise_weight`):
    tcgen05 products of each block of 128, scaled and summed in f32, rounded once to `dtype` (bfloat16, float16 or float32;
    out's where it is given). Any number of rows and columns; k a multiple of 16. x's and out's rows may be views; out overlaps nothing
    that is read; w and w_scale are contiguous. Calls of one shape give the same bits each time. A row's last bits may differ between calls of other
    numbers of rows, as sums are then taken in another order.
    ws: a workspace of the caller's, contiguous, its first 8192 bytes zero-filled once; without one the stream's is used, or
    a captured graph's own. Like `w4a16` it is no part of autograd."""
    return _calls().f8_matmul(x, x_scale, w, w_scale, None, dtype, out, ws)


def f8_expert_matmul(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor,
                     dtype=torch.bfloat16, out: torch.Tensor | None = None, ws: torch.Tensor | None = None) -> torch.Tensor:
    """`f8_matmul` by expert: rows offsets[e] to offsets[e + 1] of x (int32 [experts + 1], on the device; `expert_route`'s) take
    the matrix w[e] of [experts, n, k]. Groups are of any size, none included. Rows that no expert has are left as
    they were (undefined in a new out)."""
    if offsets is None:
        raise TypeError("offsets must be a tensor")
    return _calls().f8_matmul(x, x_scale, w, w_scale, offsets, dtype, out, ws)


def expert_route(logits: torch.Tensor, k: int, score: str = "softmax", renormalise: bool = True, gain: float = 1.0):
    """(ids, weights, rows, slots, offsets): each token's k experts of logits [tokens, experts] (float32, float16, bfloat16; at
    most 1024 experts and k of 32) and their pairs' places, laid out by expert and in each by token.

    ids int32 [tokens, k]: the experts of the largest logits, the lower of equal ones first; an expert whose logit is -inf is
    never taken, and -1 stands where none is left (a padded token has -inf everywhere). weights float32 [tokens, k]: their
    "softmax" over all experts or "sigmoid", divided by the chosen ones' sum (renormalise), times gain; 0 for -1. rows int32
    [tokens * k]: the token at each place, -1 behind the last (`f8_quantise` gathers by it). slots int32 [tokens, k]: each
    pair's place, or -1 (`expert_combine` reads it). offsets int32 [experts + 1]: where each expert's places begin
    (`f8_expert_matmul` takes it). One launch up to 64 tokens, two above; nothing comes to the host. The five are parts of one allocation
    (clone what is to be kept or saved alone). No part of autograd: the weights carry no gradient to the logits."""
    return _calls().expert_route(logits, k, score, renormalise, gain)


def expert_combine(y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor, add: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """[tokens, n] of y's type: add (a residual, or a shared expert's output) plus the sum of weights[t, j] * y[slots[t, j]] over j, in
    f32, rounded once. y [rows, n] float32, float16 or bfloat16; a slot that is no row of y adds nothing. out may be add; else it overlaps
    nothing that is read. No part of autograd."""
    return _calls().expert_combine(y, slots, weights, add, out)


def launch_count() -> int:
    return int(_lib.load().up_sm100_launch_count())
