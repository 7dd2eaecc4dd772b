"""Layers of a served language model's decoder block over the HIP backend.

  RmsNormQuantLayer     RMS norm + residual into 8-bit rows with scales
  QuantMatMulLayer      product of 8-bit rows with bias, activation, residual
  PagedKvCache          pages of keys and values, and the sequences' page table
  WindowAttentionLayer  causal attention with a sliding window and sinks over it

The C ABI (include/osh_hip.h: osh_rms_norm_quant, osh_quant_matmul,
osh_window_attention) holds the formulas and the limits.  Tensors are device
tensors; calls run on the current stream of the tensors' device, allocate only
what they return (and torch-allocated scratch), and never synchronize, so they can
be captured into a graph.  OnnxSharp has none of these operators; errors follow the
other layers: OshError for arguments that do not fit together, OshUnsupported for
sizes the backend does not take.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import torch

from . import native as N

_ROW_TYPES = {torch.float32: N.T_F32, torch.float16: N.T_F16, torch.bfloat16: N.T_BF16}
_Q_TYPES = {"int8": (N.T_I8, torch.int8), "e4m3": (N.T_E4M3, torch.float8_e4m3fn)}
_Q_CODES = {torch.int8: N.T_I8, torch.float8_e4m3fn: N.T_E4M3}
_ACTIVATIONS = {None: N.ACT_NONE, "Relu": N.ACT_RELU, "Silu": N.ACT_SILU, "Gelu": N.ACT_GELU}
_MAX_INT = 2 ** 31 - 1
# the fields of osh_window_attn in order (packing them costs a third of assigning them)
_WINDOW_ATTN = struct.Struct("@12ifiq9P8q6qq")


def _invalid(layer, message: str) -> N.OshError:
    return N.OshError(N.OSH_E_INVALID, f"{type(layer).__name__} '{layer.name}': {message}")


def _check_tensor(layer, what: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{type(layer).__name__} '{layer.name}': {what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise _invalid(layer, f"{what} must have the shape {tuple(shape)}, got {tuple(t.shape)}")


def _check_device(layer, *tensors) -> torch.device:
    """The one device of all tensors (None entries are left out)."""
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError(f"{type(layer).__name__} '{layer.name}': device tensors are needed, got {device}")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{type(layer).__name__} '{layer.name}': tensors on {device} and {t.device}")
    return device


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with its last dimension contiguous and no negative or shared rows."""
    if t.is_contiguous() or (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] == 1):
        return t
    return t.contiguous()


def _pitch(t: Optional[torch.Tensor]) -> int:
    if t is None:
        return 0
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else max(cols, 1)


def _call(device: torch.device, name: str, *args) -> None:
    """A launch on the current stream of `device`.

    Asks torch for the raw stream: the Stream object that torch.cuda.current_stream builds
    costs 4 us of the 12 that a small call takes on the host."""
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            N.check(getattr(N.lib(), name)(*args, torch._C._cuda_getCurrentRawStream(device.index)))
        return
    N.check(getattr(N.lib(), name)(*args, torch._C._cuda_getCurrentRawStream(device.index)))


class RmsNormQuantLayer:
    """h = x + residual, and its RMS norm times gamma in 8 bits with a scale a row.

    q_type "e4m3" (torch.float8_e4m3fn) or "int8"; row i stands for q[i] * scale[i]."""

    def __init__(self, eps: float = 1e-5, q_type: str = "e4m3", name: str = "rms_norm_quant"):
        if q_type not in _Q_TYPES:
            raise ValueError(f"RmsNormQuantLayer '{name}': q_type {q_type!r} is not one of {sorted(_Q_TYPES)}")
        if not eps >= 0.0:
            raise ValueError(f"RmsNormQuantLayer '{name}': eps {eps} is negative")
        self.eps, self.q_type, self.name = float(eps), q_type, name

    def forward(self, x: torch.Tensor, gamma: torch.Tensor, residual: Optional[torch.Tensor] = None,
                out_h: Optional[torch.Tensor] = None):
        """(h, q, scale) of rows x [rows, cols] of float32, float16 or bfloat16.

        h is x itself without a residual; out_h (which may be x or residual) receives
        it otherwise."""
        if x.dtype not in _ROW_TYPES:
            raise TypeError(f"RmsNormQuantLayer '{self.name}': x must be float32, float16 or bfloat16, got {x.dtype}")
        if x.dim() != 2:
            raise _invalid(self, f"x must be [rows, cols], got {tuple(x.shape)}")
        rows, cols = x.shape
        _check_tensor(self, "gamma", gamma, x.dtype, (cols,))
        if residual is not None:
            _check_tensor(self, "residual", residual, x.dtype, x.shape)
        if out_h is not None:
            if residual is None:
                raise _invalid(self, "out_h without a residual: h is x")
            _check_tensor(self, "out_h", out_h, x.dtype, x.shape)
            if out_h is not _rows(out_h):
                raise _invalid(self, "out_h must have contiguous rows")
        device = _check_device(self, x, gamma, residual, out_h)
        code, q_dtype = _Q_TYPES[self.q_type]
        q = torch.empty((rows, cols), dtype=q_dtype, device=device)
        scale = torch.empty(rows, dtype=torch.float32, device=device)
        xr, h = _rows(x), x
        if residual is not None:
            residual = _rows(residual)
            h = torch.empty((rows, cols), dtype=x.dtype, device=device) if out_h is None else out_h
        if gamma.stride(0) != 1:
            gamma = gamma.contiguous()
        _call(device, "osh_rms_norm_quant", rows, cols, _ROW_TYPES[x.dtype], xr.data_ptr(), _pitch(xr),
              None if residual is None else residual.data_ptr(), _pitch(residual), gamma.data_ptr(), self.eps,
              None if residual is None else h.data_ptr(), 0 if residual is None else _pitch(h), code, q.data_ptr(),
              _pitch(q), scale.data_ptr())
        return h, q, scale


class QuantMatMulLayer:
    """y = act((a * a_scale) @ (w * w_scale).T + bias) + residual of 8-bit a and w.

    activation None, "Relu", "Silu" or "Gelu" (with erf); out_dtype float32, float16 or
    bfloat16.  float8_e4m3fn sums are FP32 for float32 outputs (at up to 2.3 times the
    time of a 16-bit one), those of the 8-bit matrix instruction, 1.5e-5 of the result
    off, for the others."""

    def __init__(self, activation: Optional[str] = None, out_dtype: torch.dtype = torch.bfloat16,
                 name: str = "quant_matmul"):
        if activation not in _ACTIVATIONS:
            raise ValueError(f"QuantMatMulLayer '{name}': activation {activation!r} cannot be fused")
        if out_dtype not in _ROW_TYPES:
            raise ValueError(f"QuantMatMulLayer '{name}': out_dtype {out_dtype} is not float32, float16 or bfloat16")
        self.activation, self.out_dtype, self.name = activation, out_dtype, name

    def forward(self, a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y [m, n] of a [m, k], w [n, k] (both int8 or both float8_e4m3fn), a_scale [m],
        w_scale [n] and bias [n] in float32, residual [m, n] in the output's type.  out may
        be the residual."""
        if a.dtype not in _Q_CODES or w.dtype != a.dtype:
            raise TypeError(f"QuantMatMulLayer '{self.name}': a and w must both be int8 or both float8_e4m3fn, "
                            f"got {a.dtype} and {w.dtype}")
        if a.dim() != 2 or w.dim() != 2 or a.shape[1] != w.shape[1]:
            raise _invalid(self, f"a {tuple(a.shape)} and w {tuple(w.shape)} must be [m, k] and [n, k]")
        m, k = a.shape
        n = w.shape[0]
        _check_tensor(self, "a_scale", a_scale, torch.float32, (m,))
        _check_tensor(self, "w_scale", w_scale, torch.float32, (n,))
        if bias is not None:
            _check_tensor(self, "bias", bias, torch.float32, (n,))
            bias = bias.contiguous()
        if residual is not None:
            _check_tensor(self, "residual", residual, self.out_dtype, (m, n))
        if out is not None:
            _check_tensor(self, "out", out, self.out_dtype, (m, n))
            if out is not _rows(out):
                raise _invalid(self, "out must have contiguous rows")
        device = _check_device(self, a, a_scale, w, w_scale, bias, residual, out)
        a, w, a_scale, w_scale = _rows(a), _rows(w), a_scale.contiguous(), w_scale.contiguous()
        if residual is not None:
            residual = _rows(residual)
        if out is None:
            out = torch.empty((m, n), dtype=self.out_dtype, device=device)
        _call(device, "osh_quant_matmul", m, n, k, _Q_CODES[a.dtype], a.data_ptr(), _pitch(a), a_scale.data_ptr(),
              w.data_ptr(), _pitch(w), w_scale.data_ptr(), None if bias is None else bias.data_ptr(),
              _ACTIVATIONS[self.activation], _ROW_TYPES[self.out_dtype],
              None if residual is None else residual.data_ptr(), _pitch(residual), out.data_ptr(), _pitch(out))
        return out


class PagedKvCache:
    """Pages of keys and values, and which pages each sequence holds.

    k_pages and v_pages are [pages, page, kv_heads, head_dim] of float16 or bfloat16 (any
    strides with contiguous head values, no two slots in the same memory); table [batch, width] int32: position p of
    sequence b lies in slot p % page of page table[b, p // page].  Entries that no query
    sees (before the window, past the length) may hold anything."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, name: str = "kv_cache"):
        self.name = name
        if k_pages.dim() != 4:
            raise _invalid(self, f"pages must be [pages, page, kv_heads, head_dim], got {tuple(k_pages.shape)}")
        if k_pages.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"PagedKvCache '{name}': pages must be float16 or bfloat16, got {k_pages.dtype}")
        _check_tensor(self, "v_pages", v_pages, k_pages.dtype, k_pages.shape)
        if table.dtype != torch.int32:
            raise TypeError(f"PagedKvCache '{name}': table must be torch.int32, got {table.dtype}")
        if table.dim() != 2:
            raise _invalid(self, f"table must be [batch, width], got {tuple(table.shape)}")
        if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
            raise _invalid(self, "a head's values must be contiguous")
        if table.shape[1] > 1 and table.stride(1) != 1 or table.shape[0] > 1 and table.stride(0) < table.shape[1]:
            raise _invalid(self, "a sequence's table row must be contiguous")
        self.k_pages, self.v_pages, self.table = k_pages, v_pages, table


class WindowAttentionLayer:
    """Causal attention with a sliding window and sinks over a PagedKvCache.

    A query at position p sees j <= p with j > p - window (window None: all) or
    j < sinks.  scale None: 1 / sqrt(head_dim)."""

    def __init__(self, window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None,
                 name: str = "window_attention"):
        if window is not None and window < 1 or sinks < 0:
            raise ValueError(f"WindowAttentionLayer '{name}': window {window}, sinks {sinks}")
        # as a float: 0 stands for 1 / sqrt(head_dim), and times log2(e) it stays finite
        if scale is not None and not 2.0 ** -126 <= scale <= 2e38:
            raise ValueError(f"WindowAttentionLayer '{name}': scale {scale}")
        self.window, self.sinks, self.scale, self.name = window, sinks, scale, name

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedKvCache,
                cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, max_q: int, max_kv: int,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """o [tokens, q_heads, head_dim] for the new tokens' q, and k and v
        [tokens, kv_heads, head_dim], which go to their pages.

        cu_seqlens [batch + 1] int32, ascending: sequence b's tokens are rows cu_seqlens[b]
        to cu_seqlens[b + 1]; kv_lens [batch] int32: its length with them; max_q and max_kv:
        upper bounds of new and whole lengths, known to the host.  A sequence whose lengths
        contradict them gets NaN; rows of no sequence are not written."""
        kp, vp, table = cache.k_pages, cache.v_pages, cache.table
        pages, page, kv_heads, d = kp.shape
        batch, width = table.shape
        if q.dim() != 3 or q.shape[2] != d:
            raise _invalid(self, f"q must be [tokens, heads, {d}], got {tuple(q.shape)}")
        tokens, q_heads = q.shape[0], q.shape[1]
        if q.dtype != kp.dtype:
            raise TypeError(f"WindowAttentionLayer '{self.name}': q is {q.dtype}, the cache {kp.dtype}")
        _check_tensor(self, "k", k, kp.dtype, (tokens, kv_heads, d))
        _check_tensor(self, "v", v, kp.dtype, (tokens, kv_heads, d))
        _check_tensor(self, "cu_seqlens", cu_seqlens, torch.int32, (batch + 1,))
        _check_tensor(self, "kv_lens", kv_lens, torch.int32, (batch,))
        if tokens and (batch == 0 or max_q < 1):
            raise _invalid(self, f"{tokens} tokens, but {batch} sequences of at most {max_q} new ones")
        if not 0 <= max_q <= max_kv <= _MAX_INT:
            raise _invalid(self, f"max_q {max_q} and max_kv {max_kv}")
        if out is not None:
            _check_tensor(self, "out", out, kp.dtype, q.shape)
            if out.stride(2) != 1:
                raise _invalid(self, "out must have contiguous heads")
        device = _check_device(self, q, k, v, kp, vp, table, cu_seqlens, kv_lens, out)
        q, k, v = (t if t.stride(2) == 1 else t.contiguous() for t in (q, k, v))
        cu_seqlens, kv_lens = cu_seqlens.contiguous(), kv_lens.contiguous()
        if out is None:
            out = torch.empty((tokens, q_heads, d), dtype=q.dtype, device=device)
        p = N.WindowAttn.from_buffer_copy(_WINDOW_ATTN.pack(
            _ROW_TYPES[q.dtype], batch, q_heads, kv_heads, d,
            _MAX_INT if self.window is None else min(self.window, _MAX_INT), min(self.sinks, _MAX_INT),
            max_q, max_kv, pages, page, width, 0.0 if self.scale is None else self.scale, 0, tokens,
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), kp.data_ptr(), vp.data_ptr(), table.data_ptr(),
            cu_seqlens.data_ptr(), kv_lens.data_ptr(), *q.stride()[:2], *k.stride()[:2], *v.stride()[:2],
            *out.stride()[:2], *kp.stride()[:3], *vp.stride()[:3], table.stride(0)))
        size = C.c_size_t()
        N.call("osh_window_attention_scratch_bytes", C.byref(p), C.byref(size))
        scratch = torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None
        _call(device, "osh_window_attention", C.byref(p), None if scratch is None else scratch.data_ptr())
        return out
