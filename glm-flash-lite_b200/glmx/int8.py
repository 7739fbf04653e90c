"""Linear layers held in 8 bits (glmx_quantize_rows, glmx_linear_i8): int8 weights with a scale per output channel, int8
activations with a scale per token, exact 32-bit integer sums. For the linears around the routed experts: projections,
the head.

    lin = Int8Linear.from_weight(w)          # w [N, K]
    y = lin(x)                               # x [..., K] fp16 / bf16 / fp32
"""
from __future__ import annotations

import math

import torch

from . import _lib
from ._lib import check
from .ffn import _on, _raw_stream, _rows
from .layer import _dt

_PITCH = 128      # bytes between rows that are laid out here: whole lines (the product takes any multiple of 16)
_FLOAT = (torch.float16, torch.bfloat16, torch.float32)


def quantize_rows(x: torch.Tensor, stream=None):
    """x [..., K] fp16 / bf16 / fp32 -> (q int8 [..., K], scale fp32 [...]): scale = max |row| / 127, q = row / scale
    rounded to the nearest integer, ties to even (zeros and scale 0 for a row of zeros; a NaN in a row makes its scale
    NaN). Rows of q are 128 bytes aligned: the last dimension is a slice of a wider buffer where K is not a multiple
    of 128."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be [..., K] with K >= 1")
    if x.dtype not in _FLOAT:
        raise TypeError(f"x must be fp16, bf16 or fp32, not {x.dtype}")
    index = x.get_device()
    if index < 0:
        raise ValueError("x must be on a CUDA device (there is no CPU path)")
    ctx = _on(index, stream)
    if ctx is not None:
        with ctx:
            return quantize_rows(x)
    shape = x.shape
    K = shape[-1]
    x2 = x if len(shape) == 2 else x.reshape(-1, K)
    pitch, inner = x2.stride()
    if inner != 1 or pitch < K:
        x2 = x2.contiguous()
        pitch = K
    R = x2.shape[0]
    qp = (K + _PITCH - 1) // _PITCH * _PITCH
    q = x.new_empty((R, qp), dtype=torch.int8)
    s = x.new_empty(shape[:-1], dtype=torch.float32)
    rc = _lib.load().glmx_quantize_rows(x2.data_ptr(), _dt(x2), pitch, R, K, q.data_ptr(), qp, s.data_ptr(), _raw_stream(index))
    if rc:
        check(rc)
    if len(shape) != 2:
        q = q.view(*shape[:-1], qp)
    return (q if qp == K else q[..., :K]), s


def _q_rows(t: torch.Tensor, what: str, K: int) -> torch.Tensor:
    if t.dtype != torch.int8 or t.dim() < 1 or t.shape[-1] != K:
        raise ValueError(f"{what} must be int8 [..., {K}]")
    if t.dim() != 2:
        t = t.as_strided((t.numel() // K, K), (t.stride(-2), 1), t.storage_offset()) if _collapses(t) else t.reshape(-1, K)
    return _rows(t, 16, _PITCH)


def _collapses(t: torch.Tensor) -> bool:
    """Whether the leading dimensions of t are one run of equally spaced rows (quantize_rows' padded rows are)."""
    if t.dim() < 2 or t.stride(-1) != 1:
        return False
    return all(t.stride(i) == t.stride(i + 1) * t.shape[i + 1] for i in range(t.dim() - 2))


def _vec(t: torch.Tensor, shape, what: str, device) -> torch.Tensor:
    """t, fp32 with an element for each of `shape`, in its order: of that shape but for dimensions of size 1, or either of them flat"""
    if t.dtype != torch.float32 or t.get_device() != device.index or not (
            t.shape == shape or (t.numel() == math.prod(shape) and (len(shape) < 2 or t.dim() == 1 or _long(t.shape) == _long(shape)))):
        raise ValueError(f"{what} must be fp32 {list(shape)} on {device}, not {t.dtype} {list(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _long(shape) -> list:
    return [n for n in shape if n != 1]


class Int8Linear:
    """wq int8 [N, K], w_scale fp32 [N], bias fp32 [N] or None; out_dtype: fp16, bf16 or fp32, by default the input's
    dtype (bf16 for matmul). The weights are used in place; where their rows are not 16-byte aligned they are copied once."""

    def __init__(self, wq: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None, out_dtype=None):
        self.lib = _lib.load()
        if wq.dim() != 2 or wq.dtype != torch.int8 or wq.shape[0] < 1 or wq.shape[1] < 1:
            raise ValueError("wq must be int8 [N, K]")
        if wq.device.type != "cuda":
            raise ValueError("wq must be on a CUDA device (there is no CPU path)")
        if wq.shape[1] > _lib.I8_MAX_K:
            raise ValueError(f"K must be at most {_lib.I8_MAX_K} (a longer integer sum could pass 31 bits)")
        if out_dtype is not None and out_dtype not in _FLOAT:
            raise TypeError("out_dtype must be fp16, bf16 or fp32")
        self.N, self.K = int(wq.shape[0]), int(wq.shape[1])
        self.device, self.out_dtype = wq.device, out_dtype
        self._index = wq.get_device()
        with torch.cuda.device(self._index):
            self.wq = _rows(wq, 16, _PITCH)
            self.w_scale = _vec(w_scale, (self.N,), "w_scale", self.device)
            self.bias = None if bias is None else _vec(bias, (self.N,), "bias", self.device)
        self._w, self._ldw, self._ws = self.wq.data_ptr(), self.wq.stride(0), self.w_scale.data_ptr()
        self._bias = 0 if bias is None else self.bias.data_ptr()

    @classmethod
    def from_weight(cls, w: torch.Tensor, bias: torch.Tensor | None = None, out_dtype=None):
        """Quantises a weight [N, K] by its rows."""
        q, s = quantize_rows(w)
        return cls(q, s, None if bias is None else bias.float(), out_dtype)

    def matmul(self, xq: torch.Tensor, x_scale: torch.Tensor, out: torch.Tensor | None = None, out_dtype=None,
               stream=None) -> torch.Tensor:
        """y [..., N] from quantised rows xq int8 [..., K] and x_scale fp32 [...] (quantize_rows' results: one
        quantisation serves several linears; a flat x_scale has the rows' order)."""
        if xq.get_device() != self._index:
            raise ValueError(f"xq on {xq.device}, weights on {self.device}")
        ctx = _on(self._index, stream)
        if ctx is not None:
            with ctx:
                return self.matmul(xq, x_scale, out, out_dtype)
        x2 = _q_rows(xq, "xq", self.K)
        T = x2.shape[0]
        xs = _vec(x_scale, xq.shape[:-1], "x_scale", self.device)
        if out is None:
            dt = out_dtype or self.out_dtype or torch.bfloat16
            if dt not in _FLOAT:
                raise TypeError("out_dtype must be fp16, bf16 or fp32")
            out = xq.new_empty((*xq.shape[:-1], self.N), dtype=dt)
        elif out_dtype is not None and out.dtype != out_dtype:
            raise TypeError(f"out is {out.dtype}, out_dtype {out_dtype}")
        elif tuple(out.shape) != (*xq.shape[:-1], self.N) or not out.is_contiguous() or out.device != self.device or \
                out.dtype not in _FLOAT:
            raise ValueError("out must be contiguous fp16 / bf16 / fp32 [..., N] on the weights' device")
        rc = self.lib.glmx_linear_i8(x2.data_ptr(), x2.stride(0) if T else self._ldw, xs.data_ptr(), T, self.K, self.N, self._w, self._ldw,
                                     self._ws, self._bias, out.data_ptr(), self.N, _dt(out), _raw_stream(self._index))
        if rc:
            check(rc)
        return out

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """y [..., N] from x [..., K]: quantises the rows, then multiplies."""
        if x.shape[-1] != self.K:
            raise ValueError(f"x must be [..., {self.K}]")
        if x.get_device() != self._index:
            raise ValueError(f"x on {x.device}, weights on {self.device}")
        ctx = _on(self._index, stream)
        if ctx is not None:
            with ctx:
                return self(x, out)
        q, s = quantize_rows(x)
        return self.matmul(q, s, out, (self.out_dtype or x.dtype) if out is None else None)
