"""Gated feed-forward block over dense 16-bit weights (glmx_ffn_forward / glmx_ffn_backward): an unquantised shared expert
beside MoELayer's trellis experts, or one of the model's dense layers.

    g = x Wg^T, u = x Wu^T, h = min(silu(g), L) * clamp(u, -L, L), y = h Wd^T        (L = act_limit; 0 or inf: no clamp)

`GatedFFN` is the block at inference, and its forward_train / backward pair the explicit form of a training step (the one
to capture into a graph); `gated_ffn` is the same as a differentiable function.
"""
from __future__ import annotations

import ctypes as C

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib
from ._lib import check
from .layer import _dt

# the current device, and the current stream's handle without a Stream object around it; by the public way where a torch (one without
# CUDA, say) has not got these
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: int(torch.cuda.current_stream(index).cuda_stream))


def _on(index: int, stream):
    """The context in which a call allocates and launches: the tensors' device current, and `stream` (if given) current
    too, so that its temporaries belong to the stream that uses them. None where nothing has to be switched."""
    if stream is not None:
        if stream.device.index != index:
            raise ValueError(f"stream on {stream.device}, tensors on cuda:{index}")
        return torch.cuda.stream(stream)
    if index != _current_device():
        return torch.cuda.device(index)
    return None


def _rows(t: torch.Tensor, align: int, pitch_of_copy: int = 64) -> torch.Tensor:
    """t [R, n] as rows of packed elements whose distance is a multiple of `align` elements and whose start is 16-byte
    aligned; where it is not, a copy with rows a multiple of pitch_of_copy elements apart."""
    pitch, inner = t.stride()
    if inner == 1 and pitch % align == 0 and pitch >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    R, n = t.shape
    if R == 1 and inner == 1 and n % align == 0 and t.data_ptr() % 16 == 0:
        return t.as_strided((1, n), (n, 1))
    c = torch.empty((R, (n + pitch_of_copy - 1) // pitch_of_copy * pitch_of_copy), dtype=t.dtype, device=t.device)[:, :n]
    if t.dtype == torch.int8 and inner == 1 and n % 4 == 0 and pitch % 4 == 0 and pitch >= n and \
            t.storage_offset() % 4 == 0 and t.data_ptr() % 4 == 0:
        c.view(torch.int32).copy_(t.view(torch.int32))       # bytes four at a time
    else:
        c.copy_(t)
    return c


def _no_tangent(t: torch.Tensor) -> None:
    # (outside of every level no tensor has one, which is cheaper to see)
    if getattr(_forward_ad, "_current_level", 0) >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError("the gated feed-forward block has no forward-mode derivative")


def dense_check(device=None, stream=None) -> None:
    """Synchronises the stream and raises GlmxError where a dense operator on the device, on whichever stream, gave up a bounded
    wait since the last check (glmx_dense_check)."""
    index = torch.device("cuda" if device is None else device).index
    with torch.cuda.device(_current_device() if index is None else index):
        s = stream if stream is not None else torch.cuda.current_stream()
        check(_lib.load().glmx_dense_check(int(s.cuda_stream), C.byref(C.c_int())))


class GatedFFN:
    """w_gate, w_up [I, H], w_down [H, I]: bf16 or fp16 CUDA tensors of one dtype, H and I multiples of 8; act_limit as
    MoELayer's. The weights are used in place (copied once where not contiguous)."""

    def __init__(self, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, act_limit: float = 0.0):
        self.lib = _lib.load()
        if w_gate.dim() != 2 or w_up.shape != w_gate.shape or tuple(w_down.shape) != tuple(w_gate.shape[::-1]):
            raise ValueError("weights must be w_gate [I, H], w_up [I, H], w_down [H, I]")
        self.I, self.H = int(w_gate.shape[0]), int(w_gate.shape[1])
        if self.H < 8 or self.I < 8 or self.H % 8 or self.I % 8:
            raise ValueError("H and I must be positive multiples of 8")
        self.dtype, self.device = w_gate.dtype, w_gate.device
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"weights must be bf16 or fp16, not {self.dtype}")
        for w in (w_gate, w_up, w_down):
            if w.dtype != self.dtype or w.device != self.device:
                raise ValueError("weights must share one dtype and device")
        if self.device.type != "cuda":
            raise ValueError("weights must be on a CUDA device (there is no CPU path)")
        if not act_limit >= 0.0:
            raise ValueError("act_limit must be 0 (none) or positive")
        self._index = w_gate.get_device()
        self._pitch = (self.I + 63) // 64 * 64           # GLMX_FFN_PITCH: elements between hidden rows
        self.act_limit = float(act_limit)
        self._take(*(w.detach() if w.requires_grad else w for w in (w_gate, w_up, w_down)))

    def _take(self, w_gate, w_up, w_down):
        self.w_gate, self.w_up, self.w_down = self._pack(w_gate), self._pack(w_up), self._pack(w_down)
        self._desc = _lib.Ffn(self.H, self.I, _dt(w_gate), self.w_gate.data_ptr(), self.w_up.data_ptr(),
                              self.w_down.data_ptr(), self.act_limit)
        self._ref = C.byref(self._desc)

    def _bare(self):
        """The block without its weights."""
        f = GatedFFN.__new__(GatedFFN)
        f.__dict__.update(self.__dict__, w_gate=None, w_up=None, w_down=None, _desc=None, _ref=None)
        return f

    def _with(self, w_gate, w_up, w_down):
        """The same block over weights of the same shapes, dtype and device."""
        up = (self.I, self.H)
        for w, shape in ((w_gate, up), (w_up, up), (w_down, (self.H, self.I))):
            if w.dtype != self.dtype or w.get_device() != self._index or w.shape != shape:
                raise ValueError(f"weights must be the block's, {self.dtype} on {self.device}: not {w.dtype} on {w.device}")
        f = self._bare()
        f._take(w_gate, w_up, w_down)
        return f

    def _pack(self, w: torch.Tensor) -> torch.Tensor:
        _no_tangent(w)
        if w.is_contiguous() and w.data_ptr() % 16 == 0:
            return w
        with torch.cuda.device(self._index):
            return w.clone(memory_format=torch.contiguous_format)

    def _in(self, x: torch.Tensor, what: str) -> torch.Tensor:
        if x.dim() < 1 or x.shape[-1] != self.H:
            raise ValueError(f"{what} must be [..., {self.H}]")
        if x.dtype != self.dtype:
            raise TypeError(f"{what} must be {self.dtype}, not {x.dtype}")
        if x.get_device() != self._index:
            raise ValueError(f"{what} on {x.device}, weights on {self.device}")
        _no_tangent(x)
        return _rows(x if x.dim() == 2 else x.reshape(-1, self.H), 8)

    @staticmethod
    def _no_gradient(x, out) -> None:
        if torch.is_grad_enabled() and (x.requires_grad or (out is not None and out.requires_grad)):
            raise RuntimeError("GatedFFN.forward gives no gradient to x or out, which require one: use gated_ffn, or torch.no_grad()")

    def _new(self, shape, dtype=None):
        return self.w_gate.new_empty(shape) if dtype is None else self.w_gate.new_empty(shape, dtype=dtype)

    def _run(self, x, y, accumulate, h, p, q):
        rc = self.lib.glmx_ffn_forward(self._ref, x.data_ptr(), x.stride(0), x.shape[0], y.data_ptr(), self.H, _dt(y), accumulate,
                                       h.data_ptr(), p, q, _raw_stream(self._index))
        if rc:
            check(rc)

    def forward(self, x: torch.Tensor, out: torch.Tensor | None = None, out_dtype=None, accumulate: bool = False,
                stream=None) -> torch.Tensor:
        """y [..., H] for x [..., H] of the block's dtype. out_dtype: the block's dtype (default) or fp32; out: a
        contiguous tensor of x's shape to write instead, accumulate=True to add to it (a shared expert's output onto
        MoELayer.forward's). No gradient: where x or out requires one, the call is refused (gated_ffn is differentiable)."""
        self._no_gradient(x, out)
        ctx = _on(self._index, stream)
        if ctx is not None:
            with ctx:
                return self.forward(x, out, out_dtype, accumulate)
        x2 = self._in(x, "x")
        if out is None:
            if accumulate:
                raise ValueError("accumulate needs out")
            if out_dtype is not None and out_dtype not in (self.dtype, torch.float32):
                raise TypeError(f"out_dtype must be {self.dtype} or fp32")
            out = self._new(x.shape, out_dtype)
        else:
            if out.shape != x.shape or not out.is_contiguous() or out.device != self.device or out.data_ptr() % 16:
                raise ValueError("out must be contiguous, 16-byte aligned, of x's shape and device")
            if out.dtype not in (self.dtype, torch.float32) or (out_dtype is not None and out_dtype != out.dtype):
                raise TypeError(f"out must be {self.dtype} or fp32")
        n = x2.shape[0]
        if n:
            self._run(x2, out, 1 if accumulate else 0, self._new((n, self._pitch)), 0, 0)
        return out

    __call__ = forward

    # ---- training -----------------------------------------------------------------------------------------------
    def forward_train(self, x: torch.Tensor, stream=None):
        """(y, saved): y as forward's, and what backward needs: the packed input rows, the hidden rows and two fp32 factors
        per hidden value (10 bytes for each, beside x)."""
        ctx = _on(self._index, stream)
        if ctx is not None:
            with ctx:
                return self.forward_train(x)
        x2 = self._in(x, "x")
        n = x2.shape[0]
        y, h, pq = self._new(x.shape), self._new((n, self._pitch)), self._new((2, n, self.I), torch.float32)
        if n:
            p = pq.data_ptr()
            self._run(x2, y, 0, h, p, p + 4 * n * self.I)
        return y, (x2, h, pq)

    def backward(self, dy: torch.Tensor, saved, need=(True, True, True, True), stream=None):
        """(dx, dw_gate, dw_up, dw_down) for dy [..., H] from forward_train's saved; None where need says so."""
        ctx = _on(self._index, stream)
        if ctx is not None:
            with ctx:
                return self.backward(dy, saved, need)
        dy2 = self._in(dy, "dy")
        x, h, pq = saved
        n = x.shape[0]
        if dy2.shape[0] != n:
            raise ValueError("dy must have the forward call's rows")
        if x.shape != (n, self.H) or h.shape != (n, self._pitch) or pq.shape != (2, n, self.I):
            raise ValueError("saved must be of a forward_train call of this block")
        # (they may have been elsewhere in between: offloaded, or packed by a saved-tensor hook)
        for t, dt in ((x, self.dtype), (h, self.dtype), (pq, torch.float32)):
            if t.get_device() != self._index or t.dtype != dt or not (t is x or t.is_contiguous()):
                raise ValueError(f"saved must be forward_train's tensors, on {self.device}: not {t.dtype} on {t.device}")
        x = _rows(x, 8)
        H, I, new = self.H, self.I, self._new
        dx = new(dy.shape) if need[0] else None
        dwg = new((I, H)) if need[1] else None
        dwu = new((I, H)) if need[2] else None
        dwd = new((H, I)) if need[3] else None
        inner = new((2, n, self._pitch)) if n and (need[0] or need[1] or need[2]) else None
        ptr = lambda t: 0 if t is None else t.data_ptr()
        p, g = pq.data_ptr(), ptr(inner)
        rc = self.lib.glmx_ffn_backward(self._ref, dy2.data_ptr(), dy2.stride(0) if n else H, x.data_ptr(), x.stride(0) if n else H, n,
                                        h.data_ptr(), p, p + 4 * n * I, g, g and g + 2 * n * self._pitch, ptr(dx), ptr(dwg), ptr(dwu),
                                        ptr(dwd), _raw_stream(self._index))
        if rc:
            check(rc)
        return dx, dwg, dwu, dwd


class _GatedFFNFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act_limit):
        ffn = GatedFFN(w_gate, w_up, w_down, act_limit)
        if not any(ctx.needs_input_grad[:4]):
            return ffn.forward(x)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gated_ffn: a differentiated call cannot be captured into a graph (an eager graph of the "
                               "same leaves would tie the capture to another stream); capture GatedFFN.forward_train and "
                               "GatedFFN.backward")
        y, saved = ffn.forward_train(x)
        ctx.save_for_backward(*saved, w_gate, w_up, w_down)
        ctx.block = ffn._bare()
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_ffn is differentiable once (create_graph is not supported)")
        # the weights as they are unpacked here, not where they were in the forward call: their storage may have moved, or a hook may
        # have kept them elsewhere (and an error here where a weight was changed in between)
        *saved, w_gate, w_up, w_down = ctx.saved_tensors
        return (*ctx.block._with(w_gate, w_up, w_down).backward(dy, saved, ctx.needs_input_grad), None)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              act_limit: float = 0.0) -> torch.Tensor:
    """The block as a differentiable function of x and its weights (once differentiable; not in a graph capture: see
    GatedFFN.forward_train)."""
    if not torch.is_grad_enabled():              # a Function's needs_input_grad does not tell: nothing is to be kept
        return GatedFFN(w_gate, w_up, w_down, act_limit).forward(x)
    return _GatedFFNFunction.apply(x, w_gate, w_up, w_down, float(act_limit))
