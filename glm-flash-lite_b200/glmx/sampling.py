"""Sampling from the head's logits with given random numbers (glmx_sample): temperature, top-k, top-p and min-p per row.
The counterpart of Router for the vocabulary: a selection over one row per token, all on the device."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check
from .ffn import _on, _raw_stream
from .layer import _dt


def _param(v, dtype, B: int, index: int, what: str):
    """v, a number or a tensor [B], as (tensor kept alive, its device address or 0, the value for all rows)"""
    if not isinstance(v, torch.Tensor):
        return None, 0, v
    if v.dim() == 0:
        v = v.expand(B)
    if tuple(v.shape) != (B,) or v.get_device() != index:
        raise ValueError(f"{what} must be a number or a tensor [{B}] on cuda:{index}")
    if v.dtype != dtype or not v.is_contiguous():
        v = v.to(dtype).contiguous()
    return v, v.data_ptr(), 0


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out_dtype=torch.int64,
           stream=None) -> torch.Tensor:
    """ids [B] (int64 or int32) for logits [B, V] (fp16, bf16 or fp32; any row distance) and u fp32 [B] in [0, 1).

    Weights are exp((l - max) / temperature). The top_k largest logits stay (0: all; ties to the lower id); of those, in
    descending order, each whose predecessors hold less than top_p of the weight left (1: all); of those, each with at
    least min_p times the largest weight; the largest always. The pick is the lowest id at which the running sum of the
    kept weights, in id order, exceeds u times their sum. temperature 0 picks the largest logit (the lowest id of equal
    ones). -inf and NaN logits are never picked; a row without any other gives -1. An infinite temperature gives
    all others the same weight.

    temperature, top_k, top_p and min_p: one number for all rows, or a tensor [B]."""
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be [B, V] with V >= 1")
    B, V = logits.shape
    if V > _lib.SAMPLE_MAX_VOCAB:
        raise ValueError(f"at most {_lib.SAMPLE_MAX_VOCAB} logits a row")
    if logits.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f"logits must be fp16, bf16 or fp32, not {logits.dtype}")
    index = logits.get_device()
    if index < 0:
        raise ValueError("logits must be on a CUDA device (there is no CPU path)")
    if out_dtype not in (torch.int64, torch.int32):
        raise TypeError("out_dtype must be int64 or int32")
    if u.dtype != torch.float32 or tuple(u.shape) != (B,) or u.get_device() != index:
        raise ValueError(f"u must be fp32 [{B}] on cuda:{index}")
    ctx = _on(index, stream)
    if ctx is not None:
        with ctx:
            return sample(logits, u, temperature, top_k, top_p, min_p, out_dtype)
    ld, inner = logits.stride()
    if inner != 1 or (B > 1 and ld < V):
        logits = logits.contiguous()
        ld = V
    if not u.is_contiguous():
        u = u.contiguous()
    t, tp, t0 = _param(temperature, torch.float32, B, index, "temperature")
    if not isinstance(top_k, torch.Tensor):
        top_k = max(0, min(int(top_k), V))
    elif top_k.dtype != torch.int32:
        # limited before the conversion, where a larger number keeps its meaning (V itself may be beyond 8 and 16 bits)
        top_k = (top_k if top_k.is_floating_point() else top_k.long()).clamp(0, V)
    k, kp, k0 = _param(top_k, torch.int32, B, index, "top_k")
    p, pp, p0 = _param(top_p, torch.float32, B, index, "top_p")
    m, mp, m0 = _param(min_p, torch.float32, B, index, "min_p")
    ids = logits.new_empty(B, dtype=out_dtype)
    rc = _lib.load().glmx_sample(logits.data_ptr(), _dt(logits), max(ld, V), B, V, u.data_ptr(), tp, t0, kp, k0, pp, p0, mp, m0,
                                 ids.data_ptr(), _dt(ids), _raw_stream(index))
    if rc:
        check(rc)
    return ids
