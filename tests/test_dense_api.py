"""Refusals of the dense operators' entry points, before any device work (CPU only)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")


def _ffn(H=64, I=32, dtype=None, limit=0.0, wd=48):
    from glmx import _lib
    return _lib.Ffn(H, I, _lib.BF16 if dtype is None else dtype, 16, 32, wd, limit)


@pytest.mark.parametrize("kw,word", [(dict(H=60), b"multiples of 8"), (dict(I=0), b"multiples of 8"), (dict(dtype=1), b"dtype"),
                                     (dict(limit=-1.0), b"act_limit"), (dict(limit=float("nan")), b"act_limit"),
                                     (dict(wd=0), b"null weight"), (dict(wd=40), b"aligned")])
def test_ffn_block(kw, word):
    from glmx import _lib
    L = _lib.load()
    f = _ffn(**kw)
    assert L.glmx_ffn_forward(C.byref(f), 16, 64, 1, 16, 64, _lib.BF16, 0, 16, 0, 0, 0) == _lib.E_ARG
    assert word in L.glmx_last_error()
    assert L.glmx_ffn_backward(C.byref(f), 16, 64, 16, 64, 1, 16, 16, 16, 16, 16, 16, 16, 16, 16, 0) == _lib.E_ARG
    assert word in L.glmx_last_error()


def test_ffn_calls():
    from glmx import _lib
    L = _lib.load()
    f = _ffn()

    def fwd(x=16, ldx=64, n=1, y=16, ldy=64, ydt=_lib.BF16, h=16, p=0, q=0):
        return L.glmx_ffn_forward(C.byref(f), x, ldx, n, y, ldy, ydt, 0, h, p, q, 0)
    for kw in (dict(x=0), dict(y=0), dict(h=0), dict(n=-1), dict(ldx=56), dict(ldx=66), dict(ldy=63), dict(ydt=_lib.F16),
               dict(p=16), dict(x=8), dict(y=24), dict(h=20)):
        assert fwd(**kw) == _lib.E_ARG, kw
        assert b"glmx_ffn" in L.glmx_last_error()
    assert fwd(n=0) == _lib.OK
    assert L.glmx_ffn_forward(None, 16, 64, 1, 16, 64, _lib.BF16, 0, 16, 0, 0, 0) == _lib.E_ARG

    def bwd(dy=16, ld=64, x=16, n=1, h=16, p=16, q=16, dg=16, du=16, dx=16, a=16, b=16, c=16):
        return L.glmx_ffn_backward(C.byref(f), dy, ld, x, 64, n, h, p, q, dg, du, dx, a, b, c, 0)
    for kw in (dict(dy=0), dict(ld=60), dict(x=0), dict(h=0), dict(p=0), dict(q=0), dict(dg=0), dict(du=0), dict(n=-1), dict(dx=8),
               dict(c=20)):
        assert bwd(**kw) == _lib.E_ARG, kw


def test_int8_calls():
    from glmx import _lib
    L = _lib.load()

    def quant(x=16, dt=_lib.BF16, ldx=64, rows=1, K=64, q=16, ldq=64, s=16):
        return L.glmx_quantize_rows(x, dt, ldx, rows, K, q, ldq, s, 0)
    for kw in (dict(x=0), dict(dt=_lib.I32), dict(ldx=63), dict(rows=-1), dict(K=0), dict(q=0), dict(ldq=60), dict(s=0)):
        assert quant(**kw) == _lib.E_ARG, kw
    assert quant(rows=0) == _lib.OK

    def lin(x=16, ldx=64, xs=16, n=1, K=64, N=8, w=16, ldw=64, ws=16, y=16, ldy=8, dt=_lib.F32):
        return L.glmx_linear_i8(x, ldx, xs, n, K, N, w, ldw, ws, 0, y, ldy, dt, 0)
    for kw in (dict(x=0), dict(x=8), dict(ldx=72), dict(ldx=48), dict(xs=0), dict(n=-1), dict(K=0), dict(N=0), dict(w=0), dict(w=24),
               dict(ldw=68), dict(ws=0), dict(y=0), dict(ldy=7), dict(dt=_lib.I64),
               dict(K=_lib.I8_MAX_K + 1, ldx=131072, ldw=131072)):
        assert lin(**kw) == _lib.E_ARG, kw
        assert b"glmx_linear_i8" in L.glmx_last_error()
    assert lin(n=0) == _lib.OK


def test_sample_calls():
    from glmx import _lib
    L = _lib.load()

    def smp(l=16, dt=_lib.F32, ld=100, B=1, V=100, u=16, ids=16, idt=_lib.I64):
        return L.glmx_sample(l, dt, ld, B, V, u, 0, 1.0, 0, 0, 0, 1.0, 0, 0.0, ids, idt, 0)
    for kw in (dict(l=0), dict(dt=_lib.I32), dict(ld=99), dict(B=-1), dict(V=0), dict(V=_lib.SAMPLE_MAX_VOCAB + 1, ld=1 << 20), dict(u=0),
               dict(ids=0), dict(idt=_lib.F32)):
        assert smp(**kw) == _lib.E_ARG, kw
        assert b"glmx_sample" in L.glmx_last_error()
    assert smp(B=0) == _lib.OK


def test_host_refusals():
    """Shapes, dtypes and CPU tensors (there is no CPU path) are refused by name."""
    from glmx import GatedFFN, Int8Linear, quantize_rows, sample
    w, wd = torch.zeros(16, 32, dtype=torch.bfloat16), torch.zeros(32, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        GatedFFN(w, w, wd)
    with pytest.raises(ValueError, match="w_down"):
        GatedFFN(w, w, w)
    with pytest.raises(TypeError):
        GatedFFN(w.float(), w.float(), wd.float())
    with pytest.raises(ValueError, match="multiples of 8"):
        GatedFFN(w[:, :20], w[:, :20], wd[:20])
    with pytest.raises(TypeError):
        quantize_rows(torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        quantize_rows(torch.zeros(2, 3))
    with pytest.raises(ValueError, match="int8"):
        Int8Linear(torch.zeros(2, 3), torch.ones(2))
    with pytest.raises(ValueError, match="CUDA"):
        Int8Linear(torch.zeros(2, 3, dtype=torch.int8), torch.ones(2))
    with pytest.raises(ValueError, match="CUDA"):
        sample(torch.zeros(2, 3), torch.zeros(2))
    with pytest.raises(ValueError):
        sample(torch.zeros(3), torch.zeros(3))
    with pytest.raises(TypeError):
        sample(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2))
    with pytest.raises(ValueError):
        sample(torch.zeros(1, 400000), torch.zeros(1))
