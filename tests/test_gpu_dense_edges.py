"""Calls of the dense operators at the edges of what their documentation allows, on the GPU.

Tolerances count roundings. r(t) = torch.finfo(t).eps / 2 is one rounding to t."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    from glmx import dense_check
    dense_check()


def r(t):
    return torch.finfo(t).eps / 2


# ---- sampling ----------------------------------------------------------------------------------------------------------

def picks(logits, u, temperature, top_k, top_p, min_p):
    """The documented pick, row by row in 64 bits; an infinite temperature is the limit of large ones: equal weights."""
    out = []
    for b, l in enumerate(logits.double().cpu()):
        l = torch.where(l.isnan(), torch.full_like(l, -math.inf), l)
        m = float(l.max())
        if m == -math.inf:
            out.append(-1)
            continue
        if math.isinf(temperature):
            w = (l > -math.inf).double()
        else:
            w = torch.exp((l - m) / temperature)
        order = torch.sort(l, descending=True, stable=True).indices
        if 0 < top_k < l.numel():
            order = order[:top_k]
        ws = w[order]
        if top_p < 1:
            before = torch.cumsum(ws, 0) - ws
            n = max(1, int((before < top_p * ws.sum()).sum()))
            order, ws = order[:n], ws[:n]
        ok = ws >= min_p
        ok[0] = True
        ids = order[ok].sort().values
        c = torch.cumsum(w[ids], 0)
        out.append(int(ids[(c > float(u[b]) * c[-1]).nonzero()[0]]))
    return out


FILTERS = [dict(), dict(min_p=0.25), dict(top_k=5), dict(top_k=700), dict(top_p=0.5), dict(top_k=900, top_p=0.75, min_p=0.25)]


@pytest.mark.parametrize("kw", FILTERS, ids=lambda kw: "-".join(kw) + str(kw.get("top_k", "")) or "plain")
@pytest.mark.parametrize("dt", [F32, BF, HF], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,start", [(1, 0), (33, 0), (1000, 3), (4099, 1), (20011, 7)])
def test_sample_infinite_temperature(dev, V, start, dt, kw):
    """Every logit that may be picked has the same weight, and none that may not has any: masked and NaN ones, and what lies around rows
    of odd length and start."""
    from glmx import sample
    B = 6
    gen = torch.Generator(device=dev).manual_seed(V + start)
    wide = torch.full((B, start + V + 5), 100.0, device=dev, dtype=dt)
    l = wide[:, start:start + V]
    l.copy_((torch.randn(B, V, generator=gen, device=dev) * 3).to(dt))
    if V > 1:
        l[1, torch.rand(V, generator=gen, device=dev) < 0.97] = -math.inf
        l[2, ::2] = math.nan
        l[3] = -math.inf
        l[3, V // 2] = -7.0
        l[4, 1:] = -math.inf
    u = torch.rand(B, generator=gen, device=dev)
    f = dict(top_k=0, top_p=1.0, min_p=0.0) | kw
    want = picks(l, u, math.inf, **f)
    assert sample(l, u, temperature=math.inf, **kw).tolist() == want
    temps = torch.full((B,), math.inf, device=dev)
    assert sample(l, u, temperature=temps, **kw).tolist() == want
    temps[::2] = 0.8                                         # each row has its own
    got = sample(l, u, temperature=temps, **kw).tolist()
    assert got[1::2] == want[1::2] and got[::2] == picks(l[::2], u[::2], 0.8, **f)


def test_sample_logits_further_apart_than_fp32(dev):
    """The difference of two finite logits may pass the largest fp32 number; the weights of such are as of any others."""
    from glmx import sample
    l = torch.tensor([[3e38, -3e38, 0.0, 1e38]], device=dev)
    for T in (1e38, 3e38, math.inf):
        for u in (0.05, 0.3, 0.45, 0.55, 0.7, 0.95):
            assert sample(l, torch.tensor([u], device=dev), temperature=T).tolist() == picks(l, [u], float(torch.tensor(T)), 0, 1.0, 0.0)


# ---- gated feed-forward ------------------------------------------------------------------------------------------------

def block(dev, T, H, I, dt, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)
    x = rn(T, H).to(dt)
    wg, wu = (rn(I, H) * (1.2 / math.sqrt(H))).to(dt), (rn(I, H) * (1.2 / math.sqrt(H))).to(dt)
    return x, wg, wu, (rn(H, I) / math.sqrt(I)).to(dt), rn(T, H).to(dt)


def test_gated_ffn_reads_the_weights_that_were_saved(dev):
    """The backward pass takes the weights from where autograd has them: kept on the host by a hook, or in a storage that was given
    back and filled again since the forward call."""
    from glmx import gated_ffn
    for T in (5, 300):
        x, *ws, dy = block(dev, T, 256, 136, BF, 400 + T)
        for strided in (False, True):
            def leaves():
                out = [x.clone().requires_grad_(True)]
                for w in ws:
                    w = w.t().contiguous().t() if strided else w.clone()
                    out.append(w.requires_grad_(True))
                return out
            plain = leaves()
            want = torch.autograd.grad(gated_ffn(*plain, act_limit=2.0), plain, dy)
            kept = leaves()
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(dev)):
                y = gated_ffn(*kept, act_limit=2.0)
            for w in kept[1:]:
                w.data.zero_()                               # (unseen by autograd: the hook has the values)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, kept, dy), want))
            if strided:
                continue
            moved = leaves()
            y = gated_ffn(*moved, act_limit=2.0)
            sizes = [w.untyped_storage().size() for w in moved[1:]]
            for w in moved[1:]:
                w.untyped_storage().resize_(0)
            junk = [torch.full((n // 2,), math.nan, device=dev, dtype=BF) for n in sizes]
            for w, n, v in zip(moved[1:], sizes, ws):
                w.untyped_storage().resize_(n)
                w.data.copy_(v)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, moved, dy), want))
            del junk


def test_ffn_saved_tensors_that_were_elsewhere(dev):
    """What forward_train saved may be kept on the host meanwhile, and is refused unless it came back as it was."""
    from glmx import GatedFFN, gated_ffn
    x, wg, wu, wd, dy = block(dev, 40, 128, 72, HF, 431)
    ffn = GatedFFN(wg, wu, wd)
    _, saved = ffn.forward_train(x)
    want = ffn.backward(dy, saved)
    assert all(torch.equal(a, b) for a, b in zip(ffn.backward(dy, [t.cpu().to(dev) for t in saved]), want))
    wide = torch.zeros(40, 140, device=dev, dtype=HF)
    wide[:, 5:133] = x                                       # rows of another distance and alignment: laid out again
    assert all(torch.equal(a, b) for a, b in zip(ffn.backward(dy, (wide[:, 5:133], *saved[1:])), want))
    for i in range(3):
        for bad in (saved[i].cpu(), saved[i].bfloat16(), saved[i][..., :-8], saved[i][:1]):
            with pytest.raises(ValueError, match="saved|rows"):
                ffn.backward(dy, [bad if j == i else t for j, t in enumerate(saved)])
    with pytest.raises(ValueError, match="saved"):
        ffn.backward(dy, (saved[0], saved[1].t().contiguous().t(), saved[2]))
    leaf = wg.clone().requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
        y = gated_ffn(x, leaf, wu, wd)
    with pytest.raises(ValueError, match="cpu"):
        y.backward(dy)


def masks_are_exact(x, wg, wu, wd, limits):
    """forward_train's factors are zero where the value in 64 bits is past the limit, and only there or where they are by themselves: a
    sum's own error, at most 5 2^-28 (K + 96) (|x| |w| + |sum|), may make a value 0 that is not."""
    from glmx import GatedFFN
    xd, gd, ud = x.double(), wg.double(), wu.double()
    g, u = xd @ gd.t(), xd @ ud.t()
    act = g * torch.sigmoid(g)
    err = lambda w, v: 5 * 2.0 ** -28 * (x.shape[1] + 96) * (xd.norm(dim=1)[:, None] * w.norm(dim=1)[None] + v.abs())
    eg, eu = err(gd, g), err(ud, u)
    for L in limits:
        _, (_, _, pq) = GatedFFN(wg, wu, wd, act_limit=L).forward_train(x)
        p, q = pq[0], pq[1]
        inside, below = u.abs() <= L, act <= L
        assert bool((p[~inside] == 0).all()) and bool((p[inside & (g.abs() > eg)] != 0).all()), L
        # (silu' is at least 1/2 from g = 0 on)
        assert bool((q[~below] == 0).all()) and bool((q[below & (g > eg) & (u.abs() > eu)] != 0).all()), L


def near_values(x, wg, wu, lo, hi, n, seed):
    """n limits that are the fp32 numbers next to values of the block between lo and hi"""
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    v = torch.cat([(g * torch.sigmoid(g)).flatten(), u.abs().flatten()])
    v = v[(v > lo) & (v < hi)]
    pick = torch.randint(0, v.numel(), (n,), generator=torch.Generator(device=x.device).manual_seed(seed), device=x.device)
    return [float(torch.tensor(t, dtype=F32)) for t in v[pick].tolist()]


# few and many rows, with and without room for the rows' norms in the output (2 I + T against T H values)
@pytest.mark.parametrize("T,H,I", [(1, 64, 256), (3, 64, 2000), (5, 6144, 256), (70, 2048, 512), (700, 1032, 776), (900, 6144, 264)])
def test_ffn_limit_far_below_the_sums(dev, T, H, I):
    """The limit may be small beside the sums that are compared with it."""
    x, wg, wu, wd, _ = block(dev, T, H, I, BF, 600 + T)
    masks_are_exact(x, wg, wu, wd, near_values(x, wg, wu, 0.003, 0.03, 10, T))


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,H,I", [(2, 64, 256), (6, 6144, 256), (40, 1160, 488), (700, 2048, 776)])
def test_ffn_limit_with_cancelling_channels(dev, T, H, I, dt):
    """Channels that cancel, at the row's ends: the sums between them are far larger than what is compared with the limit."""
    x, wg, wu, wd, _ = block(dev, T, H, I, dt, 700 + T)
    for k, v in ((0, 1.0), (1, 1.0), (H - 2, -1.0), (H - 1, -1.0)):
        x[:, k] = v * 24
        wg[:, k] = 8
        wu[:, k] = 8
    masks_are_exact(x, wg, wu, wd, near_values(x, wg, wu, 0.5, 3.0, 6, T) + near_values(x, wg, wu, 0.01, 0.1, 6, T + 1))


def test_ffn_limit_with_an_output_that_cannot_hold_norms(dev):
    """The output serves as scratch only where it is apart from the input, packed and not added to; its values are the same."""
    import ctypes as C
    from glmx import GatedFFN, _lib
    T, H, I = 20, 512, 64
    x, wg, wu, wd, _ = block(dev, T, H, I, BF, 801)
    L = near_values(x, wg, wu, 0.01, 0.1, 1, 5)[0]
    ffn = GatedFFN(wg, wu, wd, act_limit=L)
    y, (_, h, pq) = ffn.forward_train(x)
    st = torch.cuda.current_stream().cuda_stream

    def call(xx, out, ldy, accumulate):
        h2, pq2 = torch.empty_like(h), torch.empty_like(pq)
        assert _lib.load().glmx_ffn_forward(C.byref(ffn._desc), xx.data_ptr(), xx.stride(0), T, out.data_ptr(), ldy, _lib.BF16, accumulate,
                                            h2.data_ptr(), pq2[0].data_ptr(), pq2[1].data_ptr(), st) == _lib.OK
        assert torch.equal(pq2, pq) and torch.equal(h2[:, :I], h[:, :I])
    wide = torch.full((T, H + 8), 7.0, device=dev, dtype=BF)
    call(x, wide, H + 8, 0)
    assert torch.equal(wide[:, :H], y) and bool((wide[:, H:] == 7).all())
    out = torch.zeros_like(y)
    call(x, out, H, 1)
    assert torch.equal(out, y)
    same = x.clone()
    call(same, same, H, 0)
    assert torch.equal(same, y)
    lap = torch.zeros(2 * T, H, device=dev, dtype=BF)        # the output begins in the middle of the input's rows
    lap[:T] = x
    call(lap[:T], lap[T // 2:T // 2 + T], H, 0)
    assert torch.equal(lap[T // 2:T // 2 + T], y)


def test_ffn_limit_with_rows_of_zeros_infinities_and_nan(dev):
    """Rows whose norm is 0, infinite or NaN leave the others as they are."""
    from glmx import GatedFFN
    for T in (6, 300):
        x, wg, wu, wd, dy = block(dev, T, 512, 136, BF, 811)
        ffn = GatedFFN(wg, wu, wd, act_limit=0.75)
        y, (_, h, pq) = ffn.forward_train(x)
        x[1], x[3, 5], x[4, 7], x[5, 2] = 0, math.inf, math.nan, 3e38
        y2, (_, h2, pq2) = ffn.forward_train(x)
        keep = [i for i in range(T) if i not in (1, 3, 4, 5)]
        assert torch.equal(y2[keep], y[keep]) and torch.equal(pq2[:, keep], pq[:, keep])
        assert bool((y2[1] == 0).all()) and bool((pq2[:, 1] == 0).all()) and bool(y2[4].isnan().all())
        u = (x[5:6].double() @ wu.double().t())[0]
        assert torch.equal(pq2[0, 5] == 0, (u.abs() > 0.75) | (pq2[0, 5] == 0)) and bool(torch.isfinite(y2[5]).all())


# ---- first calls -------------------------------------------------------------------------------------------------------

def test_first_calls_of_several_threads_at_once():
    """A process whose threads make their first calls together gives the bits of one that makes them one after the other."""
    import subprocess
    import sys
    from conftest import PKG
    code = """
import hashlib, sys, threading, torch
sys.path.insert(0, %r)
import glmx
d, together = 'cuda', sys.argv[1] == 'together'
g = torch.Generator(device=d).manual_seed(1)
rn = lambda *s: torch.randn(*s, generator=g, device=d)
w, wd, dy = (rn(776, 1024) / 32).bfloat16(), (rn(1024, 776) / 28).bfloat16(), rn(40, 1024).bfloat16()
xs = [rn(n, 1024).bfloat16() for n in (1, 7, 40, 40, 200, 7, 1, 200)]
u = torch.rand(200, generator=g, device=d)
wq, ws = torch.randint(-99, 99, (776, 1024), device=d, dtype=torch.int8, generator=g), torch.rand(776, device=d, generator=g)
ffn, lin = glmx.GatedFFN(w, w, wd), glmx.Int8Linear(wq, ws)
torch.cuda.synchronize()
out, start = [None] * len(xs), threading.Barrier(len(xs))
def run(i):
    torch.cuda.set_device(0)
    if together:
        start.wait()
    x = xs[i]
    with torch.cuda.stream(torch.cuda.Stream()):
        y, saved = ffn.forward_train(x)
        r = (y, *ffn.backward(x, saved), lin(x), glmx.sample(y, u[:len(x)], top_p=0.9))
        torch.cuda.current_stream().synchronize()
    out[i] = r
threads = [threading.Thread(target=run, args=(i,)) for i in range(len(xs))]
for t in threads:
    t.start()
    if not together:
        t.join()
for t in threads:
    t.join()
glmx.dense_check()
h = hashlib.sha256()
for r in out:
    for t in r:
        h.update(t.float().cpu().numpy().tobytes())
print('digest', h.hexdigest())
""" % PKG
    digest = []
    for how in ("one by one", "together", "together", "together"):
        r = subprocess.run([sys.executable, "-c", code, how], capture_output=True, text=True, timeout=240)
        assert r.returncode == 0 and "digest" in r.stdout, r.stderr[-2000:]
        digest.append(r.stdout.split("digest")[1].strip())
    assert len(set(digest)) == 1


# ---- gradients that a call does not give -------------------------------------------------------------------------------

def test_ffn_refuses_to_drop_a_gradient(dev):
    """The inference calls refuse tensors that require a gradient, unless gradients are off; nothing is written then."""
    from glmx import GatedFFN, MoELayer, gated_ffn, synth
    x, wg, wu, wd, _ = block(dev, 4, 512, 96, HF, 901)
    ffn = GatedFFN(wg.requires_grad_(True), wu, wd)          # (the weights of a block are constants of its calls)
    want = ffn(x)
    assert not want.requires_grad
    leaf, out = x.clone().requires_grad_(True), torch.zeros_like(x).requires_grad_(True)
    layer = MoELayer.from_bank(synth.make_bank(512, 256, 8, shared=False, seed=3), device=dev)
    sel, w = torch.tensor([[0, 1]] * 4, dtype=torch.int32, device=dev), torch.full((4, 2), 0.5, device=dev)
    held = torch.zeros(4, 512, device=dev)
    for call in (lambda: ffn(leaf), lambda: ffn(leaf * 2), lambda: ffn(x, out=out), lambda: ffn(x, out=out, accumulate=True),
                 lambda: ffn(leaf, stream=torch.cuda.current_stream()), lambda: layer.forward(leaf, sel, w, out=held, dense_shared=ffn)):
        with pytest.raises(RuntimeError, match="gated_ffn"):
            call()
    assert float(out.detach().abs().max()) == 0 and float(held.abs().max()) == 0
    with torch.no_grad():
        assert torch.equal(ffn(leaf), want) and torch.equal(ffn(x, out=out), want)
        assert torch.equal(layer.forward(leaf, sel, w, dense_shared=ffn), layer.forward(x, sel, w, dense_shared=ffn))
    assert torch.equal(ffn(leaf.detach()), want)
    # leading tangents are refused with gradients on and off
    import torch.autograd.forward_ad as fw
    for on in (False, True):
        with torch.set_grad_enabled(on), fw.dual_level():
            dual = fw.make_dual(x, torch.ones_like(x))
            dual_w = fw.make_dual(wu, torch.ones_like(wu))
            for call in (lambda: gated_ffn(dual, wg, wu, wd), lambda: gated_ffn(x, wg, dual_w, wd), lambda: ffn(dual),
                         lambda: ffn.forward_train(dual), lambda: GatedFFN(wg, dual_w, wd)):
                with pytest.raises((RuntimeError, NotImplementedError)):
                    call()
    assert torch.equal(ffn(x), want)


# ---- 8-bit linears -----------------------------------------------------------------------------------------------------

def test_int8_scales_have_the_rows_shape(dev):
    """A scale for each row: of the rows' leading shape, with or without dimensions of size 1, or flat in the rows' order."""
    from glmx import Int8Linear, quantize_rows
    gen = torch.Generator(device=dev).manual_seed(911)
    x, w = torch.randn(2, 3, 64, generator=gen, device=dev), torch.randn(24, 64, generator=gen, device=dev)
    lin = Int8Linear.from_weight(w, out_dtype=F32)
    want = lin(x)
    q, s = quantize_rows(x)
    for t in (s, s.reshape(6), s[..., None], s[None], s.t().contiguous().t()):
        assert torch.equal(lin.matmul(q, t), want)
    assert torch.equal(lin.matmul(q.transpose(0, 1), s.t()), want.transpose(0, 1))
    assert torch.equal(lin.matmul(q.reshape(6, 64), s), want.view(6, 24))
    for t in (s.t(), s.t().contiguous(), s.reshape(6, 1).expand(6, 2), s[:1], s[:, :2], s.double(), s.cpu(), s.reshape(1, 6, 1).expand(2, 6, 1)):
        with pytest.raises(ValueError, match="x_scale"):
            lin.matmul(q, t)
    one = lin(x[0, :1])
    q, s = quantize_rows(x[0, :1])
    for t in (s, s[0], s.reshape(1, 1, 1)):
        assert torch.equal(lin.matmul(q, t), one)
    assert torch.equal(lin.matmul(q[0], s[0]), one[0]) and torch.equal(lin.matmul(q[0], s), one[0])
    assert lin.matmul(q[:0], s[:0]).shape == (0, 24)
    b = torch.randn(24, generator=gen, device=dev)
    want = Int8Linear(lin.wq, lin.w_scale, b)(x)
    assert torch.equal(Int8Linear(lin.wq, lin.w_scale[:, None], b[None])(x), want)
    for bad in (dict(bias=b[:23]), dict(w_scale=lin.w_scale[:1]), dict(w_scale=lin.w_scale.half()), dict(bias=b.cpu())):
        with pytest.raises(ValueError, match="must be fp32"):
            Int8Linear(**(dict(wq=lin.wq, w_scale=lin.w_scale, bias=b) | bad))


# ---- the error word ----------------------------------------------------------------------------------------------------

CHECK_PROGRAM = r"""
#include "dense.cu"
#include <cstdio>
#include <thread>
namespace glmx { void set_error(const std::string&) {} }

static __global__ void or_kernel(int* p, int bits, int pause)
{
    for (int i = 0; i < pause; ++i) __nanosleep(100);
    atomicOr(p, bits);
}

int main()
{
    int* p = nullptr;
    cudaStream_t a, b;
    if (cudaStreamCreateWithFlags(&a, cudaStreamNonBlocking) || cudaStreamCreateWithFlags(&b, cudaStreamNonBlocking) || glmx::dense_err_ptr(&p)) return 1;
    int flags = -1, lost = 0, errors = 0;
    errors += glmx_dense_check(a, &flags) != GLMX_OK || flags != 0;
    or_kernel<<<1, 1, 0, a>>>(p, 5, 0);
    errors += glmx_dense_check(a, &flags) != GLMX_E_DEVICE || flags != 5;
    errors += glmx_dense_check(a, nullptr) != GLMX_OK;
    // one error is known when the check begins; another one comes from the other stream at some time during it
    for (int i = 0; i < 3000; ++i)
    {
        const int late = 1 << (1 + i % 30);
        or_kernel<<<1, 1, 0, a>>>(p, 1, 0);
        std::thread other([&] { or_kernel<<<1, 1, 0, b>>>(p, late, i / 30 % 100); });
        int first = 0, second = 0;
        glmx_dense_check(a, &first);
        other.join();
        cudaStreamSynchronize(b);
        glmx_dense_check(a, &second);
        lost += ((first | second) & late) == 0 || (first & 1) == 0;
    }
    std::printf("errors %d lost %d %s\n", errors, lost, cudaGetErrorString(cudaDeviceSynchronize()));
    return 0;
}
"""


def test_dense_check_loses_no_error(tmp_path):
    """An error of another stream that comes while a check runs is reported by that check or by the next one."""
    import os
    import shutil
    import subprocess
    from conftest import PKG, REPO
    nvcc = os.environ.get("NVCC") or shutil.which("nvcc")
    if not nvcc:
        pytest.skip("no nvcc")
    src, exe = tmp_path / "check.cu", tmp_path / "check"
    src.write_text(CHECK_PROGRAM)
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr",
                    "-I" + os.path.join(REPO, "include"), "-I" + os.path.join(PKG, "csrc"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=120).stdout
    assert out.split() == ["errors", "0", "lost", "0", "no", "error"]


@pytest.mark.parametrize("kt", [torch.uint8, torch.int8, torch.int16, torch.int64, torch.float32, torch.float16])
def test_sample_top_k_of_any_type(dev, kt):
    """top_k in any number type, also one that cannot hold the vocabulary's size."""
    from glmx import sample
    gen = torch.Generator(device=dev).manual_seed(921)
    logits, u = torch.randn(5, 70001, generator=gen, device=dev) * 3, torch.rand(5, generator=gen, device=dev)
    k = torch.tensor([0, 1, 5, 100, 127], device=dev)
    assert torch.equal(sample(logits, u, top_k=k.to(kt)), sample(logits, u, top_k=k.int()))
    if kt in (torch.float32, torch.float16):
        assert torch.equal(sample(logits, u, top_k=torch.full((5,), math.inf, device=dev, dtype=kt)), sample(logits, u))


def test_errors_of_earlier_calls_are_not_reported_again(dev):
    """A call that failed (here an allocation beyond the device's memory) has returned its error; the next ones succeed."""
    import ctypes as C
    from glmx import GatedFFN, Int8Linear, _lib, dense_check, quantize_rows, sample
    L = _lib.load()
    x, wg, wu, wd, dy = block(dev, 5, 128, 64, BF, 931)
    ffn, lin = GatedFFN(wg, wu, wd, act_limit=1.0), Int8Linear.from_weight(wg)
    u = torch.rand(5, device=dev)

    def train():
        return ffn.backward(dy, ffn.forward_train(x)[1])[0]
    for call in (lambda: quantize_rows(x)[0], lambda: quantize_rows(x[:, 1:])[0], lambda: ffn(x), train, lambda: lin(x), lambda: sample(x, u)):
        want = call()
        assert L.glmx_ipc_alloc(1 << 60, C.byref(C.c_void_p())) == _lib.E_CUDA
        assert torch.equal(call(), want)
    assert L.glmx_ipc_alloc(1 << 60, C.byref(C.c_void_p())) == _lib.E_CUDA
    dense_check()


@pytest.mark.parametrize("T", [2, 17, 100, 300, 1100])
def test_rows_do_not_depend_on_their_place(dev, T):
    """A batch's rows in another order give the same rows' bits, in that order."""
    from glmx import GatedFFN, Int8Linear, quantize_rows, sample
    x, wg, wu, wd, dy = block(dev, T, 1024, 520, BF, 941 + T)
    gen = torch.Generator(device=dev).manual_seed(T)
    perm = torch.randperm(T, generator=gen, device=dev)
    u = torch.rand(T, generator=gen, device=dev)
    for L in (0.0, 1.25):
        ffn = GatedFFN(wg, wu, wd, act_limit=L)
        y, saved = ffn.forward_train(x)
        yp, saved_p = ffn.forward_train(x[perm])
        assert torch.equal(yp, y[perm]) and torch.equal(ffn(x[perm]), y[perm])
        assert torch.equal(ffn.backward(dy[perm], saved_p)[0], ffn.backward(dy, saved)[0][perm])
    lin = Int8Linear.from_weight(wg, out_dtype=F32)
    logits = lin(x)
    assert torch.equal(lin(x[perm]), logits[perm])
    assert all(torch.equal(a, b[perm]) for a, b in zip(quantize_rows(x[perm]), quantize_rows(x)))
    assert torch.equal(sample(logits[perm], u[perm], top_p=0.9), sample(logits, u, top_p=0.9)[perm])
