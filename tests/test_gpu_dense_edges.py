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
