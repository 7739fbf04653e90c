"""The dense operators on the GPU against plain forms in 64 bits: the gated feed-forward block and its gradients, 8-bit
linears, sampling.

Tolerances count roundings. r(t) = torch.finfo(t).eps / 2 is one rounding to t; a sum of n products in fp32, in any order
and with truncation (the tensor cores'), is within (n + 8) 2^-23 sum |a b| of its value."""
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


def tiny(t):
    """half the smallest subnormal step"""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def e32(n):
    return (n + 8) * 2.0 ** -23


# ---- gated feed-forward ------------------------------------------------------------------------------------------------

def block(dev, T, H, I, dt, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)
    x = rn(T, H).to(dt)
    wg, wu = (rn(I, H) * (1.2 / math.sqrt(H))).to(dt), (rn(I, H) * (1.2 / math.sqrt(H))).to(dt)
    return x, wg, wu, (rn(H, I) / math.sqrt(I)).to(dt), rn(T, H).to(dt)


def plain(x, wg, wu, wd, L):
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    g, u = x @ wg.t(), x @ wu.t()
    act, up = g * torch.sigmoid(g), u
    if L:
        act, up = act.clamp(max=L), up.clamp(-L, L)
    return g, u, act, up, (act * up) @ wd.t()


def gap_limit(x, wg, wu):
    """A clamp in the widest gap of the values it is compared with, between their 80th and 95th hundredths: no value is so near it that
    a sum in another order would fall on its other side."""
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    v = torch.cat([(g * torch.sigmoid(g)).flatten(), u.abs().flatten()]).sort().values
    v = v[int(0.80 * v.numel()):int(0.95 * v.numel())].cpu()
    i = int((v[1:] - v[:-1]).argmax())
    # the entry takes L in fp32
    return float(torch.tensor((float(v[i]) + float(v[i + 1])) / 2, dtype=F32))


def y_bound(x, wg, wu, wd, L, dt, y_dt):
    """Largest |y - exact| of each output: the sums' errors and the rounding of h, carried through, and y's own."""
    g, u, act, up, y = plain(x, wg, wu, wd, L)
    H, I = x.shape[1], wg.shape[0]
    ax = x.double().abs()
    dg, du = e32(H) * (ax @ wg.double().abs().t()), e32(H) * (ax @ wu.double().abs().t())
    dact = 1.1 * dg + 2.0 ** -20 * act.abs()               # |silu'| <= 1.1; the exponential and the division: some ulp
    dh = dact * up.abs() + (act.abs() + dact) * du
    h = (act * up).abs() + dh
    dh = dh + r(dt) * h + tiny(dt)
    aw = wd.double().abs().t()
    dy = dh @ aw + e32(I) * (h @ aw)
    return y, dy + r(y_dt) * (y.abs() + dy) + tiny(y_dt)


def rel_rms(a, ref):
    return float((a.double() - ref.double()).norm() / ref.double().norm().clamp(min=1e-300))


# (T, H, I): one token, sizes inside one tile, ends inside tiles and one past them, more rows than a tile, wide and narrow
FFN_SIZES = [(1, 8, 8), (1, 512, 256), (2, 136, 72), (7, 264, 520), (16, 1024, 384), (33, 200, 1000), (64, 640, 320),
             (100, 1160, 488), (129, 256, 264), (200, 72, 2056), (257, 520, 136), (513, 1032, 776), (1000, 768, 512),
             (2049, 512, 264)]


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,H,I", FFN_SIZES)
def test_ffn_forward(dev, T, H, I, dt):
    from glmx import GatedFFN
    x, wg, wu, wd, _ = block(dev, T, H, I, dt, 100 + T + H)
    for L in (0.0, 1.5):
        ffn = GatedFFN(wg, wu, wd, act_limit=L)
        y, bound = y_bound(x, wg, wu, wd, L, dt, dt)
        got = ffn(x)
        assert got.dtype == dt and got.shape == x.shape
        assert bool(((got.double() - y).abs() <= bound).all())
        assert T * H < 1000 or rel_rms(got, y) <= 2 * r(dt)     # two roundings in a row, h's and y's
        y, bound = y_bound(x, wg, wu, wd, L, dt, F32)
        got = ffn(x, out_dtype=F32)
        assert bool(((got.double() - y).abs() <= bound).all())
        # added to what the output holds, fp32 and 16-bit
        base = torch.randn(T, H, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
        out = base.clone()
        assert ffn(x, out=out, accumulate=True) is out
        assert bool(((out.double() - base.double() - y).abs() <= bound + r(F32) * (out.double().abs() + bound)).all())
        b16 = base.to(dt)
        out = b16.clone()
        ffn(x, out=out, accumulate=True)
        assert bool(((out.double() - b16.double() - y).abs() <= bound + r(dt) * (out.double().abs() + bound) * 1.01).all())


@pytest.mark.parametrize("T,H,I", [(1, 6144, 1536), (64, 6144, 1536), (300, 4096, 2048)])
def test_ffn_forward_large(dev, T, H, I):
    from glmx import GatedFFN
    x, wg, wu, wd, _ = block(dev, T, H, I, BF, 7)
    y, bound = y_bound(x, wg, wu, wd, 10.0, BF, BF)
    got = GatedFFN(wg, wu, wd, act_limit=10.0)(x)
    assert bool(((got.double() - y).abs() <= bound).all())
    assert rel_rms(got, y) <= 2 * r(BF)


def grads(x, wg, wu, wd, dy, L):
    g, u, act, up, y = plain(x, wg, wu, wd, L)
    s = torch.sigmoid(g)
    dy, x, wg, wu, wd = (t.double() for t in (dy, x, wg, wu, wd))
    dh = dy @ wd
    du, dg = dh * act, dh * up * (s * (1 + g * (1 - s)))
    if L:
        du, dg = du * (u.abs() <= L), dg * (g * s <= L)
    return y, dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ (act * up)


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,H,I", FFN_SIZES)
def test_ffn_backward(dev, T, H, I, dt):
    """Against the formula: y, dx and the weights' gradients pass two roundings to 16 bits (h, dg or du, then their own)."""
    from glmx import gated_ffn
    x, wg, wu, wd, dy = block(dev, T, H, I, dt, 300 + T + H)
    for L in (0.0, gap_limit(x, wg, wu)):
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = gated_ffn(*leaves, act_limit=L)
        got = torch.autograd.grad(y, leaves, dy)
        for name, a, ref in zip(("y", "dx", "dwg", "dwu", "dwd"), (y.detach(), *got), grads(x, wg, wu, wd, dy, L)):
            assert a.dtype == dt and a.shape == ref.shape
            # each value is a sum of rounded terms: its error is at most 2 r(dt) of the sum of their magnitudes; over a whole
            # tensor, where errors are independent, 2 r(dt) of its norm
            assert ref.numel() < 1000 or rel_rms(a, ref) <= 2 * r(dt), (name, L, rel_rms(a, ref))
            assert bool(torch.isfinite(a).all())
            assert float((a.double() - ref).abs().max()) <= 40 * r(dt) * float(ref.abs().max()) + 64 * tiny(dt), (name, L)


@pytest.mark.parametrize("T,H,I", [(5, 6144, 256), (40, 1160, 488), (700, 1032, 776), (1100, 2048, 512)])
def test_ffn_limit_next_to_values(dev, T, H, I):
    """Which gradients pass the clamp is decided as in 64 bits, also where the limit is the fp32 number next to a value."""
    from glmx import GatedFFN
    x, wg, wu, wd, _ = block(dev, T, H, I, BF, 500 + T)
    g, u, act, _, _ = plain(x, wg, wu, wd, 0.0)
    vals = torch.cat([act.flatten(), u.abs().flatten()])
    vals = vals[(vals > 0.5) & (vals < 3)]
    pick = torch.randint(0, vals.numel(), (12,), generator=torch.Generator(device=dev).manual_seed(T), device=dev)
    for v in vals[pick].tolist():
        L = float(torch.tensor(v, dtype=F32))                # above or below the value, by less than a rounding
        _, (_, _, pq) = GatedFFN(wg, wu, wd, act_limit=L).forward_train(x)
        p, q = pq[0], pq[1]
        # the factors are 0 where the value is past the limit, and only there (or where they are 0 or tiny by themselves)
        assert torch.equal(p != 0, (u.abs() <= L) & (act.float() != 0))
        past = act > L
        assert bool((q[past] == 0).all()) and bool((q[~past & (act > 0.1) & (u.abs() > 1e-3)] != 0).all())


def test_ffn_backward_against_differences(dev):
    """Directional differences of the block in 64 bits: <gradient, d> = (f(p + e d) - f(p - e d)) / 2e."""
    from glmx import GatedFFN
    x, wg, wu, wd, dy = block(dev, 48, 96, 160, HF, 11)
    ffn = GatedFFN(wg, wu, wd)
    _, saved = ffn.forward_train(x)
    got = ffn.backward(dy, saved)
    params = [t.double() for t in (x, wg, wu, wd)]
    gen = torch.Generator(device=dev).manual_seed(5)
    loss = lambda ps: float((plain(*ps, 0.0)[4] * dy.double()).sum())
    for i, grad in enumerate(got):
        d = torch.randn(params[i].shape, generator=gen, device=dev, dtype=torch.float64)
        e = 1e-5
        up, dn = list(params), list(params)
        up[i], dn[i] = params[i] + e * d, params[i] - e * d
        want = (loss(up) - loss(dn)) / (2 * e)
        # independent errors of 2 r(fp16) per value over the direction: five times their root sum of squares
        assert abs(float((grad.double() * d).sum()) - want) <= 5 * 2 * r(HF) * float((grad.double() * d).norm()) + 1e-6 * abs(want)


def test_ffn_parts_strides_and_empty(dev):
    from glmx import GatedFFN
    x, wg, wu, wd, dy = block(dev, 40, 128, 192, BF, 21)
    ffn = GatedFFN(wg, wu, wd, act_limit=2.0)
    want = ffn(x)
    wide = torch.zeros(40, 200, device=dev, dtype=BF)
    wide[:, 16:144] = x                                      # rows 200 apart, 32 bytes in: used in place
    assert torch.equal(ffn(wide[:, 16:144]), want)
    odd = torch.zeros(40, 133, device=dev, dtype=BF)
    odd[:, 3:131] = x                                        # rows that are not 16-byte aligned: copied
    assert torch.equal(ffn(odd[:, 3:131]), want)
    assert torch.equal(ffn(x.t().contiguous().t()), want)
    assert torch.equal(ffn(x.view(5, 8, 128)), want.view(5, 8, 128))
    assert torch.equal(ffn(x[0]), ffn(x[:1])[0])
    assert torch.equal(GatedFFN(wg.t().contiguous().t(), wu, wd, act_limit=2.0)(x), want)
    for shape in ((0, 128), (3, 0, 128)):
        e = ffn(torch.empty(shape, device=dev, dtype=BF))
        assert e.shape == shape
    y, saved = ffn.forward_train(x)
    assert torch.equal(y, want)
    full = ffn.backward(dy, saved)
    for need in ((True, False, False, False), (False, True, False, False), (False, False, True, False),
                 (False, False, False, True), (True, False, False, True), (False, False, False, False)):
        part = ffn.backward(dy, saved, need)
        for a, b, n in zip(part, full, need):
            assert (a is None) if not n else torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(ffn.backward(dy.t().contiguous().t(), saved), full))
    y, saved = ffn.forward_train(x[:0])
    dx, *dws = ffn.backward(dy[:0], saved)
    assert y.shape == (0, 128) and dx.shape == (0, 128) and all(float(w.abs().max()) == 0 for w in dws)


def test_ffn_infinite_limit_is_none(dev):
    from glmx import GatedFFN
    x, wg, wu, wd, dy = block(dev, 20, 128, 192, BF, 23)
    a, b = GatedFFN(wg, wu, wd, act_limit=math.inf), GatedFFN(wg, wu, wd)
    (ya, sa), (yb, sb) = a.forward_train(x), b.forward_train(x)
    assert torch.equal(ya, yb) and all(torch.equal(p, q) for p, q in zip(a.backward(dy, sa), b.backward(dy, sb)))
    # no rows at the limit: zeros are not next to it
    assert float(GatedFFN(wg, wu, wd, act_limit=1e-30)(torch.zeros_like(x)).abs().max()) == 0.0


def test_ffn_in_place_and_offset_outputs(dev):
    """The output may be the input, and a slice of a larger buffer that is 16-byte aligned; others are refused."""
    from glmx import GatedFFN, Int8Linear
    for T in (3, 400):
        x, wg, wu, wd, _ = block(dev, T, 256, 128, BF, 25)
        ffn = GatedFFN(wg, wu, wd)
        want = ffn(x)
        buf = torch.zeros(T * 256 + 16, device=dev, dtype=BF)
        out = buf[8:8 + T * 256].view(T, 256)
        assert torch.equal(ffn(x, out=out), want)
        with pytest.raises(ValueError):
            ffn(x, out=buf[1:1 + T * 256].view(T, 256))
        lin = Int8Linear.from_weight(wg)
        y = lin(x)
        buf = torch.zeros(T * 128 + 16, device=dev, dtype=BF)
        assert torch.equal(lin(x, out=buf[3:3 + T * 128].view(T, 128)), y)
        assert float(buf[:3].abs().max()) == 0 and float(buf[3 + T * 128:].abs().max()) == 0
        x2 = x.clone()
        assert ffn(x2, out=x2) is x2 and torch.equal(x2, want)


def test_ffn_autograd_forms(dev):
    """A frozen weight, a broadcast gradient, two uses of one leaf, gradients that add up over two backward calls."""
    from glmx import gated_ffn
    x, wg, wu, wd, dy = block(dev, 24, 64, 96, BF, 31)
    xs = x.clone().requires_grad_(True)
    wgp = wg.clone().requires_grad_(True)
    y = gated_ffn(xs, wgp, wu, wd)
    y.sum().backward()                                       # dy is an expanded scalar
    ref = grads(x, wg, wu, wd, torch.ones_like(dy), 0.0)
    assert rel_rms(xs.grad, ref[1]) <= 2 * r(BF) and rel_rms(wgp.grad, ref[2]) <= 2 * r(BF)
    once = wgp.grad.clone()
    gated_ffn(xs, wgp, wu, wd).sum().backward()
    assert torch.equal(wgp.grad, once + once)
    # gate and up from one leaf: both gradients reach it
    w = wg.clone().requires_grad_(True)
    gated_ffn(x, w, w, wd).backward(dy)
    ref = grads(x, wg, wg, wd, dy, 0.0)
    assert rel_rms(w.grad, ref[2] + ref[3]) <= 3 * r(BF)     # one more rounding: the sum of the two
    with torch.no_grad():
        assert gated_ffn(xs, wgp, wu, wd).grad_fn is None
    # a second derivative is refused, and so is a weight that changed after the forward call
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(gated_ffn(xs, wgp, wu, wd).sum(), xs, create_graph=True)
    y = gated_ffn(xs, wgp, wu, wd)
    with torch.no_grad():
        wgp.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_ffn_infinite_and_nan_rows_stay_in_their_rows(dev):
    from glmx import GatedFFN
    for T in (5, 300):
        x, wg, wu, wd, _ = block(dev, T, 256, 128, BF, 41)
        ffn = GatedFFN(wg, wu, wd)
        want = ffn(x)
        x[1, 3] = float("nan")
        x[T - 1, 5] = float("inf")
        got = ffn(x)
        keep = [i for i in range(T) if i not in (1, T - 1)]
        assert torch.equal(got[keep], want[keep])
        assert bool(got[1].isnan().all())


def test_ffn_rows_do_not_depend_on_the_batch_order(dev):
    """Repeated calls give the same bits."""
    from glmx import GatedFFN
    for T in (1, 17, 300, 1100):
        x, wg, wu, wd, dy = block(dev, T, 1024, 512, BF, 51)
        ffn = GatedFFN(wg, wu, wd)
        y, saved = ffn.forward_train(x)
        g = ffn.backward(dy, saved)
        for _ in range(5):
            y2, saved2 = ffn.forward_train(x)
            assert torch.equal(y, y2) and torch.equal(ffn(x), y)
            assert all(torch.equal(a, b) for a, b in zip(g, ffn.backward(dy, saved2)))


# ---- 8-bit linears -----------------------------------------------------------------------------------------------------

def quant_ref(x):
    x = x.double()
    s = (x.abs().amax(-1) / 127).float()
    q = (x / torch.where(s == 0, torch.ones_like(s), s).double()[..., None]).float().round()
    return q.to(torch.int8), s


@pytest.mark.parametrize("dt", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("R,K", [(1, 1), (3, 7), (1, 6144), (17, 100), (64, 4096), (5, 8200), (2, 70001), (1030, 256)])
def test_quantize_rows(dev, R, K, dt):
    from glmx import quantize_rows
    gen = torch.Generator(device=dev).manual_seed(R + K)
    x = (torch.randn(R, K, generator=gen, device=dev) * torch.rand(R, 1, generator=gen, device=dev) * 5).to(dt)
    x[R // 2] = 0
    q, s = quantize_rows(x)
    wq, ws = quant_ref(x)
    assert torch.equal(s, ws) and torch.equal(q, wq)
    assert q.stride(0) % 16 == 0 and float(s[R // 2]) == 0
    # a slice with odd rows and an odd start, and a transposed view
    if K > 5:
        q2, s2 = quantize_rows(x[:, 3:K - 1])
        wq, ws = quant_ref(x[:, 3:K - 1])
        assert torch.equal(s2, ws) and torch.equal(q2, wq)
    assert torch.equal(quantize_rows(x.t().contiguous().t())[0], q)


def i8_ref(xq, xs, wq, ws, bias, dt):
    """y in 64 bits, and how far an output may be from it: the integer's conversion, the scales' product, their product, the bias, and the rounding to dt."""
    v = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()[None, :]
    y = v if bias is None else v + bias.double()
    d = 3.01 * 2.0 ** -24 * v.abs() + 2.0 ** -24 * y.abs()
    return y, d + r(dt) * (y.abs() + d) + tiny(dt)


I8_SIZES = [(1, 1, 1), (1, 16, 8), (1, 4096, 512), (3, 37, 130), (8, 6144, 256), (17, 100, 1000), (48, 1024, 4097), (64, 640, 333),
            (100, 4100, 129), (129, 130, 257), (256, 512, 512), (300, 2049, 1000), (513, 127, 515), (1001, 900, 1003),
            (2050, 384, 700)]


@pytest.mark.parametrize("T,K,N", I8_SIZES)
def test_linear_i8(dev, T, K, N):
    from glmx import Int8Linear
    gen = torch.Generator(device=dev).manual_seed(T + K + N)
    ri = lambda *s: torch.randint(-128, 128, s, generator=gen, device=dev, dtype=torch.int8)
    xq, wq = ri(T, K), ri(N, K)
    xs, ws = torch.rand(T, generator=gen, device=dev) * 0.1, torch.rand(N, generator=gen, device=dev) * 0.02
    bias = torch.randn(N, generator=gen, device=dev)
    for b in (None, bias):
        lin = Int8Linear(wq, ws, bias=b)
        for dt in (F32, BF, HF):
            got = lin.matmul(xq, xs, out_dtype=dt)
            y, bound = i8_ref(xq, xs, wq, ws, b, dt)
            assert got.dtype == dt and got.shape == (T, N)
            # fp16 overflows where the value does
            fine = y.abs() < 65000 if dt == HF else torch.ones_like(y, dtype=torch.bool)
            assert bool((((got.double() - y).abs() <= bound) | ~fine).all())


def test_linear_i8_longest_sum(dev):
    """K at its limit with every product at its largest: 2147221504 < 2^31, exact in the conversion's 24 bits' multiple."""
    from glmx import Int8Linear, _lib
    K = _lib.I8_MAX_K
    xq = torch.full((2, K), -128, device=dev, dtype=torch.int8)
    wq = torch.full((24, K), -128, device=dev, dtype=torch.int8)
    xq[1] = 127
    one = lambda n: torch.ones(n, device=dev)
    got = Int8Linear(wq, one(24)).matmul(xq, one(2), out_dtype=F32)
    assert bool((got[0] == float(K * 16384)).all())
    assert bool(((got[1].double() + K * 128 * 127).abs() <= K * 128 * 127 * 2.0 ** -24).all())


@pytest.mark.parametrize("T,K,N", [(1, 512, 300), (40, 1000, 77), (300, 640, 512)])
def test_int8_linear_from_weight(dev, T, K, N):
    """The whole linear from 16-bit inputs: quantise, multiply; leading dimensions and padded rows are kept."""
    from glmx import Int8Linear, quantize_rows
    gen = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn(2, T, K, generator=gen, device=dev).to(BF)
    w = (torch.randn(N, K, generator=gen, device=dev) / math.sqrt(K)).to(BF)
    lin = Int8Linear.from_weight(w)
    got = lin(x)
    xq, xs = quant_ref(x.view(-1, K))
    wq, ws = quant_ref(w)
    y, bound = i8_ref(xq, xs, wq, ws, None, BF)
    assert got.dtype == BF and got.shape == (2, T, N)
    assert bool(((got.view(-1, N).double() - y).abs() <= bound).all())
    q, s = quantize_rows(x)
    assert torch.equal(lin.matmul(q, s), got)
    assert torch.equal(lin.matmul(q[1], s[1]), got[1])
    assert torch.equal(lin.matmul(q[:, ::2], s[:, ::2]), got[:, ::2])
    out = torch.empty_like(got)
    assert lin(x, out=out) is out and torch.equal(out, got)
    assert lin(x[:, :0]).shape == (2, 0, N)
    # 8 bits carry the product: each factor is off by at most half a step of its row's largest value
    ref = x.double() @ w.double().t()
    ex = 0.5 * (xs.double()[:, None] * wq.double().abs().sum(1)[None] * ws.double()[None] + ws.double()[None] * (
        xq.double().abs().sum(1) * xs.double())[:, None] + 0.5 * K * xs.double()[:, None] * ws.double()[None]) * 1.001
    assert bool(((got.view(-1, N).double() - ref.view(-1, N)).abs() <= ex + bound).all())


def test_quantize_nan_shows_in_its_row_only(dev):
    from glmx import Int8Linear
    x = torch.randn(6, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(3)).to(BF)
    w = torch.randn(64, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(4)).to(BF)
    lin = Int8Linear.from_weight(w)
    want = lin(x)
    x[2, 7] = float("nan")
    got = lin(x)
    assert bool(got[2].isnan().all()) and torch.equal(got[[0, 1, 3, 4, 5]], want[[0, 1, 3, 4, 5]])


# ---- sampling ----------------------------------------------------------------------------------------------------------

def sample_ref(logits, u, temperature, top_k, top_p, min_p):
    """The documented pick, row by row in 64 bits."""
    out = []
    l64 = logits.double().cpu()
    B, V = l64.shape
    val = lambda v, b: float(v[b]) if isinstance(v, torch.Tensor) else float(v)
    for b in range(B):
        l = torch.where(l64[b].isnan(), torch.full_like(l64[b], -math.inf), l64[b])
        m = float(l.max())
        if m == -math.inf:
            out.append(-1)
            continue
        T = val(temperature, b)
        if T <= 0:
            out.append(int((l == m).nonzero()[0]))
            continue
        w = (l == m).double() if m == math.inf else torch.exp((l - m) / T)
        order = torch.sort(l, descending=True, stable=True).indices
        k = int(val(top_k, b))
        if 0 < k < V:
            order = order[:k]
        ws = w[order]
        p = val(top_p, b)
        if p < 1:
            before = torch.cumsum(ws, 0) - ws
            n = max(1, int((before < p * ws.sum()).sum()))
            order, ws = order[:n], ws[:n]
        ok = ws >= min(val(min_p, b), 1.0)
        ok[0] = True
        ids = order[ok].sort().values
        c = torch.cumsum(w[ids], 0)
        hit = (c > float(u[b]) * c[-1]).nonzero()
        out.append(int(ids[hit[0]]))
    return out


def head(dev, B, V, dt, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    l = torch.randn(B, V, generator=gen, device=dev) * 2
    l.scatter_add_(1, torch.randint(0, V, (B, 20), generator=gen, device=dev), 6 * torch.rand(B, 20, generator=gen, device=dev))
    return l.to(dt), torch.rand(B, generator=gen, device=dev), gen


@pytest.mark.parametrize("dt", [F32, BF, HF], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 33), (2, 1000), (16, 4099), (4, 32000), (3, 50257), (2, 131072), (1, 200001),
                                 (150, 3001), (2, 393216)])
def test_sample(dev, B, V, dt):
    from glmx import sample
    l, u, gen = head(dev, B, V, dt, B * 7 + V)
    rnd = lambda lo, hi: lo + (hi - lo) * torch.rand(B, generator=gen, device=dev)
    k = torch.randint(1, min(V, 300) + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
    for kw in (dict(), dict(temperature=0.7, top_k=50, top_p=0.9, min_p=0.05), dict(temperature=0.0),
               dict(top_k=1), dict(top_k=V), dict(top_k=5), dict(top_p=0.0), dict(top_p=0.3), dict(temperature=1.5, top_p=0.98),
               dict(min_p=0.1), dict(min_p=1.0), dict(temperature=2.0, min_p=0.001),
               dict(temperature=rnd(0.3, 1.5), top_k=k, top_p=rnd(0.2, 1.0), min_p=rnd(0.0, 0.05)),
               dict(temperature=rnd(0.3, 1.5), top_k=torch.where(k % 2 == 0, k, 0), top_p=torch.where(k % 3 == 0, 1.0, rnd(0.5, 1.0)))):
        got = sample(l, u, **kw)
        want = sample_ref(l, u, kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
        assert got.dtype == torch.int64 and got.tolist() == want, kw


def test_sample_ties_masks_and_specials(dev):
    from glmx import sample
    inf, nan = math.inf, math.nan
    row = lambda v: torch.tensor([v], device=dev, dtype=F32)
    U = lambda x: torch.tensor([x], device=dev)
    lo = torch.finfo(F32).min
    assert sample(row([-inf] * 5), U(0.5)).tolist() == [-1]
    assert sample(row([nan, -inf, nan]), U(0.5)).tolist() == [-1]
    assert sample(row([-inf, nan, 2.0, -inf]), U(0.999)).tolist() == [2]
    assert sample(row([nan, 1.0, 3.0, 3.0]), U(0.0), temperature=0).tolist() == [2]
    assert sample(row([1.0, inf, 0.0, inf]), U(0.4)).tolist() == [1] and sample(row([1.0, inf, 0.0, inf]), U(0.6)).tolist() == [3]
    assert sample(row([lo, lo, lo, lo]), U(0.6)).tolist() == [2]                 # a mask of the type's lowest value everywhere
    assert sample(row([lo, 1.0, lo, 1.0]), U(0.6), top_k=3).tolist() == [3]
    assert sample(row([0.0, -0.0, 0.0]), U(0.5), temperature=0).tolist() == [0]  # equal zeros
    # ties at the border of top-k and top-p: the lower ids stay
    flat = torch.zeros(1, 1000, device=dev)
    for k in (1, 7, 999):
        assert sample(flat, U(0.9999), top_k=k).tolist() == [k - 1]
    assert sample(flat, U(0.9999), top_p=0.5).tolist() == [499]
    assert sample(flat, U(0.9999), top_p=0.5, top_k=100).tolist() == [49]
    flat[0, 700] = 1.0
    assert sample(flat, U(0.9999), top_k=3).tolist() == [700] and sample(flat, U(0.0), top_k=3).tolist() == [0]
    # the first and the last kept id
    l, u, _ = head(dev, 1, 5000, BF, 3)
    assert sample(l, U(0.0)).tolist() == [0]
    assert sample(l, U(1.0 - 2.0 ** -24)).tolist() == sample_ref(l, U(1.0 - 2.0 ** -24), 1.0, 0, 1.0, 0.0)
    # very low and very high temperatures
    assert sample(l, U(0.7), temperature=1e-30).tolist() == [int(l.float().argmax())]
    assert sample(l, U(0.5), temperature=1e30).tolist() == [2500]


def test_sample_many_masked(dev):
    """Rows of which a grammar leaves a few tokens, some rows none."""
    from glmx import sample
    l, u, gen = head(dev, 32, 20011, BF, 77)
    l[torch.rand(32, 20011, generator=gen, device=dev) < 0.999] = -math.inf
    l[::5] = -math.inf
    for kw in (dict(), dict(top_k=5), dict(top_p=0.8), dict(top_k=500, top_p=0.95, min_p=0.02), dict(temperature=0.0)):
        want = sample_ref(l, u, kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))
        assert sample(l, u, **kw).tolist() == want


def test_sample_rows_and_types(dev):
    from glmx import sample
    l, u, _ = head(dev, 6, 999, F32, 5)
    want = sample(l, u, top_k=40)
    wide = torch.zeros(6, 1501, device=dev)
    wide[:, 7:1006] = l
    assert torch.equal(sample(wide[:, 7:1006], u, top_k=40), want)
    assert torch.equal(sample(l.t().contiguous().t(), u, top_k=40), want)
    assert torch.equal(sample(l, u, top_k=40, out_dtype=torch.int32), want.int())
    assert torch.equal(sample(l, u, top_k=torch.tensor(40, device=dev)), want)
    assert torch.equal(sample(l, u, top_k=torch.full((6,), 40, device=dev)), want)      # int64, converted
    assert torch.equal(sample(l[1:2], u[1:2], top_k=40), want[1:2])
    assert sample(l[:0], u[:0]).shape == (0,)


def test_sample_many_rows(dev):
    """More rows than one launch's grid takes."""
    from glmx import sample
    gen = torch.Generator(device=dev).manual_seed(2)
    l, u = torch.randn(66000, 5, generator=gen, device=dev), torch.rand(66000, generator=gen, device=dev)
    k = torch.randint(0, 4, (66000,), generator=gen, device=dev, dtype=torch.int32)
    got = sample(l, u, top_k=k)
    w = torch.exp(l.double() - l.double().amax(1, keepdim=True))
    rank = torch.argsort(torch.argsort(l, dim=1, descending=True), dim=1)
    w = torch.where((k[:, None] == 0) | (rank < k[:, None]), w, 0.0)
    c = w.cumsum(1)
    want = (c > u.double()[:, None] * c[:, -1:]).int().argmax(1)
    assert torch.equal(got, want)


def test_sample_frequencies(dev):
    """Many uniform numbers over one row reproduce its probabilities: counts within 5 standard deviations."""
    from glmx import sample
    n = 20000
    l = torch.randn(1, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(8))
    u = (torch.arange(n, device=dev) + 0.5) / n
    ids = sample(l.expand(n, 64).contiguous(), u, temperature=0.8)
    p = torch.softmax(l.double() / 0.8, dim=1)[0]
    # an even grid of u: each count is within one of n p
    assert float((torch.bincount(ids, minlength=64).double() - n * p).abs().max()) <= 1.0 + n * 1e-6


# ---- together, as a model's last block and head use them -----------------------------------------------------------------

def test_block_head_and_sampling_together(dev):
    """Routed experts + an unquantised shared expert added to their output, an 8-bit head, the next tokens; eager and
    captured."""
    from glmx import GatedFFN, Int8Linear, MoELayer, Router, sample, synth
    H, I, E, V, B = 512, 256, 8, 3001, 6
    layer = MoELayer.from_bank(synth.make_bank(H, I, E, shared=False, seed=3), device=dev)
    gen = torch.Generator(device=dev).manual_seed(6)
    rn = lambda *s: torch.randn(*s, generator=gen, device=dev)
    router = Router((rn(E, H) * 0.05).half(), None, 4)
    ffn = GatedFFN((rn(I, H) / 22).half(), (rn(I, H) / 22).half(), (rn(H, I) / 16).half(), act_limit=10.0)
    lin = Int8Linear.from_weight((rn(V, H) / 22).half(), out_dtype=F32)
    x, u = rn(B, H).half(), torch.rand(B, generator=gen, device=dev)

    def step():
        sel, w, _ = router(x)
        out = layer.forward(x, sel, w, dense_shared=ffn)
        logits = lin((out + x.float()).half())
        return out, logits, sample(logits, u, temperature=0.8, top_k=40, top_p=0.95)

    out, logits, ids = step()
    sel, w, _ = router(x)
    y, bound = y_bound(x, ffn.w_gate, ffn.w_up, ffn.w_down, 10.0, HF, F32)
    base = layer.forward(x, sel, w)
    assert bool(((out.double() - base.double() - y).abs() <= bound + r(F32) * (out.double().abs() + bound)).all())
    assert torch.equal(out, ffn(x, out=base.clone(), accumulate=True))
    assert torch.equal(layer.forward(x.float(), sel, w, dense_shared=ffn, stream=torch.cuda.current_stream()), out)
    with pytest.raises(ValueError):
        layer.forward(x, sel, w, dense_shared=GatedFFN(ffn.w_gate[:, :256].contiguous(), ffn.w_up[:, :256].contiguous(),
                                                       ffn.w_down[:256].contiguous()))
    with pytest.raises(TypeError):
        layer.forward(x, sel, w, out_dtype=BF, dense_shared=ffn)
    assert ids.tolist() == sample_ref(logits, u, 0.8, 40, 0.95, 0.0)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = step()
    x.copy_(rn(B, H).half())
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(cap, want))


def test_captured_calls_share_nothing(dev):
    """Two captured graphs of each operator, replayed in turn and at the same time on two streams, equal eager calls."""
    from glmx import GatedFFN, Int8Linear, sample
    x, wg, wu, wd, dy = block(dev, 70, 512, 384, BF, 61)
    ffn = GatedFFN(wg, wu, wd)
    lin = Int8Linear.from_weight(wg)
    u = torch.rand(70, device=dev, generator=torch.Generator(device=dev).manual_seed(1))

    def step(v):
        y, saved = ffn.forward_train(v)
        gr = ffn.backward(dy, saved)
        l = lin(y)
        return (y, *gr, l, sample(l, u, top_k=20), ffn(v[:1]), lin(v[:1]))

    step(x)
    torch.cuda.synchronize()
    ins = [x.clone(), (x * 0.5).to(BF)]
    want = [step(v) for v in ins]
    graphs, outs = [], []
    for v in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(v))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_streams(dev):
    """stream= runs a call there, with its temporaries; two streams at once do not disturb each other."""
    from glmx import GatedFFN, Int8Linear, quantize_rows, sample
    x, wg, wu, wd, dy = block(dev, 130, 1024, 512, BF, 71)
    ffn = GatedFFN(wg, wu, wd)
    lin = Int8Linear.from_weight(wg)
    u = torch.rand(130, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    want = ffn(x), *ffn.backward(dy, ffn.forward_train(x)[1]), lin(x), quantize_rows(x)[0], sample(x, u, top_p=0.9)
    streams = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            got.append((ffn(x, stream=s), *ffn.backward(dy, ffn.forward_train(x, stream=s)[1], stream=s), lin(x, stream=s),
                        quantize_rows(x, stream=s)[0], sample(x, u, top_p=0.9, stream=s)))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_first_calls_inside_a_capture():
    """A process whose first call of each operator is captured: nothing of their set-up disturbs the capture."""
    import subprocess
    import sys
    from conftest import PKG
    code = """
import sys, torch
sys.path.insert(0, %r)
import glmx
d = 'cuda'
w, wd, x, dy = (torch.randn(*s, device=d).bfloat16() / 8 for s in ((96, 128), (128, 96), (40, 128), (40, 128)))
u, ws = torch.rand(40, device=d), torch.rand(96, device=d)
wq = torch.randint(-9, 9, (96, 128), device=d, dtype=torch.int8)
ffn, lin = glmx.GatedFFN(w, w, wd), glmx.Int8Linear(wq, ws)
torch.cuda.synchronize()
def step():
    y, saved = ffn.forward_train(x)
    q, s = glmx.quantize_rows(x)
    return (y, *ffn.backward(dy, saved), lin.matmul(q, s), glmx.sample(x, u, top_p=0.9))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, step()))
glmx.dense_check()
print('captured')
""" % PKG
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_first_call_of_a_thread(dev):
    """A thread that has made no CUDA call of its own (an autograd worker) may make its first one here."""
    import threading
    from glmx import GatedFFN, Int8Linear, sample
    x, wg, wu, wd, dy = block(dev, 3, 64, 64, BF, 91)
    ffn, lin = GatedFFN(wg, wu, wd), Int8Linear.from_weight(wg)
    u = torch.rand(3, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    _, saved = ffn.forward_train(x)
    calls = [lambda: ffn(x), lambda: lin(x), lambda: sample(x, u), lambda: ffn.backward(dy, saved)[0]]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    got = [None] * len(calls)

    def run(i):
        got[i] = calls[i]()
        torch.cuda.synchronize()
    for i in range(len(calls)):
        t = threading.Thread(target=run, args=(i,))
        t.start()
        t.join()
    assert all(g is not None and torch.equal(g, w) for g, w in zip(got, want))


def test_refusals_with_device_tensors(dev):
    from glmx import GatedFFN, Int8Linear, gated_ffn, quantize_rows, sample
    x, wg, wu, wd, dy = block(dev, 4, 64, 32, BF, 81)
    ffn = GatedFFN(wg, wu, wd)
    with pytest.raises(ValueError):
        ffn(x[:, :56])
    with pytest.raises(TypeError):
        ffn(x.half())
    with pytest.raises(ValueError):
        ffn(x.cpu())
    with pytest.raises(TypeError):
        ffn(x, out_dtype=HF)
    with pytest.raises(ValueError):
        ffn(x, accumulate=True)
    with pytest.raises(ValueError):
        ffn(x, out=torch.empty(3, 64, device=dev, dtype=BF))
    with pytest.raises(ValueError):
        ffn(x, out=torch.empty(64, 4, device=dev, dtype=BF).t())
    with pytest.raises(ValueError):
        GatedFFN(wg, wu, wd.half())
    with pytest.raises(ValueError):
        ffn.backward(dy[:2], ffn.forward_train(x)[1])
    lin = Int8Linear.from_weight(wg)
    with pytest.raises(ValueError):
        lin(x[:, :60])
    with pytest.raises(ValueError):
        lin.matmul(quantize_rows(x)[0], torch.ones(3, device=dev))
    with pytest.raises(ValueError):
        sample(x.float(), torch.rand(3, device=dev))
    with pytest.raises(ValueError):
        sample(x.float(), torch.rand(4, device=dev), top_k=torch.ones(3, device=dev))
    # a differentiated call inside a capture is refused before anything of it is captured
    leaf = x.clone().requires_grad_(True)
    gated_ffn(leaf, wg, wu, wd)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="forward_train"):
            gated_ffn(leaf, wg, wu, wd)
        y = ffn(x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ffn(x))


def test_ffn_without_gradients_is_the_plain_call(dev):
    """Where gradients are off, leaves that ask for them change nothing: no factors kept, and the call may be captured."""
    from glmx import GatedFFN, gated_ffn
    x, wg, wu, wd, _ = block(dev, 64, 512, 1024, BF, 91)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    want = GatedFFN(wg, wu, wd, 3.0)(x)
    with torch.no_grad():
        gated_ffn(*leaves, 3.0)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = gated_ffn(*leaves, 3.0)
        assert torch.cuda.max_memory_allocated() - base <= y.nbytes + 64 * 1024 * 2      # the hidden rows, no more
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cap = gated_ffn(*leaves, 3.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(cap, want) and y.grad_fn is None


def test_refusals_of_mixed_up_calls(dev):
    from glmx import GatedFFN, Int8Linear, MoELayer, quantize_rows, synth
    x, wg, wu, wd, dy = block(dev, 4, 512, 96, HF, 92)
    ffn = GatedFFN(wg, wu, wd)
    small = GatedFFN(wg[:88], wu[:88], wd[:, :88])
    with pytest.raises(ValueError, match="saved"):
        ffn.backward(dy, small.forward_train(x)[1])
    lin = Int8Linear.from_weight(wg)
    q, s = quantize_rows(x)
    with pytest.raises(TypeError, match="out_dtype"):
        lin.matmul(q, s, out=torch.empty(4, 96, device=dev), out_dtype=BF)
    layer = MoELayer.from_bank(synth.make_bank(512, 256, 8, shared=False, seed=3), device=dev)
    sel, w = torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.full((4, 2), 0.5, device=dev)
    sel[:, 1] = 1
    kept = x.clone()
    with pytest.raises(ValueError, match="overlap"):
        layer.forward(x, sel, w, out=x, dense_shared=ffn)
    with pytest.raises(ValueError, match="aligned"):
        layer.forward(x, sel, w, out=torch.empty(4 * 512 + 1, device=dev)[1:].view(4, 512), dense_shared=ffn)
    with pytest.raises(ValueError, match="shape"):
        layer.forward(x, sel, w, out=torch.empty(5, 512, device=dev), dense_shared=ffn)
    assert torch.equal(x, kept)


def test_sample_top_k_beyond_32_bits(dev):
    """A top-k larger than the row keeps all of it, however large, as a number and as int64."""
    from glmx import sample
    gen = torch.Generator(device=dev).manual_seed(93)
    logits, u = torch.randn(64, 1000, generator=gen, device=dev), torch.rand(64, generator=gen, device=dev)
    want = sample(logits, u)
    for k in ((1 << 32) + 1, 1 << 31):
        assert torch.equal(sample(logits, u, top_k=k), want)
        assert torch.equal(sample(logits, u, top_k=torch.full((64,), k, device=dev)), want)
    assert torch.equal(sample(logits, u, top_k=-5), want) and torch.equal(sample(logits, u, top_k=torch.full((64,), -5, device=dev)), want)


@pytest.mark.parametrize("B", [40, 300, 512, 700])
def test_sample_rows_with_settings_of_their_own(dev, B):
    """Every row's pick is the one it gets alone, whatever the order in which a batch's rows are worked on."""
    from glmx import sample
    gen = torch.Generator(device=dev).manual_seed(94)
    V = 20011
    logits, u = torch.randn(B, V, generator=gen, device=dev) * 3, torch.rand(B, generator=gen, device=dev)
    row = torch.arange(B, device=dev)
    temperature = torch.where(row % 7 == 3, 0.0, 0.5 + torch.rand(B, generator=gen, device=dev))
    top_k = torch.where(row % 3 == 0, 0, torch.where(row % 5 == 0, 5000, 20 + row)).int()
    top_p = torch.where(row % 4 == 1, 1.0, 0.3 + 0.69 * torch.rand(B, generator=gen, device=dev))
    got = sample(logits, u, temperature, top_k, top_p, 0.0)
    for b in range(0, B, 1 if B < 100 else 17):
        one = sample(logits[b:b + 1], u[b:b + 1], float(temperature[b]), int(top_k[b]), float(top_p[b]), 0.0)
        assert int(got[b]) == int(one[0]), b
    assert torch.equal(got, sample(logits, u, temperature, top_k, top_p, torch.zeros(B, device=dev)))
    perm = torch.randperm(B, generator=gen, device=dev)
    assert torch.equal(got[perm], sample(logits[perm], u[perm], temperature[perm], top_k[perm], top_p[perm]))


@pytest.mark.parametrize("dt", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
def test_quantize_values_next_to_halves(dev, dt):
    """Quotients that are k + 1/2, exactly or but for their last bits: each is the fp32 quotient rounded to even, as torch has it."""
    from glmx import quantize_rows
    gen = torch.Generator(device=dev).manual_seed(95)
    R, K = 512, 2048
    s = torch.rand(R, 1, generator=gen, device=dev) + 0.5
    s[::2] = torch.randint(1, 1 << 8, (R // 2, 1), generator=gen, device=dev) / 64          # exact halves in 16 bits, too
    x = (torch.randint(-127, 127, (R, K), generator=gen, device=dev) + 0.5) * s
    x = x * (1 + torch.randint(-3, 4, (R, K), generator=gen, device=dev) * 2.0 ** -23 * (dt == F32))
    x[:, 0] = 127 * s[:, 0]
    x = x.to(dt)
    scale = x.float().abs().amax(1) / torch.full((R,), 127.0, device=dev)                   # (a scalar divisor would be a reciprocal's product)
    want = torch.round(x.float() / scale[:, None]).clamp(-127, 127).to(torch.int8)
    for rows in (slice(None), slice(1)):
        q, sc = quantize_rows(x[rows])
        assert torch.equal(q, want[rows]) and torch.equal(sc, scale[rows])
    for power in (-60, 60):                                                                 # fp32 rows far from 1
        if dt != HF:
            q, sc = quantize_rows((x.float() * 2.0 ** power).to(dt))
            assert torch.equal(q, want) and torch.equal(sc, scale * 2.0 ** power)
