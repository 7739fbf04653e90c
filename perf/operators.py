"""The dense operators beside the routed-expert layer, as cases to be timed and compared: the gated feed-forward block
(a dense layer or an unquantised shared expert) with its backward pass, the 8-bit linear (a head or a projection), and
sampling from the head's logits.

`own` False computes each operator in plain torch operations, True through the public entry points of glmx."""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_DEV = "cuda"


def _glmx():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glm-flash-lite_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import glmx
    return glmx


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence through the shared expert's geometry (H = 6144, I = 1536): latency
        dict(name="ffn_1", op="ffn", T=1, H=6144, I=1536, dtype="bf16", limit=0.0),
        # the decode batch of the benchmarked layer, with the activation clamp
        dict(name="ffn_64", op="ffn", T=64, H=6144, I=1536, dtype="fp16", limit=10.0),
        # a short prompt through the smaller geometry, ragged rows
        dict(name="ffn_777", op="ffn", T=777, H=4096, I=2048, dtype="bf16", limit=0.0),
        # a prefill batch
        dict(name="ffn_4096", op="ffn", T=4096, H=6144, I=1536, dtype="bf16", limit=0.0),
        # a small fine-tuning step on a dense layer: forward and all gradients, sizes that end inside tiles
        dict(name="ffn_train_333", op="ffn_train", T=333, H=1160, I=5000, dtype="fp16", limit=4.0),
        # a full training batch through the shared expert
        dict(name="ffn_train_4096", op="ffn_train", T=4096, H=6144, I=1536, dtype="bf16", limit=0.0),
        # one token through a projection held in 8 bits
        dict(name="i8_1", op="i8", T=1, K=6144, N=6144, dtype="bf16", out="bf16", bias=False, quantised=False),
        # a decode batch through a head of 65,536 tokens, logits in fp32
        dict(name="i8_48", op="i8", T=48, K=4096, N=65536, dtype="bf16", out="fp32", bias=False, quantised=False),
        # a ragged batch, odd sizes, with a bias; the activations come quantised (shared by several projections)
        dict(name="i8_1001", op="i8", T=1001, K=4100, N=5003, dtype="fp16", out="fp16", bias=True, quantised=True),
        # a prefill batch
        dict(name="i8_4096", op="i8", T=4096, K=6144, N=12288, dtype="bf16", out="bf16", bias=False, quantised=False),
        # the next token of one sequence
        dict(name="sample_1", op="sample", B=1, V=131072, dtype="bf16", mode="all"),
        # the next tokens of a batch whose requests each bring their own settings, an odd vocabulary
        dict(name="sample_64", op="sample", B=64, V=150001, dtype="fp32", mode="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    largest = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["ffn", "ffn", "ffn_train", "i8", "i8", "sample"])
        if op == "sample":
            return dict(op=op, B=_log(rng, 1, 128), V=_log(rng, 1000, 160000), dtype=rng.choice(["bf16", "fp16", "fp32"]),
                        mode=rng.choice(["all", "mixed", "top_k", "top_p", "min_p", "plain", "masked"]))
        if op == "i8":
            c = dict(op=op, T=_log(rng, 1, 4096), K=_log(rng, 256, 8192), N=_log(rng, 256, 65536),
                     dtype=rng.choice(["bf16", "fp16"]), out=rng.choice(["bf16", "fp16", "fp32"]),
                     bias=rng.random() < 0.5, quantised=rng.random() < 0.3)
        else:
            c = dict(op=op, T=_log(rng, 1, 4096), H=8 * _log(rng, 64, 768), I=8 * _log(rng, 32, 1536),
                     dtype=rng.choice(["bf16", "fp16"]), limit=rng.choice([0.0, 0.0, 10.0, 2.5]))
        if work(c)["flops"] <= largest:
            return c


def work(case):
    op = case["op"]
    if op in ("ffn", "ffn_train"):
        T, H, I = case["T"], case["H"], case["I"]
        if op == "ffn":
            return {"bytes": 2 * (2 * T * H + 3 * H * I), "flops": 6 * T * H * I}
        # x, dy and the weights read; y, dx and the weights' gradients written
        return {"bytes": 2 * (4 * T * H + 6 * H * I), "flops": 18 * T * H * I}
    if op == "i8":
        T, K, N = case["T"], case["K"], case["N"]
        xb = T * K + 4 * T if case["quantised"] else T * K * _SIZE[case["dtype"]]
        return {"bytes": xb + N * K + 4 * N + (4 * N if case["bias"] else 0) + T * N * _SIZE[case["out"]],
                "flops": 2 * T * N * K}
    B, V = case["B"], case["V"]
    # per logit a subtraction, a scale, an exponential, two comparisons and two additions
    return {"bytes": B * V * _SIZE[case["dtype"]] + 20 * B + 8 * B, "flops": 7 * B * V}


# ---- inputs --------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=_DEV)
    rand = lambda *s: torch.rand(*s, generator=gen, device=_DEV)
    st = dict(case=case)
    op = case["op"]
    if op in ("ffn", "ffn_train"):
        T, H, I, dt = case["T"], case["H"], case["I"], _DT[case["dtype"]]
        # normed activations of unit scale, weights that keep the pre-activations near it; a few large channels, as
        # trained models have them
        x = randn(T, H)
        x[:, ::97] *= 4.0
        st["x"] = x.to(dt)
        st["wg"] = (randn(I, H) * (1.2 / math.sqrt(H))).to(dt)
        st["wu"] = (randn(I, H) * (1.2 / math.sqrt(H))).to(dt)
        st["wd"] = (randn(H, I) * (1.0 / math.sqrt(I))).to(dt)
        if op == "ffn_train":
            st["dy"] = randn(T, H).to(dt)
    elif op == "i8":
        T, K, N, dt = case["T"], case["K"], case["N"], _DT[case["dtype"]]
        x = randn(T, K)
        x[:, ::61] *= 6.0                                  # outlier channels set the rows' scales
        x = x * (0.25 + rand(T, 1))
        w = randn(N, K) * (1.0 / math.sqrt(K))
        st["ws"] = w.abs().amax(dim=1) / 127.0
        st["wq"] = torch.round(w / st["ws"][:, None]).to(torch.int8)
        st["bias"] = randn(N) * 0.1 if case["bias"] else None
        if case["quantised"]:
            st["xs"] = x.abs().amax(dim=1) / 127.0
            st["xq"] = torch.round(x / st["xs"][:, None]).to(torch.int8)
        else:
            st["x"] = x.to(dt)
    else:
        B, V, mode = case["B"], case["V"], case["mode"]
        # a head's logits: a broad bulk and a few tokens that stand out
        l = randn(B, V) * 2.0
        n_top = min(V, 40)
        idx = torch.randint(0, V, (B, n_top), generator=gen, device=_DEV)
        l.scatter_add_(1, idx, 4.0 + 5.0 * rand(B, n_top))
        temp = 0.6 + 0.8 * rand(B)
        top_k = torch.randint(2, 400, (B,), generator=gen, device=_DEV, dtype=torch.int32)
        top_p = 0.5 + 0.49 * rand(B)
        min_p = 0.002 + 0.1 * rand(B)
        row = torch.arange(B, device=_DEV)
        off = lambda t, hit, v: torch.where(hit, torch.full_like(t, v), t)
        if mode in ("mixed", "masked"):
            # each request has its own settings, some of them off, some greedy
            top_k = off(top_k, row % 3 == 1, 0)
            top_p = off(top_p, row % 4 == 2, 1.0)
            min_p = off(min_p, row % 2 == 0, 0.0)
            temp = off(temp, row % 8 == 5, 0.0)
        if mode == "masked":
            # a grammar leaves a part of the vocabulary
            keep = rand(B, V) < 0.03
            keep[:, 0] = True
            l = torch.where(keep, l, torch.full_like(l, float("-inf")))
        every = torch.ones(B, dtype=torch.bool, device=_DEV)
        if mode in ("top_p", "min_p", "plain"):
            top_k = off(top_k, every, 0)
        if mode in ("top_k", "min_p", "plain"):
            top_p = off(top_p, every, 1.0)
        if mode in ("top_k", "top_p", "plain"):
            min_p = off(min_p, every, 0.0)
        st.update(logits=l.to(_DT[case["dtype"]]), temperature=temp, top_k=top_k, top_p=top_p, min_p=min_p, u=rand(B))
    if own:
        _handle(st)
    return st


def _handle(st):
    """What a program keeps between calls: the block or the linear over its weights."""
    if "handle" not in st:
        g = _glmx()
        if st["case"]["op"] == "ffn":
            st["handle"] = g.GatedFFN(st["wg"], st["wu"], st["wd"], act_limit=st["case"]["limit"])
        elif st["case"]["op"] == "i8":
            st["handle"] = g.Int8Linear(st["wq"], st["ws"], bias=st["bias"], out_dtype=_DT[st["case"]["out"]])
        elif st["case"]["op"] == "ffn_train":
            for k in ("x", "wg", "wu", "wd"):
                st["leaf_" + k] = st[k].detach().requires_grad_(True)
            st["handle"] = g.gated_ffn
        else:
            st["handle"] = g.sample
    return st["handle"]


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    case, h = st["case"], _handle(st)
    op = case["op"]
    if op == "ffn":
        return h(st["x"])
    if op == "ffn_train":
        leaves = [st["leaf_" + k] for k in ("x", "wg", "wu", "wd")]
        y = h(*leaves, act_limit=case["limit"])
        dx, dwg, dwu, dwd = torch.autograd.grad(y, leaves, st["dy"])
        return dict(y=y.detach(), dx=dx, dwg=dwg, dwu=dwu, dwd=dwd)
    if op == "i8":
        if case["quantised"]:
            return dict(y=h.matmul(st["xq"], st["xs"]))
        xq, xs = _glmx().quantize_rows(st["x"])
        return dict(y=h.matmul(xq, xs), q=xq, scale=xs)
    return h(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op in ("ffn", "ffn_train"):
        dt, L = _DT[case["dtype"]], case["limit"]
        x, wg, wu, wd = (st[k].float() for k in ("x", "wg", "wu", "wd"))
        g, u = x @ wg.t(), x @ wu.t()
        s = 1.0 / (1.0 + torch.exp(-g))
        a, b = g * s, u
        if L:
            a, b = torch.clamp(a, max=L), torch.clamp(u, -L, L)
        h = a * b
        y = h @ wd.t()
        if op == "ffn":
            return y.to(dt)
        dy = st["dy"].float()
        dh = dy @ wd
        dwd = dy.t() @ h
        du = dh * a
        dg = dh * b * (s * (1.0 + g * (1.0 - s)))
        if L:
            du = torch.where(u.abs() <= L, du, torch.zeros_like(du))
            dg = torch.where(g * s <= L, dg, torch.zeros_like(dg))
        dx = dg @ wg + du @ wu
        return dict(y=y.to(dt), dx=dx.to(dt), dwg=(dg.t() @ x).to(dt), dwu=(du.t() @ x).to(dt), dwd=dwd.to(dt))
    if op == "i8":
        out = {}
        if case["quantised"]:
            xq, xs = st["xq"], st["xs"]
        else:
            x = st["x"].float()
            amax = x.abs().amax(dim=1)
            xs = amax / torch.full_like(amax, 127.0)        # a true quotient: division by a number multiplies by 1 / 127
            xq = torch.round(x / torch.where(xs == 0, torch.ones_like(xs), xs)[:, None]).to(torch.int8)
            out.update(q=xq, scale=xs)
        # the integer sums pass 2^24, so they are formed in 64 bits
        acc = (xq.double() @ st["wq"].double().t()).float()
        y = acc * xs[:, None] * st["ws"][None, :]
        if case["bias"]:
            y = y + st["bias"]
        return dict(y=y.to(_DT[case["out"]]), **out)
    # sampling: weights and their sums in 64 bits, since a pick next to a border depends on their last bits
    l = st["logits"].double()
    B, V = l.shape
    temp, top_p, min_p = st["temperature"].double(), st["top_p"].double(), st["min_p"].double()
    greedy = temp <= 0
    m = l.amax(dim=1, keepdim=True)
    w = torch.exp((l - m) / torch.where(greedy, torch.ones_like(temp), temp)[:, None])
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    rank = torch.arange(V, device=l.device)
    ws = torch.gather(w, 1, order)
    k = torch.where(st["top_k"] <= 0, torch.full_like(st["top_k"], V), st["top_k"]).long()
    ws = torch.where(rank[None, :] < k[:, None], ws, torch.zeros_like(ws))
    before = torch.cumsum(ws, dim=1) - ws
    keep = (rank[None, :] < k[:, None]) & ((before < (top_p * ws.sum(dim=1))[:, None]) | (top_p >= 1.0)[:, None])
    keep &= ws >= min_p[:, None]
    keep[:, 0] = True
    keep = torch.zeros_like(keep).scatter_(1, order, keep)
    w = torch.where(keep, w, torch.zeros_like(w))
    c = torch.cumsum(w, dim=1)
    hit = (c > st["u"].double()[:, None] * c[:, -1:]) & (w > 0)
    pick = torch.where(hit, rank[None, :], torch.full_like(order, V)).amin(dim=1)
    return torch.where(greedy, order[:, 0], pick)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    f64 = lambda k: st[k].to(torch.float64)
    if op in ("ffn", "ffn_train"):
        L = case["limit"] or math.inf
        pre_g = torch.einsum("th,ih->ti", f64("x"), f64("wg"))
        pre_u = torch.einsum("th,ih->ti", f64("x"), f64("wu"))
        sig = 0.5 * (1.0 + torch.tanh(0.5 * pre_g))
        silu = pre_g * sig
        left, right = silu.clamp(max=L), pre_u.clamp(-L, L)
        y = torch.einsum("ti,hi->th", left * right, f64("wd"))
        if op == "ffn":
            return y
        d_hidden = torch.einsum("th,hi->ti", f64("dy"), f64("wd"))
        d_gate = d_hidden * right * (sig + silu * (1.0 - sig)) * (silu <= L)
        d_up = d_hidden * left * (pre_u.abs() <= L)
        return dict(y=y, dx=torch.einsum("ti,ih->th", d_gate, f64("wg")) + torch.einsum("ti,ih->th", d_up, f64("wu")),
                    dwg=torch.einsum("ti,th->ih", d_gate, f64("x")), dwu=torch.einsum("ti,th->ih", d_up, f64("x")),
                    dwd=torch.einsum("th,ti->hi", f64("dy"), left * right))
    if op == "i8":
        out = {}
        if case["quantised"]:
            q, s = f64("xq"), f64("xs")
        else:
            # the scale is a 32-bit number by definition, and so is the quotient that is rounded
            s = (f64("x").abs().max(dim=1).values / 127.0).to(torch.float32).double()
            q = (f64("x") / torch.where(s == 0, torch.ones_like(s), s)[:, None]).to(torch.float32).round().double()
            out.update(q=q.to(torch.int8), scale=s)
        y = torch.einsum("tk,nk->tn", q, f64("wq")) * torch.outer(s, f64("ws"))
        if case["bias"]:
            y = y + f64("bias")
        return dict(y=y, **out)
    import numpy as np
    l = f64("logits").cpu().numpy()
    par = {k: st[k].double().cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p", "u")}
    picks = []
    for b in range(l.shape[0]):
        row = l[b]
        if par["temperature"][b] <= 0:
            picks.append(int(np.argmax(row)))
            continue
        z = (row - row.max()) / par["temperature"][b]
        order = np.lexsort((np.arange(row.size), -row))
        if par["top_k"][b] > 0:
            order = order[:int(par["top_k"][b])]
        p = np.exp(z[order])
        if par["top_p"][b] < 1.0:
            n = 1 + int(np.count_nonzero(np.cumsum(p)[:-1] < par["top_p"][b] * p.sum()))
            order, p = order[:n], p[:n]
        ok = p >= par["min_p"][b]
        ok[0] = True
        ids = np.sort(order[ok])
        c = np.cumsum(np.exp(z[ids]))
        picks.append(int(ids[min(int(np.searchsorted(c, par["u"][b] * c[-1], side="right")), ids.size - 1)]))
    return torch.tensor(picks, dtype=torch.int64)
