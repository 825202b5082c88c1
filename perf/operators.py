"""The training operators' cases: what each computes, in plain torch, in 64
bits, and through the package's entry points.

Every pass is one training pass of an operator -- its forward, then its backward
from given output gradients -- and returns the outputs, every gradient and
(where there is one) the final state.

  gated  h_t = a_t h_{t-1} + (1 - a_t) sigmoid(g_t) x_t,  a = sigmoid(z)
  ssd    a = exp(-(dt_min + (dt_max - dt_min) sigmoid(dt))),
         h_t = a_t h_{t-1} + (1 - a_t) sigmoid(bg_t) u_t,
         y_t = (sigmoid(cg_t) h_t + D u_t) sigmoid(og_t)
  conv   y = silu(bias + causal depthwise conv_K(u))
  norm   y = x rsqrt(mean(x^2) + eps) w

A marked token (``seg``) starts a segment: the state before it, or the conv's
inputs before it, do not reach it.  With ``ckpt`` the saved activations are held
in 8 bits (e4m3, one power of two per token and 64 channels) and the backward
uses those values; the recurrence's states are kept in 32 bits every 64 tokens
and run again from there over the 8-bit values.
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
DT_MIN, DT_MAX = 0.001, 0.2  # the framework's default step range
GROUP = 64                   # channels of one token that share a scale
SPAN = 64                    # tokens from one kept state to the next


# ------------------------------------------------------------------ cases
def listed():
    c = []

    def add(name, op, B, T, C, dtype, **kw):
        c.append({"name": name, "op": op, "B": B, "T": T, "C": C, "dtype": dtype, "resets": 0, "state": False,
                  "ckpt": False, "K": 0, "chunked": False, **kw})

    # the prefill workload's shape, trained: packed windows of documents
    add("gated 16x4096x1024 bf16", "gated", 16, 4096, 1024, "bf16", resets=1024)
    # the small fp32 workload, carried state in and out (truncated back-propagation through time)
    add("gated 2x512x256 f32", "gated", 2, 512, 256, "f32", resets=160, state=True)
    # a short odd call: latency
    add("gated 3x77x100 f16", "gated", 3, 77, 100, "f16", state=True)
    # one SSD block of the 350M model, its inputs chunks of one in-projection
    add("ssd 8x2048x832 bf16", "ssd", 8, 2048, 832, "bf16", chunked=True)
    # one long sequence: few chains, many steps
    add("ssd 1x16384x832 bf16", "ssd", 1, 16384, 832, "bf16", state=True)
    # small fp32 call with packed documents
    add("ssd 2x130x96 f32", "ssd", 2, 130, 96, "f32", resets=40, state=True)
    # the same block with its activations kept in 8 bits
    add("ssd 8x2048x832 bf16 8-bit", "ssd", 8, 2048, 832, "bf16", ckpt=True, chunked=True)
    # ragged rows and channels, 8 bits
    add("ssd 3x777x200 f16 8-bit", "ssd", 3, 777, 200, "f16", ckpt=True, resets=200)
    # the block's conv, and a ragged one with packed documents
    add("conv 8x2048x832 bf16", "conv", 8, 2048, 832, "bf16", K=3, chunked=True)
    add("conv 3x501x96 f16", "conv", 3, 501, 96, "f16", K=4, resets=100)
    # the block's out-norm, plain and with its input kept in 8 bits
    add("norm 8x2048x832 bf16", "norm", 8, 2048, 832, "bf16")
    add("norm 5x1000x2000 bf16 8-bit", "norm", 5, 1000, 2000, "bf16", ckpt=True)
    return c


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["gated", "ssd", "ssd", "conv", "norm"])
    B = log(1, 16)
    T = log(1, 16384)
    C = log(8, 2048)
    if rng.random() < 0.6:
        C = max(8, C // 8 * 8)
    while B * T * C > 16 << 20:  # well inside the largest listed case's work
        if B > 1:
            B //= 2
        else:
            T //= 2
    return {"op": op, "B": B, "T": T, "C": C, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "resets": 0 if op == "norm" or rng.random() < 0.4 else log(4, 2048),
            "state": op in ("gated", "ssd") and rng.random() < 0.5,
            "ckpt": op in ("ssd", "norm") and rng.random() < 0.5,
            "K": rng.randint(1, 4) if op == "conv" else 0,
            "chunked": op in ("ssd", "conv") and rng.random() < 0.5}


def work(case):
    n = case["B"] * case["T"] * case["C"]
    es = 4 if case["dtype"] == "f32" else 2
    state = 4 * 4 * case["B"] * case["C"] if case["state"] else 0  # h0, final state, their gradients
    mask = case["B"] * case["T"] if case["resets"] else 0
    if case["op"] == "gated":    # z, g, x, dh in; h, dz, dg, dx out
        return {"bytes": 8 * es * n + state + mask, "flops": 60 * n}
    if case["op"] == "ssd":      # dt, bg, u, cg, og, dy in; y and five gradients out
        return {"bytes": 12 * es * n + state + mask + 8 * case["C"], "flops": 120 * n}
    if case["op"] == "conv":     # u, dy in; y, du out
        return {"bytes": 4 * es * n + mask + 8 * case["C"] * (case["K"] + 1), "flops": (6 * case["K"] + 30) * n}
    return {"bytes": 4 * es * n + 8 * case["C"], "flops": 16 * n}  # x, dy in; y, dx out


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    """Inputs as the block's layers hand them over: activations near N(0, 1),
    decay logits near 4 (memories of some fifty tokens), fp32 parameters."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 17)
    B, T, C, dt = case["B"], case["T"], case["C"], DT[case["dtype"]]

    def act(mean=0.0, n=1):
        t = torch.randn((B, T, n * C), generator=g, device=dev)
        return (t + mean if mean else t).to(dt)

    st = {"case": case}
    names = {"gated": ("x", "z", "g"), "ssd": ("u", "bg", "cg", "dt", "og"), "conv": ("u",), "norm": ("x",)}[case["op"]]
    if case["chunked"]:  # views into one in-projection's output, as torch.chunk gives them
        for k, t in zip(("u", "bg", "cg", "dt", "og"), act(n=5).chunk(5, dim=-1)):
            if k in names:
                st[k] = t.detach().requires_grad_()
    else:
        for k in names:
            st[k] = act(4.0 if k == "z" else 0.0).requires_grad_()
    st["gy"] = act()
    st["seg"] = None
    if case["resets"]:
        rs = np.random.RandomState(seed % (1 << 31))
        m = np.zeros((B, T), np.uint8)
        for b in range(B):
            t = 0
            while t < T:
                m[b, t] = 1
                t += int(rs.randint(1, 2 * case["resets"]))
        if case["state"]:  # the first segment goes on from the carried state
            m[:, 0] = 0
        st["seg"] = torch.from_numpy(m).to(dev)
    st["h0"] = st["ghf"] = None
    if case["state"]:
        st["h0"] = (0.5 * torch.randn((B, C), generator=g, device=dev)).requires_grad_()
        st["ghf"] = torch.randn((B, C), generator=g, device=dev)
    if case["op"] == "ssd":
        st["D"] = (1.0 + 0.1 * torch.randn(C, generator=g, device=dev)).requires_grad_()
    if case["op"] == "conv":
        st["w"] = (torch.randn((C, 1, case["K"]), generator=g, device=dev) / math.sqrt(case["K"])).requires_grad_()
        st["b"] = (0.1 * torch.randn(C, generator=g, device=dev)).requires_grad_()
    if case["op"] == "norm":
        st["w"] = (1.0 + 0.1 * torch.randn(C, generator=g, device=dev)).requires_grad_()
    return st


# ------------------------------------------------------------------ the package's operators
def run_own(st):
    from need_b200 import need_kernels as nk
    case = st["case"]
    ck = torch.float8_e4m3fn if case["ckpt"] else None
    if case["op"] == "gated":
        leaves = [st["x"], st["z"], st["g"]]
        out = nk.gated_scan_train(*leaves, seg_start=st["seg"], h0=st["h0"], return_final_state=case["state"])
    elif case["op"] == "ssd":
        leaves = [st["u"], st["bg"], st["cg"], st["dt"], st["og"], st["D"]]
        out = nk.ssd_scan_train(*leaves, DT_MIN, DT_MAX, seg_start=st["seg"], h0=st["h0"],
                                return_final_state=case["state"], checkpoint=ck)
    elif case["op"] == "conv":
        leaves = [st["u"], st["w"], st["b"]]
        out = nk.ssd_conv_silu_train(*leaves, seg_start=st["seg"])
    else:
        leaves = [st["x"], st["w"]]
        out = nk.rms_norm_train(*leaves, EPS, checkpoint=ck)
    outs, gos = ([out], [st["gy"]]) if not case["state"] else (list(out), [st["gy"], st["ghf"]])
    if case["state"]:
        leaves = leaves + [st["h0"]]
    grads = torch.autograd.grad(outs, leaves, gos)
    return [o.detach() for o in outs] + list(grads)


# ------------------------------------------------------------------ plain forms, 32 bits
def _shift(x, d):
    """x delayed by d tokens (dim 1), zeros before."""
    return torch.cat([torch.zeros_like(x[:, :d]), x[:, :max(x.shape[1] - d, 0)]], dim=1)


def _prefix(a, b):
    """Running products of a and states from zero of h_t = a_t h_{t-1} + b_t along
    dim 1, by doubling."""
    d = 1
    while d < a.shape[1]:
        pa = torch.cat([torch.ones_like(a[:, :d]), a[:, :-d]], dim=1)
        pb = torch.cat([torch.zeros_like(b[:, :d]), b[:, :-d]], dim=1)
        b = torch.where(a == 0, b, b + a * pb)
        a = a * pa
        d *= 2
    return a, b


def _spans(x, fill):
    B, T, C = x.shape
    n = -(-T // SPAN)
    if n * SPAN != T:
        x = torch.cat([x, torch.full((B, n * SPAN - T, C), fill, dtype=x.dtype, device=x.device)], dim=1)
    return x.reshape(B * n, SPAN, C), n


def _scan(a, b, h0, entering=None):
    """(h, the state entering each span of SPAN tokens) of h_t = a_t h_{t-1} + b_t."""
    B, T, C = a.shape
    sa, n = _spans(a, 1.0)
    sb, _ = _spans(b, 0.0)
    pa, pb = _prefix(sa, sb)
    if entering is None:
        ea, eb = pa[:, -1].reshape(B, n, C), pb[:, -1].reshape(B, n, C)
        eb = torch.cat([eb[:, :1] + ea[:, :1] * h0[:, None], eb[:, 1:]], dim=1)
        _, after = _prefix(ea, eb)
        entering = torch.cat([h0[:, None], after[:, :-1]], dim=1)
    h = pb + torch.where(pa == 0, torch.zeros_like(pb), pa * entering.reshape(B * n, 1, C))
    return h.reshape(B, n * SPAN, C)[:, :T], entering


def _adjoint(a, e, last):
    """(lam, mu): lam_t = e_t + mu_{t+1}, mu_t = a_t lam_t, mu_T = last."""
    fa = a.flip(1)
    mu, _ = _scan(fa, fa * e.flip(1), last)
    mu = mu.flip(1)
    return e + torch.cat([mu[:, 1:], last[:, None]], dim=1), mu


def _eight(x):
    """x rounded to e4m3 with one power of two per GROUP channels of a token."""
    C = x.shape[-1]
    p = torch.nn.functional.pad(x, (0, -C % GROUP)).reshape(*x.shape[:-1], -1, GROUP)
    m, k = torch.frexp(p.abs().amax(dim=-1, keepdim=True))
    k = (k - 9 + (m > 0.875).to(k.dtype)).clamp_min(-126)
    q = torch.ldexp(p, -k).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, k).reshape(*x.shape[:-1], -1)[..., :C]


def run_plain(st):
    case = st["case"]
    f = {k: (v.detach().float() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in st.items()}
    dt = DT[case["dtype"]]
    gy = f["gy"]
    if case["op"] in ("gated", "ssd"):
        B, T, C = gy.shape
        zero = torch.zeros((B, C), device=gy.device)
        h0 = f["h0"] if case["state"] else zero
        last = f["ghf"] if case["state"] else zero
        keep = torch.ones((B, T, 1), device=gy.device) if f["seg"] is None else (f["seg"] == 0).float()[..., None]
        if case["op"] == "gated":
            a, na = torch.sigmoid(f["z"]), torch.sigmoid(-f["z"])
            s, ns, x = torch.sigmoid(f["g"]), torch.sigmoid(-f["g"]), f["x"]
            h, _ = _scan(a * keep, na * s * x, h0)
            lam, mu = _adjoint(a * keep, gy, last)
            prev = torch.cat([h0[:, None], h[:, :-1]], dim=1) * keep
            dz = lam * (prev - s * x) * a * na
            dw = lam * na
            outs = [h.to(dt)] + ([h[:, -1]] if case["state"] else [])
            outs += [(dw * s).to(dt), dz.to(dt), (dw * x * s * ns).to(dt)]
            return outs + ([mu[:, 0]] if case["state"] else [])
        D = f["D"]

        def gates(k8):
            u, bg, cg, dtr, og = (_eight(f[k]) if k8 else f[k] for k in ("u", "bg", "cg", "dt", "og"))
            de = DT_MIN + (DT_MAX - DT_MIN) * torch.sigmoid(dtr)
            return u, bg, cg, dtr, og, torch.exp(-de), -torch.expm1(-de)

        u, bg, cg, dtr, og, a, na = gates(False)
        h, entering = _scan(a * keep, na * torch.sigmoid(bg) * u, h0)
        y = (torch.sigmoid(cg) * h + D * u) * torch.sigmoid(og)
        outs = [y.to(dt)] + ([h[:, -1]] if case["state"] else [])
        if case["ckpt"]:
            u, bg, cg, dtr, og, a, na = gates(True)
            h, _ = _scan(a * keep, na * torch.sigmoid(bg) * u, h0, entering)
        sb, sc, so, sd = (torch.sigmoid(t) for t in (bg, cg, og, dtr))
        nb, nc, no, nd = (torch.sigmoid(-t) for t in (bg, cg, og, dtr))
        gs = gy * so
        lam, mu = _adjoint(a * keep, gs * sc, last)
        prev = torch.cat([h0[:, None], h[:, :-1]], dim=1)
        if case["ckpt"]:  # at a span's first token the state before it is the kept one
            prev = prev.clone()
            prev[:, ::SPAN] = entering
        prev = prev * keep
        ddt = -lam * (prev - sb * u) * a * (DT_MAX - DT_MIN) * sd * nd
        dw = lam * na
        outs += [(dw * sb + D * gs).to(dt), (dw * u * sb * nb).to(dt), (gs * h * sc * nc).to(dt), ddt.to(dt),
                 (gy * (sc * h + D * u) * so * no).to(dt), (gs * u).sum(dim=(0, 1), dtype=torch.float64).float()]
        return outs + ([mu[:, 0]] if case["state"] else [])
    if case["op"] == "conv":
        u, w, K = f["u"], f["w"][:, 0], case["K"]
        ids = None if f["seg"] is None else torch.cumsum(f["seg"].long(), dim=1)
        ok = [1.0 if d == 0 or ids is None else (_shift(ids, d) == ids).float()[..., None] for d in range(K)]
        taps = [(u if d == 0 else _shift(u, d)) * ok[d] for d in range(K)]  # the input d tokens back
        v = f["b"] + sum(w[:, K - 1 - d] * taps[d] for d in range(K))
        s = torch.sigmoid(v)
        dv = gy * s * (1.0 + v * torch.sigmoid(-v))
        du = torch.zeros_like(u)
        for d in range(K):
            m = w[:, K - 1 - d] * dv * ok[d]
            du[:, :max(u.shape[1] - d, 0)] += m[:, d:]
        dw = torch.stack([(dv * taps[K - 1 - j]).sum(dim=(0, 1), dtype=torch.float64).float() for j in range(K)], dim=1)
        return [(v * s).to(dt), du.to(dt), dw[:, None], dv.sum(dim=(0, 1), dtype=torch.float64).float()]
    x, w = f["x"], f["w"]
    inv = torch.rsqrt(x.pow(2).mean(dim=-1, keepdim=True) + EPS)
    y = (x * inv * w).to(dt)
    xh = (_eight(x) if case["ckpt"] else x) * inv
    wg = w * gy
    dx = inv * (wg - xh * (wg * xh).mean(dim=-1, keepdim=True))
    return [y, dx.to(dt), (gy * xh).sum(dim=(0, 1), dtype=torch.float64).float()]


def run(state):
    return run_own(state) if own else run_plain(state)


# ------------------------------------------------------------------ the definition, 64 bits
def _sig64(x):
    t = torch.exp(-x.abs())
    return torch.where(x >= 0, 1.0 / (1.0 + t), t / (1.0 + t))


def _e4m3_64(x):
    """e4m3 with a power of two per GROUP channels, from the format's definition:
    four significant bits, the least exponent -6, ties to even."""
    out = torch.zeros_like(x)
    for c in range(0, x.shape[-1], GROUP):
        p = x[..., c:c + GROUP]
        top = p.abs().amax(dim=-1, keepdim=True)
        k = torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 448.0))
        k = torch.where(448.0 * torch.exp2(k - 1) >= top, k - 1, k)  # log2's own rounding
        k = torch.where(448.0 * torch.exp2(k) < top, k + 1, k).clamp(min=-126)
        v = p / torch.exp2(k)
        _, e = torch.frexp(v)
        step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
        out[..., c:c + GROUP] = torch.round(v / step) * step * torch.exp2(k)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    d = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in st.items()}
    gy = d["gy"]
    B, T, C = gy.shape
    if case["op"] == "norm":
        x, w = d["x"], d["w"]
        r = (x.square().sum(-1, keepdim=True) / C + EPS).sqrt()
        xs = _e4m3_64(x) if case["ckpt"] else x
        n = xs / r
        return [x / r * w, (w * gy - n * ((w * gy * n).sum(-1, keepdim=True) / C)) / r, (gy * n).sum((0, 1))]
    start = torch.zeros((B, T), dtype=torch.bool, device=gy.device) if d["seg"] is None else d["seg"] != 0
    if case["op"] == "conv":
        u, w, K = d["u"], d["w"], case["K"]
        pos = torch.arange(T, device=gy.device)
        first = torch.where(start, pos, torch.zeros_like(pos)).cummax(dim=1).values  # the segment's first token
        v = d["b"].expand(B, T, C).clone()
        idx = []
        for j in range(K):
            src = pos - (K - 1 - j)
            live = (src[None] >= first) & (src[None] >= 0)
            idx.append((src.clamp(min=0), live))
            v += w[:, 0, j] * u[:, src.clamp(min=0)] * live[..., None]
        s = _sig64(v)
        dv = gy * (s + v * s * _sig64(-v))
        du, dw = torch.zeros_like(u), torch.zeros_like(w)
        for j, (src, live) in enumerate(idx):
            du.index_add_(1, src, w[:, 0, j] * dv * live[..., None])
            dw[:, 0, j] = (dv * u[:, src] * live[..., None]).sum((0, 1))
        return [v * s, du, dw, dv.sum((0, 1))]

    live = (~start).double()[..., None]
    h0 = d["h0"] if case["state"] else torch.zeros_like(gy[:, 0])

    def forward(a, b, kept=None):
        """States h_t and h_{t-1}, token by token; from `kept` at every SPAN-th token."""
        at, bt = a.transpose(0, 1).contiguous(), b.transpose(0, 1).contiguous()
        hs, ps = torch.empty_like(at), torch.empty_like(at)
        h = h0
        for t in range(T):
            if kept is not None and t % SPAN == 0:
                h = kept[t // SPAN]
            ps[t] = h
            h = torch.addcmul(bt[t], at[t], h, out=hs[t])
        return hs.transpose(0, 1), ps.transpose(0, 1)

    def backward(a, e):
        at, et = a.transpose(0, 1).contiguous(), e.transpose(0, 1).contiguous()
        lam = torch.empty_like(et)
        mu = d["ghf"] if case["state"] else torch.zeros_like(gy[:, 0])
        for t in range(T - 1, -1, -1):
            torch.add(et[t], mu, out=lam[t])
            mu = at[t] * lam[t]
        return lam.transpose(0, 1), mu

    if case["op"] == "gated":
        z, g, x = d["z"], d["g"], d["x"]
        a, q = _sig64(z), _sig64(g)
        b = _sig64(-z) * q * x
        hs, ps = forward(a * live, b)
        lam, mu = backward(a * live, gy)
        res = [hs] + ([hs[:, -1]] if case["state"] else [])
        res += [lam * _sig64(-z) * q, lam * (ps * live - q * x) * a * _sig64(-z), lam * _sig64(-z) * x * q * _sig64(-g)]
        return res + ([mu] if case["state"] else [])
    D = d["D"]
    v = {k: d[k] for k in ("u", "bg", "cg", "dt", "og")}
    rate = DT_MIN + (DT_MAX - DT_MIN) * _sig64(v["dt"])
    hs, ps = forward(torch.exp(-rate) * live, -torch.expm1(-rate) * _sig64(v["bg"]) * v["u"])
    res = [(_sig64(v["cg"]) * hs + D * v["u"]) * _sig64(v["og"])] + ([hs[:, -1]] if case["state"] else [])
    if case["ckpt"]:
        kept = ps[:, ::SPAN].transpose(0, 1)
        v = {k: _e4m3_64(t) for k, t in v.items()}
        rate = DT_MIN + (DT_MAX - DT_MIN) * _sig64(v["dt"])
        hs, ps = forward(torch.exp(-rate) * live, -torch.expm1(-rate) * _sig64(v["bg"]) * v["u"], kept)
    u, a = v["u"], torch.exp(-rate)
    sb, sc, so = _sig64(v["bg"]), _sig64(v["cg"]), _sig64(v["og"])
    gv = gy * so
    lam, mu = backward(a * live, gv * sc)
    dw = lam * -torch.expm1(-rate)
    res += [dw * sb + D * gv, dw * u * sb * _sig64(-v["bg"]), gv * hs * sc * _sig64(-v["cg"]),
            lam * (sb * u - ps * live) * a * (DT_MAX - DT_MIN) * _sig64(v["dt"]) * _sig64(-v["dt"]),
            gy * (sc * hs + D * u) * so * _sig64(-v["og"]), (gv * u).sum((0, 1))]
    return res + ([mu] if case["state"] else [])
