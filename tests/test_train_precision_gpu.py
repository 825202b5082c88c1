"""The training scans' precision where a gate is saturated, a state decays far or a
stream hardly varies, element by element, on the GPU.

Every input is positive (logits aside), so that states, lam and every gradient but
the decay's are sums of positive terms: a relative error of the factors is one of the
result, however small the result.  The decay's gradient holds one difference,
h_{t-1} - w_t, whose error goes by h_{t-1} + w_t.

Bounds.  A gate (sigmoid, 1 - sigmoid, e^-r, 1 - e^-r) is off by 2^-22 for fp32
streams (library functions and an IEEE division); for 16-bit ones by 2^-21 (hardware
exp2 and reciprocal, 2 ulp each) and the rounding of the exponent's argument, 2^-24
times the logit.  A state takes a's error once per token, lam again, and at most 16
more factors and sums follow; a step r of up to dt_max carries its own error into e^-r
dt_max times over.  Then half a step of the result's dtype (an eighth more for errors
that carry a value over a tie), or a step of its subnormals."""
import pytest
import torch

import train_reference as ref
from need_b200 import need_kernels as nk

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
DTYPES = pytest.mark.parametrize("dtype", [FP, BF, HF], ids=["f32", "bf16", "f16"])
CKPTS = pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])


def gate_error(dtype, far, step=0.0):
    return (2.0 ** -22 if dtype == FP else 2.0 ** -21 + far * 2.0 ** -24) * (1 + step)


def check(what, got, want, size, arith):
    """|got - want| within `arith` of `size` and the rounding of `want`."""
    eps, small = torch.finfo(got.dtype).eps, torch.finfo(got.dtype).smallest_normal
    err = (got.detach().cpu().double() - want).abs()
    bound = arith * size + 1.125 * eps / 2 * want.abs() + small * eps
    assert bool((err <= bound).all()), (f"{what}: {int((~(err <= bound)).sum())} of {err.numel()} off; worst "
                                        f"{float((err / bound).max()):.3g} of the bound")


def states(a, b, h0, start, kept=None):
    """h_t and h_{t-1} of h_t = [start ? 0 : a_t h_{t-1}] + b_t, from `kept` at every chunk."""
    h, hs, ps = h0, [], []
    for t in range(a.shape[1]):
        if kept is not None and t % ref.SPAN == 0:
            h = kept[:, t]
        prev = torch.where(start[:, t, None], torch.zeros_like(h), h)
        ps.append(prev)
        h = a[:, t] * prev + b[:, t]
        hs.append(h)
    return torch.stack(hs, 1), torch.stack(ps, 1)


def adjoint(a, e, last, start):
    mu, lams = last, []
    for t in range(a.shape[1] - 1, -1, -1):
        lam = e[:, t] + mu
        lams.append(lam)
        mu = torch.where(start[:, t, None], torch.zeros_like(lam), a[:, t] * lam)
    return torch.stack(lams[::-1], 1), mu


def entering(a, b, h0, start):
    """The state before every token, resets aside (what a chunk starts from)."""
    h, _ = states(a, b, h0, start)
    return torch.cat([h0[:, None], h[:, :-1]], 1)


def gated64(x, z, g, h0, go, gf, start, ckpt):
    """Outputs and gradients with their sizes: (value, size) by name."""
    s = torch.sigmoid
    a, b = s(z), s(-z) * s(g) * x
    h, prev = states(a, b, h0, start)
    res = {"h": (h, h), "final": (h[:, -1], h[:, -1])}
    if ckpt:
        kept = entering(a, b, h0, start)
        x, z, g = (ref.e4m3(t) for t in (x, z, g))
        a, b = s(z), s(-z) * s(g) * x
        h, prev = states(a, b, h0, start, kept)
    lam, mu = adjoint(a, go, gf, start)
    w, f = s(g) * x, lam * a * s(-z)
    res["dx"] = (lam * s(-z) * s(g),) * 2
    res["dz"] = (f * (prev - w), f * (prev + w.abs()))
    res["dg"] = (lam * s(-z) * x * s(g) * s(-g),) * 2
    res["dh0"] = (mu, mu)
    return res


def ssd64(u, bg, cg, dt, og, D, h0, go, gf, lo, hi, start, ckpt):
    s = torch.sigmoid

    def maps(u, bg, dt):
        r = lo + (hi - lo) * s(dt)
        return torch.exp(-r), -torch.expm1(-r), -torch.expm1(-r) * s(bg) * u

    a, n, b = maps(u, bg, dt)
    h, prev = states(a, b, h0, start)
    y = (s(cg) * h + D * u) * s(og)
    res = {"y": (y, y), "final": (h[:, -1], h[:, -1])}
    if ckpt:
        kept = entering(a, b, h0, start)
        u, bg, cg, dt, og = (ref.e4m3(t) for t in (u, bg, cg, dt, og))
        a, n, b = maps(u, bg, dt)
        h, prev = states(a, b, h0, start, kept)
    gs = go * s(og)
    lam, mu = adjoint(a, gs * s(cg), gf, start)
    w, f = s(bg) * u, lam * a * (hi - lo) * s(dt) * s(-dt)
    res["du"] = (lam * n * s(bg) + D * gs,) * 2
    res["dbg"] = (lam * n * u * s(bg) * s(-bg),) * 2
    res["dcg"] = (gs * h * s(cg) * s(-cg),) * 2
    res["ddt"] = (f * (w - prev), f * (w + prev))
    res["dog"] = (go * (s(cg) * h + D * u) * s(og) * s(-og),) * 2
    res["dD"] = ((gs * u).sum((0, 1)),) * 2
    res["dh0"] = (mu, mu)
    return res


def positive(gen, *shape):
    return 0.1 + torch.rand(*shape, generator=gen)


def run_gated(cuda, case, dtype, ckpt, arith, seg=None, parts=None):
    x, z, g, h0, go, gf = case
    start = torch.zeros(x.shape[:2], dtype=torch.bool) if seg is None else seg != 0
    want = gated64(*(t.double() for t in case), start, ckpt is not None)
    ls = [t.to(cuda).requires_grad_() for t in (x, z, g, h0)]
    outs = nk.gated_scan_train(*ls[:3], seg_start=None if seg is None else seg.to(cuda), h0=ls[3],
                               return_final_state=True, checkpoint=ckpt)
    grads = torch.autograd.grad(outs, ls, [go.to(cuda), gf.to(cuda)])
    for what, got in zip(("h", "final", "dx", "dz", "dg", "dh0"), [*outs, *grads]):
        if parts is None or what in parts:
            check(what, got, *want[what], arith)


def run_ssd(cuda, case, lo, hi, dtype, ckpt, arith, seg=None, parts=None):
    u, bg, cg, dt, og, D, h0, go, gf = case
    start = torch.zeros(u.shape[:2], dtype=torch.bool) if seg is None else seg != 0
    want = ssd64(*(t.double() for t in case), lo, hi, start, ckpt is not None)
    ls = [t.to(cuda).requires_grad_() for t in (u, bg, cg, dt, og, D, h0)]
    outs = nk.ssd_scan_train(*ls[:6], lo, hi, seg_start=None if seg is None else seg.to(cuda), h0=ls[6],
                             return_final_state=True, checkpoint=ckpt)
    grads = torch.autograd.grad(outs, ls, [go.to(cuda), gf.to(cuda)])
    for what, got in zip(("y", "final", "du", "dbg", "dcg", "ddt", "dog", "dD", "dh0"), [*outs, *grads]):
        if parts is None or what in parts:
            check(what, got, *want[what], arith)


# ------------------------------------------------------------------ decaying states

def decaying(dtype, B):
    """Nothing comes in: h_t = a^t h_0, down to 1e-31 of h_0."""
    gen = torch.Generator().manual_seed(1)
    T, C = 24, 40
    zero = torch.zeros(B, T, C, dtype=dtype)
    h0, go, gf = positive(gen, B, C), positive(gen, B, T, C).to(dtype), positive(gen, B, C)
    z = (-3 + 0.1 * torch.randn(B, T, C, generator=gen)).to(dtype)
    gates = [torch.randn(B, T, C, generator=gen).to(dtype) for _ in range(4)]
    return (zero, z, zero, h0, go, gf), (zero, *gates, torch.zeros(C), h0, go, gf), T


@CKPTS
@DTYPES
@pytest.mark.parametrize("B", [2, 200])
def test_decayed_states(cuda, dtype, B, ckpt):
    """Each to the last bit of its dtype, however far it has decayed inside a tile."""
    gated, ssd, T = decaying(dtype, B)
    run_gated(cuda, gated, dtype, ckpt, (T + 16) * gate_error(dtype, 4), parts=("h", "final"))
    run_ssd(cuda, ssd, 2.5, 3.5, dtype, ckpt, (T + 16) * gate_error(dtype, 4, 3.5), parts=("y", "final"))


@DTYPES
@pytest.mark.parametrize("B", [2, 200])
def test_decayed_states_in_the_backward(cuda, dtype, B):
    """Gradients that hold such states."""
    gated, ssd, T = decaying(dtype, B)
    run_gated(cuda, gated, dtype, None, (T + 16) * gate_error(dtype, 4))
    run_ssd(cuda, ssd, 2.5, 3.5, dtype, None, (T + 16) * gate_error(dtype, 4, 3.5))


# ------------------------------------------------------------------ streams that hardly vary

@DTYPES
@pytest.mark.parametrize("B", [2, 200])
def test_constant_stream(cuda, dtype, B):
    """A stream at its own limit: h_t = w for good, so the decay's gradient, lam a (1 -
    a) (h_{t-1} - w_t), is 0 but for the rounding of states to fp32 -- not of anything
    held in 16 bits between the passes."""
    gen = torch.Generator().manual_seed(2)
    T, C = 16, 40
    x = (100 * positive(gen, B, 1, C)).to(dtype).expand(B, T, C).contiguous()
    g = torch.randn(B, 1, C, generator=gen).to(dtype).expand(B, T, C).contiguous()
    z = (1 + 3 * torch.rand(B, T, C, generator=gen)).to(dtype)
    h0 = (torch.sigmoid(g[:, 0].double()) * x[:, 0].double()).float()
    go, gf = positive(gen, B, T, C).to(dtype), positive(gen, B, C)
    run_gated(cuda, (x, z, g, h0, go, gf), dtype, None, (T + 16) * gate_error(dtype, 4))
    xs = [x, g] + [torch.randn(B, T, C, generator=gen).to(dtype) for _ in range(3)]
    run_ssd(cuda, (*xs, positive(gen, C), h0, go, gf), 0.001, 0.2, dtype, None, (T + 16) * gate_error(dtype, 4, 0.2))


# ------------------------------------------------------------------ saturated gates

def marks(gen, B, T):
    m = (torch.rand(B, T, generator=gen) < 0.3).to(torch.uint8)
    m[:, -1] = 1
    return m


# B, T, C, resets: whole rows of warps and none; tiles of 32 and of 64 channels
SHAPES = pytest.mark.parametrize("B,T,C,resets", [(1, 70, 40, False), (2, 21, 72, True), (200, 64, 24, False)])


@CKPTS
@DTYPES
@SHAPES
def test_saturated_gates_gated(cuda, B, T, C, resets, dtype, ckpt):
    """Logits to +-20: every gradient to its own last bits, where s, 1 - s or both
    their products are as small as 1e-17."""
    gen = torch.Generator().manual_seed(3)
    z, g = (40 * torch.rand(B, T, C, generator=gen) - 20 for _ in range(2))
    case = [positive(gen, B, T, C), z, g, positive(gen, B, C), positive(gen, B, T, C), positive(gen, B, C)]
    case = [t.to(dtype) if t.dim() == 3 else t for t in case]
    run_gated(cuda, case, dtype, ckpt, (T + 16) * gate_error(dtype, 20), marks(gen, B, T) if resets else None)


@CKPTS
@DTYPES
@SHAPES
@pytest.mark.parametrize("lo,hi", [(0.001, 0.2), (0.0, 12.0)])
def test_saturated_gates_ssd(cuda, B, T, C, resets, lo, hi, dtype, ckpt):
    """The same; with steps to 12, where e^-r is small too."""
    gen = torch.Generator().manual_seed(4)
    logits = [40 * torch.rand(B, T, C, generator=gen) - 20 for _ in range(4)]
    case = [positive(gen, B, T, C), *logits, positive(gen, C), positive(gen, B, C), positive(gen, B, T, C), positive(gen, B, C)]
    case = [t.to(dtype) if t.dim() == 3 else t for t in case]
    run_ssd(cuda, case, lo, hi, dtype, ckpt, (T + 16) * gate_error(dtype, 20, hi), marks(gen, B, T) if resets else None)


# ------------------------------------------------------------------ ordinary inputs

def turned(got, want):
    """How many bf16 results are not `want` rounded."""
    return float((got.detach().cpu() != want.detach().to(BF)).float().mean())


@CKPTS
def test_ssd_is_rounded_once(cuda, ckpt):
    """bf16 results on ordinary inputs are the 64-bit ones rounded, but for values next
    to a tie: an error e in fp32 turns e / (eps / 2) of them, and e is some 2^-17 of the
    value (tens of tokens at 2^-21 each, and differences).  A factor rounded to 11 bits
    between the passes would turn 2^-12 / 2^-8 = 1 in 16 of them."""
    gen = torch.Generator().manual_seed(5)
    B, T, C = 4, 200, 64
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    xs, D, h0, go, gf = [r(B, T, C).to(BF) for _ in range(5)], 1 + 0.1 * r(C), r(B, C), r(B, T, C).to(BF), r(B, C)
    ls = [t.double().requires_grad_() for t in (*xs, D, h0)]
    w = ref.ssd(*ls, 0.001, 0.2, None, ckpt is not None)
    want = [w[0], *torch.autograd.grad(w, ls, [go.double(), gf.double()])[:5]]
    ls = [t.to(cuda).requires_grad_() for t in (*xs, D, h0)]
    o = nk.ssd_scan_train(*ls[:6], 0.001, 0.2, h0=ls[6], return_final_state=True, checkpoint=ckpt)
    got = [o[0], *torch.autograd.grad(o, ls, [go.to(cuda), gf.to(cuda)])[:5]]
    off = [turned(a, b) for a, b in zip(got, want)]
    assert max(off) <= 0.02, off


@CKPTS
def test_gated_is_rounded_once(cuda, ckpt):
    """As test_ssd_is_rounded_once."""
    gen = torch.Generator().manual_seed(6)
    B, T, C = 4, 200, 64
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    case, go, gf = [r(B, T, C).to(BF), (r(B, T, C) + 4).to(BF), r(B, T, C).to(BF), r(B, C)], r(B, T, C).to(BF), r(B, C)
    ls = [t.double().requires_grad_() for t in case]
    w = ref.gated(*ls, None, ckpt is not None)
    want = [w[0], *torch.autograd.grad(w, ls, [go.double(), gf.double()])[:3]]
    ls = [t.to(cuda).requires_grad_() for t in case]
    o = nk.gated_scan_train(*ls[:3], h0=ls[3], return_final_state=True, checkpoint=ckpt)
    got = [o[0], *torch.autograd.grad(o, ls, [go.to(cuda), gf.to(cuda)])[:3]]
    off = [turned(a, b) for a, b in zip(got, want)]
    assert max(off) <= 0.02, off
