"""The training operators in plain torch, any dtype (the tests use float64),
written for autograd: token by token, with selections for resets.  Also the
8-bit rounding, and how far a kernel's result may lie from these."""
import torch

SPAN, GROUP = 64, 64


def e4m3(x):
    """x in e4m3 with one power of two per GROUP channels of a token: four
    significant bits, least exponent -6, ties to even."""
    out = torch.empty_like(x)
    for c in range(0, x.shape[-1], GROUP):
        g = x[..., c:c + GROUP]
        top = g.abs().amax(-1, keepdim=True)
        m, e = torch.frexp(top)
        e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126)  # the least e with top <= 448 * 2^e
        v = torch.ldexp(g, -e)
        step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 1).clamp(min=-6) - 3)
        out[..., c:c + GROUP] = torch.ldexp(torch.round(v / step) * step, e)
    return out


def scan(a, b, h0, seg, kept=None):
    """h_t = [seg_t ? 0 : a_t h_{t-1}] + b_t over [B, T, C]; the states before each
    token too.  `kept` [B, chunks, C]: values that replace the state entering each
    chunk (the gradient still flows through it)."""
    h, hs, before = h0, [], []
    for t in range(a.shape[1]):
        if kept is not None and t % SPAN == 0:
            h = h + (kept[:, t // SPAN] - h).detach()
        before.append(h)
        cur = a[:, t] * h
        if seg is not None:
            cur = torch.where(seg[:, t, None] != 0, torch.zeros_like(cur), cur)
        h = cur + b[:, t]
        hs.append(h)
    return torch.stack(hs, 1), torch.stack(before, 1)


def _through(x, value):
    """x with another value, the gradient straight through."""
    return x + (value - x).detach()


def gated(x, z, g, h0, seg=None, ckpt=False):
    def run(x, z, g, kept=None):
        return scan(torch.sigmoid(z), torch.sigmoid(-z) * torch.sigmoid(g) * x, h0, seg, kept)

    h, before = run(x, z, g)
    if not ckpt:
        return h, h[:, -1]
    h8, _ = run(*(_through(t, e4m3(t.detach())) for t in (x, z, g)), before[:, ::SPAN].detach())
    return _through(h8, h.detach()), _through(h8[:, -1], h[:, -1].detach())


def ssd(u, bg, cg, dt, og, D, h0, lo, hi, seg=None, ckpt=False):
    def run(u, bg, cg, dt, og, kept=None):
        r = lo + (hi - lo) * torch.sigmoid(dt)
        h, before = scan(torch.exp(-r), -torch.expm1(-r) * torch.sigmoid(bg) * u, h0, seg, kept)
        return (torch.sigmoid(cg) * h + D * u) * torch.sigmoid(og), h[:, -1], before

    xs = (u, bg, cg, dt, og)
    y, f, before = run(*xs)
    if not ckpt:
        return y, f
    y8, f8, _ = run(*(_through(t, e4m3(t.detach())) for t in xs), before[:, ::SPAN].detach())
    return _through(y8, y.detach()), _through(f8, f.detach())


def conv_silu(u, w, b, seg=None):
    B, T, C = u.shape
    K = w.shape[1]
    v = torch.zeros_like(u) if b is None else b.expand(B, T, C)
    ids = torch.zeros(B, T, dtype=torch.long) if seg is None else torch.cumsum(seg.long(), 1)
    for d in range(min(K, T)):
        src = torch.cat([torch.zeros_like(u[:, :d]), u[:, :T - d]], 1)
        sid = torch.cat([torch.full((B, d), -1), ids[:, :T - d]], 1)
        src = torch.where((sid == ids)[..., None], src, torch.zeros_like(src))
        v = v + w[:, K - 1 - d] * src
    return v * torch.sigmoid(v)


def rms_norm(x, w, eps, ckpt=False):
    if not ckpt:
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    # y's value is the true one's; its gradient r (g - n mean(g n)), n = r x8, w dy = g
    r = torch.rsqrt(x.detach().square().mean(-1, keepdim=True) + eps)
    n8 = r * e4m3(x.detach())
    lin = r * x - n8 * (n8 * r * x).mean(-1, keepdim=True)
    y = lin * w.detach() + n8 * w
    return _through(y, (x * r * w).detach())


def close(got, want, dtype, reach, what=""):
    """Whether `got` may be `want` computed in fp32 from streams of `dtype` and
    rounded once, element by element and in the 2-norm.

    Rounding: half a step, eps / 2 of the value; an eighth more because the error
    below can carry a value over a tie.
    Arithmetic: a gate's relative error d is a few ulp -- 2^-22 for fp32 streams
    (library exp and expm1, divisions, the products after them), 2^-21 for 16-bit
    streams (hardware exp2 and reciprocal, about 2 ulp each, and the products).  A
    state that reaches back `reach` tokens takes a's error once per step, so it is
    off by at most reach * d of the largest state; lam by as much again, and the
    products of the two by both.  Differences (h - w) and slopes (s (1 - s) <= 1/4)
    put the operands at up to 4 times the largest result.  Sums over all tokens
    are trees whose steps round by 2^-24, less than this.
    In the 2-norm the steps' errors have independent signs: sqrt(reach) for reach.
    Kept sigmoids: a bf16 gradient of the scans is a product of at most four that the
    kernel holds in f16 from its first pass to its second, 2^-12 off each (of the
    value, and in the difference h - w of the larger operand): 4 * 2^-12, half of
    bf16's own half step."""
    d = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -21
    eps = torch.finfo(got.dtype).eps
    reach = max(reach, 4)
    w = want.detach().to(torch.float64)
    assert got.shape == w.shape, (what, got.shape, w.shape)
    if w.numel() == 0:
        return
    err = (got.detach().cpu().to(torch.float64) - w).abs()
    top = float(w.abs().max())
    tiny = float(torch.finfo(got.dtype).smallest_normal) * eps  # a step of the subnormals
    kept = 4 * 2.0 ** -12 if got.dtype == torch.bfloat16 else 0.0
    bound = 1.125 * (eps / 2 + kept) * w.abs() + (2 * 4 * reach * d + kept) * top + tiny
    assert bool((err <= bound).all()), (f"{what}: {int((~(err <= bound)).sum())} of {err.numel()} beyond; worst "
                                        f"{float((err / bound).max()):.2f} of the bound, error {float(err.max()):.3e}, "
                                        f"largest {top:.3e}")
    norm = float(torch.linalg.norm(w))
    assert float(torch.linalg.norm(err)) <= (eps / 2 + kept + 2 * 4 * reach ** 0.5 * d) * norm + tiny * w.numel() ** 0.5, (
        f"{what}: 2-norm off by {float(torch.linalg.norm(err)) / norm:.3e}")
