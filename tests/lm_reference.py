"""The language-model operators in 64 bits, from their definitions, and the sums of
magnitudes that their rounding errors are bounded by."""
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def expand(t, H):
    """[..., heads, features] with each head for H / heads consecutive ones, in 64 bits."""
    return t.double().repeat_interleave(H // t.shape[-2], dim=-2)


def attention(q, k, v, log_decay, scale=1.0, seg_start=None, state=None):
    """(out, final state, magnitudes of out's terms, of the state's): token by token."""
    H = log_decay.shape[-1]
    q, k, v = (expand(t, H) for t in (q, k, v))
    B, T, _, dk = q.shape
    dv = v.shape[-1]
    a = torch.exp(log_decay.double()).expand(B, T, H)
    drop = torch.isneginf(log_decay).expand(B, T, H)
    if seg_start is not None:
        drop = drop | (seg_start != 0)[..., None]
    s = torch.zeros(B, H, dk, dv, dtype=torch.float64, device=q.device) if state is None else state.double().clone()
    m = s.abs()
    out, mag = torch.empty_like(v), torch.empty_like(v)
    for t in range(T):
        at, dt = a[:, t, :, None, None], drop[:, t, :, None, None]
        kv = k[:, t, :, :, None] * v[:, t, :, None, :]
        s = torch.where(dt, kv, at * s + kv)
        m = torch.where(dt, kv.abs(), at * m + kv.abs())
        out[:, t] = scale * (q[:, t, :, :, None] * s).sum(-2)
        mag[:, t] = abs(scale) * (q[:, t, :, :, None].abs() * m).sum(-2)
    return out, s, mag, m


def residual_norm(x, y, w, eps, scale):
    """(r in x's dtype, n in 64 bits)."""
    r = (x.double() + float(torch.tensor(scale, dtype=torch.float32)) * y.double()).to(x.dtype)
    f = r.double()
    return r, f / (f.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def log_probs(logits, tokens, temperature=1.0):
    """(log p, entropy, all log probabilities)."""
    x = logits.double() / temperature
    lp = torch.log_softmax(x, dim=-1)
    empty = torch.isneginf(x).all(-1)
    lp = torch.where(empty[..., None], -torch.inf, lp)
    p = torch.exp(lp)
    h = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    h = torch.where(torch.isnan(lp).any(-1), torch.nan, h)
    t = tokens.long()
    got = lp.gather(-1, t.clamp(0, x.shape[-1] - 1)[..., None])[..., 0]
    return torch.where(t < 0, 0.0, torch.where(t >= x.shape[-1], torch.nan, got)), h, lp


def log_probs_grad(logits, tokens, g, gh, temperature=1.0):
    x = logits.double() / temperature
    _, h, lp = log_probs(logits, tokens, temperature)
    p = torch.exp(lp)
    given = tokens >= 0
    hit = torch.zeros_like(p).scatter(-1, tokens.long().clamp_min(0)[..., None], 1.0) * given[..., None]
    d = (g.double() * given)[..., None] * (hit - p) - gh.double()[..., None] * torch.where(p > 0, p * (lp + h[..., None]), 0.0)
    return torch.where(torch.isneginf(x).all(-1, keepdim=True), 0.0, d) / temperature
