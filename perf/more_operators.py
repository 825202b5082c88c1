"""The language-model operators' cases: what each computes, in plain torch, in 64
bits, and through the package's entry points.

  attention  S_t = exp(log_decay_t) S_{t-1} + k_t^T v_t,  o_t = scale q_t S_t  for each
             head, over whole prompts (linear_attention)
  step       the same for one token of each sequence, its state in a pool
             (linear_attention_step)
  norm       r = x + scale y,  n = r rsqrt(mean(r^2) + eps) w, n in x's type or in
             8 bits with scales (residual_rms_norm)
  logp       log p(token), the entropy and the largest log probabilities of each
             row of logits, and the gradient (token_log_probs)

A marked token (``seg``) starts a segment: the state before it does not reach it.
Heads of q, k and v are shared by runs of consecutive heads of the decay.  8 bits:
e4m3 under one power of two per token and group of channels, the least that fits.
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
CHUNK = 64  # tokens of the plain form's chunks
TOP = 448.0  # e4m3's largest value


# ------------------------------------------------------------------ cases
def listed():
    c = []

    def attention(name, B, T, H, dk, dv, dtype, **kw):
        c.append({"name": name, "op": "attention", "B": B, "T": T, "H": H, "Hq": H, "Hk": H, "Hv": H, "dk": dk, "dv": dv,
                  "dtype": dtype, "decay": "token", "resets": 0, "state": False, "chunked": False, **kw})

    def step(name, N, H, dk, dv, dtype, **kw):
        c.append({"name": name, "op": "step", "N": N, "H": H, "Hq": H, "Hk": H, "Hv": H, "dk": dk, "dv": dv,
                  "dtype": dtype, "decay": "token", **kw})

    def norm(name, B, T, C, dtype, group):
        c.append({"name": name, "op": "norm", "B": B, "T": T, "C": C, "dtype": dtype, "group": group})

    def logp(name, N, V, dtype, **kw):
        c.append({"name": name, "op": "logp", "N": N, "V": V, "dtype": dtype, "top": 0, "grad": False, "masked": False,
                  "temperature": 1.0, **kw})

    # the prefill workload's shape: packed windows of documents
    attention("attention 16x4096 16x64 bf16", 16, 4096, 16, 64, 64, "bf16", resets=1024)
    # one layer of the 350M model's width over its batch, q, k and v chunks of one projection
    attention("attention 8x2048 13x64 bf16", 8, 2048, 13, 64, 64, "bf16", chunked=True)
    # one long prompt with wide heads and a fixed decay for each head, its state kept for decoding
    attention("attention 1x16384 32x128 bf16", 1, 16384, 32, 128, 128, "bf16", decay="head", state=True)
    # ragged rows and heads, q and k shared by three heads each, a state carried in and out
    attention("attention 3x777 6x40x72 f16", 3, 777, 6, 40, 72, "f16", Hq=2, Hk=2, resets=200, state=True)
    # a short fp32 call
    attention("attention 2x300 4x64 f32", 2, 300, 4, 64, 64, "f32", state=True)
    # one token for a full decoding batch
    step("step 256 13x64 bf16", 256, 13, 64, 64, "bf16")
    # one token of three sequences: latency
    step("step 3 8x128x96 f16", 3, 8, 128, 96, "f16", Hk=4, Hq=4, decay="head")
    # the 350M model's block over its batch, the norm's output in 8 bits for the next projection
    norm("norm 8x2048x832 bf16 8-bit", 8, 2048, 832, "bf16", 32)
    # the same for a decoding batch, in 16 bits
    norm("norm 64x1x832 f16", 64, 1, 832, "f16", 0)
    # a training batch's loss and policy terms over the model's vocabulary, with the gradient
    logp("logp 16384x784 bf16 grad", 16384, 784, "bf16", grad=True)
    # scores of drafted tokens over a wide odd vocabulary, part of it masked, with alternatives
    logp("logp 1024x50021 bf16 top 20", 1024, 50021, "bf16", top=20, masked=True, temperature=0.7)
    # one step of a small batch: few rows, a long vocabulary
    logp("logp 4x131072 f32 top 5", 4, 131072, "f32", top=5)
    return c


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attention", "attention", "step", "norm", "logp"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("attention", "step"):
        H = log(1, 32)
        dk, dv = log(8, 128), log(8, 128)
        if rng.random() < 0.6:
            dk, dv = max(8, dk // 8 * 8), max(8, dv // 8 * 8)
        part = [d for d in range(1, H + 1) if H % d == 0]
        case = {"op": op, "H": H, "Hq": H, "Hk": H, "Hv": H, "dk": dk, "dv": dv, "dtype": dtype,
                "decay": rng.choice(["token", "token", "head"])}
        if rng.random() < 0.4:
            case["Hk"] = case["Hq"] = rng.choice(part)
        elif rng.random() < 0.4:
            case["Hk"] = case["Hv"] = rng.choice(part)
        if op == "step":
            N = log(1, 512)
            while N * H * dk * dv > 20 << 20:
                N = N // 2
            return {**case, "N": max(1, N)}
        B, T = log(1, 16), log(1, 16384)
        while B * T * H * (dk + dv) > 48 << 20:  # well inside the largest listed case's work
            if B > 1:
                B //= 2
            else:
                T //= 2
        return {**case, "B": B, "T": T, "resets": 0 if rng.random() < 0.5 else log(4, 2048),
                "state": rng.random() < 0.5, "chunked": rng.random() < 0.4}
    if op == "norm":
        B, T, C = log(1, 16), log(1, 4096), log(8, 8192)
        if rng.random() < 0.6:
            C = max(8, C // 8 * 8)
        while B * T * C > 24 << 20:
            if B > 1:
                B //= 2
            else:
                T //= 2
        return {"op": op, "B": B, "T": T, "C": C, "dtype": dtype, "group": rng.choice([0, 32, 64, 128, -1])}
    N, V = log(1, 8192), log(256, 131072)
    while N * V > 40 << 20:
        N //= 2
    grad = rng.random() < 0.4
    return {"op": op, "N": max(1, N), "V": V, "dtype": dtype, "top": 0 if grad else rng.choice([0, 1, 5, 20]), "grad": grad,
            "masked": rng.random() < 0.4, "temperature": rng.choice([1.0, 1.0, 0.7])}


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("attention", "step"):
        H, dk, dv = case["H"], case["dk"], case["dv"]
        n = case["N"] if case["op"] == "step" else case["B"] * case["T"]
        row = es * (case["Hq"] * dk + case["Hk"] * dk + case["Hv"] * dv + H * dv)
        per = n if case["decay"] == "token" else 1
        state = 4 * H * dk * dv
        if case["op"] == "step":
            held = 2 * n * state
        else:
            held = 2 * case["B"] * state if case["state"] else 0
        mask = n if case.get("resets") else 0
        return {"bytes": n * row + 4 * H * per + held + mask, "flops": 4 * n * H * dk * dv}  # the update, the read
    if case["op"] == "norm":
        n = case["B"] * case["T"] * case["C"]
        out = es * n
        if case["group"]:
            size = case["C"] if case["group"] < 0 else case["group"]
            out = n + 4 * case["B"] * case["T"] * -(-case["C"] // size)
        return {"bytes": 3 * es * n + out + 4 * case["C"], "flops": 8 * n}  # x, y in; r, n out
    n = case["N"] * case["V"]
    return {"bytes": es * n * (2 if case["grad"] else 1) + 16 * case["N"], "flops": (16 if case["grad"] else 6) * n}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    """Inputs as the layers hand them over: activations near N(0, 1), decays near
    those of the recurrent block (memories of some fifty tokens; fixed ones of 8 to
    256), logits with a spread of 3."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 6113 + 29)
    dt = DT[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    st = {"case": case}
    if case["op"] in ("attention", "step"):
        H, dk, dv = case["H"], case["dk"], case["dv"]
        lead = (case["N"],) if case["op"] == "step" else (case["B"], case["T"])
        heads, sizes = (case["Hq"], case["Hk"], case["Hv"]), (dk, dk, dv)
        wide = [h * s for h, s in zip(heads, sizes)]
        if case.get("chunked"):  # views into one projection's output
            parts = randn(*lead, sum(wide)).to(dt).split(wide, dim=-1)
        else:
            parts = [randn(*lead, w).to(dt) for w in wide]
        for name, t, h, s in zip("qkv", parts, heads, sizes):
            st[name] = t.unflatten(-1, (h, s))
        if case["decay"] == "token":
            st["decay"] = torch.nn.functional.logsigmoid(4.0 + randn(*lead, H))
        else:
            st["decay"] = torch.log1p(-torch.exp2(-(3.0 + 5.0 * torch.arange(H, device=dev) / H)))
        st["scale"] = dk ** -0.5
        if case["op"] == "step":
            pool = case["N"] + case["N"] // 4 + 1
            st["pool"] = randn(pool, H, dk, dv)
            st["slot"] = torch.randperm(pool, generator=g, device=dev)[:case["N"]].to(torch.int32)
            return st
        st["state"] = 0.5 * randn(case["B"], H, dk, dv) if case["state"] else None
        st["seg"] = None
        if case["resets"]:
            rs = np.random.RandomState(seed % (1 << 31))
            m = np.zeros(lead, np.uint8)
            for b in range(lead[0]):
                t = 0
                while t < lead[1]:
                    m[b, t] = 1
                    t += int(rs.randint(1, 2 * case["resets"]))
            if case["state"]:  # the first segment goes on from the carried state
                m[:, 0] = 0
            st["seg"] = torch.from_numpy(m).to(dev)
        return st
    if case["op"] == "norm":
        shape = (case["B"], case["T"], case["C"])
        st["x"], st["y"] = randn(*shape).to(dt), randn(*shape).to(dt)
        st["w"] = 1.0 + 0.1 * randn(case["C"])
        st["scale"] = 0.5
        return st
    N, V = case["N"], case["V"]
    x = 3.0 * randn(N, V)
    if case["masked"]:  # tokens that a grammar or a filter rules out
        x = x.masked_fill(torch.rand((N, V), generator=g, device=dev) < 0.3, -math.inf)
    st["logits"] = x.to(dt)
    st["tokens"] = torch.multinomial(torch.softmax(x, dim=-1), 1, generator=g)[:, 0]
    if case["grad"]:
        st["logits"].requires_grad_()
        st["g"], st["gh"] = randn(N) / N, 0.01 * randn(N) / N
    return st


# ------------------------------------------------------------------ the package's operators
def run_own(st):
    from need_b200 import need_kernels as nk
    case = st["case"]
    if case["op"] == "attention":
        out = nk.linear_attention(st["q"], st["k"], st["v"], st["decay"], scale=st["scale"], seg_start=st["seg"],
                                  state=st["state"], return_final_state=case["state"])
        return list(out) if case["state"] else [out]
    if case["op"] == "step":
        out = nk.linear_attention_step(st["q"], st["k"], st["v"], st["decay"], st["pool"], scale=st["scale"],
                                       slot=st["slot"])
        return [out, st["pool"]]
    if case["op"] == "norm":
        if not case["group"]:
            return list(nk.residual_rms_norm(st["x"], st["y"], st["w"], EPS, scale=st["scale"]))
        r, q, s = nk.residual_rms_norm(st["x"], st["y"], st["w"], EPS, scale=st["scale"], out_dtype=torch.float8_e4m3fn,
                                       group=case["group"] if case["group"] > 0 else None)
        return [r, _values(q, s, case), s]
    p = nk.token_log_probs(st["logits"], st["tokens"], temperature=case["temperature"], top=case["top"])
    out = [p.log_prob, p.entropy]
    if case["top"]:
        out += [p.top_log_probs, p.top_tokens]
    if case["grad"]:
        out = [t.detach() for t in out] + list(torch.autograd.grad(out, [st["logits"]], [st["g"], st["gh"]]))
    return out


def _values(q, s, case):
    """What 8-bit values stand for; four bits and a power of two fit bf16."""
    size = case["C"] if case["group"] < 0 else case["group"]
    return q.bfloat16() * s.repeat_interleave(size, dim=-1)[..., :case["C"]].bfloat16()


# ------------------------------------------------------------------ plain forms, 32 bits
def _heads(t, H):
    """[B, T, h, d] with each head for its H / h consecutive ones, as [B, H, T, d] in 32 bits."""
    return t.float().repeat_interleave(H // t.shape[2], dim=2).transpose(1, 2)


def _chunks(t, fill=0.0):
    """[B, H, T, ...] as [B, H, chunks, CHUNK, ...]."""
    pad = -t.shape[2] % CHUNK
    if pad:
        t = torch.cat([t, torch.full((*t.shape[:2], pad, *t.shape[3:]), fill, dtype=t.dtype, device=t.device)], dim=2)
    return t.unflatten(2, (-1, CHUNK))


def _attention_plain(st):
    case = st["case"]
    H, dt = case["H"], DT[case["dtype"]]
    q, k, v = (_chunks(_heads(st[n], H)) for n in "qkv")
    B, T = st["q"].shape[:2]
    d = st["decay"].double()
    d = _chunks((d.expand(B, T, H) if d.dim() == 1 else d).transpose(1, 2))  # [B, H, n, CHUNK]
    g = torch.cumsum(d, dim=-1)  # in 64 bits: differences of long sums follow
    if st["seg"] is None:
        seg = torch.zeros((1, 1, g.shape[2], CHUNK), dtype=torch.long, device=d.device)
    else:
        seg = torch.cumsum(_chunks((st["seg"] != 0).long()[:, None], 0), dim=-1)
    at = torch.arange(CHUNK, device=d.device)
    same = (seg[..., :, None] == seg[..., None, :]) & (at[:, None] >= at)
    # the later tokens' places are left out before exp: they may overflow
    w = torch.exp(torch.where(same, g[..., :, None] - g[..., None, :], -math.inf).float())
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * w, v)
    whole = (seg[..., -1] == 0)
    out_of = torch.where(whole, g[..., -1], -math.inf).exp().float()  # of the entering state, over the chunk
    left = torch.where(seg == seg[..., -1:], g[..., -1:] - g, -math.inf).exp().float()
    own_part = torch.matmul((k * left[..., None]).transpose(-1, -2), v)
    # the state that enters each chunk: a scan over the chunks, by doubling
    first = torch.zeros_like(own_part[:, :, 0]) if st["state"] is None else st["state"]
    a, s = out_of.expand(B, H, -1), own_part
    s = torch.cat([s[:, :, :1] + a[:, :, :1, None, None] * first[:, :, None], s[:, :, 1:]], dim=2)
    step = 1
    while step < s.shape[2]:
        s = torch.cat([s[:, :, :step], s[:, :, step:] + a[:, :, step:, None, None] * s[:, :, :-step]], dim=2)
        a = torch.cat([a[:, :, :step], a[:, :, step:] * a[:, :, :-step]], dim=2)
        step *= 2
    entering = torch.cat([first[:, :, None], s[:, :, :-1]], dim=2)
    into = torch.where(seg == 0, g, -math.inf).exp().float()
    o = (o + into[..., None] * torch.matmul(q, entering)) * st["scale"]
    o = o.flatten(2, 3)[:, :, :T].transpose(1, 2).to(dt)
    return [o, s[:, :, -1]] if case["state"] else [o]


def _step_plain(st):
    case = st["case"]
    H = case["H"]
    q, k, v = (st[n].float().repeat_interleave(H // st[n].shape[1], dim=1) for n in "qkv")
    at = st["slot"].long()
    s = st["pool"][at] * torch.exp(st["decay"])[..., None, None] + k[..., :, None] * v[..., None, :]
    st["pool"][at] = s
    return [((q[..., :, None] * s).sum(-2) * st["scale"]).to(DT[case["dtype"]]), st["pool"]]


def _norm_plain(st):
    case = st["case"]
    C, dt = case["C"], DT[case["dtype"]]
    r = (st["x"].float() + st["scale"] * st["y"].float()).to(dt)
    f = r.float()
    n = f * torch.rsqrt(f.pow(2).mean(dim=-1, keepdim=True) + EPS) * st["w"]
    if not case["group"]:
        return [r, n.to(dt)]
    size = C if case["group"] < 0 else case["group"]
    p = torch.nn.functional.pad(n, (0, -C % size)).unflatten(-1, (-1, size))
    m, e = torch.frexp(p.abs().amax(dim=-1, keepdim=True))
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp_min(-126)  # 448 is 0.875 2^9
    q = torch.ldexp(p, -e).to(torch.float8_e4m3fn)
    s = torch.ldexp(torch.ones_like(m), e)[..., 0]
    return [r, _values(q.flatten(-2)[..., :C], s, case), s]


def _logp_plain(st):
    case = st["case"]
    tau = case["temperature"]
    x = st["logits"].detach().float()
    m, top = x.max(dim=-1, keepdim=True)
    z = (x - m) / tau
    e = torch.exp(z).scatter(1, top, 0.0)  # without the largest, whose term is 1
    rest = e.sum(dim=-1, dtype=torch.float64)[:, None]
    lse = torch.log1p(rest).float()
    lp = z - lse
    h = (lse.double() - torch.where(e > 0, e * z, 0.0).sum(dim=-1, keepdim=True, dtype=torch.float64) / (1.0 + rest)).float()
    out = [lp.gather(1, st["tokens"][:, None])[:, 0], h[:, 0]]
    if case["top"]:
        v, i = torch.sort(x, dim=-1, descending=True, stable=True)
        out += [lp.gather(1, i[:, :case["top"]]), i[:, :case["top"]].clone()]
    if case["grad"]:
        p = torch.exp(lp)
        hit = torch.zeros_like(p).scatter(1, st["tokens"][:, None], 1.0)
        dx = st["g"][:, None] * (hit - p) - st["gh"][:, None] * torch.where(p > 0, p * (lp + h), 0.0)
        out.append((dx / tau).to(DT[case["dtype"]]))
    return out


PLAIN = {"attention": _attention_plain, "step": _step_plain, "norm": _norm_plain, "logp": _logp_plain}


def run(state):
    return run_own(state) if own else PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definition, 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    d = {n: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for n, t in st.items()}
    if case["op"] in ("attention", "step"):
        H = case["H"]
        at = [torch.arange(H, device=d["q"].device) // (H // d[n].shape[-2]) for n in "qkv"]
        q, k, v = (d[n].index_select(-2, i) for n, i in zip("qkv", at))
        if case["op"] == "step":
            s = torch.exp(d["decay"])[..., None, None] * d["pool"][st["slot"].long()]
            s += torch.einsum("nhi,nhj->nhij", k, v)
            pool = d["pool"].clone()
            pool[st["slot"].long()] = s
            return [st["scale"] * torch.einsum("nhi,nhij->nhj", q, s), pool]
        B, T, _, dk = q.shape
        dv = v.shape[-1]
        a = torch.exp(d["decay"]).expand(B, T, H).clone()
        if st["seg"] is not None:
            a[st["seg"] != 0] = 0.0
        # token by token, all sequences and heads at once
        a = a.permute(1, 0, 2).reshape(T, B * H, 1, 1)
        q = st["scale"] * q.permute(1, 0, 2, 3).reshape(T, B * H, 1, dk)
        k = k.permute(1, 0, 2, 3).reshape(T, B * H, dk, 1)
        v = v.permute(1, 0, 2, 3).reshape(T, B * H, 1, dv)
        s = q.new_zeros(B * H, dk, dv) if st["state"] is None else d["state"].reshape(B * H, dk, dv).clone()
        o = torch.empty_like(v)
        for t in range(T):
            s.mul_(a[t]).baddbmm_(k[t], v[t])
            torch.bmm(q[t], s, out=o[t])
        o = o.reshape(T, B, H, dv).permute(1, 0, 2, 3)
        return [o, s.reshape(B, H, dk, dv)] if case["state"] else [o]
    if case["op"] == "norm":
        C = case["C"]
        r = d["x"] + st["scale"] * d["y"]
        f = r.to(DT[case["dtype"]]).double()  # the stream as it is kept
        n = d["w"] * f / (f.square().sum(-1, keepdim=True) / C + EPS).sqrt()
        if not case["group"]:
            return [r, n]
        size = C if case["group"] < 0 else case["group"]
        vals, scales = torch.empty_like(n), []
        for c in range(0, C, size):
            x = n[..., c:c + size]
            top = x.abs().amax(-1, keepdim=True)
            e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / TOP))
            e = torch.where(TOP * torch.exp2(e - 1) >= top, e - 1, e)  # log2's own rounding
            e = torch.where(TOP * torch.exp2(e) < top, e + 1, e).clamp(min=-126)
            u = x / torch.exp2(e)
            _, b = torch.frexp(u)
            ulp = torch.exp2((b - 1).clamp(min=-6).double() - 3)  # four significant bits, the least exponent -6
            vals[..., c:c + size] = torch.round(u / ulp) * ulp * torch.exp2(e)
            scales.append(torch.exp2(e))
        return [r, vals, torch.cat(scales, dim=-1)]
    x = d["logits"] / case["temperature"]
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m)
    lse = torch.log(p.sum(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    lp = x - m - lse
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    rows = torch.arange(case["N"], device=x.device)
    h = -plp.sum(-1)
    out = [lp[rows, st["tokens"]], h]
    if case["top"]:
        out += [torch.topk(lp, case["top"], dim=-1).values, None]
    if case["grad"]:
        dx = -(p * d["g"][:, None]) - d["gh"][:, None] * (plp + p * h[:, None])
        dx[rows, st["tokens"]] += d["g"]
        out.append(dx / case["temperature"])
    return out
