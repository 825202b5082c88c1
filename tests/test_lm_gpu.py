"""The language-model operators on the GPU against 64 bits.

Bounds.  A result in a type is off by half a step of it at most (HALF_STEP of the value)
plus what its sums lose, which is bounded by the sum of their terms' magnitudes:

* attention, 16 bits: the scores and the entering state are sums of two bf16 values
  (2^-17 of a value each), fp32 sums of at most 64 + 128 terms in steps of 16 (12 truncated
  additions of 2^-23), decays from ex2 (2^-22): under 2^-15 of the magnitudes;
* fp32: three values (2^-25), the same sums for each of their products, decays of 2^-22 and
  their exponents' own 2^-24 |log decay| e^-|log decay|: under 2^-18;
* states: one fp32 addition a chunk (2^-24 each, at most 64 chunks here; their mean sign is
  not fixed), products as for fp32: under 2^-18.
"""
import math

import pytest
import torch

import lm_reference as ref
from need_b200 import need_kernels as nk

pytestmark = pytest.mark.gpu

BF, HF, F32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
SUMS = {BF: 2.0 ** -15, HF: 2.0 ** -15, F32: 2.0 ** -18}
STATE = 2.0 ** -18
TINY = 1e-37  # below it values may be flushed to 0


def gen(seed, dev):
    return torch.Generator(device=dev).manual_seed(seed)


def close(got, want, mag, sums, half=0.0):
    err = (got.double() - want).abs()
    lim = half * want.abs() * (1 + 2.0 ** -7) + sums * mag + TINY
    bad = ~(err <= lim)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).nan_to_num(math.inf).max()):.3g} of the bound"


def check_attention(q, k, v, ld, scale=1.0, seg=None, state=None, twice=True):
    out, fin = nk.linear_attention(q, k, v, ld, scale=scale, seg_start=seg, state=state, return_final_state=True)
    want, s, mag, m = ref.attention(q, k, v, ld, float(torch.tensor(scale, dtype=F32)), seg, state)
    assert out.dtype == q.dtype and out.shape == want.shape and fin.shape == s.shape
    small = 2.0 ** -24 if q.dtype == HF else 0.0  # f16 numbers below its least normal one
    close(out, want, mag + small / SUMS[q.dtype], SUMS[q.dtype], ref.HALF_STEP[q.dtype])
    close(fin, s, m, STATE)
    alone = nk.linear_attention(q, k, v, ld, scale=scale, seg_start=seg, state=state)
    if q.dtype == BF:  # without a state to return its sums may hold 2^-17 of their terms (as the scores do), within the bound
        close(alone, want, mag, SUMS[BF], ref.HALF_STEP[BF])
        alone, out2 = (nk.linear_attention(q, k, v, ld, scale=scale, seg_start=seg, state=state) for _ in range(2))
        assert torch.equal(alone, out2) or not twice
    else:
        assert torch.equal(alone, out)
    return out, fin


def make(cuda, B, T, H, dk, dv, dtype, seed=0, heads=None, decay="token", state=False, resets=0):
    g = gen(seed, cuda)
    hq, hk, hv = heads or (H, H, H)
    q, k, v = (torch.randn(B, T, h, d, device=cuda, generator=g).to(dtype) for h, d in ((hq, dk), (hk, dk), (hv, dv)))
    z = torch.randn(B, T, H, device=cuda, generator=g)
    ld = {"token": lambda: torch.nn.functional.logsigmoid(3 + z), "head": lambda: -torch.rand(H, device=cuda, generator=g) / 8,
          "none": lambda: torch.zeros(H, device=cuda), "strong": lambda: -60 * torch.rand(B, T, H, device=cuda, generator=g) ** 4,
          "mixed": lambda: torch.where(z > 1.2, torch.full_like(z, -1e5), torch.where(z < -1.2, torch.full_like(z, -math.inf), -z.abs() / 50)),
          "grow": lambda: 0.02 * z}[decay]()
    seg = None
    if resets:
        seg = (torch.rand(B, T, device=cuda, generator=g) < 1 / resets).to(torch.uint8)
    s0 = torch.randn(B, H, dk, dv, device=cuda, generator=g) if state else None
    return q, k, v, ld, seg, s0


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("T", [1, 2, 15, 63, 64, 65, 200])
def test_attention_lengths(cuda, T, dtype):
    q, k, v, ld, seg, s0 = make(cuda, 2, T, 3, 64, 64, dtype, state=True, resets=30)
    check_attention(q, k, v, ld, 0.125, seg, s0)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("dk,dv", [(1, 1), (8, 16), (16, 8), (40, 72), (33, 65), (128, 64), (64, 128), (100, 200), (72, 56)])
def test_attention_sizes(cuda, dk, dv, dtype):
    q, k, v, ld, seg, s0 = make(cuda, 2, 130, 2, dk, dv, dtype, state=True)
    check_attention(q, k, v, ld, dk ** -0.5, None, s0)


@pytest.mark.parametrize("heads", [(6, 6, 6), (2, 2, 6), (6, 1, 1), (3, 2, 1), (1, 6, 2)])
def test_attention_shared_heads(cuda, heads):
    q, k, v, ld, _, _ = make(cuda, 2, 100, 6, 32, 48, BF, heads=heads)
    check_attention(q, k, v, ld)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("decay", ["token", "head", "none", "strong", "mixed", "grow"])
def test_attention_decays(cuda, decay, dtype):
    """Decays down to e^-100000, dropped states between, none at all, growing states."""
    q, k, v, ld, seg, s0 = make(cuda, 2, 300, 4, 32, 32, dtype, decay=decay, state=True)
    check_attention(q, k, v, ld, 1.0, None, s0)
    check_attention(q, k, v, ld, 1.0, (torch.arange(300, device=cuda) % 37 == 5).expand(2, 300), s0)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("scale", [-0.125, -3.0, 0.0])
@pytest.mark.parametrize("B,T,H,dk,dv", [(2, 65, 3, 64, 64), (2, 300, 3, 64, 72), (1, 300, 2, 128, 64), (1, 3000, 2, 64, 64)])
def test_attention_scales(cuda, B, T, H, dk, dv, scale, dtype):
    """Of either sign and 0, with a state, whole and cut into parts."""
    q, k, v, ld, seg, s0 = make(cuda, B, T, H, dk, dv, dtype, state=True, resets=170)
    check_attention(q, k, v, ld, scale, None, s0)
    check_attention(q, k, v, ld, scale, seg, s0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [64, 300])
@pytest.mark.parametrize("decay", [-0.34, 0.5])
def test_attention_large_scale(cuda, T, decay, dtype):
    """A scale that no decay may be multiplied with first: small q and k, rows of no key among them."""
    q, k, v, _, _, s0 = make(cuda, 2, T, 2, 64, 64, dtype, state=True)
    q, k = q * 2.0 ** -36, k * 2.0 ** -34
    k[:, 10:60] = 0
    ld = torch.zeros(2, T, 2, device=cuda)
    ld[:, 10:120] = decay
    check_attention(q, k, v, ld, 2.0 ** 70, None, None)
    check_attention(q, k, v, ld, -2.0 ** 70, None, s0 * 2.0 ** -34)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("grow,n,then,m", [(0.5, 120, -100.0, 1), (0.5, 100, -90.0, 1), (0.4, 90, -90.0, 1), (0.5, 40, -20.0, 1),
                                           (-1.0, 80, 0.5, 80), (0.5, 128, 0.0, 1)])
def test_attention_grows_and_forgets(cuda, grow, n, then, m, dtype):
    """`n` tokens of one log decay, `m` of another sign, then none; within a chunk, across two,
    and with segments' starts between.  An exponent of 2 below 128 is off by 2^-18 as a float, so
    that each of the three factors of a term (to a chunk's end, over a chunk, from its start) is
    off by ln 2 2^-18 beside what the bounds count: under 2^-16 together."""
    q, k, v, _, _, s0 = make(cuda, 2, 384, 2, 64, 64, dtype, state=True)
    one = torch.zeros(384, device=cuda)
    one[:n], one[n:n + m] = grow, then
    ld = torch.zeros(2, 384, 2, device=cuda)
    ld[0, :, 0] = ld[1, :, 1] = one
    ld[0, 70:, 1], ld[1, 17:, 0] = one[:314], one[:367]
    seg = torch.zeros(2, 384, dtype=torch.uint8, device=cuda)
    seg[:, [60, 200]] = 1
    for marks in (None, seg):
        out, fin = nk.linear_attention(q, k, v, ld, scale=0.125, seg_start=marks, state=s0, return_final_state=True)
        want, s, mag, ms = ref.attention(q, k, v, ld, 0.125, marks, s0)
        close(out, want, mag, SUMS[dtype] + 2.0 ** -16, ref.HALF_STEP[dtype])
        close(fin, s, ms, STATE + 2.0 ** -16)
        close(nk.linear_attention(q, k, v, ld, scale=0.125, seg_start=marks, state=s0), want, mag, SUMS[dtype] + 2.0 ** -16, ref.HALF_STEP[dtype])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("T", [64, 128, 300])
def test_attention_grows_back(cuda, T, dtype):
    """Tokens forgotten to e^-100 that grow back to e^-52: all that the later rows hold is theirs.
    Decays below 2^-126 (the first rows') may be taken for 0, which costs 2^-126 of a term without
    its decay; three exponents below 256 a term lose ln 2 2^-17 each."""
    q, k, v, _, _, _ = make(cuda, 1, T, 2, 32, 32, dtype)
    k[:, 8:64] = 0
    v[:, :8] = v[:, :8] * 2.0 ** 10  # with the scale the last rows' results are normal numbers in f16 too
    ld = torch.zeros(1, T, 2, device=cuda)
    ld[:, 8] = -100.0
    ld[:, 16:64] = 1.0
    scale = 2.0 ** 60
    out, fin = nk.linear_attention(q, k, v, ld, scale=scale, return_final_state=True)
    want, s, mag, m = ref.attention(q, k, v, ld, scale)
    bare = ref.attention(q, k, v, 0 * ld, scale)[2:]
    rows, sums = slice(20, 64), SUMS[dtype] + 2.0 ** -15
    small = 2.0 ** -24 if dtype == HF else 0.0
    close(out[:, rows], want[:, rows], mag[:, rows] + (small + 2.0 ** -126 * bare[0][:, rows]) / sums, sums, ref.HALF_STEP[dtype])
    close(fin, s, m + 2.0 ** -126 * bare[1] / STATE, STATE + 2.0 ** -15)


def test_attention_decay_strides(cuda):
    q, k, v, ld, _, _ = make(cuda, 2, 100, 4, 32, 32, BF)
    want = nk.linear_attention(q, k, v, ld)
    assert torch.equal(nk.linear_attention(q, k, v, ld.transpose(1, 2).contiguous().transpose(1, 2)), want)
    assert torch.equal(nk.linear_attention(q, k, v, ld.double()), want)
    one = ld[:1, :1].expand(2, 100, 4)
    assert torch.equal(nk.linear_attention(q, k, v, one), nk.linear_attention(q, k, v, ld[0, 0].contiguous()))


@pytest.mark.parametrize("B,T,H,dk,dv,dtype", [(1, 4096, 1, 64, 64, BF), (1, 3000, 2, 128, 96, BF), (1, 2500, 3, 40, 40, HF),
                                               (2, 1500, 1, 64, 64, F32), (1, 2000, 1, 33, 17, BF)])
@pytest.mark.parametrize("resets", [0, 400])
def test_attention_few_chains(cuda, B, T, H, dk, dv, dtype, resets):
    """Prompts that are cut into parts."""
    q, k, v, ld, seg, s0 = make(cuda, B, T, H, dk, dv, dtype, decay="head", state=True, resets=resets)
    check_attention(q, k, v, ld, dk ** -0.5, seg, s0)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("T", [129, 192, 193, 320, 900, 1024])
def test_attention_short_parts(cuda, T, dtype):
    """Down to a chunk each, the last one short."""
    q, k, v, ld, seg, s0 = make(cuda, 1, T, 2, 64, 64, dtype, state=True, resets=150)
    check_attention(q, k, v, ld, 0.125, seg, s0)


@pytest.mark.parametrize("H,T,dk,dv", [(52, 4000, 64, 64), (30, 2200, 128, 128), (40, 2700, 40, 64)])
@pytest.mark.parametrize("resets", [0, 500])
def test_attention_some_chains(cuda, H, T, dk, dv, resets):
    """Two or three parts side by side, the first one's outputs ahead of the others'."""
    q, k, v, ld, seg, s0 = make(cuda, 1, T, H, dk, dv, BF, state=True, resets=resets)
    out, fin = check_attention(q, k, v, ld, dk ** -0.5, seg, s0)
    bad = [t.clone() for t in (k, v)]
    bad[0][0, 20, 1, 3], bad[1][0, 2000, 2, 5] = math.inf, math.nan  # in the first part, in a later one
    got, last = nk.linear_attention(q, *bad, ld, scale=dk ** -0.5, seg_start=seg, state=s0, return_final_state=True)
    rest = [h for h in range(H) if h not in (1, 2)]
    assert torch.equal(got[:, :, rest], out[:, :, rest]) and torch.equal(last[:, rest], fin[:, rest])
    _, _, mag, _ = ref.attention(q, k, v, ld, dk ** -0.5, seg, s0)
    for h, t in ((1, 20), (2, 2000)):  # another kernel's sums there
        close(got[:, :t, h], out[:, :t, h].double(), mag[:, :t, h], 2 * SUMS[BF], 2 * ref.HALF_STEP[BF])
        assert not torch.isfinite(got[:, t, h]).all()
        later = [] if seg is None else (seg[0, t + 1:] != 0).nonzero().flatten().tolist()
        if later:  # the next segment is free of it
            after = t + 1 + later[0]
            close(got[:, after:, h], out[:, after:, h].double(), mag[:, after:, h], 2 * SUMS[BF], 2 * ref.HALF_STEP[BF])


def test_attention_parts_and_batches_agree(cuda):
    """One sequence alone (cut into parts) and among many (not cut): the same but for fp32 sums."""
    q, k, v, ld, _, _ = make(cuda, 1, 2048, 2, 64, 64, F32, decay="head")
    a, sa = nk.linear_attention(q, k, v, ld, return_final_state=True)
    b, sb = nk.linear_attention(*(t.expand(150, *t.shape[1:]) for t in (q, k, v)), ld, return_final_state=True)
    assert (b == b[:1]).all() and (sb == sb[:1]).all()
    _, _, mag, m = ref.attention(q, k, v, ld)
    close(b[:1], a.double(), mag, 2 * SUMS[F32])
    close(sb[:1], sa.double(), m, 2 * STATE)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_attention_parts_grow_from_nothing(cuda, dtype):
    """A growing prefix of zero keys (padding on the left): a state of 0 stays 0, though what the
    prefix would multiply it with is past fp32 (e^256 a part and more)."""
    q, k, v, _, _, _ = make(cuda, 1, 2200, 30, 64, 64, dtype)
    k[:, :1400] = 0
    ld = torch.zeros(1, 2200, 30, device=cuda)
    ld[:, :1400] = 0.5
    out, fin = check_attention(q, k, v, ld, 0.125)
    assert (out[:, :1400] == 0).all() and torch.isfinite(fin).all()


@pytest.mark.parametrize("dtype,grow,start,n", [(BF, 0.2, 256, 700), (F32, 0.5, 0, 280)])
def test_attention_parts_grow_from_little(cuda, dtype, grow, start, n):
    """States of 1e-30 that grow by e^140, over e^88 of it in one part: 1e30 is left.  The chunks'
    exponents (202 together, 2^-24 of each lost: ln 2 2^-16.3) and their ex2 (2^-22 each of 22) beside
    what the bounds count: under 2^-15."""
    q, k, v, _, _, s0 = make(cuda, 1, 2200, 30, 64, 64, dtype, state=True)
    k[:, :start + n] = 0
    ld = torch.zeros(1, 2200, 30, device=cuda)
    ld[:, start:start + n] = grow
    s0 = s0 * 1e-30
    out, fin = nk.linear_attention(q, k, v, ld, scale=0.125, state=s0, return_final_state=True)
    want, s, mag, m = ref.attention(q, k, v, ld, 0.125, None, s0)
    close(out, want, mag, SUMS[dtype] + 2.0 ** -15, ref.HALF_STEP[dtype])
    close(fin, s, m, STATE + 2.0 ** -15)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_attention_views(cuda, dtype):
    """Chunks of a projection, heads before tokens, features apart, rows at odd offsets."""
    g = gen(3, cuda)
    B, T, H, d = 2, 150, 3, 40
    p = torch.randn(B, T, 3 * H * d, device=cuda, generator=g).to(dtype)
    ld = -torch.rand(B, T, H, device=cuda, generator=g) / 10
    q, k, v = (t.unflatten(-1, (H, d)) for t in p.chunk(3, -1))
    want = nk.linear_attention(*(t.contiguous() for t in (q, k, v)), ld)
    assert torch.equal(nk.linear_attention(q, k, v, ld), want)
    bh = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(nk.linear_attention(*bh, ld), want)
    apart = [torch.stack([t, t], -1)[..., 0] for t in (q, k, v)]
    assert torch.equal(nk.linear_attention(*apart, ld), want)
    odd = []
    for t in (q, k, v):
        buf = torch.zeros(B, T, H * d + 1, dtype=dtype, device=cuda)
        buf[..., 1:] = t.flatten(2)
        odd.append(buf[..., 1:].unflatten(-1, (H, d)))
    if dtype != BF:  # unaligned bf16 rows go through the kernel of shorter chunks: other sums, within the same bound
        assert torch.equal(nk.linear_attention(*odd, ld), want)
    check_attention(*odd, ld)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", ["q", "k", "v", "decay", "state"])
def test_attention_infinities_stay(cuda, where, bad, dtype):
    """One of them reaches neither the tokens before it nor the next segment."""
    q, k, v, ld, _, s0 = make(cuda, 2, 300, 2, 32, 40, dtype, state=True)
    seg = torch.zeros(2, 300, dtype=torch.uint8, device=cuda)
    seg[0, 140] = 1  # a segment start in the middle of a chunk
    clean, cfin = nk.linear_attention(q, k, v, ld, seg_start=seg, state=s0, return_final_state=True)
    t = 131
    if where == "decay":
        ld = ld.clone()
        ld[0, t, 0] = abs(bad)
    elif where == "state":
        t, s0 = 0, s0.clone()
        s0[0, 0, 3, 5] = bad
    else:
        x = {"q": q, "k": k, "v": v}[where]
        x[0, t, 0, 5] = bad
    out, fin = nk.linear_attention(q, k, v, ld, seg_start=seg, state=s0, return_final_state=True)
    tol = dict(rtol=4 * ref.HALF_STEP[dtype], atol=1e-2 if dtype != F32 else 1e-4)
    keep = torch.ones(2, 300, 2, dtype=torch.bool, device=cuda)
    keep[0, t:140, 0] = False
    assert torch.isfinite(out[keep]).all() and torch.isfinite(fin).all()
    assert torch.allclose(out[keep].float(), clean[keep].float(), **tol)
    assert torch.allclose(fin, cfin, rtol=1e-4, atol=1e-4)
    assert not torch.isfinite(out[0, t, 0]).all()
    if where in ("k", "v", "decay", "state"):
        assert not torch.isfinite(out[0, 139, 0]).all()
    else:
        assert torch.isfinite(out[0, t + 1:140, 0]).all()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", ["q", "k", "v", "state"])
@pytest.mark.parametrize("B,T,H,dk,dv", [(2, 64, 2, 32, 40), (2, 300, 2, 64, 72), (1, 900, 2, 128, 64)])
def test_attention_infinities_are_the_definition_s(cuda, B, T, H, dk, dv, where, bad, dtype):
    """Infinities stay infinities, with their signs, and NaN what is NaN in the recurrence: in the
    rows that see them, in the chunks and parts that follow, in the final state."""
    q, k, v, ld, _, s0 = make(cuda, B, T, H, dk, dv, dtype, state=True)
    if where == "state":
        s0[0, 1, 3, 5] = bad
        s0[-1, 0, 7, 1] = -bad
    else:
        x = {"q": q, "k": k, "v": v}[where]
        x[0, 20, 0, 5], x[-1, T - 40, 1, 9] = bad, -bad
    seg = torch.zeros(B, T, dtype=torch.uint8, device=cuda)
    seg[0, T - 20] = 1
    small = 2.0 ** -24 if dtype == HF else 0.0
    for marks in (None, seg):
        out, fin = nk.linear_attention(q, k, v, ld, scale=0.125, seg_start=marks, state=s0, return_final_state=True)
        alone = nk.linear_attention(q, k, v, ld, scale=0.125, seg_start=marks, state=s0)
        want, s, mag, m = ref.attention(q, k, v, ld, 0.125, marks, s0)
        for got, exact, terms, sums, half in ((out, want, mag, SUMS[dtype], ref.HALF_STEP[dtype]), (fin, s, m, STATE, 0.0),
                                              (alone, want, mag, SUMS[dtype], ref.HALF_STEP[dtype])):
            assert torch.equal(torch.isnan(got), torch.isnan(exact))
            assert torch.equal(torch.isposinf(got), torch.isposinf(exact)) and torch.equal(torch.isneginf(got), torch.isneginf(exact))
            fine = torch.isfinite(exact)
            close(got[fine], exact[fine], terms[fine] + small / sums, sums, half)
    # a state that a segment's start at the first token drops is not looked at
    if where == "state":
        seg[:, 0] = 1
        a, b = (nk.linear_attention(q, k, v, ld, seg_start=seg, state=x, return_final_state=True) for x in (s0, None))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,H,dk,dv", [(2, 64, 2, 32, 40), (2, 300, 2, 64, 72), (1, 900, 2, 128, 64)])
def test_attention_scores_past_fp32(cuda, B, T, H, dk, dv, dtype):
    """q . k past fp32 where the states and the results are not.  Such chunks run token by token: two
    roundings of the state (2^-24 of its terms) a token, dk of the product with q."""
    q, k, v, ld, seg, s0 = make(cuda, B, T, H, dk, dv, dtype, state=True, resets=100)
    q, k, v = q * 2.0 ** 66, k * 2.0 ** 64, v * 2.0 ** -66
    q[:, T // 2:T // 2 + 70] *= 2.0 ** -66  # and some where they are in range
    more = (2 * T + dk) * 2.0 ** -24
    for marks in (None, seg):
        out, fin = nk.linear_attention(q, k, v, ld, scale=0.125, seg_start=marks, state=s0, return_final_state=True)
        alone = nk.linear_attention(q, k, v, ld, scale=0.125, seg_start=marks, state=s0)
        want, s, mag, m = ref.attention(q, k, v, ld, 0.125, marks, s0)
        for got in (out, alone):
            close(got, want, mag, SUMS[dtype] + more, ref.HALF_STEP[dtype])
        close(fin, s, m, STATE + more)


def test_attention_large_values(cuda):
    """Values whose bf16 rounding would be infinite, and products past 65504 in f16."""
    q, k, v, ld, _, _ = make(cuda, 1, 100, 1, 8, 8, F32)
    big = torch.finfo(F32).max
    v[0, 50, 0, 3] = big
    k[0, 50:] = 0
    k[0, 50, 0, 0] = 0.5
    out = nk.linear_attention(q * 2.0 ** -10, k, v, ld)
    want, _, mag, _ = ref.attention(q * 2.0 ** -10, k, v, ld)
    assert torch.isfinite(out).all()
    close(out, want, mag, SUMS[F32], ref.HALF_STEP[F32])
    q, k, v, ld, _, _ = make(cuda, 1, 100, 1, 64, 64, HF)
    check_attention(q * 100, k * 100, v * 2.0 ** -10, ld)
    check_attention(q * 2.0 ** -8, k * 2.0 ** -8, v * 64, ld)


def test_attention_long_sums_of_one_sign(cuda):
    """No decay, all terms positive: the state's rounding may not drift."""
    g = gen(5, cuda)
    q, k, v = (torch.rand(1, 4096, 1, 16, device=cuda, generator=g).to(BF) for _ in range(3))
    _, fin = nk.linear_attention(q, k, v, torch.zeros(1, device=cuda), return_final_state=True)
    want = torch.einsum("bthi,bthj->bhij", k.double(), v.double())
    err = float(((fin.double() - want).abs() / want).max())
    assert err < 2.0 ** -20  # 64 additions, 2^-24 at most and of either sign: 8 of them


def test_attention_waits_given_up(cuda):
    """Blocks of the tensor-core kernel that give a wait up are run again: nothing is lost
    (which do so depends on their timing, and two kernels' sums differ within the bounds)."""
    from need_b200 import abi
    cases = [make(cuda, 2, 500, 3, 64, 64, BF, state=True, resets=90), make(cuda, 1, 3000, 1, 128, 72, BF, decay="head", state=True)]
    torch.cuda.synchronize()
    for polls in (1, 3, 0):
        abi.load().need_test_linear_attention_polls(polls)
        try:
            for c in cases:
                check_attention(*c[:4], 0.125, *c[4:], twice=False)
            torch.cuda.synchronize()
        finally:
            abi.load().need_test_linear_attention_polls(0)


def test_attention_waits_given_up_in_parts(cuda):
    from need_b200 import abi
    lib = abi.load()
    q, k, v, ld, seg, s0 = make(cuda, 1, 4000, 52, 64, 64, BF, state=True, resets=500)
    try:
        lib.need_test_linear_attention_polls(1)
        check_attention(q, k, v, ld, 0.125, seg, s0, twice=False)
    finally:
        lib.need_test_linear_attention_polls(0)
    check_attention(q, k, v, ld, 0.125, seg, s0)


def test_attention_empty(cuda):
    z = lambda *s: torch.zeros(s, device=cuda)  # noqa: E731
    s0 = torch.randn(2, 3, 8, 8, device=cuda)
    out, fin = nk.linear_attention(z(2, 0, 3, 8), z(2, 0, 3, 8), z(2, 0, 3, 8), z(3), state=s0, return_final_state=True)
    assert out.shape == (2, 0, 3, 8) and torch.equal(fin, s0) and fin.data_ptr() != s0.data_ptr()
    out, fin = nk.linear_attention(z(0, 5, 3, 8), z(0, 5, 3, 8), z(0, 5, 3, 8), z(3), return_final_state=True)
    assert out.shape == (0, 5, 3, 8) and fin.shape == (0, 3, 8, 8)


def test_attention_refusals(cuda):
    q, k, v, ld, _, s0 = make(cuda, 2, 10, 4, 8, 8, BF, state=True)
    for bad in (lambda: nk.linear_attention(q[0], k, v, ld), lambda: nk.linear_attention(q, k[:, :9], v, ld),
                lambda: nk.linear_attention(q, k[..., :4], v, ld), lambda: nk.linear_attention(q[:, :, :3], k, v, ld),
                lambda: nk.linear_attention(q, k, v, ld[:, :9]), lambda: nk.linear_attention(q, k, v, ld[0]),
                lambda: nk.linear_attention(q, k, v, ld, state=s0[:1]), lambda: nk.linear_attention(q, k, v, ld, seg_start=ld[..., 0].T)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        nk.linear_attention(q, k.float(), v, ld)
    with pytest.raises(TypeError):
        nk.linear_attention(q.double(), k.double(), v.double(), ld)
    with pytest.raises(RuntimeError):
        nk.linear_attention(q, k.cpu(), v, ld)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        nk.linear_attention(torch.autograd.forward_ad.make_dual(q, torch.ones_like(q)), k, v, ld)


# ------------------------------------------------------------------ the step
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("N,H,dk,dv,heads", [(1, 1, 1, 1, (1, 1, 1)), (5, 4, 64, 64, (4, 4, 4)), (3, 6, 128, 96, (2, 2, 6)), (7, 3, 33, 65, (1, 3, 1)),
                                             (2, 2, 16, 300, (2, 1, 2)), (300, 2, 8, 20, (2, 2, 2))])
def test_step(cuda, N, H, dk, dv, heads, dtype):
    q, k, v, ld, _, _ = make(cuda, N, 1, H, dk, dv, dtype, heads=heads)
    S = N + 3
    pool = torch.randn(S, H, dk, dv, device=cuda)
    slot = torch.randperm(S, device=cuda)[:N].to(torch.int32)
    before = pool.clone()
    version = pool._version
    out = nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], pool, scale=0.3, slot=slot)
    assert pool._version > version
    want, s, mag, m = ref.attention(q, k, v, ld, float(torch.tensor(0.3, dtype=F32)), None, before[slot.long()])
    small = 2.0 ** -24 if dtype == HF else 0.0
    # fp32 products and sums of dk terms: in 8 groups of rows at least, or few of them
    close(out[:, None], want, mag + small * 2 ** 18, 2.0 ** -18, ref.HALF_STEP[dtype])
    close(pool[slot.long()], s, m, 2.0 ** -21)
    rest = torch.ones(S, dtype=torch.bool, device=cuda)
    rest[slot.long()] = False
    assert torch.equal(pool[rest], before[rest])
    again = before[slot.long()].clone()
    out2 = nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], again, scale=0.3)
    assert torch.equal(out2, out) and torch.equal(again, pool[slot.long()])


@pytest.mark.parametrize("N,H,dk,dv", [(3, 5, 16, 16), (2, 3, 32, 64), (4, 7, 9, 5), (600, 2, 128, 128)])
def test_step_shared_blocks(cuda, N, H, dk, dv):
    """Small states, some heads of a sequence side by side; slots of none, twice and past the pool among them."""
    q, k, v, ld, _, _ = make(cuda, N, 1, H, dk, dv, BF)
    pool = torch.randn(N, H, dk, dv, device=cuda)
    before = pool.clone()
    slot = torch.arange(N, device=cuda, dtype=torch.int32)
    slot[1] = -1
    if N > 2:
        slot[2] = 0
    if N > 3:
        slot[3] = N
    out = nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], pool, slot=slot)
    want, s, mag, m = ref.attention(q, k, v, ld, 1.0, None, before)
    good = [0] + list(range(4, N))
    close(out[good, None], want[good], mag[good], 2.0 ** -18, ref.HALF_STEP[BF])
    close(pool[good], s[good], m[good], 2.0 ** -21)
    assert torch.equal(pool[1:4], before[1:4])
    assert (out[1] == 0).all() and torch.isnan(out[2:4]).all()


def test_step_slots(cuda):
    """No sequence, a slot twice, a slot past the pool: nothing else is touched."""
    q, k, v, ld, _, _ = make(cuda, 7, 1, 2, 16, 24, F32)
    q, k, v, ld = q[:, 0], k[:, 0], v[:, 0], ld[:, 0]
    pool = torch.randn(5, 2, 16, 24, device=cuda)
    before = pool.clone()
    slot = torch.tensor([3, -1, 0, 3, 5, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=cuda)
    out = nk.linear_attention_step(q, k, v, ld, pool, slot=slot)
    want = before.clone()
    good = nk.linear_attention_step(q[[0, 2]], k[[0, 2]], v[[0, 2]], ld[[0, 2]], want, slot=slot[[0, 2]])
    assert torch.equal(pool, want) and torch.equal(out[[0, 2]], good)
    assert (out[[1, 6]] == 0).all() and torch.isnan(out[[3, 4, 5]]).all()
    assert torch.equal(pool[[1, 2, 4]], before[[1, 2, 4]])


def test_step_empty_pool(cuda):
    """No state at all: rows without a sequence are 0, the others NaN."""
    q, k, v, ld, _, _ = make(cuda, 4, 1, 2, 16, 24, BF)
    slot = torch.tensor([-1, 0, -5, 3], dtype=torch.int32, device=cuda)
    out = nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], torch.zeros(0, 2, 16, 24, device=cuda), slot=slot)
    assert (out[[0, 2]] == 0).all() and torch.isnan(out[[1, 3]]).all()
    with pytest.raises(ValueError):
        nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], torch.zeros(0, 2, 16, 24, device=cuda))


def test_step_decays(cuda):
    """A log decay of -infinity drops the state, whatever it holds; pool rows apart."""
    q, k, v, _, _, _ = make(cuda, 2, 1, 2, 16, 16, F32)
    wide = torch.full((2, 3, 2, 16, 16), math.nan, device=cuda)
    pool = wide[:, 1]
    pool[1] = 1.0
    ld = torch.tensor([[-math.inf, -math.inf], [-0.5, 0.0]], device=cuda)
    out = nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, pool)
    kv = k[:, 0, :, :, None] * v[:, 0, :, None, :]
    assert torch.equal(pool[0], kv[0]) and torch.isfinite(out).all()
    assert torch.isnan(wide[:, [0, 2]]).all()
    assert torch.allclose(pool[1], torch.exp(ld[1])[:, None, None] + kv[1])


def test_step_refusals(cuda):
    q, k, v, ld, _, _ = make(cuda, 4, 1, 2, 8, 8, BF)
    q, k, v, ld = q[:, 0], k[:, 0], v[:, 0], ld[:, 0]
    pool = torch.zeros(6, 2, 8, 8, device=cuda)
    slot = torch.arange(4, dtype=torch.int32, device=cuda)
    for bad in (lambda: nk.linear_attention_step(q, k, v, ld, pool[:3]), lambda: nk.linear_attention_step(q, k, v, ld, pool[:, :1]),
                lambda: nk.linear_attention_step(q, k, v, ld, pool.transpose(2, 3)),
                lambda: nk.linear_attention_step(q, k, v, ld, pool[:1].expand(6, 2, 8, 8)),
                lambda: nk.linear_attention_step(q, k, v, ld, pool, slot=slot[:3]), lambda: nk.linear_attention_step(q, k, v, ld[:3], pool)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        nk.linear_attention_step(q, k, v, ld, pool.to(BF))
    with pytest.raises(TypeError):
        nk.linear_attention_step(q, k, v, ld, pool, slot=slot.long())
    assert nk.linear_attention_step(q[:0], k[:0], v[:0], ld[:0], pool).shape == (0, 2, 8)


# ------------------------------------------------------------------ the norm
def scales_of(n, size):
    """The least powers of two that fit each group of |n| under 448 of them, in 64 bits."""
    C = n.shape[-1]
    p = torch.nn.functional.pad(n, (0, -C % size)).unflatten(-1, (-1, size)).abs().amax(-1)
    e = torch.ceil(torch.log2(p.clamp_min(1e-300) / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= p, e - 1, e)
    e = torch.where(448.0 * torch.exp2(e) < p, e + 1, e)
    return torch.exp2(e.clamp_min(-126))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 7), (5, 64), (2, 100), (9, 832), (3, 830), (2, 2000), (1, 4096), (2, 8191), (4, 8192)])
def test_norm(cuda, rows, C, dtype):
    g = gen(C, cuda)
    x, y = (torch.randn(rows, C, device=cuda, generator=g).to(dtype) for _ in range(2))
    w = 1 + 0.1 * torch.randn(C, device=cuda, generator=g)
    r, n = nk.residual_rms_norm(x, y, w, 1e-6, scale=0.7)
    wr, _ = ref.residual_norm(x, y, w, 1e-6, 0.7)
    # r: one fp32 rounding before its own: half a step, and 2^-24
    close(r, x.double() + float(torch.tensor(0.7)) * y.double(), x.double().abs() + y.double().abs(), 2.0 ** -24, ref.HALF_STEP[dtype])
    f = r.double()
    want = f / (f.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    small = 2.0 ** -24 if dtype == HF else 0.0
    # the sum's additions (under 40 on a path, 2^-24 each, halved by the root), rsqrt 2^-22, three products
    close(n, want, want.abs() + small * 2 ** 18, 2.0 ** -18, ref.HALF_STEP[dtype])
    for group in (32, 64, 128, None):
        r8, q, s = nk.residual_rms_norm(x, y, w, 1e-6, scale=0.7, out_dtype=F8, group=group)
        size = group or C
        assert torch.equal(r8, r) and q.dtype == F8 and s.shape == (rows, -(-C // size)) and s.dtype == F32
        ws = scales_of(want, size)
        same = ws == s.double()
        # a largest value within 2^-18 of the border may round to either side of it
        near = torch.nn.functional.pad(want, (0, -C % size)).unflatten(-1, (-1, size)).abs().amax(-1) / (448.0 * torch.minimum(ws, s.double()))
        assert (same | ((near - 1).abs() < 2.0 ** -17)).all()
        d = q.double() * s.double().repeat_interleave(size, -1)[:, :C]
        # e4m3: half a step is 2^-4 of a normal value, 2^-10 of the scale below 2^-6
        lim = want.abs() * (2.0 ** -4 + 2.0 ** -17) + 2.0 ** -10 * s.double().repeat_interleave(size, -1)[:, :C]
        assert ((d - want).abs() <= lim).all()


def test_norm_shapes_and_strides(cuda):
    g = gen(1, cuda)
    x, y = (torch.randn(2, 3, 5, 64, device=cuda, generator=g).to(BF) for _ in range(2))
    w = torch.randn(64, device=cuda, generator=g)
    r, n = nk.residual_rms_norm(x, y, w)
    flat = nk.residual_rms_norm(x.reshape(-1, 64), y.reshape(-1, 64), w)
    assert torch.equal(r.reshape(-1, 64), flat[0]) and torch.equal(n.reshape(-1, 64), flat[1])
    assert torch.equal(nk.residual_rms_norm(x.transpose(0, 2), y.transpose(0, 2), w)[1], n.transpose(0, 2))
    buf = torch.zeros(30, 65, dtype=BF, device=cuda)
    buf[:, 1:] = x.reshape(-1, 64)
    for out in (nk.residual_rms_norm(buf[:, 1:], y.reshape(-1, 64), w), nk.residual_rms_norm(x.reshape(-1, 64), y.reshape(-1, 64), w.to(BF).float())):
        assert out[0].shape == (30, 64)
    assert torch.equal(nk.residual_rms_norm(buf[:, 1:], y.reshape(-1, 64), w)[1], flat[1])
    a, b, c = nk.residual_rms_norm(buf[:, 1:], y.reshape(-1, 64), w, out_dtype=F8, group=32)
    a2, b2, c2 = nk.residual_rms_norm(x.reshape(-1, 64), y.reshape(-1, 64), w, out_dtype=F8, group=32)
    assert torch.equal(a, a2) and torch.equal(b.float(), b2.float()) and torch.equal(c, c2)
    one = nk.residual_rms_norm(x[0, 0, 0], y[0, 0, 0], w)
    assert torch.equal(one[1], n[0, 0, 0])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("C,stride,at", [(1324, 1324, 0), (1324, 1326, 0), (1324, 1328, 2), (1326, 1326, 0), (64, 64, 1), (60, 68, 4), (2052, 2056, 8)])
def test_norm_alignments(cuda, C, stride, at, dtype):
    """Rows, weights and channels that 8, 4 or 2 bytes divide."""
    g = gen(C + at, cuda)
    flat = [torch.randn(5 * stride + at, device=cuda, generator=g).to(dtype) for _ in range(2)]
    x, y = (t[at:].unflatten(0, (5, stride))[:, :C] for t in flat)
    w = (1 + 0.1 * torch.randn(C + at, device=cuda, generator=g))[at:]
    r, n = nk.residual_rms_norm(x, y, w, 1e-6, scale=0.7)
    # one fp32 rounding of the sum (torch's expression has two: a tie may fall the other way) before r's own
    close(r, x.double() + float(torch.tensor(0.7)) * y.double(), x.double().abs() + y.double().abs(), 2.0 ** -24, ref.HALF_STEP[dtype])
    f = r.double()
    want = f / (f.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    close(n, want, want.abs(), 2.0 ** -18, ref.HALF_STEP[dtype])
    for group in (32, 128, None):
        r8, q, s = nk.residual_rms_norm(x, y, w, 1e-6, scale=0.7, out_dtype=F8, group=group)
        size = group or C
        val = q.double() * s.double().repeat_interleave(size, -1)[:, :C]
        # e4m3: half a step of the value, or of its least step under the scale
        lim = want.abs() * 2.0 ** -4 * (1 + 2.0 ** -7) + s.double().repeat_interleave(size, -1)[:, :C] * 2.0 ** -10
        assert torch.equal(r8, r) and ((val - want).abs() <= lim).all()


@pytest.mark.parametrize("group", [32, None])
def test_norm_special_values(cuda, group):
    """Rows of zeros, a NaN, an infinity; the others are left as they are."""
    g = gen(2, cuda)
    x, y = (torch.randn(6, 128, device=cuda, generator=g) for _ in range(2))
    w = torch.ones(128, device=cuda)
    clean = nk.residual_rms_norm(x, y, w, out_dtype=F8, group=group)
    x[1], y[1] = 0, 0
    x[2, 40] = math.nan
    x[4, 40] = math.inf
    r, q, s = nk.residual_rms_norm(x, y, w, out_dtype=F8, group=group)
    for i in (0, 3, 5):
        assert torch.equal(q[i].float(), clean[1][i].float()) and torch.equal(s[i], clean[2][i])
    assert (q[1].float() == 0).all() and (s[1] == 2.0 ** -126).all()
    assert torch.isnan(s[2]).all()
    assert torch.isnan(s[4, 40 // group if group else 0])
    assert (nk.residual_rms_norm(x[1:2], y[1:2], w)[1] == 0).all()


def test_norm_refusals(cuda):
    x, w = torch.zeros(3, 64, device=cuda), torch.ones(64, device=cuda)
    for bad in (lambda: nk.residual_rms_norm(x, x[:2], w), lambda: nk.residual_rms_norm(x, x, w[:32]),
                lambda: nk.residual_rms_norm(x, x, w, -1.0), lambda: nk.residual_rms_norm(x, x, w, math.nan)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        nk.residual_rms_norm(x, x.to(BF), w)
    r, n = nk.residual_rms_norm(x[:0], x[:0], w)
    assert r.shape == n.shape == (0, 64)
    r, q, s = nk.residual_rms_norm(x[:0], x[:0], w, out_dtype=F8, group=32)
    assert q.shape == (0, 64) and s.shape == (0, 2)


# ------------------------------------------------------------------ log probabilities
def check_logp(logits, tokens, temperature=1.0, top=0):
    p = nk.token_log_probs(logits, tokens, temperature=temperature, top=top)
    want, h, lp = ref.log_probs(logits, tokens, temperature)
    # (x - m) / t: 2^-23; the sum: ex2 2^-22, its additions 2^-24 each on a path of under 600
    close(p.log_prob, want.nan_to_num(0, 0, 0), want.nan_to_num(0, 0, 0).abs() + h.nan_to_num(0), 2.0 ** -17) if torch.isfinite(want).all() \
        else close(p.log_prob[torch.isfinite(want)], want[torch.isfinite(want)], want[torch.isfinite(want)].abs() + 1, 2.0 ** -17)
    assert torch.equal(torch.isnan(p.log_prob), torch.isnan(want)) and torch.equal(torch.isneginf(p.log_prob), torch.isneginf(want))
    fin = torch.isfinite(h)
    close(p.entropy[fin], h[fin], h[fin], 2.0 ** -16)
    assert torch.equal(torch.isnan(p.entropy), torch.isnan(h))
    if top == 0:
        assert p.top_log_probs is None and p.top_tokens is None
        return p
    x = logits.float()
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][..., :top]
    at = x.gather(-1, order)
    ids = torch.where(torch.isneginf(at), -1, order)
    assert torch.equal(p.top_tokens, ids)
    wl = torch.where(ids < 0, -torch.inf, lp.gather(-1, order))
    wl = torch.where(torch.isnan(lp).any(-1, keepdim=True), torch.nan, wl)
    ok = torch.isfinite(wl)
    close(p.top_log_probs[ok], wl[ok], wl[ok].abs() + 1, 2.0 ** -17)
    assert torch.equal(torch.isnan(p.top_log_probs), torch.isnan(wl)) and torch.equal(torch.isneginf(p.top_log_probs), torch.isneginf(wl))
    return p


def logits_of(cuda, N, V, dtype, seed=0, spread=3.0):
    g = gen(seed, cuda)
    return (spread * torch.randn(N, V, device=cuda, generator=g)).to(dtype), torch.randint(0, V, (N,), device=cuda, generator=g)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (3, 2, 2), (2, 7, 5), (9, 784, 5), (5, 1000, 32), (3, 2048, 20), (2, 2049, 20), (1, 8191, 32),
                                     (7, 32001, 20), (200, 5003, 3), (1, 131072, 32), (3, 131071, 1)])
def test_logp(cuda, N, V, top, dtype):
    x, t = logits_of(cuda, N, V, dtype, N + V)
    check_logp(x, t, top=top)
    check_logp(x, t.int(), temperature=0.6)


@pytest.mark.parametrize("N,V,top,dtype", [(700, 20001, 9, BF), (600, 70001, 20, F32), (310, 9000, 32, HF), (4096, 300, 17, BF), (1, 1 << 21, 32, BF)])
def test_logp_many(cuda, N, V, top, dtype):
    """Rows uncut and cut, many pieces of a thread, blocks for short rows."""
    x, t = logits_of(cuda, N, V, dtype, N + V)
    check_logp(x, t, top=top)


@pytest.mark.parametrize("V", [100, 784, 5001, 70000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_logp_masks(cuda, V, dtype):
    """Rows that a mask leaves nothing, one, a few, or in which it is the type's lowest value."""
    x, t = logits_of(cuda, 8, V, dtype, V)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, V // 3] = 2.0
    t[1] = V // 3
    x[2] = -math.inf
    x[2, [5, V - 1, 17]] = torch.tensor([1.0, 3.0, 3.0], device=cuda, dtype=dtype)
    x[3] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    x[4, 9] = 0.5
    x[5, ::2] = -math.inf
    x[6] = 0.0
    p = check_logp(x, t, top=20)
    assert p.log_prob[0] == -math.inf and p.entropy[0] == 0 and (p.top_tokens[0] == -1).all()
    assert p.log_prob[1] == 0 and p.entropy[1] == 0
    assert p.top_tokens[2, :4].tolist() == [17, V - 1, 5, -1]
    assert p.top_tokens[6].tolist() == list(range(20))


@pytest.mark.parametrize("V", [100, 5001])
def test_logp_infinities(cuda, V):
    x, t = logits_of(cuda, 6, V, F32, V)
    want = nk.token_log_probs(x, t, top=5)
    x[1, 3] = math.nan
    x[2, V - 1] = math.inf
    x[3] = -math.inf
    x[3, 7] = math.nan
    p = check_logp(x, t, top=5)
    assert torch.isnan(p.log_prob[1:4]).all() and p.top_tokens[1, 0] == 3 and p.top_tokens[2, 0] == V - 1 and p.top_tokens[3, :2].tolist() == [7, -1]
    for a, b in zip(p, want):
        assert torch.equal(a[[0, 4, 5]], b[[0, 4, 5]])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("V,top", [(300, 5), (784, 16), (784, 32), (3000, 5), (131072, 20)])
def test_logp_rows_of_nan(cuda, V, top, dtype):
    """NaN are the largest, the lower token first: rows of nothing else, and one at token 0 of a row
    of equal logits (more than are put into order at once)."""
    x = torch.full((4, V), math.nan, device=cuda, dtype=dtype)
    x[1] = 0.5
    x[1, 0] = math.nan
    x[2] = 0.5
    x[2, V - 1] = math.nan
    x[3] = 0.5
    r = nk.token_log_probs(x, torch.zeros(4, dtype=torch.long, device=cuda), top=top)
    lowest = torch.arange(top, device=cuda)
    assert torch.equal(r.top_tokens[0], lowest) and torch.equal(r.top_tokens[1], lowest) and torch.equal(r.top_tokens[3], lowest)
    assert r.top_tokens[2, 0] == V - 1 and torch.equal(r.top_tokens[2, 1:], lowest[:-1])
    assert torch.isnan(r.top_log_probs[:3]).all() and torch.isnan(r.log_prob[:3]).all() and torch.isnan(r.entropy[:3]).all()
    assert torch.allclose(r.top_log_probs[3], torch.full((top,), -math.log(V), device=cuda), rtol=1e-6)


def test_logp_tokens(cuda):
    """None given, and past the vocabulary."""
    x, t = logits_of(cuda, 4, 784, BF)
    t[1], t[2] = -100, 784
    p = nk.token_log_probs(x, t)
    assert p.log_prob[1] == 0 and torch.isnan(p.log_prob[2]) and torch.isfinite(p.entropy).all()


@pytest.mark.parametrize("V", [784, 40000])
def test_logp_ties(cuda, V):
    """More equal logits than the blocks gather: the lower token first."""
    g = gen(V, cuda)
    x = torch.randint(-2, 3, (6, V), device=cuda, generator=g).to(BF)
    x[0] = 1.0
    x[1, :] = torch.arange(V, device=cuda) // 2000
    check_logp(x, torch.zeros(6, dtype=torch.long, device=cuda), top=32)
    y = torch.sort(torch.randn(3, V, device=cuda, generator=g), dim=-1)[0]  # the largest next to each other
    check_logp(y, torch.zeros(3, dtype=torch.long, device=cuda), top=32)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("V,top", [(50, 32), (700, 5), (30000, 20)])
def test_logp_zeros_of_both_signs(cuda, V, top, dtype):
    """-0 and 0 are equal: the lower token first."""
    g = gen(V, cuda)
    x = -torch.rand(5, V, device=cuda, generator=g)
    x[torch.rand(5, V, device=cuda, generator=g) < 0.5] = 0.0
    x[torch.rand(5, V, device=cuda, generator=g) < 0.4] = -0.0
    check_logp(x.to(dtype), torch.zeros(5, dtype=torch.long, device=cuda), top=top)


def test_logp_sure_of_it(cuda):
    """Probabilities near 1: log p and the entropy keep their relative precision."""
    for V in (784, 20000):
        x = torch.zeros(5, V, device=cuda)
        x[:, 11] = torch.tensor([12.0, 20.0, 40.0, 60.0, 80.0], device=cuda)
        t = torch.full((5,), 11, device=cuda)
        p = nk.token_log_probs(x, t)
        r = (V - 1) * torch.exp(-x[:, 11].double())
        want, h = -torch.log1p(r), torch.log1p(r) + x[:, 11].double() * r / (1 + r)
        assert ((p.log_prob.double() - want).abs() <= 2.0 ** -17 * want.abs()).all()
        assert ((p.entropy.double() - h).abs() <= 2.0 ** -16 * h).all()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("N,V", [(3, 1), (2, 7), (9, 784), (5, 2047), (3, 5003), (2, 131072)])
def test_logp_gradient(cuda, N, V, dtype):
    x, t = logits_of(cuda, N, V, dtype, N + V)
    t[0] = -1
    if V > 100:
        x[1, ::3] = -math.inf
        t[1] = 1
    g = gen(7, cuda)
    gl, gh = torch.randn(N, device=cuda, generator=g), torch.randn(N, device=cuda, generator=g)
    for tau, use in ((1.0, (True, True)), (0.7, (True, False)), (1.3, (False, True))):
        x = x.detach().requires_grad_()
        p = nk.token_log_probs(x, t, temperature=tau, top=min(V, 3))
        assert p.log_prob.requires_grad and p.entropy.requires_grad and not p.top_log_probs.requires_grad
        loss = (p.log_prob * gl).sum() * use[0] if use == (True, False) else (p.entropy * gh).sum() if use == (False, True) else \
            (p.log_prob * gl + p.entropy * gh).sum()
        got, = torch.autograd.grad(loss, x)
        a, b = gl * use[0], gh * use[1]
        want = ref.log_probs_grad(x.detach(), t, a, b, tau)
        _, h, lp = ref.log_probs(x.detach(), t, tau)
        q = torch.exp(lp)
        # p: 2^-22 and its exponent's 2^-23 |log p|; the products of the two terms
        mag = (q * (a.abs()[:, None] + b.abs()[:, None] * (lp.clamp_min(-200).abs() + h[:, None]))) / tau
        mag = mag + torch.where(torch.arange(V, device=cuda) == t[:, None], a.abs()[:, None] / tau, 0.0)
        small = 2.0 ** -24 if dtype == HF else 0.0
        assert got.dtype == dtype
        close(got, want, mag + small * 2 ** 17, 2.0 ** -17, ref.HALF_STEP[dtype])


def test_logp_gradient_against_differences(cuda):
    x, t = logits_of(cuda, 2, 9, F32, spread=1.0)
    x = x.requires_grad_()
    p = nk.token_log_probs(x, t)
    got, = torch.autograd.grad((p.log_prob * 0.5 - 2.0 * p.entropy).sum(), x)
    step = 1e-5
    for j in range(9):
        d = torch.zeros(2, 9, dtype=torch.float64, device=cuda)
        d[:, j] = step
        f = [ref.log_probs(x.detach().double() + s * d, t) for s in (1, -1)]
        num = ((f[0][0] - f[1][0]) * 0.5 - 2.0 * (f[0][1] - f[1][1])) / (2 * step)
        assert ((got[:, j] - num).abs() < 1e-5).all()


def test_logp_gradient_of_empty_and_bad_rows(cuda):
    x, t = logits_of(cuda, 4, 300, F32)
    x[1] = -math.inf
    x[2, 5] = math.nan
    t[3] = 300
    x = x.requires_grad_()
    p = nk.token_log_probs(x, t)
    got, = torch.autograd.grad((p.log_prob, p.entropy), x, (torch.ones(4, device=cuda),) * 2)
    assert torch.isfinite(got[0]).all() and (got[1] == 0).all() and torch.isnan(got[2]).all() and torch.isnan(got[3]).all()


def test_logp_views(cuda):
    """Padded vocabularies, odd offsets, more dims, no rows."""
    x, t = logits_of(cuda, 6, 1001, BF)
    want = nk.token_log_probs(x, t, top=4)
    buf = torch.zeros(6, 1024, dtype=BF, device=cuda)
    for off in (0, 1, 8):
        buf[:, off:off + 1001] = x
        view = buf[:, off:off + 1001]
        for a, b in zip(nk.token_log_probs(view, t, top=4), want):
            assert torch.equal(a, b) or (a.dtype == F32 and torch.allclose(a, b, rtol=1e-6, atol=1e-6))
        leaf = view.detach().requires_grad_()
        g1, = torch.autograd.grad(nk.token_log_probs(leaf, t).log_prob.sum(), leaf)
        y = x.detach().requires_grad_()
        g2, = torch.autograd.grad(nk.token_log_probs(y, t).log_prob.sum(), y)
        assert g1.shape == g2.shape and torch.allclose(g1.float(), g2.float(), rtol=2 ** -7, atol=1e-6)
    p = nk.token_log_probs(x.reshape(2, 3, 1001).transpose(0, 1), t.reshape(2, 3).T, top=4)
    for a, b in zip(p, want):  # the copied rows lie elsewhere within 16 bytes: sums in another order, as check_logp bounds them
        a = a.transpose(0, 1).reshape(b.shape)
        assert torch.equal(a, b) if a.dtype != F32 else ((a - b).abs() <= 2.0 ** -16 * (b.abs() + 1)).all()
    p = nk.token_log_probs(x[:0], t[:0], top=4)
    assert p.log_prob.shape == (0,) and p.top_tokens.shape == (0, 4)
    p = nk.token_log_probs(x[0], t[0])
    assert p.log_prob.shape == () and torch.equal(p.log_prob, want.log_prob[0])


def test_logp_refusals(cuda):
    x, t = logits_of(cuda, 4, 50, BF)
    for bad in (lambda: nk.token_log_probs(x, t[:3]), lambda: nk.token_log_probs(x, t, temperature=0.0),
                lambda: nk.token_log_probs(x, t, temperature=math.inf), lambda: nk.token_log_probs(x, t, temperature=-1.0),
                lambda: nk.token_log_probs(x[:, :3], t, top=4), lambda: nk.token_log_probs(x, t, top=-1), lambda: nk.token_log_probs(x[:, :0], t)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        nk.token_log_probs(x, t.float())
    with pytest.raises(RuntimeError):
        nk.token_log_probs(x, t.cpu())
    y = x.float().requires_grad_()
    g, = torch.autograd.grad(nk.token_log_probs(y, t).log_prob.sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


# ------------------------------------------------------------------ together, and how they are run
def layer(p, w, seg=None, state=None):
    """A layer's mixer over whole prompts."""
    H, d = w["H"], w["d"]
    q, k, v = (t.unflatten(-1, (H, d)) for t in (p @ w["qkv"]).chunk(3, -1))
    ld = torch.nn.functional.logsigmoid(3 + p.float() @ w["decay"])
    return nk.linear_attention(q, k, v, ld, scale=d ** -0.5, seg_start=seg, state=state, return_final_state=True)


def test_prompt_then_tokens(cuda):
    """A small model, as it is served: a prompt in two pieces, then tokens one by one from a
    pool of states, against the whole text at once; the scores of drafted tokens at the end."""
    g = gen(11, cuda)
    r = lambda *s: torch.randn(*s, device=cuda, generator=g)  # noqa: E731
    B, T, V, H, d = 3, 90, 784, 4, 32
    C = H * d
    w = {"H": H, "d": d, "qkv": r(C, 3 * C) / C ** 0.5, "decay": r(C, H) / C ** 0.5, "out": r(C, C) / C ** 0.5}
    emb, head, nw = r(V, C), r(C, V) / C ** 0.5, 1 + 0.1 * r(C)
    ids = torch.randint(0, V, (B, T), device=cuda, generator=g)
    x = emb[ids]
    y, fin = layer(x, w)
    h, n = nk.residual_rms_norm(x, y.flatten(2) @ w["out"], nw, scale=0.5)
    want = nk.token_log_probs(n[:, :-1] @ head, ids[:, 1:], top=5)
    pool = torch.zeros(B + 2, H, d, d, device=cuda)
    slot = torch.tensor([4, 0, 2], dtype=torch.int32, device=cuda)
    y1, s1 = layer(x[:, :40], w)
    y2, s2 = layer(x[:, 40:70], w, state=s1)
    pool[slot.long()] = s2
    ys = [y1, y2]
    for t in range(70, T):
        q, k, v = (u.unflatten(-1, (H, d)) for u in (x[:, t] @ w["qkv"]).chunk(3, -1))
        ld = torch.nn.functional.logsigmoid(3 + x[:, t] @ w["decay"])
        ys.append(nk.linear_attention_step(q, k, v, ld, pool, scale=d ** -0.5, slot=slot)[:, None])
    assert torch.allclose(torch.cat(ys, 1), y, rtol=1e-3, atol=1e-4)
    assert torch.allclose(pool[slot.long()], fin, rtol=1e-3, atol=1e-4)
    h2, n2 = nk.residual_rms_norm(x, torch.cat(ys, 1).flatten(2) @ w["out"], nw, scale=0.5)
    got = nk.token_log_probs(n2[:, :-1] @ head, ids[:, 1:], top=5)
    assert torch.allclose(got.log_prob, want.log_prob, rtol=1e-3, atol=1e-3)
    _, n8, s = nk.residual_rms_norm(x, y.flatten(2) @ w["out"], nw, scale=0.5, out_dtype=F8, group=32)
    assert torch.allclose(n8.float() * s.repeat_interleave(32, -1), n, rtol=2 ** -4, atol=1e-3)


def calls(cuda, seed, few=False):
    """One call of each operator with everything on, its inputs, and what it gives."""
    q, k, v, ld, seg, s0 = make(cuda, 1 if few else 3, 700, 2, 64, 64, BF, seed, state=True, resets=200, decay="token")
    x, t = logits_of(cuda, 3, 9000, BF, seed)
    x.requires_grad_()
    g = gen(seed, cuda)
    a, b = (torch.randn(40, 832, device=cuda, generator=g).to(BF) for _ in range(2))
    w = torch.ones(832, device=cuda)
    pool = torch.randn(5, 2, 64, 64, device=cuda, generator=g)
    slot = torch.tensor([1], dtype=torch.int32, device=cuda) if few else torch.tensor([4, 0, 2], dtype=torch.int32, device=cuda)

    def run():
        p = nk.token_log_probs(x, t, top=20)
        dx, = torch.autograd.grad((p.log_prob, p.entropy), x, (torch.ones(3, device=cuda), torch.ones(3, device=cuda)))
        st = pool.clone()
        o = nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], st, slot=slot)
        r, n8, s = nk.residual_rms_norm(a, b, w, out_dtype=F8, group=64)
        return [*nk.linear_attention(q, k, v, ld, seg_start=seg, state=s0, return_final_state=True), *(u.detach() for u in p), dx, st, o,
                r, n8.view(torch.uint8), s]
    return run


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_repeatable(cuda):
    for few in (False, True):
        run = calls(cuda, 1, few)
        want = run()
        for _ in range(5):
            assert same(run(), want)


def test_streams(cuda):
    """Calls at once on streams of their own."""
    runs = [calls(cuda, s, s % 2 == 0) for s in range(4)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [[] for _ in runs]
    for _ in range(3):
        for i, (r, s) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(s):
                got[i].append(r())
    torch.cuda.synchronize()
    assert all(same(x, w) for xs, w in zip(got, want) for x in xs)


def test_graphs(cuda):
    """Two captured graphs of all operators, replayed at once, again and again."""
    runs = [calls(cuda, 10, True), calls(cuda, 11, False)]
    want = [r() for r in runs]
    graphs, outs = [], []
    for r in runs:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            r()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(r())
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(same(o, w) for o, w in zip(outs, want))
    for gr in graphs:
        gr.reset()


def test_first_call_captured():
    """A process whose first calls are captured into a graph."""
    code = """
import torch
from need_b200 import need_kernels as nk
q = torch.randn(1, 300, 2, 64, device="cuda").bfloat16()
ld = torch.full((2,), -0.1, device="cuda")
x, t, w, pool = q.flatten(2), torch.zeros(1, 300, dtype=torch.long, device="cuda"), torch.ones(128, device="cuda"), torch.zeros(1, 2, 64, 64, device="cuda")
def calls():
    y = nk.linear_attention(q, q, q, ld, scale=0.125)
    z = nk.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], ld, pool)
    r, n = nk.residual_rms_norm(x, y.flatten(2), w)
    return [y, z, r, n, *nk.token_log_probs(n, t, top=3)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = calls()
g.replay()
torch.cuda.synchronize()
pool.zero_()
assert all(torch.equal(a, b) for a, b in zip(got, calls()))
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_step_under_inference_mode(cuda):
    q, k, v, ld, _, _ = make(cuda, 2, 1, 2, 32, 32, BF)
    with torch.inference_mode():
        pool = torch.zeros(2, 2, 32, 32, device=cuda)
        nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], pool)
    before = pool.clone()
    with pytest.raises(RuntimeError, match="inference tensor"):
        nk.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], pool)
    assert torch.equal(pool, before) and before.any()


def test_attention_broadcast_batch(cuda):
    """Strides of 0: one k and v for the whole batch."""
    q, k, v, ld, _, _ = make(cuda, 3, 200, 4, 64, 64, BF)
    k1, v1 = (t[:1].expand(3, -1, -1, -1) for t in (k, v))
    check_attention(q, k1, v1, ld, 0.125)
    one = q[:, :1].expand(-1, 200, -1, -1)
    check_attention(one, k, v, ld, 0.125)


def test_no_synchronisation(cuda):
    run = calls(cuda, 3)
    run()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        run()
    finally:
        torch.cuda.set_sync_debug_mode("default")
