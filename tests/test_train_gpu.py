"""The training operators (gated_scan_train, ssd_scan_train,
ssd_conv_silu_train, rms_norm_train) on the GPU against float64 references."""
import numpy as np
import pytest
import torch

import train_reference as ref
from need_b200 import abi
from need_b200 import need_kernels as nk

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
LO, HI = 0.001, 0.2


def rnd(gen, *shape, mean=0.0, dtype=FP):
    return (torch.randn(*shape, generator=gen) + mean).to(dtype)


def marks(gen, B, T, every):
    if not every:
        return None
    m = (torch.rand(B, T, generator=gen) < 1.0 / every).to(torch.uint8)
    for t in (0, 7, 8, 63, 64, T - 1):  # rows at the edges of warps and chunks
        if t < T:
            m[0, t] = (t + B) % 2
    return m


def grads64(fn, leaves, gos):
    """Outputs and gradients of fn(*leaves) in float64."""
    ls = [x.detach().double().requires_grad_() for x in leaves]
    outs = fn(*ls)
    outs = outs if isinstance(outs, tuple) else (outs,)
    return outs, torch.autograd.grad(outs, ls, [g.double() for g in gos])


def on(dev, ts):
    return [t.detach().to(dev).requires_grad_() for t in ts]


def compare(outs, grads, wouts, wgrads, dtype, reach):
    for k, (a, b) in enumerate(zip(list(outs) + list(grads), list(wouts) + list(wgrads))):
        ref.close(a, b, dtype, reach, f"result {k}")


# ------------------------------------------------------------------ the recurrences

SHAPES = [  # B, T, C, reset every
    (1, 1, 8, 0), (2, 1, 72, 1), (1, 3, 64, 0), (2, 8, 64, 3), (3, 63, 40, 0), (2, 64, 64, 9), (2, 65, 136, 0),
    (1, 129, 200, 20), (2, 200, 13, 0), (1, 330, 100, 50), (1, 700, 64, 0),
    (200, 70, 24, 15), (97, 131, 70, 0), (70, 90, 40, 0),  # chains enough for the wide tiles
]


def gated_case(B, T, C, every, dtype, seed=0):
    gen = torch.Generator().manual_seed(1000 * B + T + C + seed)
    x, z, g = rnd(gen, B, T, C, dtype=dtype), rnd(gen, B, T, C, mean=2.0, dtype=dtype), rnd(gen, B, T, C, dtype=dtype)
    return [x, z, g, rnd(gen, B, C)], marks(gen, B, T, every), [rnd(gen, B, T, C, dtype=dtype), rnd(gen, B, C)]


def ssd_case(B, T, C, every, dtype, seed=0):
    gen = torch.Generator().manual_seed(2000 * B + T + C + seed)
    leaves = [rnd(gen, B, T, C, dtype=dtype) for _ in range(5)] + [1 + 0.1 * rnd(gen, C), rnd(gen, B, C)]
    return leaves, marks(gen, B, T, every), [rnd(gen, B, T, C, dtype=dtype), rnd(gen, B, C)]


def reach_of(T):
    return min(T, 1000)  # 1 / (1 - a): 2 to 400 tokens at decay logits near 2, at most 1000 at dt_min = 0.001


@pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])
@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,C,every", SHAPES)
def test_gated(cuda, B, T, C, every, dtype, ckpt):
    leaves, seg, gos = gated_case(B, T, C, every, dtype)
    want = grads64(lambda x, z, g, h0: ref.gated(x, z, g, h0, seg, ckpt is not None), leaves, gos)
    ls = on(cuda, leaves)
    outs = nk.gated_scan_train(*ls[:3], seg_start=None if seg is None else seg.to(cuda), h0=ls[3],
                               return_final_state=True, checkpoint=ckpt)
    grads = torch.autograd.grad(outs, ls, [g.to(cuda) for g in gos])
    assert outs[0].dtype == dtype and outs[1].dtype == FP and [g.dtype for g in grads] == [l.dtype for l in ls]
    compare(outs, grads, *want, dtype, reach_of(T))


@pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])
@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,C,every", SHAPES)
def test_ssd(cuda, B, T, C, every, dtype, ckpt):
    leaves, seg, gos = ssd_case(B, T, C, every, dtype)
    want = grads64(lambda *a: ref.ssd(*a, LO, HI, seg, ckpt is not None), leaves, gos)
    ls = on(cuda, leaves)
    outs = nk.ssd_scan_train(*ls[:6], LO, HI, seg_start=None if seg is None else seg.to(cuda), h0=ls[6],
                             return_final_state=True, checkpoint=ckpt)
    grads = torch.autograd.grad(outs, ls, [g.to(cuda) for g in gos])
    compare(outs, grads, *want, dtype, reach_of(T))


@pytest.mark.parametrize("lo,hi", [(0.0, 0.2), (0.0, 3.0), (0.5, 0.5), (0.0, 0.0)])
@pytest.mark.parametrize("dtype", [FP, BF], ids=["f32", "bf16"])
def test_ssd_step_ranges(cuda, lo, hi, dtype):
    """Steps from none (a = 1) to many e-folds a token."""
    leaves, seg, gos = ssd_case(2, 150, 64, 30, dtype, seed=5)
    want = grads64(lambda *a: ref.ssd(*a, lo, hi, seg), leaves, gos)
    ls = on(cuda, leaves)
    outs = nk.ssd_scan_train(*ls[:6], lo, hi, seg_start=seg.to(cuda), h0=ls[6], return_final_state=True)
    compare(outs, torch.autograd.grad(outs, ls, [g.to(cuda) for g in gos]), *want, dtype, 150)


@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=["f32", "bf16", "f16"])
def test_far_logits(cuda, dtype):
    """Saturated gates: logits to +-200, where 1 - sigmoid must not be a difference."""
    gen = torch.Generator().manual_seed(3)
    B, T, C = 1, 70, 64
    x, g = rnd(gen, B, T, C, dtype=dtype), (100 * rnd(gen, B, T, C)).to(dtype)
    z = torch.linspace(-200, 200, T * C).reshape(B, T, C)[:, torch.randperm(T, generator=gen)].to(dtype)
    leaves, gos = [x, z, g, rnd(gen, B, C)], [rnd(gen, B, T, C, dtype=dtype), rnd(gen, B, C)]
    want = grads64(lambda *a: ref.gated(*a), leaves, gos)
    ls = on(cuda, leaves)
    outs = nk.gated_scan_train(*ls[:3], h0=ls[3], return_final_state=True)
    compare(outs, torch.autograd.grad(outs, ls, [g.to(cuda) for g in gos]), *want, dtype, T)


def test_chunks_of_one_projection(cuda):
    """Views into a packed in-projection: no copies, and the gradient reaches it."""
    gen = torch.Generator().manual_seed(4)
    B, T, C = 2, 100, 72
    proj = rnd(gen, B, T, 5 * C, dtype=BF)
    D, go = 1 + rnd(gen, C), rnd(gen, B, T, C, dtype=BF)
    h0 = torch.zeros(B, C, dtype=torch.float64)
    want = grads64(lambda p, d: ref.ssd(*p.chunk(5, -1), d, h0, LO, HI)[0], [proj, D], [go])
    p, d = on(cuda, [proj, D])
    y = nk.ssd_scan_train(*p.chunk(5, -1), d, LO, HI)
    compare([y], torch.autograd.grad(y, [p, d], go.to(cuda)), *want, BF, T)


def test_layouts(cuda):
    """Transposed, offset and expanded inputs and output gradients."""
    gen = torch.Generator().manual_seed(5)
    B, T, C = 3, 90, 64
    leaves, seg, gos = gated_case(B, T, C, 20, BF, seed=9)
    want = grads64(lambda *a: ref.gated(*a, seg), leaves, gos)
    x = leaves[0].to(cuda).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()   # [T, B, C] in memory
    z = torch.empty(B * T * C + 1, dtype=BF, device=cuda)[1:].view(B, T, C).copy_(leaves[1]).requires_grad_()  # odd offset
    g = leaves[2].to(cuda).transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()   # channel stride T
    h0 = leaves[3].to(cuda).t().contiguous().t().requires_grad_()
    mask = seg.to(cuda).t().contiguous().t()
    outs = nk.gated_scan_train(x, z, g, seg_start=mask, h0=h0, return_final_state=True)
    go = [gos[0].to(cuda).transpose(0, 1).contiguous().transpose(0, 1), gos[1].to(cuda).t().contiguous().t()]
    compare(outs, torch.autograd.grad(outs, [x, z, g, h0], go), *want, BF, T)

    ls = on(cuda, leaves[:3])  # .sum(): the output's gradient is one expanded number
    one = torch.ones(B, T, C)
    want = grads64(lambda *a: ref.gated(*a, torch.zeros(B, C, dtype=torch.float64))[0], leaves[:3], [one])
    y = nk.gated_scan_train(*ls)
    compare([y], torch.autograd.grad(y.float().sum(), ls), *want, BF, T)
    y = nk.gated_scan_train(*ls)
    y.sum().backward()
    compare([y], [t.grad for t in ls], *want, BF, T)

    # one row given to every sequence (batch stride 0), and one sequence's gates for all
    xe = leaves[0][:1].to(cuda).requires_grad_()
    ye = nk.gated_scan_train(xe.expand(B, T, C), ls[1], ls[2])
    want = grads64(lambda x, z, g: ref.gated(x.expand(B, T, C), z, g, torch.zeros(B, C, dtype=torch.float64))[0],
                   [leaves[0][:1], *leaves[1:3]], [gos[0]])
    got = torch.autograd.grad(ye, [xe, ls[1], ls[2]], gos[0].to(cuda))
    compare([ye], got[1:], want[0], want[1][1:], BF, T)
    # autograd adds B rounded gradients and rounds the sum: B half steps of each, and one of the sum
    assert float((got[0].cpu().double() - want[1][0]).abs().max()) <= (B + 1) * 2 ** -8 * float(want[1][0].abs().max()) * 2


@pytest.mark.parametrize("dtype", [FP, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,T,C", [(2, 150, 100), (3, 70, 98), (2, 131, 97), (1, 1, 100)])
def test_alignments(cuda, B, T, C, dtype):
    """Every stream at its own alignment: 16, 8, 4 bytes and one element; the results are those of aligned copies."""
    leaves, seg, gos = ssd_case(B, T, C, 40, dtype, seed=9)
    ls = on(cuda, leaves)

    def view(t, off, width):  # a copy that lies off elements into rows of `width`
        buf = torch.full((B * T * width + 16,), float("nan"), dtype=dtype, device=cuda)
        v = buf[off:].as_strided((B, T, C), (T * width, width, 1))
        v.copy_(t)
        return v

    def run(place, go):
        with torch.no_grad():
            xs = [place(k, x) for k, x in enumerate(ls[:5])]
        xs = [x.requires_grad_() for x in xs]
        out = nk.ssd_scan_train(*xs, ls[5], LO, HI, seg_start=seg.to(cuda), h0=ls[6])
        return [out, *torch.autograd.grad(out, [*xs, ls[5], ls[6]], go)]

    go = gos[0].to(cuda)
    want = run(lambda k, x: x.clone(), go)
    spots = [(0, 128), (4, 108), (2, 102), (1, 101), (3, 128)]
    for turn in range(5):
        got = run(lambda k, x: view(x, *spots[(k + turn) % 5]), view(go, *spots[turn]))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_mixed_dtypes(cuda):
    """Gates in another dtype take x's; gradients come back in their own."""
    leaves, _, gos = gated_case(2, 40, 64, 0, BF, seed=2)
    x, z, g = leaves[0].to(cuda).requires_grad_(), leaves[1].float().to(cuda).requires_grad_(), leaves[2].to(cuda)
    y = nk.gated_scan_train(x, z, g)
    gx, gz = torch.autograd.grad(y, [x, z], gos[0].to(cuda))
    assert y.dtype == gx.dtype == BF and gz.dtype == FP
    want = grads64(lambda x, z: ref.gated(x, z, leaves[2].double(), torch.zeros(2, 64, dtype=torch.float64))[0],
                   leaves[:2], gos[:1])
    ref.close(y, want[0][0], BF, 40)
    ref.close(gx, want[1][0], BF, 40)
    ref.close(gz.to(BF), want[1][1], BF, 40)


def test_parts_of_the_graph(cuda):
    """Only the final state, only h0, only one gate: the rest is left out."""
    leaves, seg, gos = ssd_case(2, 100, 64, 30, BF, seed=7)
    ls = on(cuda, leaves)
    run = lambda *a: nk.ssd_scan_train(*a[:6], LO, HI, seg_start=seg.to(cuda), h0=a[6], return_final_state=True)  # noqa: E731
    full = run(*ls)
    f = torch.autograd.grad(full[1], ls, gos[1].to(cuda))
    z = [torch.zeros_like(gos[0]), gos[1]]
    _, want = grads64(lambda *a: ref.ssd(*a, LO, HI, seg), leaves, z)
    compare([], f, [], want, BF, 100)
    only = [t.detach() for t in ls]
    only[3] = ls[3]
    both = run(*only)
    (g,) = torch.autograd.grad(both, [ls[3]], [t.to(cuda) for t in gos])
    (g2,) = torch.autograd.grad(run(*ls), [ls[3]], [t.to(cuda) for t in gos])
    assert torch.equal(g, g2)
    with torch.no_grad():
        y, _ = run(*ls)
    assert not y.requires_grad and torch.equal(y, full[0])
    y8 = nk.ssd_scan_train(*ls[:6], LO, HI, seg_start=seg.to(cuda), h0=ls[6], checkpoint=F8)
    assert torch.equal(y8, full[0])  # a checkpoint changes no output


@pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_bad_values_stay_in_their_segment(cuda, value, ckpt):
    """An infinity or NaN in one segment reaches neither the states after the next
    start nor the gradients before its own."""
    B, T, C = 1, 200, 64
    leaves, _, gos = gated_case(B, T, C, 0, FP, seed=11)
    seg = torch.zeros(B, T, dtype=torch.uint8)
    seg[0, 70] = seg[0, 140] = 1
    clean = on(cuda, leaves)
    call = lambda ls: nk.gated_scan_train(*ls[:3], seg_start=seg.to(cuda), h0=ls[3], return_final_state=True, checkpoint=ckpt)  # noqa: E731
    co = call(clean)
    cg = torch.autograd.grad(co, clean, [g.to(cuda) for g in gos])
    out_of = torch.ones(T, dtype=torch.bool)
    out_of[70:140] = False
    for which in range(4):  # x, z, g, and the output's gradient
        ls = [t.clone() for t in leaves]
        go = [t.clone() for t in gos]
        (ls[which] if which < 3 else go[0])[0, 100, 5] = value
        ls = on(cuda, ls)
        o = call(ls)
        g = torch.autograd.grad(o, ls, [t.to(cuda) for t in go])
        for a, b in zip([o[0], *g[:3]], [co[0], *cg[:3]]):
            assert torch.equal(a[:, out_of], b[:, out_of]), which
        assert torch.equal(o[1], co[1]) and torch.equal(g[3], cg[3])
        if which < 3 and value != value:
            assert bool(o[0][0, 100:140, 5].isnan().all())


@pytest.mark.parametrize("dtype", [FP, BF], ids=["f32", "bf16"])
def test_gradient_against_differences(cuda, dtype):
    """The kernel's own outputs, moved along a direction in each input: the change of
    <outputs, gos> against <gradient, direction>.  Central differences with step s
    leave a third-derivative term of s^2 / 6 times the direction's size cubed
    (gates have derivatives below 1) and twice the outputs' rounding over 2 s."""
    B, T, C = 2, 90, 64
    gen = torch.Generator().manual_seed(21)
    leaves, seg, gos = ssd_case(B, T, C, 30, FP, seed=13)
    seg = seg.to(cuda)
    gos = [g.to(cuda).double() for g in gos]
    ls = on(cuda, leaves)
    f = lambda a: nk.ssd_scan_train(*a[:6], LO, HI, seg_start=seg, h0=a[6], return_final_state=True)  # noqa: E731
    if dtype == BF:  # a bf16 gradient at bf16 points, the differences in fp32 around them
        ls = [t.detach().to(BF).requires_grad_() if t.dim() == 3 else t for t in ls]
        gl = [gos[0].to(BF), gos[1].float()]
        grads = torch.autograd.grad(f(ls), ls, gl)
        gos = [g.double() for g in gl]
        ls = [t.detach().float() for t in ls]
    else:
        grads = torch.autograd.grad(f(ls), ls, [g.float() for g in gos])
    s = 2.0 ** -6
    for k in range(7):
        v = torch.randn(ls[k].shape, generator=gen).to(cuda)
        v /= v.norm()
        dots = []
        for sign in (1, -1):
            moved = [t.detach() + sign * s * v if j == k else t.detach() for j, t in enumerate(ls)]
            dots.append(sum(float((o.double() * g).sum()) for o, g in zip(f(moved), gos)))
        got = float((grads[k].double() * v.double()).sum())
        num = (dots[0] - dots[1]) / (2 * s)
        # rounding: each output off by 2^-22 of its size, independent; the bf16 gradient by 2^-9 of its own
        size = sum(float((o.double() * g).norm()) for o, g in zip(f([t.detach() for t in ls]), gos))
        slack = 2 * 2.0 ** -22 * 16 * size / (2 * s) + s * s * float(grads[k].double().norm()) + (
            2.0 ** -8 * float(grads[k].double().norm()) if dtype == BF else 0)
        assert abs(got - num) <= slack + 1e-3 * abs(num), (k, got, num, slack)


def test_repeats_are_identical(cuda):
    leaves, seg, gos = ssd_case(3, 1000, 328, 100, BF, seed=3)
    ls, seg, gos = on(cuda, leaves), seg.to(cuda), [g.to(cuda) for g in gos]
    first = None
    for _ in range(5):
        outs = nk.ssd_scan_train(*ls[:6], LO, HI, seg_start=seg, h0=ls[6], return_final_state=True)
        res = list(outs) + list(torch.autograd.grad(outs, ls, gos))
        if first is None:
            first = res
        assert all(torch.equal(a, b) for a, b in zip(first, res))


@pytest.mark.parametrize("B,T,C", [(1, 20000, 64), (7, 2113, 328)])
def test_long_against_the_scan_kernels(cuda, B, T, C):
    """Many chunks: fp32 outputs against the forward-only fp32 scans, whose gates are
    fp32 too, and the adjoint against a run over halves joined by the carried state."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    z, g, x, go = (torch.randn(B, T, C, device=cuda, generator=gen) for _ in range(4))
    z += 4
    h, f = nk.gated_scan_train(x, z, g, return_final_state=True)
    h2, f2 = nk.gated_scan(x, z, g, return_final_state=True)
    assert float((h - h2).abs().max()) <= 64 * 2.0 ** -22 * 4 * float(h2.abs().max())
    ls = [t.requires_grad_() for t in (x, z, g)]
    whole = torch.autograd.grad(nk.gated_scan_train(*ls), ls, go)
    cut = T // 2 + 5
    h1, s1 = nk.gated_scan_train(*[t[:, :cut] for t in ls], return_final_state=True)
    h2 = nk.gated_scan_train(*[t[:, cut:] for t in ls], h0=s1)
    halves = torch.autograd.grad([h1, h2], ls, [go[:, :cut], go[:, cut:]])
    for a, b in zip(whole, halves):
        assert float((a - b).abs().max()) <= 64 * 2.0 ** -22 * 4 * float(a.abs().max())


def test_more_tiles_than_a_grid_dimension(cuda):
    """A sequence of more than 65535 tiles, against its two halves joined by the state."""
    T, C = 65536 * 128 + 300, 8
    gen = torch.Generator(device=cuda).manual_seed(2)
    x, z, g, go = (torch.randn(1, T, C, device=cuda, generator=gen).to(BF) for _ in range(4))
    ls = [t.requires_grad_() for t in (x, z, g)]
    h, f = nk.gated_scan_train(*ls, return_final_state=True)
    whole = torch.autograd.grad(h, ls, go)
    cut = 128 * 40000  # at a tile: both runs then round alike
    h1, s1 = nk.gated_scan_train(*[t[:, :cut] for t in ls], return_final_state=True)
    h2, f2 = nk.gated_scan_train(*[t[:, cut:] for t in ls], h0=s1, return_final_state=True)
    halves = torch.autograd.grad([h1, h2], ls, [go[:, :cut], go[:, cut:]])
    # the carries into a tile compose other tiles' maps in the halves: a few fp32
    # roundings, which turn at most the rare value next to a tie
    for a, b in zip([h, f, *whole], [torch.cat([h1, h2], 1), f2, *halves]):
        assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.float().abs().max())
        assert float((a != b).float().mean()) <= 0.01


def test_look_back_gives_up_and_says_so(cuda):
    """A wait that runs out (4 polls, far less than a tile needs to load): the launch
    ends, the error word says so, the outputs past the break are NaN and not wrong
    numbers, and the next call is right."""
    lib = abi.load()
    B, T, C = 2, 2048, 512
    gen = torch.Generator(device=cuda).manual_seed(1)
    x, z, g = (torch.randn(B, T, C, device=cuda, generator=gen).to(BF) for _ in range(3))
    good, _ = nk.gated_scan_train(x, z, g, return_final_state=True)
    lib.need_test_set_lookback_polls(4)
    try:
        bad = nk.gated_scan_train(x, z, g)
        torch.cuda.synchronize()
    finally:
        lib.need_test_set_lookback_polls(0)
    wrong = ~((bad == good) | bad.isnan())
    assert not bool(wrong.any()) and bool(bad.isnan().any())
    assert torch.equal(nk.gated_scan_train(x, z, g), good)


# ------------------------------------------------------------------ streams and graphs

def test_other_stream(cuda):
    leaves, seg, gos = ssd_case(2, 300, 136, 50, BF, seed=1)
    ls, gos, seg = on(cuda, leaves), [g.to(cuda) for g in gos], seg.to(cuda)
    run = lambda: nk.ssd_scan_train(*ls[:6], LO, HI, seg_start=seg, h0=ls[6], return_final_state=True)  # noqa: E731
    here = run()
    want = list(here) + list(torch.autograd.grad(here, ls, gos))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    got = []
    for s in streams:  # two at once
        with torch.cuda.stream(s):
            o = run()
            got.append(list(o) + list(torch.autograd.grad(o, ls, gos)))
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_graphs_share_nothing(cuda):
    """Two captured training passes of different sizes, replayed in turn and with new
    inputs, give what eager calls give."""
    graphs = []
    for T, seed in ((500, 1), (130, 2)):
        leaves, seg, gos = ssd_case(2, T, 200, 60, BF, seed=seed)
        ls, gos, seg = on(cuda, leaves), [g.to(cuda) for g in gos], seg.to(cuda)

        def run(ls=ls, gos=gos, seg=seg):
            o = nk.ssd_scan_train(*ls[:6], LO, HI, seg_start=seg, h0=ls[6], return_final_state=True, checkpoint=F8)
            return list(o) + list(torch.autograd.grad(o, ls, gos))

        s = torch.cuda.Stream(cuda)
        with torch.cuda.stream(s):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run()
        graphs.append((graph, res, run, ls))
    for step in range(4):
        for _, _, _, ls in graphs:
            with torch.no_grad():
                for t in ls:
                    t.mul_(0.9)
        for graph, _, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, res, run, _ in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, run()))


# ------------------------------------------------------------------ the conv

@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,C,K,every,bias", [
    (1, 1, 8, 4, 0, True), (2, 2, 12, 3, 0, False), (1, 3, 4, 4, 1, True), (3, 31, 40, 2, 5, True), (2, 33, 128, 4, 0, True),
    (2, 128, 132, 3, 11, False), (1, 129, 100, 4, 3, True), (2, 300, 13, 1, 9, True), (1, 261, 264, 3, 40, True),
])
def test_conv(cuda, B, T, C, K, every, bias, dtype):
    gen = torch.Generator().manual_seed(B + T + C + K)
    leaves = [rnd(gen, B, T, C, dtype=dtype), rnd(gen, C, K)] + ([rnd(gen, C)] if bias else [])
    seg = marks(gen, B, T, every)
    go = rnd(gen, B, T, C, dtype=dtype)
    want = grads64(lambda u, w, b=None: ref.conv_silu(u, w, b, seg), leaves, [go])
    ls = on(cuda, leaves)
    y = nk.ssd_conv_silu_train(ls[0], ls[1][:, None], *ls[2:], seg_start=None if seg is None else seg.to(cuda))
    # sums over B * T tokens and at most 128 in a row: 128 roundings
    compare([y], torch.autograd.grad(y, ls, go.to(cuda)), *want, dtype, 128 if T > 4 else 4)


@pytest.mark.parametrize("B,T,C,K,every,dtype", [(3, 333, 10530, 3, 0, BF), (3, 333, 10529, 4, 40, HF), (9, 150, 14040, 3, 60, BF),
                                                 (9, 150, 14041, 2, 0, HF), (3, 333, 2880, 3, 50, FP), (3, 333, 2881, 4, 0, BF)])
def test_conv_wide(cuda, B, T, C, K, every, dtype):
    """Widths at which a thread walks 32 and 64 tokens, backward or both ways."""
    gen = torch.Generator().manual_seed(C)
    leaves = [rnd(gen, B, T, C, dtype=dtype), rnd(gen, C, K), rnd(gen, C)]
    seg, go = marks(gen, B, T, every), rnd(gen, B, T, C, dtype=dtype)
    want = grads64(lambda u, w, b: ref.conv_silu(u, w, b, seg), leaves, [go])
    ls = on(cuda, leaves)
    y = nk.ssd_conv_silu_train(ls[0], ls[1][:, None], ls[2], seg_start=None if seg is None else seg.to(cuda))
    compare([y], torch.autograd.grad(y, ls, go.to(cuda)), *want, dtype, 128)


@pytest.mark.parametrize("dtype", [FP, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,T,C,K", [(2, 150, 100, 3), (3, 70, 98, 4), (2, 131, 97, 2), (1, 1, 101, 3)])
def test_conv_alignments(cuda, B, T, C, K, dtype):
    """Rows aligned to 16 bytes down to one element: the results are those of aligned copies."""
    gen = torch.Generator().manual_seed(C)
    u, go, w, b = rnd(gen, B, T, C, dtype=dtype), rnd(gen, B, T, C, dtype=dtype), rnd(gen, C, K), rnd(gen, C)
    seg = marks(gen, B, T, 30).to(cuda)

    def view(t, off, width):
        buf = torch.full((B * T * width + 16,), float("nan"), dtype=dtype, device=cuda)
        return buf[off:].as_strided((B, T, C), (T * width, width, 1)).copy_(t)

    def run(spot, gspot):
        ls = [view(u, *spot).requires_grad_(), *on(cuda, [w, b])]
        y = nk.ssd_conv_silu_train(*ls, seg_start=seg)
        return [y, *torch.autograd.grad(y, ls, view(go, *gspot))]

    want = run((0, 128), (0, 128))
    spots = [(4, 108), (2, 102), (1, 101), (3, 128)]
    for k, spot in enumerate(spots):
        for gspot in (spots[(k + 1) % 4], (0, 128)):
            assert all(torch.equal(x, y) for x, y in zip(run(spot, gspot), want))


def test_conv_chunk_and_repeat(cuda):
    gen = torch.Generator().manual_seed(8)
    proj = rnd(gen, 2, 400, 5 * 72, dtype=BF)
    w, b, go = rnd(gen, 72, 1, 3), rnd(gen, 72), rnd(gen, 2, 400, 72, dtype=BF)
    want = grads64(lambda p, w, b: ref.conv_silu(p.chunk(5, -1)[1], w[:, 0], b), [proj, w, b], [go])
    ls = on(cuda, [proj, w, b])
    y = nk.ssd_conv_silu_train(ls[0].chunk(5, -1)[1], ls[1], ls[2])
    g = torch.autograd.grad(y, ls, go.to(cuda), retain_graph=True)
    compare([y], g, *want, BF, 128)
    assert all(torch.equal(a, c) for a, c in zip(g, torch.autograd.grad(y, ls, go.to(cuda))))


# ------------------------------------------------------------------ the norm

@pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])
@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 8), (17, 64), (5, 100), (9, 264), (700, 832), (6, 2000), (33, 4104), (2, 8192)])
def test_norm(cuda, rows, C, dtype, ckpt):
    gen = torch.Generator().manual_seed(rows + C)
    leaves = [(3 * rnd(gen, rows, C)).to(dtype), 1 + 0.1 * rnd(gen, C)]
    go = rnd(gen, rows, C, dtype=dtype)
    want = grads64(lambda x, w: ref.rms_norm(x, w, 1e-6, ckpt is not None), leaves, [go])
    ls = on(cuda, leaves)
    y = nk.rms_norm_train(*ls, 1e-6, checkpoint=ckpt)
    # C = 1: y = sign(x) w, whose true gradient is eps / x^2 of its two terms: a difference of equals
    compare([y], torch.autograd.grad(y, ls, go.to(cuda)), *want, dtype, 64) if C > 1 else ref.close(y, want[0][0], dtype, 64)


@pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])
@pytest.mark.parametrize("C", [6136, 6144, 6152])
def test_norm_at_the_default_shared_memory(cuda, C, ckpt):
    """Rows whose backward takes just under, all of and just over the shared memory a launch has unasked."""
    gen = torch.Generator().manual_seed(C)
    leaves, go = [rnd(gen, 5, C, dtype=BF), 1 + 0.1 * rnd(gen, C)], rnd(gen, 5, C, dtype=BF)
    want = grads64(lambda x, w: ref.rms_norm(x, w, 1e-6, ckpt is not None), leaves, [go])
    ls = on(cuda, leaves)
    y = nk.rms_norm_train(*ls, 1e-6, checkpoint=ckpt)
    compare([y], torch.autograd.grad(y, ls, go.to(cuda)), *want, BF, 64)


def test_norm_longest_row_and_layouts(cuda):
    gen = torch.Generator().manual_seed(4)
    for C, dtype in ((16384, BF), (8192, FP)):
        x, w, go = rnd(gen, 2, C, dtype=dtype), rnd(gen, C), rnd(gen, 2, C, dtype=dtype)
        want = grads64(lambda x, w: ref.rms_norm(x, w, 1e-6), [x, w], [go])
        ls = on(cuda, [x, w])
        y = nk.rms_norm_train(*ls)
        compare([y], torch.autograd.grad(y, ls, go.to(cuda)), *want, dtype, 64)
        with pytest.raises(NotImplementedError):
            nk.rms_norm_train(torch.cat([ls[0], ls[0]], -1), torch.cat([ls[1], ls[1]]))
    x = rnd(gen, 4, 6, 80, dtype=BF)
    w, go = rnd(gen, 72), rnd(gen, 4, 6, 72, dtype=BF)
    want = grads64(lambda x, w: ref.rms_norm(x[..., 8:], w, 1e-6), [x, w], [go])
    ls = on(cuda, [x, w])
    y = nk.rms_norm_train(ls[0][..., 8:], ls[1])
    compare([y], torch.autograd.grad(y, ls, go.to(cuda)), *want, BF, 64)


def test_norm_bad_row_stays_alone(cuda):
    gen = torch.Generator().manual_seed(6)
    x, w, go = rnd(gen, 40, 256, dtype=BF), rnd(gen, 256), rnd(gen, 40, 256, dtype=BF).to(cuda)
    for ckpt in (None, F8):
        ls = on(cuda, [x, w])
        y = nk.rms_norm_train(*ls, checkpoint=ckpt)
        (g,) = torch.autograd.grad(y, ls[:1], go)
        xb = x.clone()
        xb[7, 9] = float("inf")
        lb = on(cuda, [xb, w])
        yb = nk.rms_norm_train(*lb, checkpoint=ckpt)
        (gb,) = torch.autograd.grad(yb, lb[:1], go)
        rest = torch.arange(40) != 7
        assert torch.equal(y[rest], yb[rest]) and torch.equal(g[rest], gb[rest])
        assert bool(gb[7].isnan().any())


# ------------------------------------------------------------------ empty calls, refusals

def test_empty(cuda):
    for B, T, C in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        x = [torch.randn(B, T, C, device=cuda, dtype=BF).requires_grad_() for _ in range(5)]
        h0 = torch.randn(B, C, device=cuda).requires_grad_()
        D = torch.ones(C, device=cuda).requires_grad_()
        y, f = nk.gated_scan_train(*x[:3], h0=h0, return_final_state=True)
        assert y.shape == (B, T, C) and torch.equal(f, h0)
        g = torch.autograd.grad([y, f], [*x[:3], h0], [torch.zeros_like(y), torch.ones_like(f)])
        assert torch.equal(g[3], torch.ones_like(h0))
        y, f = nk.ssd_scan_train(*x, D, LO, HI, return_final_state=True)
        assert y.dtype == BF and not bool(f.any())
        assert not bool(torch.autograd.grad(y.sum(), D)[0].any())
        w = torch.ones(C, 1, 3, device=cuda).requires_grad_()
        yc = nk.ssd_conv_silu_train(x[0], w, D)
        assert yc.dtype == BF and not bool(torch.autograd.grad(yc.sum(), w)[0].any())
        yn = nk.rms_norm_train(x[0], D)
        assert yn.dtype == BF and not bool(torch.autograd.grad(yn.sum(), D)[0].any())


def test_refusals(cuda):
    x = torch.randn(2, 6, 16, device=cuda)
    D = torch.ones(16, device=cuda)
    with pytest.raises(ValueError):
        nk.gated_scan_train(x, x, x[:, :5])
    with pytest.raises(ValueError):
        nk.gated_scan_train(x[0], x[0], x[0])
    with pytest.raises(ValueError):
        nk.gated_scan_train(x, x, x, seg_start=torch.zeros(2, 5, device=cuda))
    with pytest.raises(ValueError):
        nk.gated_scan_train(x, x, x, h0=torch.zeros(2, 15, device=cuda))
    with pytest.raises(ValueError):
        nk.gated_scan_train(x, x, x, checkpoint=torch.float8_e5m2)
    with pytest.raises(TypeError):
        nk.gated_scan_train(x.double(), x.double(), x.double())
    with pytest.raises(RuntimeError):
        nk.gated_scan_train(x, x.cpu(), x)
    with pytest.raises(RuntimeError):
        nk.gated_scan_train(x, x, x, h0=torch.zeros(2, 16))
    with pytest.raises(ValueError):
        nk.ssd_scan_train(x, x, x, x, x, D[:15], LO, HI)
    for lo, hi in ((-0.1, 0.2), (0.2, 0.1), (0.0, float("nan")), (0.0, float("inf"))):
        with pytest.raises(ValueError):
            nk.ssd_scan_train(x, x, x, x, x, D, lo, hi)
    with pytest.raises(ValueError):
        nk.ssd_conv_silu_train(x, torch.ones(16, 1, 5, device=cuda))
    with pytest.raises(ValueError):
        nk.ssd_conv_silu_train(x, torch.ones(15, 1, 3, device=cuda))
    with pytest.raises(ValueError):
        nk.ssd_conv_silu_train(x, torch.ones(16, 1, 3, device=cuda), D[:8])
    with pytest.raises(ValueError):
        nk.rms_norm_train(x, D[:8])
    with pytest.raises(ValueError):
        nk.rms_norm_train(x, D, -1.0)
    # gradients of gradients
    xr = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(nk.gated_scan_train(xr, x, x).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    # an input changed between the forward and the backward
    xr = x.clone().requires_grad_()
    z = x.clone()
    y = nk.gated_scan_train(xr, z, x)
    z.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


# ------------------------------------------------------------------ the block

@pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])
def test_block(cuda, ckpt):
    """The block as it trains: conv + SiLU, SSD scan, out_norm over chunks of one
    projection, with packed documents, against the same in float64.  Each operator
    hands 16-bit values on, so errors add: a half step of each tensor between them,
    carried through factors that the norm keeps near 1 -- 3 % of the 2-norm for the
    full form covers four such roundings with the norm's 1 / rms.  With the 8-bit
    checkpoint a stored value is off by 2^-4 at most (2^-5 in the middle), and a
    gradient is a product of several: 15 % of the 2-norm."""
    gen = torch.Generator().manual_seed(31)
    B, T, C = 2, 150, 72
    proj, seg = rnd(gen, B, T, 5 * C, dtype=BF), marks(gen, B, T, 40)
    leaves = [proj, rnd(gen, C, 1, 3) / 3 ** 0.5, 0.1 * rnd(gen, C), 1 + 0.1 * rnd(gen, C), 1 + 0.1 * rnd(gen, C)]
    go = rnd(gen, B, T, C, dtype=BF)

    def block64(p, w, b, D, nw):
        u, bg, cg, dt, og = p.chunk(5, -1)
        u = ref.conv_silu(u, w[:, 0], b, seg)
        return ref.rms_norm(ref.ssd(u, bg, cg, dt, og, D, torch.zeros(B, C, dtype=torch.float64), LO, HI, seg)[0], nw, 1e-6)

    want, wg = grads64(block64, leaves, [go])
    ls, s = on(cuda, leaves), seg.to(cuda)
    u, bg, cg, dt, og = ls[0].chunk(5, -1)
    u = nk.ssd_conv_silu_train(u, ls[1], ls[2], seg_start=s)
    y = nk.ssd_scan_train(u, bg, cg, dt, og, ls[3], LO, HI, seg_start=s, checkpoint=ckpt)
    y = nk.rms_norm_train(y, ls[4], checkpoint=ckpt)
    for a, b in zip([y, *torch.autograd.grad(y, ls, go.to(cuda))], [*want, *wg]):
        off = float(torch.linalg.norm(a.detach().cpu().double() - b.detach()) / torch.linalg.norm(b.detach()))
        assert off <= (0.03 if ckpt is None else 0.15), off


def test_saved_memory(cuda):
    """What an 8-bit checkpoint is for: the activations held between forward and
    backward, 10 bytes an element for the SSD scan, come down to 5 and the scales."""
    B, T, C = 2, 2048, 512
    n = B * T * C

    def held(ckpt):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated(cuda)
        xs = [torch.randn(B, T, C, device=cuda).to(BF).requires_grad_() for _ in range(5)]
        y = nk.ssd_scan_train(*[x * 1 for x in xs], torch.ones(C, device=cuda), LO, HI, checkpoint=ckpt)
        del xs[:]
        return torch.cuda.memory_allocated(cuda) - before, y

    full, y1 = held(None)
    small, y2 = held(F8)
    del y1, y2
    leaf = 5 * 2 * n  # the leaves live in the graph either way
    assert full >= leaf + 10 * n and small <= leaf + 2 * n + 5 * n * 1.1
