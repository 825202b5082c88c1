"""The training operators at the edges of their documentation, on the GPU: values that
are not finite or the type's lowest, calls that they refuse, waits that run out."""
import threading

import pytest
import torch

import train_reference as ref
from need_b200 import abi
from need_b200 import need_kernels as nk

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
DTYPES = pytest.mark.parametrize("dtype", [FP, BF, HF], ids=["f32", "bf16", "f16"])


# ------------------------------------------------------------------ not a number

@DTYPES
@pytest.mark.parametrize("B", [1, 200])  # tiles of 32 and of 64 channels
@pytest.mark.parametrize("segments", [False, True])
def test_a_bad_value_lasts_to_the_end_of_its_segment(cuda, dtype, B, segments):
    """With a reset mask as without: where the product of a over a tile has underflowed,
    a NaN in the state (or, backward, in mu) still reaches all that depends on it."""
    T, C = 600, 40
    gen = torch.Generator().manual_seed(12)
    x, g, go, u, cg, og = (torch.randn(B, T, C, generator=gen).to(dtype) for _ in range(6))
    z = torch.full((B, T, C), -3.0, dtype=dtype)  # a = 0.047, 1e-85 over 64 tokens
    for t in (x, u):
        t[0, 20, 5] = float("nan")
    go[0, 560, 6] = float("nan")
    seg = torch.zeros(B, T, dtype=torch.uint8)
    if segments:
        seg[0, 10] = seg[0, 580] = 1
    first, last = (10, 580) if segments else (0, T)
    rows = torch.arange(T)
    for call in (lambda a, b, c: nk.gated_scan_train(a, b, c, seg_start=seg.to(cuda), return_final_state=True),
                 lambda a, b, c: nk.ssd_scan_train(a, c, cg.to(cuda), b, og.to(cuda), torch.ones(C, device=cuda), 3.0, 3.1,
                                                   seg_start=seg.to(cuda), return_final_state=True)):
        ls = [t.to(cuda).requires_grad_() for t in (x, z, g)]
        h, f = call(*ls)
        dx = torch.autograd.grad(h, ls, go.to(cuda))[0]
        assert torch.equal(h[0, :, 5].isnan().cpu(), (rows >= 20) & (rows < last))
        assert int(h.isnan().sum()) == last - 20 and bool(f[0, 5].isnan()) != segments
        assert torch.equal(dx[0, :, 6].isnan().cpu(), (rows >= first) & (rows <= 560))


# ------------------------------------------------------------------ the type's lowest value

@DTYPES
@pytest.mark.parametrize("K", [1, 3])
def test_conv_of_the_lowest_value(cuda, dtype, K):
    """silu and its slope are 0 far below 0, however far: nothing is left of the type's
    lowest value, which padding may hold (and whose s = 2^-126 would leave 4).  Bound: half
    a step and 2^-18 (a gate's few ulp and six products) of the largest result."""
    B, T, C = 2, 37, 24
    gen = torch.Generator().manual_seed(5)
    u, go = (torch.randn(B, T, C, generator=gen).to(dtype) for _ in range(2))
    w = 0.1 + 0.2 * torch.rand(C, K, generator=gen)
    u[0, 10] = torch.finfo(dtype).min
    u[1, 20] = -90.0
    l64 = [t.double().requires_grad_() for t in (u, w)]
    y64 = ref.conv_silu(*l64, None)
    want = [y64, torch.autograd.grad(y64, l64, go.double())[0]]
    ls = [t.to(cuda).requires_grad_() for t in (u, w)]
    y = nk.ssd_conv_silu_train(*ls)
    got = [y, torch.autograd.grad(y, ls, go.to(cuda))[0]]
    for a, b in zip(got, want):
        off = (a.detach().cpu().double() - b.detach()).abs()
        assert float(off.max()) <= (torch.finfo(dtype).eps / 2 + 2.0 ** -18) * float(b.detach().abs().max())


@DTYPES
@pytest.mark.parametrize("B", [1, 200])
def test_a_closed_decay_gate_drops_the_lowest_value(cuda, dtype, B):
    """decay_logit far below 0 (-1000, -inf): nothing of the state before is left, though
    it is near the type's largest."""
    T, C = 70, 40
    z = torch.full((B, T, C), 3.0, dtype=dtype)
    x, g = torch.zeros(B, T, C, dtype=dtype), torch.full((B, T, C), 30.0, dtype=dtype)
    x[:, 4] = torch.finfo(dtype).min
    z[:, 5], z[:, 4] = -1000.0, -1000.0
    z[:, 5, 7] = -float("inf")
    with torch.no_grad():
        h, f = nk.gated_scan_train(x.to(cuda), z.to(cuda), g.to(cuda), return_final_state=True)
    assert bool((h[:, 4] <= 0.99 * torch.finfo(dtype).min).all())
    assert not bool(h[:, 5:].any()) and not bool(f.any())


@pytest.mark.parametrize("dtype", [FP, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 2, 5, 64, 67])
def test_conv_rows_behind_the_sequence(cuda, dtype, T):
    """The last input overflows only in rows that the sequence does not have: its own
    gradient is w[K-1] dv, dv = 1 (silu's slope far above 0), and no NaN."""
    u = torch.zeros(2, T, 8, dtype=dtype, device=cuda)
    u[:, T - 1] = 2.0 ** 126
    w = torch.tensor([[8.0, 8.0, 0.5]], device=cuda).repeat(8, 1).requires_grad_()
    u.requires_grad_()
    y = nk.ssd_conv_silu_train(u, w)
    du, dw = torch.autograd.grad(y, [u, w], torch.ones_like(y))
    assert bool((y[:, T - 1] == 2.0 ** 125).all()) and bool((du[:, T - 1] == 0.5).all())
    assert bool(du.isfinite().all()) and bool(dw.isfinite().all())


# ------------------------------------------------------------------ other kinds of differentiation

@pytest.mark.parametrize("op", ["gated", "ssd", "conv", "norm"])
def test_forward_mode_and_transforms_raise(cuda, op):
    """A tangent is refused, not dropped, also where nothing asks for a gradient; so are
    torch.func's transforms."""
    import torch.autograd.forward_ad as fa
    x, D = torch.randn(2, 6, 16, device=cuda), torch.ones(16, device=cuda)
    w = torch.ones(16, 1, 3, device=cuda)
    f = {"gated": lambda t: nk.gated_scan_train(x, t, x), "ssd": lambda t: nk.ssd_scan_train(x, x, t, x, x, D, 0.001, 0.2),
         "conv": lambda t: nk.ssd_conv_silu_train(t, w), "norm": lambda t: nk.rms_norm_train(t, D)}[op]
    with fa.dual_level():
        dual = fa.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError):
            f(dual)
        with torch.no_grad(), pytest.raises(RuntimeError):
            f(dual)
    if op == "gated":
        h0 = torch.zeros(2, 16, device=cuda)
        with fa.dual_level(), pytest.raises(RuntimeError):
            nk.gated_scan_train(x, x, x, h0=fa.make_dual(h0, torch.ones_like(h0)))
    for transform in (lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.vmap(f)(torch.stack([x, x])),
                      lambda: torch.func.grad(lambda t: f(t).sum())(x)):
        with pytest.raises(RuntimeError):
            transform()
    assert not f(x).requires_grad
    with torch.inference_mode():
        assert torch.equal(f(x), f(x.clone()))


@DTYPES
@pytest.mark.parametrize("far", [-86.0, -87.5, -88.5, -1000.0, -float("inf")])
def test_a_closed_gate_drops_the_lowest_value(cuda, dtype, far):
    """An input gate as far below 0: the type's lowest input leaves nothing, in the output
    or in any gradient that the true one (e^far of it) does not."""
    B, T, C = 2, 40, 24
    x = torch.full((B, T, C), torch.finfo(dtype).min, dtype=dtype, device=cuda).requires_grad_()
    g = torch.full((B, T, C), far, dtype=dtype, device=cuda).requires_grad_()
    z = torch.zeros(B, T, C, dtype=dtype, device=cuda).requires_grad_()
    o, D = torch.zeros_like(z, requires_grad=True), torch.zeros(C, device=cuda)
    # half of e^far of the input enters, twice that is in the state
    size = float(torch.exp(torch.tensor(far, dtype=torch.float64).to(dtype).double())) * torch.finfo(dtype).max
    for call in (lambda: nk.gated_scan_train(x, z, g), lambda: nk.ssd_scan_train(x, g, o, z, o, D, 0.7, 0.7)):
        y = call()
        assert float(y.detach().abs().max()) <= 1.01 * size
        for d in torch.autograd.grad(y, [x, z, g], torch.ones_like(y)):
            assert bool(d.isfinite().all()) and float(d.abs().max()) <= 2.02 * size + 2.0 ** -20


# ------------------------------------------------------------------ waits that run out

ERR_LOOKBACK, ERR_LOAD = 1, 2


@pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])
def test_look_back_that_gives_up_is_reported(cuda, ckpt):
    """4 polls, far less than a tile needs to load: forward or backward, the launch ends,
    the error word says so, what depends on the break is NaN, and the next call is right."""
    lib = abi.load()
    gen = torch.Generator(device=cuda).manual_seed(1)
    ls = [torch.randn(2, 2048, 512, device=cuda, generator=gen).to(BF).requires_grad_() for _ in range(3)]
    go = torch.randn(2, 2048, 512, device=cuda, generator=gen).to(BF)
    run = lambda: nk.gated_scan_train(*ls, checkpoint=ckpt)  # noqa: E731
    nk.workspace_error()
    h = run()
    good = [h, *torch.autograd.grad(h, ls, go, retain_graph=True)]
    assert nk.workspace_error() == 0
    for call in (lambda: [run()], lambda: torch.autograd.grad(h, ls, go, retain_graph=True)):
        lib.need_test_set_lookback_polls(4)
        try:
            bad = call()
            torch.cuda.synchronize()
        finally:
            lib.need_test_set_lookback_polls(0)
        for a, b in zip(bad, good[:1] if len(bad) == 1 else good[1:]):
            assert bool(((a == b) | a.isnan()).all()) and bool(a.isnan().any())
        assert nk.workspace_error() == ERR_LOOKBACK and nk.workspace_error() == 0
    assert all(torch.equal(a, b) for a, b in zip([run(), *torch.autograd.grad(h, ls, go)], good))


@pytest.mark.parametrize("ckpt", [None, F8], ids=["full", "8bit"])
@DTYPES
@pytest.mark.parametrize("B", [2, 200])
def test_load_that_gives_up_is_reported(cuda, dtype, B, ckpt):
    """Every load wait gives up: all results are NaN, none a number made of whatever the
    rows held, and the error word says so, for a call on any stream."""
    lib = abi.load()
    T, C = 100, 40
    gen = torch.Generator(device=cuda).manual_seed(2)
    xs = [torch.randn(B, T, C, device=cuda, generator=gen).to(dtype).requires_grad_() for _ in range(5)]
    D, h0 = torch.ones(C, device=cuda, requires_grad=True), torch.zeros(B, C, device=cuda, requires_grad=True)
    go = torch.randn(B, T, C, device=cuda, generator=gen).to(dtype)
    for leaves, run in (([*xs[:3], h0], lambda *a: nk.gated_scan_train(*a[:3], h0=a[3], return_final_state=True, checkpoint=ckpt)),
                        ([*xs, D, h0], lambda *a: nk.ssd_scan_train(*a[:6], 0.001, 0.2, h0=a[6], return_final_state=True,
                                                                    checkpoint=ckpt))):
        nk.workspace_error()
        good = run(*leaves)
        want = torch.autograd.grad(good[0], leaves, go, retain_graph=True)
        assert nk.workspace_error() == 0
        s = torch.cuda.Stream(cuda)
        s.wait_stream(torch.cuda.current_stream(cuda))
        lib.need_test_scan_train_load_give_up(1)
        try:
            with torch.cuda.stream(s):
                bad = run(*(t.detach() for t in leaves))
                kept = run(*leaves)  # with what the backward keeps
            grads = torch.autograd.grad(good[0], leaves, go, retain_graph=True)
            torch.cuda.synchronize()
        finally:
            lib.need_test_scan_train_load_give_up(0)
        assert all(bool(t.isnan().all()) for t in (*bad, *kept, *grads))
        assert nk.workspace_error() == ERR_LOAD and nk.workspace_error() == 0
        after = torch.autograd.grad(kept[0], leaves[:-1], go)
        if ckpt:  # the copies it made are NaN,
            assert all(bool(t.isnan().all()) for t in after)
        assert any(bool(t.isnan().any()) for t in after)  # and the state it kept at token 64 is
        again = torch.autograd.grad(good[0], leaves, go)
        assert all(torch.equal(a, b) for a, b in zip(again, want))


# ------------------------------------------------------------------ empty calls

@pytest.mark.parametrize("B,T,C", [(2, 0, 8), (0, 4, 8), (2, 4, 0)])
def test_an_empty_call_returns_a_state_of_its_own(cuda, B, T, C):
    """The final state of an empty call is a new tensor, as that of any other: updated in
    place it leaves the caller's h0 alone."""
    x, D = torch.zeros(B, T, C, device=cuda), torch.ones(C, device=cuda)
    h0 = torch.ones(B, C, device=cuda)
    for call in (lambda: nk.gated_scan_train(x, x, x, h0=h0, return_final_state=True),
                 lambda: nk.ssd_scan_train(x, x, x, x, x, D, 0.001, 0.2, h0=h0, return_final_state=True)):
        out, final = call()
        assert out.shape == x.shape and torch.equal(final, h0)
        final.add_(1)
        assert bool((h0 == 1).all())


# ------------------------------------------------------------------ calls at once

def test_calls_at_once(cuda):
    """Threads on streams of their own, and captured passes replayed on two streams at
    once: every result is that of the call alone."""
    gen = torch.Generator(device=cuda).manual_seed(7)
    jobs = []
    for B, T, C, dtype, ckpt in ((2, 700, 200, BF, None), (3, 333, 136, FP, F8), (40, 150, 64, HF, None), (1, 2000, 328, BF, F8)):
        xs = [torch.randn(B, T, C, device=cuda, generator=gen).to(dtype).requires_grad_() for _ in range(5)]
        D, go = torch.ones(C, device=cuda, requires_grad=True), torch.randn(B, T, C, device=cuda, generator=gen).to(dtype)

        def job(xs=xs, D=D, go=go, ckpt=ckpt):
            ls = [t.detach().requires_grad_() for t in (*xs, D)]  # leaves of its own: their streams are the caller's
            y = nk.ssd_scan_train(*ls, 0.001, 0.2, checkpoint=ckpt)
            h = nk.gated_scan_train(*ls[:3], checkpoint=ckpt)
            return [y, h, *torch.autograd.grad([y, h], ls, [go, go])]

        jobs.append((job, [t.detach() for t in job()]))
    torch.cuda.synchronize()
    wrong = []

    def work(job, want):
        with torch.cuda.stream(torch.cuda.Stream(cuda)):
            for _ in range(10):
                got = job()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(job)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    graphs = []
    for job, want in jobs[:2]:
        s = torch.cuda.Stream(cuda)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = job()
        graphs.append((graph, s, got, want))
    for _ in range(5):
        for graph, s, _, _ in graphs:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, want in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert nk.workspace_error() == 0
