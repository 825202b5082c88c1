"""The block on the training operators: what it holds between forward and backward."""
import pytest
import torch

from need_b200 import need_kernels as nk

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def block(proj, w, b, D, nw, ckpt, own_u):
    """conv + SiLU, scan and norm over the five chunks of `proj`; `own_u`: the conv is given
    a u of its own instead of the chunk."""
    u, bg, cg, dt, og = proj.chunk(5, dim=-1)
    u = nk.ssd_conv_silu_train(u.contiguous() if own_u else u, w, b)
    y = nk.ssd_scan_train(u, bg, cg, dt, og, D, 0.001, 0.2, checkpoint=ckpt)
    return nk.rms_norm_train(y, nw, 1e-6, checkpoint=ckpt)


def test_what_the_block_holds(cuda):
    """Bytes per 16-bit element.  Without copies: the projection 10, the conv's output 2,
    the norm's input 2.  With 8-bit copies: u 2 for the conv, five streams 5, the norm's
    input 1, a byte a group of 64 for each of the six, fp32 states every 64 tokens and a
    row's 1 / rms -- if the conv's u is a tensor of its own: a chunk keeps all five alive.
    The allocator rounds each of some ten tensors up to 2 MB at most."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    B, T, C = 4, 2048, 832
    n, slack = B * T * C, 10 << 21
    x = torch.randn(B, T, 5 * C, device=cuda, generator=gen).to(torch.bfloat16).requires_grad_()
    ps = [torch.randn(s, device=cuda, generator=gen).requires_grad_() for s in ((C, 1, 3), (C,), (C,), (C,))]
    go = torch.randn(B, T, C, device=cuda, generator=gen).to(torch.bfloat16)

    def run(ckpt, own_u):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated(cuda)
        y = block(x * 1, *ps, ckpt, own_u)  # the projection itself is held by the block alone
        held = torch.cuda.memory_allocated(cuda) - before - 2 * n
        return held, [y, *torch.autograd.grad(y, [x, *ps], go)]

    full, want = run(None, False)
    held, got = run(None, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    chunk, want = run(F8, False)
    small, got = run(F8, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    extra = 6 * n / 64 + 4 * n / 64 + 4 * B * T
    assert 14 * n <= full <= 14.2 * n + slack
    assert 8 * n <= small <= 8 * n + extra + slack
    assert chunk >= 16 * n
