"""The training operators at the edges of their documentation, on the GPU: values that
are not finite or the type's lowest, calls that they refuse, waits that run out."""
import pytest
import torch

import train_reference as ref
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
