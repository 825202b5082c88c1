"""The training operators without a GPU: refusals (host checks that make no
CUDA call), the ctypes layouts, and the tests' own references against
differences."""
import ctypes
import os
import subprocess

import pytest
import torch

import train_reference as ref
from need_b200 import abi, build
from need_b200 import need_kernels as nk

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "need_scan.h")


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


def test_struct_layout_matches_header(tmp_path):
    structs = {"need_scan_train_args": abi.NeedScanTrainArgs, "need_conv_train_args": abi.NeedConvTrainArgs,
               "need_norm_train_args": abi.NeedNormTrainArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for n, *_ in cls._fields_:
            lines.append(f'printf("{name}.{n} %zu\\n", offsetof({name}, {"in" if n == "in_" else n}));')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for n, *_ in cls._fields_:
            assert int(got[f"{name}.{n}"]) == getattr(cls, n).offset, f"{name}.{n}"


def test_sizes(lib):
    assert lib.need_scan_train_chunk_len() == ref.SPAN
    assert lib.need_scan_train_group() == ref.GROUP
    ws = lib.need_scan_train_workspace_size
    gated, ssd, bf, f32 = abi.FORM_GATED, abi.FORM_SSD, abi.BF16, abi.F32
    assert ws(gated, bf, 0, 0, 2, 128, 64) == 128                                 # one tile: no records
    assert ws(gated, bf, 0, 1, 2, 129, 65) == 128 + 2 * 3 * 2 * 32 * 12           # few chains: 32 channels x 128 tokens
    assert ws(ssd, bf, 0, 1, 2, 129, 65) == 128 + 2 * 3 * 2 * 32 * 12 + 2 * 2 * 65 * 4
    assert ws(gated, bf, 0, 1, 96, 129, 65) == 128 + 96 * 2 * 2 * 64 * 12         # many: 64 x 128
    assert ws(gated, f32, 0, 1, 96, 65, 65) == 128 + 96 * 2 * 2 * 64 * 12         # 64 x 64
    assert ws(ssd, bf, 1, 1, 2, 65, 65) == 128 + 2 * 2 * 2 * 64 * 12 + 2 * 2 * 65 * 4
    assert ws(ssd, bf, 0, 1, 40, 65, 65) == 128 + 40 * 2 * 2 * 64 * 12 + 40 * 2 * 65 * 4  # 80 chains: wide backward,
    assert ws(ssd, bf, 0, 0, 40, 129, 65) == 128 + 40 * 3 * 2 * 32 * 12                  # narrow forward
    assert ws(ssd, bf, 0, 1, 0, 65, 65) == 128
    conv = lib.need_conv_silu_train_workspace_size
    assert conv(3, 2, 129, 8) == 2 * 3 * 8 * 4 * 4            # 16 tokens a thread, 4 threads a block
    assert conv(3, 3, 333, 2880) == 3 * 3 * 2880 * 4 * 4      # 32
    assert conv(3, 3, 333, 10530) == 3 * 2 * 10530 * 4 * 4    # 64
    assert lib.need_rms_norm_train_workspace_size(3, 8) == 3 * 8 * 4


P = 1 << 20  # an aligned address that no refused call reads


def scan_args(form=abi.FORM_SSD, **kw):
    a = abi.NeedScanTrainArgs()
    a.form, a.dtype, a.nb, a.T, a.C = form, abi.BF16, 2, 100, 64
    a.dt_min, a.dt_max = 0.001, 0.2
    for k in range(5):
        a.in_[k] = abi.NeedView(P, 6400, 0, 64)
        a.grad[k] = P
    a.gout = abi.NeedView(P, 6400, 0, 64)
    a.d_skip = a.states = a.out = a.workspace = a.grad_d = P
    a.out_stride_b, a.out_stride_t, a.workspace_bytes = 6400, 64, 1 << 30
    a.grad_stride_b, a.grad_stride_t = 6400, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change,code", [
    ({"form": abi.FORM_AFFINE}, abi.ERR_INVALID), ({"dtype": 7}, abi.ERR_UNSUPPORTED),
    ({"checkpoint": 2}, abi.ERR_INVALID), ({"T": 0}, abi.ERR_INVALID), ({"nb": -1}, abi.ERR_INVALID),
    ({"C": 1 << 32}, abi.ERR_UNSUPPORTED),
    ({"nb": 1 << 27, "T": 1 << 29}, abi.ERR_UNSUPPORTED),
    ({"states": None}, abi.ERR_INVALID), ({"d_skip": None}, abi.ERR_INVALID),
    ({"dt_min": -0.1}, abi.ERR_INVALID), ({"dt_max": 0.0}, abi.ERR_INVALID),
    ({"dt_max": float("nan")}, abi.ERR_INVALID), ({"dt_max": float("inf")}, abi.ERR_INVALID),
    ({"checkpoint": 1}, abi.ERR_INVALID), ({"workspace": None}, abi.ERR_WORKSPACE),
    ({"workspace": P + 8}, abi.ERR_WORKSPACE), ({"workspace_bytes": 127}, abi.ERR_WORKSPACE),
])
def test_scan_refuses(lib, backward, change, code):
    fn = lib.need_scan_train_backward if backward else lib.need_scan_train_forward
    assert fn(ctypes.byref(scan_args(**change)), None) == code
    assert lib.need_last_error()


def test_scan_refuses_outputs(lib):
    fwd, bwd = lib.need_scan_train_forward, lib.need_scan_train_backward
    assert fwd(None, None) == bwd(None, None) == abi.ERR_INVALID
    assert fwd(ctypes.byref(scan_args(out=None)), None) == abi.ERR_INVALID
    assert fwd(ctypes.byref(scan_args(out=P + 2)), None) == abi.ERR_INVALID
    for bad in (60, 56, 63):  # not 16 bytes apart, or shorter than C
        assert fwd(ctypes.byref(scan_args(out_stride_t=bad)), None) == abi.ERR_INVALID
        assert bwd(ctypes.byref(scan_args(grad_stride_t=bad)), None) == abi.ERR_INVALID
    assert fwd(ctypes.byref(scan_args(out_stride_b=0)), None) == abi.ERR_INVALID
    assert bwd(ctypes.byref(scan_args(grad_d=None)), None) == abi.ERR_INVALID
    a = scan_args()
    a.grad[3] = None
    assert bwd(ctypes.byref(a), None) == abi.ERR_INVALID
    a = scan_args()
    a.in_[2].ptr = None
    assert fwd(ctypes.byref(a), None) == bwd(ctypes.byref(a), None) == abi.ERR_INVALID
    a = scan_args()
    a.gout.ptr = None
    assert bwd(ctypes.byref(a), None) == abi.ERR_INVALID


def conv_args(**kw):
    a = abi.NeedConvTrainArgs()
    a.dtype, a.K, a.nb, a.T, a.C = abi.BF16, 3, 2, 100, 64
    a.u = a.weight = a.out = a.gout = a.grad_u = a.grad_wb = a.workspace = P
    a.u_stride_b = a.gout_stride_b = 6400
    a.u_stride_t = a.gout_stride_t = a.out_stride_t = 64
    a.out_stride_b = 6400
    a.workspace_bytes = 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code,both", [
    ({"dtype": 5}, abi.ERR_UNSUPPORTED, True), ({"K": 0}, abi.ERR_UNSUPPORTED, True), ({"K": 5}, abi.ERR_UNSUPPORTED, True),
    ({"T": 0}, abi.ERR_INVALID, True), ({"u": None}, abi.ERR_INVALID, True), ({"out_stride_t": 63}, abi.ERR_INVALID, True),
    ({"weight": None}, abi.ERR_INVALID, True), ({"nb": 1 << 40}, abi.ERR_UNSUPPORTED, True),
    ({"gout": None}, abi.ERR_INVALID, False), ({"grad_u": None}, abi.ERR_INVALID, False),
    ({"grad_wb": None}, abi.ERR_INVALID, False), ({"workspace_bytes": 8}, abi.ERR_WORKSPACE, False),
])
def test_conv_refuses(lib, change, code, both):
    assert lib.need_conv_silu_train_backward(ctypes.byref(conv_args(**change)), None) == code
    if both:
        assert lib.need_conv_silu_train_forward(ctypes.byref(conv_args(**change)), None) == code


def norm_args(**kw):
    a = abi.NeedNormTrainArgs()
    a.dtype, a.rows, a.C, a.eps = abi.BF16, 10, 64, 1e-6
    a.x = a.weight = a.out = a.rstd = a.gout = a.grad_x = a.grad_weight = a.workspace = P
    a.x_stride = a.gout_stride = a.out_stride = 64
    a.workspace_bytes = 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code,both", [
    ({"dtype": 5}, abi.ERR_UNSUPPORTED, True), ({"rows": 0}, abi.ERR_INVALID, True), ({"C": 0}, abi.ERR_INVALID, True),
    ({"C": 16385}, abi.ERR_UNSUPPORTED, True), ({"eps": -1.0}, abi.ERR_INVALID, True),
    ({"eps": float("nan")}, abi.ERR_INVALID, True), ({"checkpoint": 1}, abi.ERR_INVALID, True),
    ({"weight": None}, abi.ERR_INVALID, True), ({"rstd": None}, abi.ERR_INVALID, True),
    ({"x": None}, abi.ERR_INVALID, True), ({"out_stride": 60}, abi.ERR_INVALID, True),
    ({"gout": None}, abi.ERR_INVALID, False), ({"grad_x": None}, abi.ERR_INVALID, False),
    ({"grad_weight": None}, abi.ERR_INVALID, False), ({"workspace_bytes": 8}, abi.ERR_WORKSPACE, False),
])
def test_norm_refuses(lib, change, code, both):
    assert lib.need_rms_norm_train_backward(ctypes.byref(norm_args(**change)), None) == code
    if both:
        assert lib.need_rms_norm_train_forward(ctypes.byref(norm_args(**change)), None) == code


def test_python_refuses_cpu_tensors():
    x = torch.randn(2, 3, 8)
    with pytest.raises(RuntimeError):
        nk.gated_scan_train(x, x, x)
    with pytest.raises(RuntimeError):
        nk.ssd_scan_train(x, x, x, x, x, torch.ones(8), 0.001, 0.2)
    with pytest.raises(RuntimeError):
        nk.ssd_conv_silu_train(x, torch.ones(8, 1, 3))
    with pytest.raises(RuntimeError):
        nk.rms_norm_train(x, torch.ones(8))


# ------------------------------------------------------------------ the references themselves

def test_reference_gradients_against_differences():
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64, requires_grad=True)  # noqa: E731
    seg = torch.zeros(2, 7, dtype=torch.uint8)
    seg[0, 3] = seg[1, 0] = seg[1, 6] = 1
    assert torch.autograd.gradcheck(lambda *a: ref.gated(*a, seg=seg), [r(2, 7, 3) for _ in range(3)] + [r(2, 3)])
    assert torch.autograd.gradcheck(lambda *a: ref.ssd(*a, 0.001, 0.2, seg=seg),
                                    [r(2, 7, 3) for _ in range(5)] + [r(3), r(2, 3)])
    assert torch.autograd.gradcheck(lambda *a: ref.conv_silu(*a, seg=seg), [r(2, 7, 3), r(3, 4), r(3)])
    assert torch.autograd.gradcheck(lambda *a: ref.rms_norm(*a, 1e-6), [r(4, 6), r(6)])


def test_reference_norm_gradient_form():
    """The form of the norm's gradient written out for the 8-bit reference is the true
    gradient when the stored values are the true ones."""
    gen = torch.Generator().manual_seed(1)
    x = ref.e4m3(torch.randn(5, 70, generator=gen, dtype=torch.float64)).requires_grad_()
    w = torch.randn(70, generator=gen, dtype=torch.float64, requires_grad=True)
    g = torch.randn(5, 70, generator=gen, dtype=torch.float64)
    for a, b in zip(torch.autograd.grad(ref.rms_norm(x, w, 1e-6), (x, w), g),
                    torch.autograd.grad(ref.rms_norm(x, w, 1e-6, ckpt=True), (x, w), g)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_reference_e4m3_against_torch():
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(64, 130, generator=gen) * torch.exp(3 * torch.randn(64, 1, generator=gen))
    x[0] = 0
    x[1, :64] *= 1e-30
    q = ref.e4m3(x)
    for c in range(0, 130, 64):
        g, top = x[:, c:c + 64], x[:, c:c + 64].abs().amax(-1, keepdim=True)
        for e in range(-126, 20):  # the least exponent that fits, by trial
            rows = ((top <= 448 * 2.0 ** e) & ((top > 448 * 2.0 ** (e - 1)) | (e == -126)))[:, 0]
            want = (g[rows] * 2.0 ** -e).to(torch.float8_e4m3fn).float() * 2.0 ** e
            assert torch.equal(q[rows, c:c + 64], want)
