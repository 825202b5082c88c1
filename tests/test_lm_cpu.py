"""The language-model operators without a GPU: refusals (host checks that make no CUDA
call), the ctypes layouts, and the tests' own references against differences."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import lm_reference as ref
from need_b200 import abi, build, lm
from need_b200 import need_kernels as nk

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "need_scan.h")
P = 1 << 20  # an aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


def test_struct_layout_matches_header(tmp_path):
    structs = {"need_heads": abi.NeedHeads, "need_linear_attention_args": abi.NeedLinearAttentionArgs,
               "need_linear_attention_step_args": abi.NeedLinearAttentionStepArgs,
               "need_residual_norm_args": abi.NeedResidualNormArgs, "need_token_log_probs_args": abi.NeedTokenLogProbsArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for n, *_ in cls._fields_:
            lines.append(f'printf("{name}.{n} %zu\\n", offsetof({name}, {n}));')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for n, *_ in cls._fields_:
            assert int(got[f"{name}.{n}"]) == getattr(cls, n).offset, f"{name}.{n}"


def attention_args(**kw):
    a = abi.NeedLinearAttentionArgs()
    a.dtype, a.scale, a.nb, a.T, a.H, a.dk, a.dv = abi.BF16, 1.0, 2, 100, 4, 64, 64
    for x in (a.q, a.k, a.v):
        x.ptr, x.stride_b, x.stride_t, x.stride_h, x.heads = P, 25600, 256, 64, 4
    a.log_decay = a.out = a.workspace = P
    a.ld_stride_h, a.workspace_bytes = 1, 1 << 40
    a.out_stride_b, a.out_stride_t, a.out_stride_h = 25600, 256, 64
    for k, v in kw.items():
        if "." in k:
            setattr(getattr(a, k.split(".")[0]), k.split(".")[1], v)
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    ({"dtype": 7}, abi.ERR_UNSUPPORTED), ({"T": 0}, abi.ERR_INVALID), ({"nb": -1}, abi.ERR_INVALID), ({"dk": 0}, abi.ERR_INVALID),
    ({"dk": 129}, abi.ERR_UNSUPPORTED), ({"T": 1 << 40}, abi.ERR_UNSUPPORTED), ({"H": 1 << 30}, abi.ERR_UNSUPPORTED),
    ({"nb": 1 << 40}, abi.ERR_UNSUPPORTED), ({"q.ptr": None}, abi.ERR_INVALID), ({"v.ptr": None}, abi.ERR_INVALID),
    ({"k.heads": 3}, abi.ERR_INVALID), ({"k.heads": 0}, abi.ERR_INVALID), ({"v.heads": 8}, abi.ERR_INVALID),
    ({"log_decay": None}, abi.ERR_INVALID), ({"out": None}, abi.ERR_INVALID), ({"out_stride_t": 63}, abi.ERR_INVALID),
    ({"workspace": None}, abi.ERR_WORKSPACE), ({"T": 4096, "workspace": None}, abi.ERR_WORKSPACE), ({"T": 4096, "workspace_bytes": 1000}, abi.ERR_WORKSPACE),
])
def test_attention_refuses(lib, change, code):
    assert lib.need_linear_attention(ctypes.byref(attention_args(**change)), None) == code
    assert lib.need_last_error()


@pytest.mark.parametrize("T,dtype", [(1, abi.F32), (100, abi.BF16), (4096, abi.F16)])
@pytest.mark.parametrize("shift", [0, 4, 2 * 4 * 64 * 64 * 4 - 4, -4])
def test_attention_refuses_a_state_in_place(lib, T, dtype, shift):
    """Blocks may read it again after the final one has been written."""
    a = attention_args(T=T, dtype=dtype, state=P, final_state=P + shift)
    assert lib.need_linear_attention(ctypes.byref(a), None) == abi.ERR_INVALID
    assert b"overlap" in lib.need_last_error()


def test_attention_takes_states_side_by_side(lib):
    """Next to each other they are taken: what is refused here is the workspace."""
    for shift in (2 * 4 * 64 * 64 * 4, -2 * 4 * 64 * 64 * 4):
        a = attention_args(T=4096, state=P, final_state=P + shift, workspace=None)
        assert lib.need_linear_attention(ctypes.byref(a), None) == abi.ERR_WORKSPACE


def step_args(**kw):
    a = abi.NeedLinearAttentionStepArgs()
    a.dtype, a.scale, a.n, a.H, a.dk, a.dv = abi.BF16, 1.0, 10, 4, 64, 64
    for x in (a.q, a.k, a.v):
        x.ptr, x.stride_b, x.stride_h, x.heads = P, 256, 64, 4
    a.log_decay = a.out = a.state = a.slot = P
    a.state_stride, a.slots, a.out_stride_n, a.out_stride_h = 4 * 64 * 64, 20, 256, 64
    for k, v in kw.items():
        if "." in k:
            setattr(getattr(a, k.split(".")[0]), k.split(".")[1], v)
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    ({"dtype": 7}, abi.ERR_UNSUPPORTED), ({"n": 0}, abi.ERR_INVALID), ({"dv": 0}, abi.ERR_INVALID), ({"slots": -1}, abi.ERR_INVALID),
    ({"dk": 2049}, abi.ERR_UNSUPPORTED), ({"n": 1 << 40}, abi.ERR_UNSUPPORTED), ({"k.ptr": None}, abi.ERR_INVALID),
    ({"q.heads": 3}, abi.ERR_INVALID), ({"state": None}, abi.ERR_INVALID), ({"out": None}, abi.ERR_INVALID),
    ({"log_decay": None}, abi.ERR_INVALID), ({"slot": None, "slots": 9}, abi.ERR_INVALID),
    ({"state_stride": 4 * 64 * 64 - 1}, abi.ERR_INVALID),
])
def test_step_refuses(lib, change, code):
    assert lib.need_linear_attention_step(ctypes.byref(step_args(**change)), None) == code
    assert lib.need_last_error()


def norm_args(**kw):
    a = abi.NeedResidualNormArgs()
    a.dtype, a.out8, a.rows, a.C, a.group, a.eps, a.scale = abi.BF16, 1, 10, 100, 32, 1e-6, 1.0
    a.x = a.y = a.weight = a.stream = a.out = a.scales = P
    a.x_stride = a.y_stride = a.stream_stride = a.out_stride = 100
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    ({"dtype": 5}, abi.ERR_UNSUPPORTED), ({"rows": 0}, abi.ERR_INVALID), ({"C": 0}, abi.ERR_INVALID),
    ({"C": 16385}, abi.ERR_UNSUPPORTED), ({"dtype": abi.F32, "C": 8193}, abi.ERR_UNSUPPORTED), ({"rows": 1 << 31}, abi.ERR_UNSUPPORTED),
    ({"eps": -1.0}, abi.ERR_INVALID), ({"eps": float("nan")}, abi.ERR_INVALID), ({"x": None}, abi.ERR_INVALID),
    ({"y": None}, abi.ERR_INVALID), ({"weight": None}, abi.ERR_INVALID), ({"stream": None}, abi.ERR_INVALID),
    ({"out": None}, abi.ERR_INVALID), ({"scales": None}, abi.ERR_INVALID), ({"group": 16}, abi.ERR_INVALID),
    ({"group": 0}, abi.ERR_INVALID), ({"out8": 2}, abi.ERR_INVALID), ({"out_stride": 99}, abi.ERR_INVALID),
    ({"stream_stride": 99}, abi.ERR_INVALID),
])
def test_norm_refuses(lib, change, code):
    assert lib.need_residual_rms_norm(ctypes.byref(norm_args(**change)), None) == code
    assert lib.need_last_error()


def logp_args(**kw):
    a = abi.NeedTokenLogProbsArgs()
    a.dtype, a.top, a.rows, a.V, a.stride, a.temperature = abi.BF16, 5, 10, 100, 100, 1.0
    a.logits = a.tokens = a.log_prob = a.entropy = a.stats = a.top_log_probs = a.top_tokens = a.grad = a.workspace = P
    a.grad_stride, a.workspace_bytes = 100, 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    ({"dtype": 5}, abi.ERR_UNSUPPORTED), ({"rows": 0}, abi.ERR_INVALID), ({"V": 0}, abi.ERR_INVALID),
    ({"V": 1 << 31}, abi.ERR_UNSUPPORTED), ({"rows": 1 << 31}, abi.ERR_UNSUPPORTED), ({"logits": None}, abi.ERR_INVALID),
    ({"tokens": None}, abi.ERR_INVALID), ({"entropy": None}, abi.ERR_INVALID), ({"temperature": 0.0}, abi.ERR_INVALID),
    ({"temperature": float("inf")}, abi.ERR_INVALID), ({"temperature": float("nan")}, abi.ERR_INVALID),
])
def test_logp_refuses(lib, change, code):
    assert lib.need_token_log_probs(ctypes.byref(logp_args(**change)), None) == code
    assert lib.need_token_log_probs_backward(ctypes.byref(logp_args(**change)), None) == code


@pytest.mark.parametrize("change,code", [
    ({"top": -1}, abi.ERR_INVALID), ({"top": 33}, abi.ERR_UNSUPPORTED), ({"V": 4}, abi.ERR_INVALID),
    ({"top_tokens": None}, abi.ERR_INVALID), ({"log_prob": None}, abi.ERR_INVALID),
    ({"V": 100000, "stride": 100000, "workspace": None}, abi.ERR_WORKSPACE),
    ({"V": 100000, "stride": 100000, "workspace_bytes": 8}, abi.ERR_WORKSPACE),
])
def test_logp_forward_refuses(lib, change, code):
    assert lib.need_token_log_probs(ctypes.byref(logp_args(**change)), None) == code


@pytest.mark.parametrize("change", [{"stats": None}, {"grad": None}, {"grad_stride": 99}])
def test_logp_backward_refuses(lib, change):
    assert lib.need_token_log_probs_backward(ctypes.byref(logp_args(**change)), None) == abi.ERR_INVALID


def test_null_args(lib):
    for fn in (lib.need_linear_attention, lib.need_linear_attention_step, lib.need_residual_rms_norm, lib.need_token_log_probs,
               lib.need_token_log_probs_backward):
        assert fn(None, None) == abi.ERR_INVALID


def test_workspaces(lib):
    size = lib.need_linear_attention_workspace_size
    assert size(abi.F32, 16, 4096, 32, 64, 64) == 16  # chains enough: nothing between parts
    assert size(abi.F32, 1, 64, 1, 64, 64) == 16      # one chunk
    assert size(abi.F32, 1, 16384, 4, 32, 48) > 16 and size(abi.F32, 0, 1, 1, 1, 1) == 16 and size(9, 1, 16384, 4, 32, 48) == 16
    assert size(abi.BF16, 16, 4096, 16, 64, 64) == 16 + 4 * 256  # a word a block
    size = lib.need_token_log_probs_workspace_size
    assert size(abi.BF16, 1000, 50000, 20) == 16 and size(abi.BF16, 4, 784, 20) == 16
    assert size(abi.F32, 4, 131072, 5) > 16 and size(9, 4, 131072, 5) == 16


# ------------------------------------------------------------------ the Python layer
def test_python_refusals():
    """All before any CUDA call."""
    x = torch.zeros(2, 3, 4, 8)
    d, s = torch.zeros(4), torch.zeros(2, 4, 8, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nk.linear_attention(x, x, x, d)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nk.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], d, s)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nk.residual_rms_norm(x, x, torch.ones(8))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nk.token_log_probs(x, torch.zeros(2, 3, 4, dtype=torch.long))
    with pytest.raises(NotImplementedError, match="no backward"):
        nk.linear_attention(x.clone().requires_grad_(), x, x, d)
    with pytest.raises(NotImplementedError, match="no backward"):
        nk.linear_attention(x, x, x, d.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="no backward"):
        nk.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], d, s.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="no backward"):
        nk.residual_rms_norm(x, x, torch.ones(8).requires_grad_())
    wide = torch.zeros(1, 1, 1, 129)
    with pytest.raises(NotImplementedError, match="128 features"):
        nk.linear_attention(wide, wide, wide, torch.zeros(1))
    with pytest.raises(NotImplementedError, match="2048 features"):
        nk.linear_attention_step(torch.zeros(1, 1, 2049), torch.zeros(1, 1, 2049), wide[0], torch.zeros(1), s)
    with pytest.raises(NotImplementedError, match="32768 bytes"):
        nk.residual_rms_norm(torch.zeros(1, 8193), torch.zeros(1, 8193), torch.ones(8193))
    with pytest.raises(ValueError, match="group"):
        nk.residual_rms_norm(x, x, torch.ones(8), out_dtype=torch.float8_e4m3fn, group=16)
    with pytest.raises(ValueError, match="group"):
        nk.residual_rms_norm(x, x, torch.ones(8), group=32)
    with pytest.raises(ValueError, match="out_dtype"):
        nk.residual_rms_norm(x, x, torch.ones(8), out_dtype=torch.float8_e5m2)
    with pytest.raises(NotImplementedError, match="32 alternatives"):
        nk.token_log_probs(x, torch.zeros(2, 3, 4, dtype=torch.long), top=33)


def test_limits_agree():
    text = open(HEADER).read()
    assert f"NEED_LINEAR_ATTENTION_MAX_DK {lm._MAX_FEATURES}\n" in text
    assert f"NEED_TOKEN_LOG_PROBS_MAX_TOP {lm._MAX_TOP}\n" in text


def test_the_module_runs_on_the_shared_cpp_library():
    build.build()
    ext = os.path.join(build.LIBDIR, "_lm.so")
    with open(ext, "rb") as f:
        assert b"\0libstdc++.so.6\0" in f.read()
    assert "-nostdlib++" in build._ext_command(ext)


def test_error_texts_format_numbers():
    """In a process of its own: a second C++ library in it would end it."""
    code = ("import torch\nfrom need_b200 import need_kernels as nk\nx = torch.zeros(2, 3, 4, 8)\n"
            "try:\n    nk.linear_attention(x, x, x, torch.zeros(4))\nexcept RuntimeError as e:\n    print(e)\n")
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=build.ROOT)
    assert p.returncode == 0 and "[2, 3, 4, 8] on cpu" in p.stdout, p.stderr[-500:]


# ------------------------------------------------------------------ the references
def test_attention_reference_is_the_sum():
    """Against the sum over tokens that the recurrence stands for."""
    g = torch.Generator().manual_seed(0)
    B, T, H, dk, dv = 2, 9, 2, 3, 4
    q, k, v = (torch.randn(B, T, h, d, generator=g, dtype=torch.float64) for h, d in ((2, dk), (1, dk), (2, dv)))
    ld = -torch.rand(B, T, H, generator=g, dtype=torch.float64)
    seg = torch.zeros(B, T, dtype=torch.uint8)
    seg[1, 4] = 1
    s0 = torch.randn(B, H, dk, dv, generator=g, dtype=torch.float64)
    out, s, _, _ = ref.attention(q, k, v, ld, 0.5, seg, s0)
    for b in range(B):
        for h in range(H):
            for t in range(T):
                first = 4 if b == 1 and t >= 4 else 0
                acc = torch.zeros(dv, dtype=torch.float64)
                if first == 0:
                    acc = torch.exp(ld[b, :t + 1, h].sum()) * (q[b, t, h] @ s0[b, h])
                for u in range(first, t + 1):
                    acc = acc + torch.exp(ld[b, u + 1:t + 1, h].sum()) * (q[b, t, h] @ k[b, u, 0]) * v[b, u, h]
                assert torch.allclose(out[b, t, h], 0.5 * acc, rtol=1e-12, atol=1e-12)


def test_log_probs_reference_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 7, generator=g, dtype=torch.float64)
    tok = torch.tensor([2, 6, -1])
    gl, gh = torch.randn(3, generator=g, dtype=torch.float64), torch.randn(3, generator=g, dtype=torch.float64)

    def loss(y):
        lp, h, _ = ref.log_probs(y, tok, 0.7)
        return (gl * lp + gh * h).sum()

    want, step = ref.log_probs_grad(x, tok, gl, gh, 0.7), 1e-6
    for i in range(3):
        for j in range(7):
            d = torch.zeros_like(x)
            d[i, j] = step
            num = (loss(x + d) - loss(x - d)) / (2 * step)
            assert abs(num - want[i, j]) < 1e-8
