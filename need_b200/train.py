"""The recurrent block's operators for training: each with its gradient.

``gated_scan_train`` and ``ssd_scan_train`` are the recurrences of
``gated_scan`` and ``ssd_scan``, ``ssd_conv_silu_train`` the block's causal
depthwise conv + SiLU, ``rms_norm_train`` its out_norm (need_core.py:1618-1643
computes them with torch ops under grad).  ``need_kernels`` re-exports them.

They differ from the forward-only functions in precision: gates, states and
gradients are fp32, rounded once to the input's dtype, as the reference's GPU
kernels compute (need_kernels.py:99-144) -- the forward-only functions round
every gate op as its torch path does.

``checkpoint=torch.float8_e4m3fn`` keeps the activations the backward needs in 8
bits (one power-of-two scale per token and 64 channels) instead of the inputs
themselves: half the memory of 16-bit inputs, provided nothing else holds them.
The forward's results are unchanged.  The gradient is the formula's at the
stored values; the recurrences start every 64-token chunk from the true fp32
state.  A group that holds an infinity or NaN gives NaN gradients.

All take CUDA tensors of one device in fp32, bf16 or f16, run on the current
stream, allocate their scratch per call, and can be captured into CUDA graphs.
Gradients of gradients are not available.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import abi

_DT = {torch.float32: abi.F32, torch.bfloat16: abi.BF16, torch.float16: abi.F16}
_MAX_NORM_BYTES = 32768  # need_rms_norm_train_forward's longest row
_SPAN, _GROUP = 64, 64   # need_scan_train_chunk_len(), need_scan_train_group()


def _check(*ts: Optional[torch.Tensor]) -> None:
    dev = ts[0].device
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"need_b200 kernels take CUDA tensors only (no CPU fallback); got a {t.device} tensor")
        if t.device != dev:
            raise RuntimeError("all tensors must be on the same CUDA device")


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _DT.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} takes fp32, bf16 or f16 data; got {t.dtype}")
    return code


def _checkpoint(checkpoint) -> bool:
    if checkpoint is None:
        return False
    if checkpoint is torch.float8_e4m3fn:
        return True
    raise ValueError(f"checkpoint must be None or torch.float8_e4m3fn; got {checkpoint}")


def _on(dev: torch.device):
    return contextlib.nullcontext() if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _call(name: str, a, dev: torch.device) -> None:
    abi.check(name, getattr(abi.load(), name)(ctypes.byref(a), torch.cuda.current_stream(dev).cuda_stream))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with channel stride 1, a 16-byte aligned base and positive row strides of
    whole 16 bytes (dims of size 1 excepted); a copy if it is laid out otherwise."""
    es = t.element_size()
    ok = t.data_ptr() % 16 == 0 and (t.stride(-1) == 1 or t.shape[-1] == 1)
    for n, s in zip(t.shape[:-1], t.stride()[:-1]):
        ok = ok and (n == 1 or (s > 0 and s * es % 16 == 0))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _mask(seg_start: Optional[torch.Tensor], B: int, T: int, dev) -> Optional[torch.Tensor]:
    if seg_start is None:
        return None
    if tuple(seg_start.shape) != (B, T):
        raise ValueError(f"seg_start must be [B, T] = [{B}, {T}]; got {tuple(seg_start.shape)}")
    return seg_start.to(device=dev, dtype=torch.uint8)


# --------------------------------------------------------------------------
# the recurrences
# --------------------------------------------------------------------------

class _ScanTrainFn(torch.autograd.Function):
    """(out, final state) of the GATED or SSD scan; streams in the C ABI's in[] order."""

    @staticmethod
    def forward(ctx, form, ckpt, dt_min, dt_max, seg, h0, d_skip, *streams):
        xs = [_rows(x) for x in streams]
        B, T, C = xs[0].shape
        dev, dt = xs[0].device, xs[0].dtype
        ckpt = ckpt and any(ctx.needs_input_grad)
        lib = abi.load()
        out = torch.empty((B, T, C), dtype=dt, device=dev)
        final = torch.empty((B, C), dtype=torch.float32, device=dev)
        states = torch.empty((B, -(-T // _SPAN), C), dtype=torch.float32, device=dev)
        a = abi.NeedScanTrainArgs()
        _ScanTrainFn._common(a, form, dt, ckpt, dt_min, dt_max, seg, d_skip, states, B, T, C)
        for k, x in enumerate(xs):
            a.in_[k] = abi.NeedView(x.data_ptr(), x.stride(0), 0, x.stride(1))
        q = qs = None
        if ckpt:
            groups = -(-C // _GROUP)
            q = torch.empty((len(xs), B, T, groups * _GROUP), dtype=torch.uint8, device=dev)
            qs = torch.empty((len(xs), B, T, groups), dtype=torch.uint8, device=dev)
            a.ckpt_values, a.ckpt_scales = q.data_ptr(), qs.data_ptr()
        if h0 is not None:
            h0 = h0.contiguous()
            a.h0 = h0.data_ptr()
        a.out, a.out_stride_b, a.out_stride_t = out.data_ptr(), out.stride(0), out.stride(1)
        a.h_final = final.data_ptr()
        ws = torch.empty(lib.need_scan_train_workspace_size(form, 0, B, T, C), dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        with _on(dev):
            _call("need_scan_train_forward", a, dev)
        ctx.save_for_backward(states, seg, d_skip, *((q, qs) if ckpt else xs))
        ctx.info = (form, ckpt, dt_min, dt_max, dt, B, T, C, h0 is not None)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def _common(a, form, dt, ckpt, dt_min, dt_max, seg, d_skip, states, B, T, C):
        a.form, a.dtype, a.checkpoint = form, _DT[dt], int(ckpt)
        a.nb, a.T, a.C = B, T, C
        a.dt_min, a.dt_max = dt_min, dt_max
        a.states = states.data_ptr()
        if d_skip is not None:
            a.d_skip = d_skip.data_ptr()
        if seg is not None:
            a.seg_start = seg.data_ptr()
            a.seg_stride_b, a.seg_stride_t = seg.stride()

    @staticmethod
    @once_differentiable
    def backward(ctx, gout, gfinal):
        form, ckpt, dt_min, dt_max, dt, B, T, C, has_h0 = ctx.info
        states, seg, d_skip, *saved = ctx.saved_tensors
        dev = states.device
        nin = 3 if form == abi.FORM_GATED else 5
        gout = torch.zeros((B, T, C), dtype=dt, device=dev) if gout is None else _rows(gout)
        a = abi.NeedScanTrainArgs()
        _ScanTrainFn._common(a, form, dt, ckpt, dt_min, dt_max, seg, d_skip, states, B, T, C)
        if ckpt:
            a.ckpt_values, a.ckpt_scales = saved[0].data_ptr(), saved[1].data_ptr()
        else:
            for k, x in enumerate(saved):
                a.in_[k] = abi.NeedView(x.data_ptr(), x.stride(0), 0, x.stride(1))
        a.gout = abi.NeedView(gout.data_ptr(), gout.stride(0), 0, gout.stride(1))
        if gfinal is not None:
            gfinal = gfinal.contiguous()
            a.g_final = gfinal.data_ptr()
        grads = [torch.empty((B, T, C), dtype=dt, device=dev) for _ in range(nin)]
        for k, g in enumerate(grads):
            a.grad[k] = g.data_ptr()
        gh0 = gd = None
        if has_h0:
            gh0 = torch.empty((B, C), dtype=torch.float32, device=dev)
            a.grad_h0 = gh0.data_ptr()
        if d_skip is not None:
            gd = torch.empty(C, dtype=torch.float32, device=dev)
            a.grad_d = gd.data_ptr()
        ws = torch.empty(abi.load().need_scan_train_workspace_size(form, 1, B, T, C), dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        with _on(dev):
            _call("need_scan_train_backward", a, dev)
        return (None, None, None, None, None, gh0, gd, *grads)


def _scan_train(form, streams, seg_start, h0, checkpoint, return_final_state, d_skip=None, dt_min=0.0, dt_max=0.0):
    x = streams[0]
    ckpt = _checkpoint(checkpoint)
    B, T, C = x.shape
    if h0 is not None:
        if tuple(h0.shape) != (B, C):
            raise ValueError(f"h0 must be [B, C] = [{B}, {C}]; got {tuple(h0.shape)}")
        h0 = h0.float()
    seg = _mask(seg_start, B, T, x.device)
    if x.numel() == 0:  # nothing to scan: the state passes through
        out = x
        for s in streams[1:]:
            out = out * s
        if d_skip is not None:
            out = (out * d_skip).to(x.dtype)
        final = h0 if h0 is not None else torch.zeros((B, C), device=x.device)
        return (out, final) if return_final_state else out
    pad = -C % (16 // x.element_size())
    if pad:
        streams = [F.pad(s, (0, pad)) for s in streams]
        h0 = None if h0 is None else F.pad(h0, (0, pad))
        d_skip = None if d_skip is None else F.pad(d_skip, (0, pad))
    out, final = _ScanTrainFn.apply(form, ckpt, dt_min, dt_max, seg, h0,
                                    None if d_skip is None else d_skip.contiguous(), *streams)
    if pad:
        out, final = out[..., :C], final[:, :C]
    return (out, final) if return_final_state else out


def gated_scan_train(x: torch.Tensor, decay_logit: torch.Tensor, gate_logit: torch.Tensor, *,
                     seg_start: Optional[torch.Tensor] = None, h0: Optional[torch.Tensor] = None,
                     return_final_state: bool = False, checkpoint: Optional[torch.dtype] = None):
    """:func:`need_kernels.gated_scan` with gradients: ``a = sigmoid(decay_logit)``,
    ``h_t = a_t h_{t-1} + (1 - a_t) sigmoid(gate_logit_t) x_t`` over [B, T, C];
    returns ``h`` in ``x.dtype``, with ``return_final_state`` also the fp32 state
    [B, C] after the last token.

    Differentiable in ``x``, both logits and ``h0`` [B, C], through ``h`` and the
    final state.  ``seg_start`` [B, T] (bool / uint8): the state before a marked
    token does not reach it, nor do later gradients reach back across it, even
    where either is an infinity or NaN.  ``checkpoint``: see the module.
    """
    _check(x, decay_logit, gate_logit, seg_start, h0)
    _dtype(x, "gated_scan_train")
    if x.dim() != 3 or not (x.shape == decay_logit.shape == gate_logit.shape):
        raise ValueError("x, decay_logit and gate_logit must have the same [B, T, C] shape")
    return _scan_train(abi.FORM_GATED, [decay_logit.to(x.dtype), gate_logit.to(x.dtype), x], seg_start, h0, checkpoint,
                       return_final_state)


def ssd_scan_train(u: torch.Tensor, b_gate: torch.Tensor, c_gate: torch.Tensor, dt_raw: torch.Tensor,
                   out_gate: torch.Tensor, d_skip: torch.Tensor, dt_min: float, dt_max: float, *,
                   seg_start: Optional[torch.Tensor] = None, h0: Optional[torch.Tensor] = None,
                   return_final_state: bool = False, checkpoint: Optional[torch.dtype] = None):
    """:func:`need_kernels.ssd_scan` with gradients, all [B, T, D]:

    ``a = exp(-(dt_min + (dt_max - dt_min) * sigmoid(dt_raw)))``,
    ``h_t = a_t h_{t-1} + (1 - a_t) sigmoid(b_gate_t) u_t``,
    ``y = (sigmoid(c_gate) * h + d_skip * u) * sigmoid(out_gate)``;
    returns ``y`` in ``u.dtype``, with ``return_final_state`` also the fp32 state
    [B, D] after the last token.  ``0 <= dt_min <= dt_max``; ``d_skip`` holds D values.

    Differentiable in the five streams, ``d_skip`` and ``h0``, through ``y`` and the
    final state.  ``seg_start`` as for :func:`gated_scan_train`; ``checkpoint``: see
    the module.  The streams may be chunks of one in-projection (no copy is made
    of views whose rows are 16-byte aligned).
    """
    streams = (u, b_gate, c_gate, dt_raw, out_gate)
    _check(*streams, d_skip, seg_start, h0)
    _dtype(u, "ssd_scan_train")
    if u.dim() != 3 or any(s.shape != u.shape for s in streams):
        raise ValueError("u, b_gate, c_gate, dt_raw and out_gate must have the same [B, T, D] shape")
    if d_skip.numel() != u.shape[-1]:
        raise ValueError(f"d_skip must have D={u.shape[-1]} elements; got {tuple(d_skip.shape)}")
    if not 0.0 <= float(dt_min) <= float(dt_max):
        raise ValueError(f"0 <= dt_min <= dt_max expected; got {dt_min}, {dt_max}")
    order = [s.to(u.dtype) for s in (dt_raw, b_gate, u, c_gate, out_gate)]
    return _scan_train(abi.FORM_SSD, order, seg_start, h0, checkpoint, return_final_state,
                       d_skip.reshape(-1).float(), float(dt_min), float(dt_max))


# --------------------------------------------------------------------------
# the conv + SiLU before the scan
# --------------------------------------------------------------------------

class _ConvTrainFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, weight, bias, seg):
        u = _rows(u)
        B, T, C = u.shape
        w = weight.contiguous()
        b = None if bias is None else bias.contiguous()
        out = torch.empty((B, T, C), dtype=u.dtype, device=u.device)
        a = _ConvTrainFn._args(u, w, b, seg)
        a.out = out.data_ptr()
        with _on(u.device):
            _call("need_conv_silu_train_forward", a, u.device)
        ctx.save_for_backward(u, w, b, seg)
        return out

    @staticmethod
    def _args(u, w, b, seg):
        a = abi.NeedConvTrainArgs()
        a.dtype, a.K = _DT[u.dtype], w.shape[1]
        a.nb, a.T, a.C = u.shape
        a.u, a.u_stride_b, a.u_stride_t = u.data_ptr(), u.stride(0), u.stride(1)
        a.weight = w.data_ptr()
        if b is not None:
            a.bias = b.data_ptr()
        if seg is not None:
            a.seg_start = seg.data_ptr()
            a.seg_stride_b, a.seg_stride_t = seg.stride()
        return a

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        u, w, b, seg = ctx.saved_tensors
        B, T, C = u.shape
        K = w.shape[1]
        gout = _rows(gout)
        a = _ConvTrainFn._args(u, w, b, seg)
        a.gout, a.gout_stride_b, a.gout_stride_t = gout.data_ptr(), gout.stride(0), gout.stride(1)
        gu = torch.empty((B, T, C), dtype=u.dtype, device=u.device)
        gwb = torch.empty((C, K + 1), dtype=torch.float32, device=u.device)
        ws = torch.empty(abi.load().need_conv_silu_train_workspace_size(K, B, T, C), dtype=torch.uint8, device=u.device)
        a.grad_u, a.grad_wb = gu.data_ptr(), gwb.data_ptr()
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        with _on(u.device):
            _call("need_conv_silu_train_backward", a, u.device)
        return gu, gwb[:, :K], gwb[:, K] if b is not None else None, None


def ssd_conv_silu_train(u: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                        seg_start: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`need_kernels.ssd_conv_silu` with gradients: ``silu(conv1d(u, weight,
    bias, padding=K-1, groups=C)[..., :T])`` over ``u`` [B, T, C] (channels last),
    in fp32, rounded once to ``u.dtype``.  ``weight`` is the Conv1d weight [C, 1,
    K] (or [C, K]), K <= 4, ``bias`` [C] or None, both used in fp32.  Differentiable
    in all three.  ``seg_start`` [B, T]: inputs before a token's segment start do
    not feed it."""
    _check(u, weight, bias, seg_start)
    _dtype(u, "ssd_conv_silu_train")
    if u.dim() != 3:
        raise ValueError(f"u must be [B, T, C]; got {tuple(u.shape)}")
    B, T, C = u.shape
    if weight.dim() not in (2, 3) or weight.shape[0] != C or (weight.dim() == 3 and weight.shape[1] != 1):
        raise ValueError(f"weight must be [C, 1, K] or [C, K] with C={C}; got {tuple(weight.shape)}")
    K = weight.shape[-1]
    if not 1 <= K <= 4:
        raise ValueError(f"1 to 4 taps expected; got {K}")
    if bias is not None and tuple(bias.shape) != (C,):
        raise ValueError(f"bias must be [C] = [{C}]; got {tuple(bias.shape)}")
    seg = _mask(seg_start, B, T, u.device)
    w = weight.reshape(C, K).float()
    b = None if bias is None else bias.float()
    if u.numel() == 0:
        out = u * w.sum(dim=1) if b is None else u * w.sum(dim=1) + b
        return out.to(u.dtype)
    pad = -C % (16 // u.element_size())
    if pad:
        u = F.pad(u, (0, pad))
        w = F.pad(w, (0, 0, 0, pad))
        b = None if b is None else F.pad(b, (0, pad))
    out = _ConvTrainFn.apply(u, w, b, seg)
    return out[..., :C] if pad else out


# --------------------------------------------------------------------------
# the norm after the scan
# --------------------------------------------------------------------------

class _NormTrainFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, ckpt, c_mean):
        x = _rows(x)
        rows, C = x.shape
        ckpt = ckpt and any(ctx.needs_input_grad)
        w = weight if weight.is_contiguous() and weight.data_ptr() % 16 == 0 else weight.clone(
            memory_format=torch.contiguous_format)
        out = torch.empty((rows, C), dtype=x.dtype, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        a = _NormTrainFn._args(x.dtype, rows, C, c_mean, w, rstd, eps, ckpt)
        a.x, a.x_stride, a.out = x.data_ptr(), x.stride(0), out.data_ptr()
        q = qs = None
        if ckpt:
            q = torch.empty((rows, C), dtype=torch.uint8, device=x.device)
            qs = torch.empty((rows, -(-C // _GROUP)), dtype=torch.uint8, device=x.device)
            a.ckpt_values, a.ckpt_scales = q.data_ptr(), qs.data_ptr()
        with _on(x.device):
            _call("need_rms_norm_train_forward", a, x.device)
        ctx.save_for_backward(w, rstd, *((q, qs) if ckpt else (x,)))
        ctx.info = (x.dtype, rows, C, c_mean, eps, ckpt)
        return out

    @staticmethod
    def _args(dt, rows, C, c_mean, w, rstd, eps, ckpt):
        a = abi.NeedNormTrainArgs()
        a.dtype, a.checkpoint = _DT[dt], int(ckpt)
        a.rows, a.C, a.C_mean = rows, C, c_mean
        a.weight, a.rstd, a.eps = w.data_ptr(), rstd.data_ptr(), eps
        return a

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        dt, rows, C, c_mean, eps, ckpt = ctx.info
        w, rstd, *saved = ctx.saved_tensors
        dev = rstd.device
        gout = _rows(gout)
        a = _NormTrainFn._args(dt, rows, C, c_mean, w, rstd, eps, ckpt)
        if ckpt:
            a.ckpt_values, a.ckpt_scales = saved[0].data_ptr(), saved[1].data_ptr()
        else:
            a.x, a.x_stride = saved[0].data_ptr(), saved[0].stride(0)
        a.gout, a.gout_stride = gout.data_ptr(), gout.stride(0)
        gx = torch.empty((rows, C), dtype=dt, device=dev)
        gw = torch.empty(C, dtype=torch.float32, device=dev)
        ws = torch.empty(abi.load().need_rms_norm_train_workspace_size(rows, C), dtype=torch.uint8, device=dev)
        a.grad_x, a.grad_weight = gx.data_ptr(), gw.data_ptr()
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        with _on(dev):
            _call("need_rms_norm_train_backward", a, dev)
        return gx, gw, None, None, None


def rms_norm_train(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                   checkpoint: Optional[torch.dtype] = None) -> torch.Tensor:
    """:func:`need_kernels.rms_norm` with gradients: ``x / sqrt(mean(x^2) + eps) *
    weight`` over the last dim, in fp32, rounded once to ``x.dtype``; ``weight`` [C] is
    used in fp32.  Differentiable in both.  Rows of up to 32 KB.  ``checkpoint``: x is
    kept in 8 bits for the backward, 1 / sqrt(...) in fp32; see the module."""
    _check(x, weight)
    _dtype(x, "rms_norm_train")
    ckpt = _checkpoint(checkpoint)
    C = x.shape[-1] if x.dim() else 0
    if x.dim() < 1 or weight.numel() != C:
        raise ValueError(f"weight must have as many elements as x's last dim; got {tuple(weight.shape)} for {tuple(x.shape)}")
    if not float(eps) >= 0.0:
        raise ValueError(f"eps must be >= 0; got {eps}")
    w = weight.reshape(-1).float()
    if x.numel() == 0:
        return (x * w).to(x.dtype)
    pad = -C % (16 // x.element_size())
    if (C + pad) * x.element_size() > _MAX_NORM_BYTES:
        raise NotImplementedError(f"rms_norm_train takes rows of at most {_MAX_NORM_BYTES} bytes; got C={C} of {x.dtype}")
    rows = x.reshape(-1, C)
    if pad:
        rows, w = F.pad(rows, (0, pad)), F.pad(w, (0, pad))
    y = _NormTrainFn.apply(rows, w, float(eps), ckpt, C)
    return (y[:, :C] if pad else y).reshape(x.shape)
