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
themselves: half the memory of 16-bit inputs, provided nothing else holds them -- a
chunk of a projection that another operator saves holds all of it, so give
``ssd_conv_silu_train`` a ``u`` of its own there (see it).  Outputs are those without
it, but for the order of a few fp32 sums (such a call may take other tiles).  The
gradient is the formula's at the stored values; the recurrences start every 64-token
chunk from the true fp32 state.  A group that holds an infinity or NaN gives NaN
gradients.

All take CUDA tensors of one device in fp32, bf16 or f16, run on the current
stream, allocate their scratch per call, and can be captured into CUDA graphs.
Rows of their results are 16-byte aligned: where C elements are not a whole number
of 16 bytes, the rows lie further apart than C and the result is not contiguous.
Gradients of gradients and forward-mode tangents raise.  The autograd nodes are
compiled (csrc/train_autograd.cpp, ``_lib/_train.so``); there is no other path.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import abi

_MAX_NORM_BYTES = 32768  # need_rms_norm_train_forward's longest row
_EXT = None


def _ext():
    """The compiled autograd module (raises if it has not been built)."""
    global _EXT
    if _EXT is None:
        abi.load()  # the library it runs on: present, and of this ABI version
        try:
            from ._lib import _train
        except ImportError as e:
            raise RuntimeError("need_b200/_lib/_train.so is missing or does not load: build it with "
                               f"`python -m need_b200.build` ({e})") from e
        _EXT = _train
    return _EXT


def _checkpoint(checkpoint) -> bool:
    if checkpoint is not None and checkpoint is not torch.float8_e4m3fn:
        raise ValueError(f"checkpoint must be None or torch.float8_e4m3fn; got {checkpoint}")
    return checkpoint is not None


# --------------------------------------------------------------------------
# the recurrences
# --------------------------------------------------------------------------

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
    out, final = _ext().gated_scan_train(x, decay_logit, gate_logit, seg_start, h0, _checkpoint(checkpoint))
    return (out, final) if return_final_state else out


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
    the module.  The streams may be chunks of one in-projection: no copy is made of
    views with channel stride 1.
    """
    out, final = _ext().ssd_scan_train(u, b_gate, c_gate, dt_raw, out_gate, d_skip, dt_min, dt_max, seg_start, h0,
                                       _checkpoint(checkpoint))
    return (out, final) if return_final_state else out


# --------------------------------------------------------------------------
# the conv + SiLU before the scan
# --------------------------------------------------------------------------

def ssd_conv_silu_train(u: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                        seg_start: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`need_kernels.ssd_conv_silu` with gradients: ``silu(conv1d(u, weight,
    bias, padding=K-1, groups=C)[..., :T])`` over ``u`` [B, T, C] (channels last),
    in fp32, rounded once to ``u.dtype``.  ``weight`` is the Conv1d weight [C, 1,
    K] (or [C, K]), K <= 4, ``bias`` [C] or None, both used in fp32.  Differentiable
    in all three.  ``seg_start`` [B, T]: inputs before a token's segment start do
    not feed it.

    The backward keeps ``u`` as it is given, in the memory it lies in.  Where ``u`` is
    a chunk of a projection whose other chunks are kept in 8 bits only, pass
    ``u.contiguous()``: the projection can then be freed (2 bytes an element instead
    of 10)."""
    return _ext().conv_train(u, weight, bias, seg_start)


# --------------------------------------------------------------------------
# the norm after the scan
# --------------------------------------------------------------------------

def rms_norm_train(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                   checkpoint: Optional[torch.dtype] = None) -> torch.Tensor:
    """:func:`need_kernels.rms_norm` with gradients: ``x / sqrt(mean(x^2) + eps) *
    weight`` over the last dim, in fp32, rounded once to ``x.dtype``; ``weight`` [C] is
    used in fp32.  Differentiable in both.  Rows of up to 32 KB.  ``checkpoint``: x is
    kept in 8 bits for the backward, 1 / sqrt(...) in fp32; see the module."""
    if x.dim() and x.shape[-1] * x.element_size() > _MAX_NORM_BYTES:
        raise NotImplementedError(f"rms_norm_train takes rows of at most {_MAX_NORM_BYTES} bytes; got {tuple(x.shape)} "
                                  f"of {x.dtype}")
    return _ext().norm_train(x, weight, eps, _checkpoint(checkpoint))
