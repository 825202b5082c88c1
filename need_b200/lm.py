"""Operators of a language model around the recurrent block's.

``linear_attention`` is the matrix-state form of the retention scan
(``recurrent_retention_scan`` keeps ``k * v`` by element, need_core.py:1590-1592; here
the state of a head is ``k^T v``), for whole prompts; ``linear_attention_step`` is its
decode step, on a pool of states.  ``residual_rms_norm`` is ``residual_scale_add`` with
the ``rms_norm`` that follows it, optionally with its output in 8 bits for the next
projection.  ``token_log_probs`` scores given tokens under a row of logits -- drafted
ones for the verification that ``ragged_verify`` and ``commit_states`` carry out, or a
training batch's, with its gradient.  ``need_kernels`` re-exports them.

All take CUDA tensors of one device in fp32, bf16 or f16, sum in fp32 and round their
results once, run on the current stream, allocate their scratch per call and keep nothing
between calls, and can be captured into CUDA graphs.  The calls are compiled
(csrc/lm_autograd.cpp, ``_lib/_lm.so``); there is no other path.  Only
``token_log_probs`` has a gradient: the others refuse inputs that require one.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import abi

_MAX_FEATURES = 128  # NEED_LINEAR_ATTENTION_MAX_DK
_MAX_STEP_FEATURES = 2048
_MAX_NORM_BYTES = 32768
_MAX_TOP = 32  # NEED_TOKEN_LOG_PROBS_MAX_TOP
_GROUPS = (32, 64, 128)
_EXT = None


def _ext():
    """The compiled module (raises if it has not been built)."""
    global _EXT
    if _EXT is None:
        abi.load()  # the library it runs on: present, and of this ABI version
        try:
            from ._lib import _lm
        except ImportError as e:
            raise RuntimeError("need_b200/_lib/_lm.so is missing or does not load: build it with "
                               f"`python -m need_b200.build` ({e})") from e
        _EXT = _lm
    return _EXT


def _no_grad(name: str, *ts: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise NotImplementedError(f"need_b200: {name} has no backward; call it under torch.no_grad() or with tensors "
                                  "that do not require grad")


# --------------------------------------------------------------------------
# linear attention with a decay for each head
# --------------------------------------------------------------------------

def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *, scale: float = 1.0,
                     seg_start: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                     return_final_state: bool = False):
    """``S_t = exp(log_decay_t) S_{t-1} + k_t^T v_t``, ``o_t = scale * q_t S_t`` for each
    of H heads, over whole prompts; returns ``o`` [B, T, H, dv] in q's dtype, with
    ``return_final_state`` also the fp32 state [B, H, dk, dv] after the last token.

    ``q``, ``k`` [B, T, heads, dk] (dk <= 128) and ``v`` [B, T, heads, dv] of one dtype; the
    heads of each divide H, and one is then shared by consecutive heads.  Any strides
    with features next to each other are read in place (chunks of one projection, or
    [B, heads, T, features] transposed); 16-byte aligned rows of whole 16 bytes are
    fastest.  ``log_decay`` [H] or [B, T, H]: natural logarithms, used in fp32; values above
    0 grow the state, -infinity drops it.  ``state`` [B, H, dk, dv]: before the first
    token.  ``seg_start`` [B, T] (bool / uint8): the state before a marked token does not
    reach it, even where it holds an infinity or NaN.

    Precision: products run on bf16 tensor cores, their operands as sums of bf16 values: 2 for
    the scores ``q k^T`` and the entering state under 16-bit results (2^-17 of a value; the
    result's own rounding is 2^-8 in bf16, 2^-11 in f16), 3 for fp32 results and the returned
    state (2^-25).  Without ``return_final_state`` a bf16 call keeps what its states sum to 2^-17
    too, so its ``o`` may differ by a rounding from that of a call with it.  Decays are fp32, and
    0 below 2^-126.  Infinities, NaN, scores past fp32 and log decays over 0.5 are right but slow
    (token by token).  Calls in bf16 of more than 64 tokens run fastest: on tcgen05, if rows are
    whole, aligned 16 bytes and no stride of a dim of more than one is 0 -- heads that share one
    are passed as fewer heads, not expanded."""
    _no_grad("linear_attention", q, k, v, log_decay, state)
    if q.dim() and q.shape[-1] > _MAX_FEATURES:
        raise NotImplementedError(f"linear_attention: at most {_MAX_FEATURES} features a head; got {q.shape[-1]}")
    out, final = _ext().linear_attention(q, k, v, log_decay, scale, seg_start, state, return_final_state)
    return (out, final) if return_final_state else out


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *,
                          scale: float = 1.0, slot: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of :func:`linear_attention` for each of N sequences: returns ``o``
    [N, H, dv], and updates their rows of ``state`` in place.

    ``q``, ``k`` [N, heads, dk], ``v`` [N, heads, dv]; ``log_decay`` [H] or [N, H];
    ``state`` [S, H, dk, dv] fp32, each [H, dk, dv] contiguous.  ``slot`` [N] int32 picks
    rows of the pool (default row i).  A negative slot is a row of the batch without a
    sequence: its output is 0 and nothing is updated.  A slot outside the pool, or one
    that an earlier row of the same call has, gives NaN and updates nothing: a state takes
    one token a call (each block looks through the slots before its own, which thousands of
    rows show: 4096 of 8 heads take 185 us, 158 without ``slot``).  The state is fp32 throughout."""
    _no_grad("linear_attention_step", q, k, v, log_decay, state)
    if q.dim() and q.shape[-1] > _MAX_STEP_FEATURES:
        raise NotImplementedError(f"linear_attention_step: at most {_MAX_STEP_FEATURES} features a head; got {q.shape[-1]}")
    return _ext().linear_attention_step(q, k, v, log_decay, state, scale, slot)


# --------------------------------------------------------------------------
# the residual's addition and the norm
# --------------------------------------------------------------------------

def residual_rms_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, scale: float = 1.0,
                      out_dtype: Optional[torch.dtype] = None, group: Optional[int] = None):
    """``r = x + scale * y`` and its RMSNorm ``n = r / sqrt(mean(r^2) + eps) * weight``
    over the last dim, one pass; returns (r, n), both in x's dtype.  r is rounded once,
    and n is of the rounded r: the stream that goes on.  ``weight`` [C] is used in fp32, and
    the squares are summed in it; rows of up to 32 KB.

    ``out_dtype=torch.float8_e4m3fn`` returns (r, n8, scales): n in 8 bits, one fp32 scale
    -- a power of two, the least that fits the values -- for each ``group`` channels (32,
    64 or 128), or with ``group=None`` one a row; n is ``n8 * scales``, ``scales``
    [..., ceil(C / group)].  A group with an infinity or NaN has the scale NaN."""
    _no_grad("residual_rms_norm", x, y, weight)
    if x.dim() and x.shape[-1] * x.element_size() > _MAX_NORM_BYTES:
        raise NotImplementedError(f"residual_rms_norm takes rows of at most {_MAX_NORM_BYTES} bytes; got {tuple(x.shape)} of "
                                  f"{x.dtype}")
    if out_dtype is torch.float8_e4m3fn:
        if group is not None and group not in _GROUPS:
            raise ValueError(f"group must be None or one of {_GROUPS}; got {group}")
        return _ext().residual_norm(x, y, weight, eps, scale, group or 0)
    if out_dtype is not None and out_dtype is not x.dtype:
        raise ValueError(f"out_dtype must be None, x's dtype or torch.float8_e4m3fn; got {out_dtype}")
    if group is not None:
        raise ValueError("group goes with out_dtype=torch.float8_e4m3fn")
    return _ext().residual_norm(x, y, weight, eps, scale, -1)[:2]


# --------------------------------------------------------------------------
# scores of tokens
# --------------------------------------------------------------------------

class TokenLogProbs(NamedTuple):
    """What :func:`token_log_probs` returns, all but the tokens in fp32."""
    log_prob: torch.Tensor                 # [...]
    entropy: torch.Tensor                  # [...]
    top_log_probs: Optional[torch.Tensor]  # [..., top]
    top_tokens: Optional[torch.Tensor]     # [..., top] int64


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, top: int = 0) -> TokenLogProbs:
    """Of each row of ``p = softmax(logits / temperature)`` [..., V]: the log probability
    of its token (``tokens`` [...], int64 or int32), the entropy, and with ``top`` (at most
    32) the largest log probabilities and their tokens, in order, the lower token first
    where they are equal.  Differentiable in ``logits`` through ``log_prob`` and ``entropy``.

    A logit of -infinity is a token that cannot be: p is 0, and it is no alternative
    (where fewer than ``top`` are left, the rest are -infinity with token -1).  A row of
    nothing else has ``log_prob`` -infinity, entropy 0 and no gradient; one with a NaN or
    +infinity gives NaN (among the alternatives a NaN is the largest).  A negative token:
    none is given, ``log_prob`` is 0.  A token past the vocabulary: NaN."""
    if top > _MAX_TOP:
        raise NotImplementedError(f"token_log_probs: at most {_MAX_TOP} alternatives; got {top}")
    return TokenLogProbs(*_ext().token_log_probs(logits, tokens, temperature, top))
