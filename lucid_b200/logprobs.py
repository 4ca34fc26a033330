"""Log probabilities of given tokens, entropy and the most likely alternatives of rows of
logits, from one pass over them, with the gradient of the first two."""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib
from .paged import _on, _raw_stream

__all__ = ["token_logprobs", "TokenLogprobs", "MAX_TOP"]

MAX_TOP = 64
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class TokenLogprobs(NamedTuple):
    """Per row of logits: fp32 ``logprobs`` of the given tokens (None without tokens) and
    ``entropy``, fp32 ``top_logprobs`` and int64 ``top_tokens`` [..., top]."""
    logprobs: torch.Tensor | None
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def _row_view(logits: torch.Tensor):
    """(logits, R0, R1, s0, s1): the rows as two strided dimensions, without a copy where
    the leading dimensions merge into two."""
    if logits.numel() == 0:               # contiguous() leaves the strides of an empty tensor alone
        return logits, 0, 0, 0, 0
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    dims = []
    for n, s in zip(logits.shape[:-1], logits.stride()[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s:
            dims[-1] = (dims[-1][0] * n, s)
        else:
            dims.append((n, s))
    if len(dims) > 2:
        return _row_view(logits.contiguous())
    (r0, s0), (r1, s1) = [(1, 0)] * (2 - len(dims)) + dims
    return logits, r0, r1, s0, s1


def _forward(logits, tokens, top, keep):
    """The outputs, and with ``keep`` the rows' statistics for the backward."""
    lib = _lib._lib or _lib.load()
    index, lead = logits.get_device(), logits.shape[:-1]
    view, r0, r1, s0, s1 = _row_view(logits)
    entropy = logits.new_empty(lead, dtype=torch.float32)
    logprobs = torch.empty_like(entropy) if tokens is not None else None
    stats = entropy.new_empty((*lead, 3)) if keep else None
    top_lp = entropy.new_empty((*lead, top))
    top_tok = logits.new_empty((*lead, top), dtype=torch.int64)
    with _on(index):
        rc = lib.lucid_token_logprobs(
            r0, r1, logits.shape[-1], _DTYPES[logits.dtype], view.data_ptr(), s0, s1,
            None if tokens is None else tokens.data_ptr(), top, None if tokens is None else logprobs.data_ptr(),
            entropy.data_ptr(), stats.data_ptr() if keep else None, top_lp.data_ptr(), top_tok.data_ptr(),
            _lib.STATUS.device_word(index), _raw_stream(index))
    _lib.check(rc, "lucid_token_logprobs")
    _lib.STATUS.settle()
    return logprobs, entropy, top_lp, top_tok, stats


class TokenLogprobsFunction(torch.autograd.Function):
    """logprobs and entropy with the gradient of the logits.  The alternatives carry none:
    they go into the list ``beside`` and stay out of the graph."""

    @staticmethod
    def forward(ctx, logits, tokens, top: int, beside: list):
        logprobs, entropy, top_lp, top_tok, ctx.stats = _forward(logits, tokens, top, True)
        ctx.save_for_backward(logits, tokens)
        ctx.set_materialize_grads(False)
        beside += (top_lp, top_tok)
        return logprobs, entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprobs, g_entropy):
        if g_logprobs is None and g_entropy is None:
            return None, None, None, None
        lib = _lib._lib or _lib.load()
        logits, tokens = ctx.saved_tensors
        index = logits.get_device()
        view, r0, r1, s0, s1 = _row_view(logits)
        gl, ge = (None if g is None else g.float().contiguous() for g in (g_logprobs, g_entropy))
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with _on(index):
            rc = lib.lucid_token_logprobs_bwd(
                r0, r1, logits.shape[-1], _DTYPES[logits.dtype], view.data_ptr(), s0, s1,
                None if tokens is None else tokens.data_ptr(), ctx.stats.data_ptr(),
                None if gl is None else gl.data_ptr(), None if ge is None else ge.data_ptr(), dlogits.data_ptr(),
                _raw_stream(index))
        _lib.check(rc, "lucid_token_logprobs_bwd")
        return dlogits, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None, top: int = 0) -> TokenLogprobs:
    """log softmax(logits)[tokens], the entropy -sum p log p, and the ``top`` most likely
    tokens (at most 64; likeliest first, ties to the lowest index) of each row.

    logits [..., V] bf16, fp16 or fp32 on CUDA, V at most 2^30 (any row strides: a view such
    as logits[:, :-1] is read in place); tokens [...] integers in [0, V), or -100 for rows
    without one (log probability 0, no gradient through it), or None.  Entries of -inf
    have probability 0; a row without a distribution (all -inf, a NaN or +inf in it)
    gives NaN and top tokens -1.  A token outside the vocabulary is reported by the next
    call or ``check_status()``.  Differentiable once in logits through ``logprobs`` and
    ``entropy``, in reverse mode; the arithmetic is fp32, the gradient has the logits' type.
    To capture the backward into a CUDA graph use torch.autograd.grad: ``backward()`` on a
    leaf that an eager graph also holds makes torch wait for another stream, which a capture
    cannot."""
    if unpack_dual(logits).tangent is not None:
        raise NotImplementedError("token_logprobs: no forward mode, only the gradient of logprobs and entropy")
    if not logits.is_cuda:
        raise RuntimeError("logits: LUCID B200 kernels need CUDA tensors (no CPU fallback)")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits: expected bfloat16, float16 or float32, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits: expected [..., V], got shape {tuple(logits.shape)}")
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"top: expected 0 to {min(MAX_TOP, logits.shape[-1])}, got {top}")
    if tokens is not None:
        if tokens.device != logits.device or tokens.shape != logits.shape[:-1]:
            raise ValueError(f"tokens {tuple(tokens.shape)} on {tokens.device} must match the rows of logits "
                             f"{tuple(logits.shape)} on {logits.device}")
        if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
            raise TypeError(f"tokens: expected integers, got {tokens.dtype}")
        if tokens.dtype != torch.int64 or not tokens.is_contiguous():
            tokens = tokens.to(torch.int64).contiguous()
    _lib.STATUS.poll()
    if torch.is_grad_enabled() and logits.requires_grad:
        beside: list = []
        logprobs, entropy = TokenLogprobsFunction.apply(logits, tokens, top, beside)
        return TokenLogprobs(logprobs, entropy, *beside)
    return TokenLogprobs(*_forward(logits, tokens, top, False)[:4])
