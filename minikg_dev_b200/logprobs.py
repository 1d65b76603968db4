"""Log probabilities of given columns in rows of logits, with entropy and top alternatives.

``target_logprobs`` is what a rule model is trained on and read with: rows of logits over the
channels (``rules.build_rule_logits``) or over the entities, a softmax at temperature ``tau`` over
each row's candidates, and of it the log probability of the given columns, the entropy, the log of
the normaliser and the ``topk`` best columns.  Forward and backward run in the library
(``mkg_logprob_forward`` / ``mkg_logprob_backward``): one pass over the logits each, no softmax
in memory.  Gradients flow to the logits through every floating output.

``rules.rule_logprobs`` applies it to the rules of a query, ``decode.tail_logprobs`` to a query's
answers.  The product path has no CPU implementation.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N


class TargetLogprobs(NamedTuple):
    logprobs: torch.Tensor      # targets' shape, fp32
    entropy: torch.Tensor       # [...] fp32
    lse: torch.Tensor           # [...] fp32: log sum exp(logits / tau) over the candidates
    top_ids: torch.Tensor       # [..., topk] int64, -1 padded
    top_logprobs: torch.Tensor  # [..., topk] fp32, -inf padded


def _row_stride(t: torch.Tensor) -> int | None:
    """Elements from one row of ``t`` [..., V] to the next; None where the rows have no common stride or
    no unit column stride.  0 where there is one row, or one row stands for all."""
    shape, strides = t.shape, t.stride()
    if strides[-1] != 1 and shape[-1] != 1:
        return None
    step, rows = 0, 1
    for n, st in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if rows == 1:
            step = st
        elif st != step * rows:
            return None
        rows *= n
    return step


def _as_rows(t: torch.Tensor | None):
    """(t, row stride) of a tensor the library can read, copied only where it cannot be read as it is."""
    if t is None:
        return None, 0
    if t.is_neg():  # lazily negated: memory holds the opposite
        t = t.resolve_neg()
    stride = _row_stride(t)
    if stride is None:
        t = t.contiguous()
        stride = _row_stride(t)
    return t, stride


def _forward(logits, targets, mask, tau: float, topk: int, stats):
    """(parameters, logprobs, entropy, lse, top_ids, top_logprobs); targets int64, contiguous; ``stats``
    (fp32 [..., 2] or None) receives what the backward needs."""
    lib, dev, lead = N.load(), logits.device, logits.shape[:-1]
    x, stride = _as_rows(logits)
    m, m_stride = _as_rows(mask)
    p = N.LogprobParams(math.prod(lead), logits.shape[-1], stride, m_stride,
                        targets.shape[-1] if targets.dim() > len(lead) else 1, topk, tau, N.DTYPES[logits.dtype], 0)
    logprobs = torch.empty_like(targets, dtype=torch.float32)
    entropy, lse = (torch.empty(lead, dtype=torch.float32, device=dev) for _ in range(2))
    top_logprobs = torch.empty((*lead, topk), dtype=torch.float32, device=dev)
    top_ids = torch.empty((*lead, topk), dtype=torch.int64, device=dev)
    with N.on_device(dev):
        need = lib.mkg_logprob_workspace_bytes(p)
        ws = N.workspace(need, dev) if need else None
        N.check(lib.mkg_logprob_forward(p, x.data_ptr(), N.ptr(m), targets.data_ptr(), logprobs.data_ptr(),
                                        entropy.data_ptr(), lse.data_ptr(), top_ids.data_ptr(),
                                        top_logprobs.data_ptr(), N.ptr(stats), N.ptr(ws), need,
                                        N.error_word(dev).data_ptr(), N.stream_handle(dev)), "logprob_forward")
    return p, logprobs, entropy, lse, top_ids, top_logprobs


def _as_saved(p, device: int, logits, targets, mask, top_ids, entropy, stats) -> bool:
    """Whether these are of the sizes, types and device that a backward with these parameters reads."""
    rows, width = p.rows, p.width
    if logits.shape[-1:] != (width,) or N.DTYPES.get(logits.dtype) != p.dtype:
        return False
    if mask is not None and (mask.shape[-1:] != (width,) or mask.numel() not in (rows * width, width)
                             or mask.dtype is not torch.uint8 or mask.get_device() != device):
        return False
    for t, n, dtype in ((logits, rows * width, logits.dtype), (targets, rows * p.targets, torch.int64),
                        (top_ids, rows * p.topk, torch.int64), (entropy, rows, torch.float32),
                        (stats, 2 * rows, torch.float32)):
        if t.numel() != n or t.dtype is not dtype or t.get_device() != device:
            return False
    return True


class _TargetLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, tau: float, topk: int):
        stats = torch.empty((*logits.shape[:-1], 2), dtype=torch.float32, device=logits.device)
        p, logprobs, entropy, lse, top_ids, top_logprobs = _forward(logits, targets, mask, tau, topk, stats)
        ctx.save_for_backward(logits, targets, mask, top_ids, entropy, stats)
        ctx.call = p, logits.get_device()
        ctx.mark_non_differentiable(top_ids)
        ctx.set_materialize_grads(False)
        return logprobs, entropy, lse, top_ids, top_logprobs

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprobs, g_entropy, g_lse, _g_ids, g_top):
        p, device = ctx.call
        logits, targets, mask, top_ids, entropy, stats = saved = ctx.saved_tensors
        # hooks on saved tensors (checkpointing, offloading) may hand back copies, with other strides
        if not _as_saved(p, device, *saved):
            raise RuntimeError("target_logprobs: a saved tensor came back with another shape, type or device")
        x, stride = _as_rows(logits)
        m, m_stride = _as_rows(mask)
        if stride != p.row_stride or m_stride != p.mask_row_stride:
            p = N.LogprobParams.from_buffer_copy(p)
            p.row_stride, p.mask_row_stride = stride, m_stride
        dev = logits.device
        targets, top_ids, entropy, stats = (t.contiguous() for t in (targets, top_ids, entropy, stats))
        ups = [g if g is None else g.resolve_neg().contiguous() if g.is_neg() else g.contiguous()
               for g in (g_logprobs, g_entropy, g_lse, g_top)]
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        with N.on_device(dev):
            N.check(N.load().mkg_logprob_backward(p, x.data_ptr(), N.ptr(m), targets.data_ptr(),
                                                  top_ids.data_ptr(), entropy.data_ptr(), stats.data_ptr(),
                                                  *map(N.ptr, ups), grad.data_ptr(), N.stream_handle(dev)),
                    "logprob_backward")
        return grad, None, None, None, None


def target_logprobs(logits: torch.Tensor, targets: torch.Tensor, tau: float = 1.0,
                    mask: torch.Tensor | None = None, topk: int = 0) -> TargetLogprobs:
    """Log probabilities of ``targets`` under ``softmax(logits / tau)`` over each row's candidates.

    ``logits [..., V]`` float32, bfloat16 or float16 (V up to 2^30); ``targets [...]`` or
    ``[..., S]`` int64 / int32 columns (S up to 1024; -1 is padding: log probability 0, no gradient);
    ``mask [..., V]`` or ``[V]`` bool, True = candidate; ``topk`` up to 32.  Statistics are fp32,
    logits are never copied where their rows have one stride and unit column stride.

    A target that is no candidate has log probability -inf.  A row without a candidate above -inf
    has ``lse`` -inf, entropy 0, every log probability -inf and gradient 0.  A row with NaN or +inf
    among its candidates is NaN throughout, with no alternatives.  Alternatives are ordered by logit,
    ties to the lowest column; candidates at -inf are not listed.  A target outside [-1, V) gets NaN
    and sets the device error word (``_native.raise_device_errors``).  Logits with a forward-mode tangent
    are refused: the derivative is reverse-mode, once, and of the logits alone (``tau`` is a number).
    """
    if logits.dtype not in N.DTYPES:
        raise TypeError(f"target_logprobs: logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"target_logprobs: targets must be int64 or int32, got {targets.dtype}")
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise NotImplementedError("target_logprobs: no forward-mode derivative")
    if logits.dim() < 1 or logits.shape[-1] < 1 or logits.shape[-1] > 1 << 30:
        raise ValueError(f"target_logprobs: logits must be [..., V] with 1 <= V <= 2^30, got {tuple(logits.shape)}")
    lead = tuple(logits.shape[:-1])
    if tuple(targets.shape[:len(lead)]) != lead or targets.dim() - len(lead) not in (0, 1):
        raise ValueError(f"target_logprobs: targets must be {lead} or {lead + ('S',)}, got {tuple(targets.shape)}")
    s = int(targets.shape[-1]) if targets.dim() > len(lead) else 1
    if s > N.LOGPROB_TARGETS_MAX:
        raise ValueError(f"target_logprobs: at most {N.LOGPROB_TARGETS_MAX} targets per row, got {s}")
    if not 0 <= int(topk) <= N.LOGPROB_TOPK_MAX:
        raise ValueError(f"target_logprobs: topk must be in [0, {N.LOGPROB_TOPK_MAX}], got {topk}")
    if isinstance(tau, torch.Tensor) and ((tau.requires_grad and torch.is_grad_enabled())
                                          or forward_ad.unpack_dual(tau).tangent is not None):
        raise NotImplementedError("target_logprobs: tau is a number and has no derivative")
    tau = float(tau)
    if not 2.0 ** -60 <= tau <= 2.0 ** 60:
        raise ValueError(f"target_logprobs: tau must be in [2^-60, 2^60], got {tau}")
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError(f"target_logprobs: mask must be bool, got {mask.dtype}")
        if tuple(mask.shape) not in (tuple(logits.shape), tuple(logits.shape[-1:])):
            raise ValueError(f"target_logprobs: mask must be {tuple(logits.shape)} or {tuple(logits.shape[-1:])}, "
                             f"got {tuple(mask.shape)}")
    for t, what in ((logits, "logits"), (targets, "targets"), (mask, "mask")):
        if t is not None:
            N.require_cuda(t, what)
            if t.device != logits.device:
                raise ValueError(f"target_logprobs: {what} on {t.device}, logits on {logits.device}")
    t = targets.to(torch.int64).contiguous()
    m = None if mask is None else mask.view(torch.uint8)
    if logits.requires_grad and torch.is_grad_enabled():
        return TargetLogprobs(*_TargetLogprobs.apply(logits, t, m, tau, int(topk)))
    return TargetLogprobs(*_forward(logits, t, m, tau, int(topk), None)[1:])
