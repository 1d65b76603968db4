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
from torch.autograd.function import once_differentiable

from . import _native as N


class TargetLogprobs(NamedTuple):
    logprobs: torch.Tensor      # targets' shape, fp32
    entropy: torch.Tensor       # [...] fp32
    lse: torch.Tensor           # [...] fp32: log sum exp(logits / tau) over the candidates
    top_ids: torch.Tensor       # [..., topk] int64, -1 padded
    top_logprobs: torch.Tensor  # [..., topk] fp32, -inf padded


def _rows(t: torch.Tensor, width: int, zero_ok: bool):
    """(t as rows of unit column stride, their common stride in elements); copied only where the
    leading dimensions have no common stride."""
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if zero_ok and t.numel() and all(st == 0 or n == 1 for st, n in zip(t.stride()[:-1], t.shape[:-1])) \
            and (t.stride(-1) == 1 or width == 1):
        return t, 0
    if t.stride(-1) == 1 or width == 1:
        try:
            v = t.view(-1, width)
            return v, v.stride(0) if v.shape[0] > 1 else width
        except RuntimeError:
            pass
    t = t.contiguous()
    return t.view(-1, width), width


class _TargetLogprobs(torch.autograd.Function):
    """Flat form: logits [..., V], targets [N, S] int64, mask [..., V] uint8 or None."""

    @staticmethod
    def forward(ctx, logits, targets, mask, tau: float, topk: int):
        lib = N.load()
        dev, width = logits.device, int(logits.shape[-1])
        x, stride = _rows(logits.detach(), width, False)
        rows, s = int(targets.shape[0]), int(targets.shape[1])
        m, m_stride = (None, 0) if mask is None else _rows(mask, width, True)
        if stride < 0 or m_stride < 0:
            raise ValueError("target_logprobs: negative strides")
        p = N.LogprobParams(rows, width, stride, m_stride, s, topk, tau, N.DTYPES[x.dtype], 0)
        f32 = dict(dtype=torch.float32, device=dev)
        logprobs, top_logprobs = torch.empty((rows, s), **f32), torch.empty((rows, topk), **f32)
        entropy, lse, stats = torch.empty(rows, **f32), torch.empty(rows, **f32), torch.empty((rows, 2), **f32)
        top_ids = torch.empty((rows, topk), dtype=torch.int64, device=dev)
        with torch.cuda.device(dev):
            ws = N.workspace(lib.mkg_logprob_workspace_bytes(p), dev)
            N.check(lib.mkg_logprob_forward(p, x.data_ptr(), N.ptr(m), targets.data_ptr(), logprobs.data_ptr(),
                                            entropy.data_ptr(), lse.data_ptr(), top_ids.data_ptr(),
                                            top_logprobs.data_ptr(), stats.data_ptr(), ws.data_ptr(), ws.numel(),
                                            N.error_word(dev).data_ptr(), N.stream_handle(dev)), "logprob_forward")
        ctx.p = p
        ctx.save_for_backward(logits, targets, mask, top_ids, entropy, stats)
        ctx.mark_non_differentiable(top_ids)
        ctx.set_materialize_grads(False)
        return logprobs, entropy, lse, top_ids, top_logprobs

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprobs, g_entropy, g_lse, _g_ids, g_top):
        logits, targets, mask, top_ids, entropy, stats = ctx.saved_tensors
        dev, p = logits.device, ctx.p
        x, _ = _rows(logits.detach(), int(p.width), False)
        m = None if mask is None else _rows(mask, int(p.width), True)[0]
        ups = [None if g is None else g.to(torch.float32).contiguous() for g in (g_logprobs, g_entropy, g_lse, g_top)]
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        with torch.cuda.device(dev):
            N.check(N.load().mkg_logprob_backward(p, x.data_ptr(), N.ptr(m), targets.data_ptr(), top_ids.data_ptr(),
                                                  entropy.data_ptr(), stats.data_ptr(), *(N.ptr(g) for g in ups),
                                                  grad.data_ptr(), N.stream_handle(dev)), "logprob_backward")
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
    and sets the device error word (``_native.raise_device_errors``).
    """
    if logits.dtype not in N.DTYPES:
        raise TypeError(f"target_logprobs: logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"target_logprobs: targets must be int64 or int32, got {targets.dtype}")
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
    tau = float(tau)
    if not (tau > 0.0 and math.isfinite(tau)):
        raise ValueError(f"target_logprobs: tau must be positive and finite, got {tau}")
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
    rows = math.prod(lead)
    t = targets.reshape(rows, s).to(torch.int64).contiguous()
    m = None if mask is None else mask.view(torch.uint8)
    lp, h, lse, ids, top = _TargetLogprobs.apply(logits, t, m, tau, int(topk))
    k = (int(topk),)
    return TargetLogprobs(lp.view(targets.shape), h.view(lead), lse.view(lead), ids.view(lead + k), top.view(lead + k))
