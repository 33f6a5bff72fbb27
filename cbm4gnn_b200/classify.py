"""What the logits of a stack are turned into: class log probabilities, their entropy and the most probable classes.

``class_log_probs(logits, labels, top)`` gives for every row the log probability of its label, the entropy of the row's
distribution and the ``top`` most probable classes with their log probabilities, from one pass over the logits, and is
differentiable in them.  The reference stops at the logits (benchmark/parallel/benchmark_gcn_cpu.py:92-103 sums them).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .dense import _call, _ld, _rows
from .norm import TYPES, _data, needs_function, only_once, rows_like

MAX_TOP = 32           # include/cbm_b200.h, CBM_B200_MAX_TOP
MAX_CLASSES = 1 << 30  # on the GPU


class ClassLogProbs(NamedTuple):
    log_prob: torch.Tensor        # [N] fp32: of each row's label, 0 where the label is negative
    entropy: torch.Tensor         # [N] fp32
    top_log_probs: torch.Tensor   # [N, top] fp32, falling
    top_classes: torch.Tensor     # [N, top] int64; of equal logits the lower class comes first


def _forward(x, labels, top, keep):
    n, c = x.shape
    log_prob = torch.empty(n, dtype=torch.float32, device=x.device)
    entropy = torch.empty_like(log_prob)
    stats = torch.empty((n, 2), dtype=torch.float32, device=x.device) if keep else None
    best = torch.empty((n, top), dtype=torch.float32, device=x.device)
    classes = torch.empty((n, top), dtype=torch.int64, device=x.device)
    _call("cbm_b200_class_log_probs", x.get_device(), x.data_ptr(), _ld(x), TYPES[x.dtype], labels.data_ptr(), labels.dtype is torch.int64, n, c, top,
          log_prob.data_ptr(), entropy.data_ptr(), _data(stats), best.data_ptr(), classes.data_ptr())
    return log_prob, entropy, best, classes, stats


class _ClassLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, labels, top):
        log_prob, entropy, best, classes, stats = _forward(x, labels, top, True)
        ctx.save_for_backward(x, labels, stats, entropy, classes)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(classes)
        return log_prob, entropy, best, classes

    @only_once
    def backward(ctx, *grads):
        x, *kept = ctx.saved_tensors
        # (a saved-tensor hook may hand them back in another layout)
        x = _rows(x)
        labels, stats, entropy, classes = (t.contiguous() for t in kept)
        g_log, g_entropy, g_top = (None if g is None else g.contiguous() for g in grads[:3])
        n, c = x.shape
        gx = rows_like(x)
        _call("cbm_b200_class_log_probs_grad", x.get_device(), x.data_ptr(), _ld(x), TYPES[x.dtype], labels.data_ptr(), labels.dtype is torch.int64, n, c,
              classes.size(1), stats.data_ptr(), entropy.data_ptr(), classes.data_ptr(), _data(g_log), _data(g_entropy), _data(g_top), gx.data_ptr(),
              _ld(gx))
        return gx, None, None


def _on_host(logits, labels, top):
    """The same by torch's elementary operations, for CPU tensors."""
    x = logits.float()
    c = x.size(1)
    m = x.detach().max(dim=1, keepdim=True).values
    closed = m == -torch.inf
    d = torch.where(closed, 0.0, x) - torch.where(closed, 0.0, m)
    lp = d - torch.exp(d).sum(1, keepdim=True).log()
    p = torch.exp(lp)
    entropy = torch.where(closed[:, 0], 0.0, -(p * torch.where(p > 0, lp, 0.0)).sum(1))
    lp = torch.where(closed, -torch.inf, lp)
    known = labels >= 0
    log_prob = torch.where(known, lp.gather(1, labels.long().clamp(0, c - 1)[:, None])[:, 0], 0.0)
    log_prob = torch.where(labels >= c, torch.nan, log_prob)
    best = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :top]
    return ClassLogProbs(log_prob, entropy, lp.gather(1, best), best)


def class_log_probs(logits: torch.Tensor, labels: torch.Tensor, top: int = 0) -> ClassLogProbs:
    """For every row of ``logits`` [N, C] (fp32, bf16 or fp16; rows at any pitch): the log probability of its class
    ``labels`` [N] (int64 or int32), the entropy of the row and its ``top`` most probable classes (0 to 32).  On the GPU up to
    2^31 - 1 rows and 2^30 classes; rows of more than 1 024 classes up to 2^31 - 1 stretches of 4 096.

    A negative label stands for none: log probability 0, no gradient.  One of C or more gives NaN.  A logit of -inf closes a
    class; a row without an open class has log probabilities -inf, entropy 0 and no gradient.  A row with NaN or +inf is
    NaN throughout, and its gradient is, with a label or without.  Differentiable once in ``logits``, through all three results.
    """
    shape = logits.shape
    if len(shape) != 2 or shape[1] < 1 or labels.shape != shape[:1]:
        raise RuntimeError(f"class log probabilities: shape mismatch, logits of {tuple(shape)} and labels of {tuple(labels.shape)}")
    if logits.dtype not in TYPES:
        raise RuntimeError(f"class log probabilities: fp32, bf16 or fp16 logits expected, not {logits.dtype}")
    if labels.dtype is not torch.int64 and labels.dtype is not torch.int32:
        raise RuntimeError(f"class log probabilities: int64 or int32 labels expected, not {labels.dtype}")
    if labels.device != logits.device:
        raise RuntimeError(f"class log probabilities: logits on {logits.device} and labels on {labels.device}")
    if not 0 <= top <= min(MAX_TOP, shape[1]):
        raise ValueError(f"top must be between 0 and {min(MAX_TOP, shape[1])}")
    if not logits.is_cuda:
        return _on_host(logits, labels, top)
    if shape[1] > MAX_CLASSES:  # (asked here: the library's sizes have 32 bits)
        raise RuntimeError(f"class log probabilities: {shape[1]} classes, at most {MAX_CLASSES} on the GPU")
    x, labels = _rows(logits), labels.contiguous()
    if needs_function(x):
        return ClassLogProbs(*_ClassLogProbs.apply(x, labels, int(top)))
    return ClassLogProbs(*_forward(x, labels, int(top), False)[:4])
