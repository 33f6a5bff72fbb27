"""Group norm with an activation between the layers of a stack.

Rows are nodes and the last dimension holds the channels, as everywhere in this package.  A sample is a graph: all rows of a
two-dimensional operand, the rows ``ptr[s] .. ptr[s + 1]`` of a batch of graphs of uneven sizes, or the rows of each
entry of a three-dimensional operand; ``x.unsqueeze(1)`` normalises every node by itself.  The reference has a ReLU and
no normalisation between its layers (benchmark/parallel/benchmark_gcn_cpu.py:70-89).
"""
from __future__ import annotations

import functools

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .dense import _call, _ld, _rows

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # CBM_B200_FP32, ...
ACTIVATIONS = {None: 0, "relu": 1, "silu": 2}                      # CBM_B200_ACT_NONE, ...
MAX_CHANNELS = 1 << 22                                             # on the GPU


def rows_like(x: torch.Tensor) -> torch.Tensor:
    """An uninitialised tensor of rows that lie as those of ``x`` do; without gaps where its rows are a window of far wider ones."""
    n, c = x.shape
    pitch = _ld(x)
    if pitch == c or (pitch - c) * x.element_size() >= 128:
        return x.new_empty((n, c))
    return x.new_empty((n, pitch))[:, :c]


def needs_function(*tensors) -> bool:
    """Whether an autograd function has to be applied: a backward pass can follow, or forward-mode differentiation is
    going on, which has to meet (and be refused by) it.  Applying one costs the host 10 us of 25."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def only_once(backward):
    """``once_differentiable``, asked for only where a second derivative might be: its bookkeeping takes the host as long as the launches."""
    guarded = once_differentiable(backward)

    @staticmethod
    def checked(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return checked


@functools.lru_cache(maxsize=256)
def _workspace(n, samples, c, groups, gradient):
    return _lib.lib().cbm_b200_group_norm_workspace(n, samples, c, groups, gradient)


def _data(t):
    return 0 if t is None else t.data_ptr()


def _forward(x, weight, bias, ptr, samples, rows_each, groups, eps, act, wide, keep):
    """The result and, where ``keep`` asks for them, mean and 1 / deviation of every sample's group."""
    n, c = x.shape
    y = rows_like(x)
    stats = None
    if keep and (ptr is not None or rows_each != 1):  # (of single rows the gradient computes them anew)
        stats = torch.empty((2, samples, groups), dtype=torch.float32, device=x.device)
    space = _workspace(n, -samples if ptr is None else samples, c, groups, 0)
    ws = torch.empty(space, dtype=torch.uint8, device=x.device) if space else None
    mean = _data(stats)
    _call("cbm_b200_group_norm", x.get_device(), x.data_ptr(), _ld(x), TYPES[x.dtype], n, c, groups, _data(ptr), samples, rows_each, _data(weight),
          _data(bias), wide, eps, act, y.data_ptr(), _ld(y), mean, mean and mean + 4 * samples * groups, _data(ws), space)
    return y, stats


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, ptr, *sizes):
        y, stats = _forward(x, weight, bias, ptr, *sizes, True)
        ctx.save_for_backward(x, weight, bias, ptr, stats)
        ctx.sizes = sizes
        return y

    @only_once
    def backward(ctx, gy):
        x, weight, bias, ptr, stats = ctx.saved_tensors
        # (a saved-tensor hook may hand them back in another layout)
        x, gy = _rows(x), _rows(gy)
        weight, bias, ptr, stats = (None if t is None else t.contiguous() for t in (weight, bias, ptr, stats))
        samples, rows_each, groups, eps, act, wide = ctx.sizes
        n, c = x.shape
        gx = rows_like(x)
        _, want_w, want_b, *_ = ctx.needs_input_grad
        gw = torch.empty(c, dtype=torch.float32, device=x.device) if want_w else None
        gb = torch.empty(c, dtype=torch.float32, device=x.device) if want_b else None
        space = _workspace(n, -samples if ptr is None else samples, c, groups, 1)
        ws = torch.empty(space, dtype=torch.uint8, device=x.device) if space else None
        mean = _data(stats)
        _call("cbm_b200_group_norm_grad", x.get_device(), x.data_ptr(), _ld(x), gy.data_ptr(), _ld(gy), TYPES[x.dtype], n, c, groups, _data(ptr),
              samples, rows_each, _data(weight), _data(bias), wide, eps, act, mean, mean and mean + 4 * samples * groups, gx.data_ptr(), _ld(gx),
              _data(gw), _data(gb), _data(ws), space)
        if gw is not None and not wide:
            gw = gw.to(weight.dtype)
        if gb is not None and not wide:
            gb = gb.to(bias.dtype)
        return gx, gw, gb, None, None, None, None, None, None, None


def _on_host(x, weight, bias, ptr, samples, rows_each, groups, eps, act):
    """The same by torch's elementary operations, for CPU tensors; a sample's rows are added up in 64 bits."""
    n, c = x.shape
    v = x.float()
    if ptr is None:
        row = torch.arange(n) // max(rows_each, 1)
    else:
        row = torch.bucketize(torch.arange(n), ptr[1:].contiguous(), right=True)
        row = torch.where((row >= samples) | (torch.arange(n) < (ptr[0] if samples else 0)), samples, row)
        v = torch.where((row < samples)[:, None], v, 0.0)  # (whatever rows of no sample hold does not come into sums of gradients)
    size = (torch.bincount(row, minlength=samples + 1) * (c // groups)).clamp_min(1)[:, None]

    def mean(t):
        of_row = t.reshape(n, groups, c // groups).sum(2, dtype=torch.float64)
        of_sample = of_row.new_zeros((samples + 1, groups)).index_add(0, row, of_row) / size
        return of_sample[row].float().repeat_interleave(c // groups, dim=1)

    d = v - mean(v)
    z = d * torch.rsqrt(mean(d * d) + eps)
    z = z if weight is None else z * weight.float()
    z = z if bias is None else z + bias.float()
    y = z.relu() if act == 1 else torch.nn.functional.silu(z) if act == 2 else z
    return torch.where((row < samples)[:, None], y, 0.0).to(x.dtype)


def group_norm(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               ptr: torch.Tensor | None = None, eps: float = 1e-5, activation: str | None = None) -> torch.Tensor:
    """``act(weight * (x - mean) / sqrt(var + eps) + bias)`` with mean and variance of each sample's ``groups`` equal ranges of
    channels (on the GPU up to 2^22 channels).  ``x``: [N, C], one sample or, with ``ptr``, the samples
    ``ptr[s] .. ptr[s + 1]``; or [B, n, C], B samples.
    fp32, bf16 or fp16; ``weight`` and ``bias`` [C] of that type or fp32; ``activation`` None, "relu" or "silu".

    ``ptr`` (int64 or int32, rising, on x's device; its values are not looked at on the host) may leave samples
    empty; rows before its first and behind its last entry belong to no sample: 0, and no gradient.  Differentiable once in
    ``x``, ``weight`` and ``bias``; statistics and sums are kept in fp32.
    """
    shape, device = x.shape, x.device
    if len(shape) != 2 and (len(shape) != 3 or ptr is not None):
        raise RuntimeError(f"group norm: [N, C] or [B, n, C] expected, [N, C] with ptr, not {tuple(shape)}")
    c = shape[-1]
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"group norm: {c} channels do not make {groups} groups")
    if x.dtype not in TYPES:
        raise RuntimeError(f"group norm: fp32, bf16 or fp16 expected, not {x.dtype}")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    wide = 1
    for t in (weight, bias):
        if t is None:
            continue
        if t.shape != (c,) or t.device != device:
            raise RuntimeError(f"group norm: shape mismatch, parameters of {tuple(t.shape)} on {t.device} for {c} channels on {device}")
        if t.dtype is not torch.float32:
            if t.dtype is not x.dtype:
                raise RuntimeError(f"group norm: parameters of x's type or fp32 expected, not {t.dtype}")
            wide = 0
    if not wide and weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise RuntimeError("group norm: weight and bias of one type expected")
    if ptr is not None:
        if ptr.dim() != 1 or ptr.numel() < 1 or ptr.dtype not in (torch.int64, torch.int32) or ptr.device != device:
            raise RuntimeError(f"group norm: ptr must be a vector of int64 or int32 on {device}")
        samples, rows_each, rows = ptr.numel() - 1, 0, x
        ptr = ptr.to(torch.int64).contiguous()
    elif len(shape) == 3:
        samples, rows_each = shape[0], shape[1]
        rows = x.reshape(-1, c)  # (a view where the entries' rows follow one another at one pitch)
    else:
        samples, rows_each, rows = 1, shape[0], x
    if not x.is_cuda:
        return _on_host(rows, weight, bias, ptr, samples, rows_each, groups, eps, act).view(shape)
    if c > MAX_CHANNELS:  # (asked here: the library's sizes have 32 bits)
        raise RuntimeError(f"group norm: bad sizes, {c} channels, at most {MAX_CHANNELS} on the GPU")
    rows = _rows(rows)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    sizes = (samples, rows_each, groups, float(eps), act, wide)
    if needs_function(rows, weight, bias):
        y = _GroupNorm.apply(rows, weight, bias, ptr, *sizes)
    else:
        y = _forward(rows, weight, bias, ptr, *sizes, False)[0]
    return y if len(shape) == 2 else y.view(shape)


class GroupNorm(nn.Module):
    """``group_norm`` with weight (ones) and bias (zeros) of its own."""

    def __init__(self, groups: int, channels: int, eps: float = 1e-5, activation: str | None = None):
        super().__init__()
        if groups < 1 or channels % groups:
            raise ValueError(f"group norm: {channels} channels do not make {groups} groups")
        self.groups, self.channels, self.eps, self.activation = groups, channels, eps, activation
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels))

    def forward(self, x, ptr=None):
        return group_norm(x, self.groups, self.weight, self.bias, ptr, self.eps, self.activation)

    def extra_repr(self):
        return f"{self.groups}, {self.channels}, eps={self.eps}, activation={self.activation!r}"
