"""The batch-independent normaliser and the regulariser of the decoder's activations, next to ``batch_norm_elu``:

    group_norm_act    group norm (channels last), an activation and, if asked for, a dropout mask, in the same passes
    dropout           the mask alone
    DropoutMask       which mask: a function of (seed, step, layer, item, place), never stored (csrc/norm_drop.h)

Both are differentiable (torch.autograd; once), take fp32, bf16 and fp16 activations with fp32 parameters, compute in fp32 and
round a 16-bit result once.  Like the rest of the package they have no CPU path.  Group norm takes its statistics from one item:
it is the same function for any batch size, in training and in serving, and needs no collective under data parallelism.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import call, ptr, stream_of
from .aspp import BN_EPSILON, _grad_out
from .utils import _check, _same_device

Tensor = torch.Tensor
GN_EPSILON = BN_EPSILON
ACTIVATIONS = {None: 0, "none": 0, "elu": 1, "relu": 2, "silu": 3}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HERE = contextlib.nullcontext()


def _on(device):
    """the device of the tensors as the current one (entering a device context costs more than asking)"""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _check_activation(x, name: str) -> int:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(x).__name__}")
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    if not x.is_cuda:
        raise TypeError(f"{name} is on {x.device}; sfm_amd runs on ROCm devices only (no CPU fallback)")
    if x.dim() < 2:
        raise ValueError(f"{name} must be [B, ..., C] with at least two dimensions, got shape {tuple(x.shape)}")
    return dt


def _rows(x: Tensor) -> Tuple[Tensor, int]:
    """x [B, ..., C] as rows of C channels ld elements apart: itself if it is dense or a channel slice of a dense buffer, else a copy"""
    if x.is_contiguous():
        return x, x.shape[-1]
    shape, stride = x.shape, x.stride()
    if shape[-1] == 1 or stride[-1] == 1:
        ld, want = None, None
        for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
            if n == 1:
                continue
            if ld is None:
                ld = want = s
            elif s != want:
                break
            want *= n
        else:
            if ld is None:
                return x, shape[-1]
            if ld >= shape[-1]:
                return x, ld
    return x.contiguous(), shape[-1]


def _refuse_second_order(name: str) -> None:
    if torch.is_grad_enabled():  # a backward runs with gradients on under create_graph=True alone: what it returns would lack its history
        raise RuntimeError(f"{name} is differentiable once: its backward was called with create_graph=True")


class DropoutMask:
    """Which elements are dropped: a function of counters, evaluated wherever it is needed and never stored.

    ``p``: the probability of being dropped, 0 <= p < 1, taken to the nearest of the 65536ths (``mask.probability``); what is kept is
    multiplied by 1 / (1 - that).  ``rng``: ``(seed, step)``, as two Python ints or as a device tensor int64 [2] that the kernels read
    when they run - a captured graph follows the tensor, while ints are frozen into it.  Of ``step`` the low 32 bits count.  Advance
    the step when a step's backward is done: a backward that finds the tensor changed since its forward raises, as for any
    saved tensor.  ``layer``: 0 <= layer < 2^32, another one for each place that draws in a step.  ``per_channel``: whole channels
    of an item are dropped.  ``first_item``: the index of this call's first item in the global batch: ranks that hold shards of
    one batch then draw what one device would have drawn."""

    __slots__ = ("threshold", "rng", "seed", "step", "layer", "per_channel", "first_item")

    def __init__(self, p: float, rng: Union[Tensor, Tuple[int, int]], layer: int = 0, per_channel: bool = False, first_item: int = 0):
        if not 0.0 <= float(p) < 1.0:
            raise ValueError(f"p must be in [0, 1), got {p}")
        self.threshold = int(round(float(p) * 65536))
        if self.threshold > 65535:
            raise ValueError(f"p = {p} rounds to 1: everything would be dropped")
        if isinstance(rng, torch.Tensor):
            if rng.dtype != torch.int64 or tuple(rng.shape) != (2,):
                raise TypeError(f"rng must be an int64 tensor [2] (seed, step), got {rng.dtype} {tuple(rng.shape)}")
            if not rng.is_cuda:
                raise TypeError(f"rng is on {rng.device}: give (seed, step) as ints, or a tensor on the device of the activations")
            if not rng.is_contiguous():
                raise ValueError("rng must be contiguous: the kernels read it in place")
            self.rng, self.seed, self.step = rng, 0, 0
        else:
            seed, step = rng
            self.rng, self.seed, self.step = None, int(seed) % 2 ** 64, int(step) % 2 ** 32
        for name, v in (("layer", layer), ("first_item", first_item)):
            if not 0 <= int(v) < 2 ** 32:
                raise ValueError(f"{name} must be in [0, 2^32), got {v}")
        self.layer, self.per_channel, self.first_item = int(layer), bool(per_channel), int(first_item)

    @property
    def probability(self) -> float:
        return self.threshold / 65536

    def for_layer(self, layer: int) -> "DropoutMask":
        """The same draw for another place of the model."""
        return DropoutMask(self.probability, self.rng if self.rng is not None else (self.seed, self.step), layer, self.per_channel,
                           self.first_item)

    def _args(self):
        return (ptr(self.rng), self.seed, self.step, self.layer, self.first_item, self.threshold, int(self.per_channel))


_NO_MASK = (None, 0, 0, 0, 0, 0, 0)


def _check_mask(mask, x: Tensor) -> None:
    if not isinstance(mask, DropoutMask):
        raise TypeError(f"a DropoutMask is needed, got {type(mask).__name__}")
    if mask.rng is not None and mask.rng.device != x.device:
        raise TypeError(f"the mask's rng is on {mask.rng.device}, the activations on {x.device}")
    if mask.first_item + x.shape[0] > 2 ** 32:
        raise ValueError("first_item plus the batch size must not pass 2^32")


# ----------------------------------------------------------------------------- group norm
@functools.lru_cache(maxsize=1024)
def _workspace_floats(B, N, C, G, dt, backward) -> int:
    n = _lib.load().sfm_group_norm_workspace_floats(B, N, C, G, dt, backward)
    if n < 0:
        raise ValueError(f"unsupported group-norm shape B={B} N={N} C={C} G={G} (rc {n})")
    return n


def _workspace(B, N, C, G, dt, backward, device) -> Tensor:
    return torch.empty((_workspace_floats(B, N, C, G, dt, backward) + 1) // 2, dtype=torch.float64, device=device)


def _raw_gn(x, ld_x, gamma, beta, groups, epsilon, act, mask, y, ld_y, stats):
    """-> (mean, rstd) [B, G] if stats; y: a tensor of its own or a channel slice (row stride ld_y)"""
    B, C = x.shape[0], x.shape[-1]
    N = x.numel() // (B * C)
    dt = _DTYPES[x.dtype]
    ws = _workspace(B, N, C, groups, dt, 0, x.device)
    mean = rstd = None
    if stats:
        mean = torch.empty(B, groups, dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
    call("sfm_group_norm_act_fwd", ptr(x), ld_x, dt, ptr(gamma), ptr(beta), B, N, C, groups, epsilon, act,
         *(_NO_MASK if mask is None else mask._args()), ptr(y), ld_y, ptr(mean), ptr(rstd), ptr(ws), stream_of(x))
    return mean, rstd


def _raw_gn_bwd(x, ld_x, srcs, gamma, beta, stats, groups, act, mask, need_x=True, need_params=True):
    """srcs: [(tensor whose data pointer is the slice's first channel at row 0, row stride)], summed while loading"""
    B, C = x.shape[0], x.shape[-1]
    N = x.numel() // (B * C)
    dt = _DTYPES[x.dtype]
    ws = _workspace(B, N, C, groups, dt, 1, x.device)
    gx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
    gg, gb = (_grad_out(gamma), _grad_out(beta)) if need_params else (None, None)
    n = len(srcs)
    gy = (ctypes.c_void_p * n)(*[t.data_ptr() for t, _ in srcs])
    ld = (ctypes.c_longlong * n)(*[int(l) for _, l in srcs])
    call("sfm_group_norm_act_bwd", ptr(x), ld_x, dt, gy, ld, n, ptr(gamma), ptr(beta), ptr(stats[0]), ptr(stats[1]), B, N, C,
         groups, act, *(_NO_MASK if mask is None else mask._args()), ptr(gx), ptr(gg), ptr(gb), ptr(ws), stream_of(x))
    return gx, gg, gb


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, groups, epsilon, act, mask):
        with _on(x.device):
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            if x.numel() == 0:
                mean = rstd = None
            else:
                rows, ld = _rows(x)
                mean, rstd = _raw_gn(rows, ld, gamma, beta, groups, epsilon, act, mask, y, x.shape[-1], True)
        ctx.save_for_backward(x, gamma, beta, mean, rstd, None if mask is None else mask.rng)
        ctx.cfg = (groups, act, mask)
        return y

    @staticmethod
    def backward(ctx, gy):
        _refuse_second_order("group_norm_act")
        x, gamma, beta, mean, rstd, _ = ctx.saved_tensors  # (unpacking checks that the mask's rng is what the forward read)
        groups, act, mask = ctx.cfg
        need_x, need_params = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        with _on(x.device):
            if x.numel() == 0:
                gx, gg, gb = torch.zeros_like(x), torch.zeros_like(gamma), torch.zeros_like(beta)
            else:
                rows, ld = _rows(x)
                gx, gg, gb = _raw_gn_bwd(rows, ld, [_rows(gy)], gamma, beta, (mean, rstd), groups, act, mask, need_x, need_params)
        return gx, gg, gb, None, None, None, None


def group_norm_act(x: Tensor, gamma: Tensor, beta: Tensor, groups: int, epsilon: float = GN_EPSILON,
                   activation: Optional[str] = "elu", dropout: Optional[DropoutMask] = None) -> Tensor:
    """``dropout(activation(group_norm(x)))`` with the parameters ``gamma``, ``beta`` [C] (fp32), channels last.

    x [B, ..., C] (fp32, bf16 or fp16; a channel slice of a dense buffer is read in place): for every item and group of C / groups
    adjacent channels the mean and the population variance over all rows, z = gamma (x - mean) / sqrt(var + epsilon) + beta, the
    activation ("elu", "relu", "silu" or None), and, with a ``DropoutMask``, the mask.  Statistics and parameter gradients are
    fp32 for every type.  Differentiable once, in x, gamma and beta; the backward reads x and forms z and the mask again."""
    dt = _check_activation(x, "x")
    C = x.shape[-1]
    gamma = _check(gamma, "gamma", 1, C)
    beta = _check(beta, "beta", 1, C)
    _same_device(x, gamma, beta)
    groups, epsilon = int(groups), float(epsilon)
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"groups must divide the {C} channels, got {groups}")
    if not 0.0 < epsilon < float("inf"):
        raise ValueError(f"epsilon must be positive and finite, got {epsilon}")
    act = ACTIVATIONS.get(activation, -1) if activation is None or isinstance(activation, str) else -1
    if act < 0:
        raise ValueError(f"activation must be one of {[a for a in ACTIVATIONS if a]} or None, got {activation!r}")
    if dropout is not None:
        _check_mask(dropout, x)
        if dropout.threshold == 0:
            dropout = None
    if x.numel():
        _workspace_floats(x.shape[0], x.numel() // (x.shape[0] * C), C, groups, dt, 0)
    if torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad or beta.requires_grad):
        return _GroupNormAct.apply(x, gamma, beta, groups, epsilon, act, dropout)
    with _on(x.device):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if x.numel():
            rows, ld = _rows(x.detach())
            _raw_gn(rows, ld, gamma, beta, groups, epsilon, act, dropout, y, C, False)
    return y


# ----------------------------------------------------------------------------- dropout
def _raw_dropout(x, mask):
    x = x.contiguous()
    y = torch.empty_like(x)
    if x.numel():
        call("sfm_dropout", ptr(x), _DTYPES[x.dtype], x.shape[0], x.numel() // x.shape[0], x.shape[-1], *mask._args(), ptr(y),
             stream_of(x))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, mask):
        ctx.save_for_backward(mask.rng)
        ctx.mask = mask
        with _on(x.device):
            return _raw_dropout(x, mask)

    @staticmethod
    def backward(ctx, gy):
        _refuse_second_order("dropout")
        ctx.saved_tensors  # (checks that the mask's rng is what the forward read)
        with _on(gy.device):
            return _raw_dropout(gy, ctx.mask), None


def dropout(x: Tensor, mask: DropoutMask) -> Tensor:
    """``x`` [B, ..., C] (fp32, bf16 or fp16) with the elements, or the channels, that ``mask`` drops set to 0 and the others
    multiplied by 1 / (1 - mask.probability).  What is dropped is 0 even where x is infinite or NaN.  Differentiable once: the backward
    draws the same mask again, nothing is kept for it."""
    _check_activation(x, "x")
    _check_mask(mask, x)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dropout.apply(x, mask)
    with _on(x.device):
        return _raw_dropout(x.detach(), mask)
