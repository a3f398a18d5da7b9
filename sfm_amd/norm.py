"""The batch-independent normaliser and the regulariser of the decoder's activations, next to ``batch_norm_elu``:

    group_norm_act    group norm (channels last), an activation and, if asked for, a dropout mask, in the same passes
    dropout           the mask alone
    DropoutMask       which mask: a function of (seed, step, layer, item, place), never stored (csrc/norm_drop.h)

Both are differentiable (torch.autograd; once), take fp32, bf16 and fp16 activations with fp32 parameters, compute in fp32 and
round a 16-bit result once.  Like the rest of the package they have no CPU path.  Group norm takes its statistics from one item:
it is the same function for any batch size, in training and in serving, and needs no collective under data parallelism.
"""
from __future__ import annotations

import ctypes
import functools
import operator
from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import call, ptr, stream_of
from .aspp import BN_EPSILON, _grad_out, _sink_of
from .utils import _check, _same_device

Tensor = torch.Tensor
GN_EPSILON = BN_EPSILON
ACTIVATIONS = {None: 0, "none": 0, "elu": 1, "relu": 2, "silu": 3}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FP32 = torch.finfo(torch.float32)
_autograd = None


def _nodes():
    """sfm_amd._autograd: the operators' autograd nodes (csrc/autograd.cpp)"""
    global _autograd
    if _autograd is None:
        _lib.load()
        try:
            from . import _autograd as built
        except ImportError as e:
            raise ImportError("sfm_amd/_autograd.so is missing or was built for another torch - build it first (python -c 'import "
                              "__graft_entry__ as g; g.build()' or make -C sfm_amd/csrc)") from e
        _autograd = built
    return _autograd


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
    if x.shape[-1] > 2 ** 31 - 1:
        raise ValueError(f"{name} has {x.shape[-1]} channels, more than 2^31 - 1")
    return dt


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
            self.rng, self.seed, self.step = None, operator.index(seed) % 2 ** 64, operator.index(step) % 2 ** 32
        for name, v in (("layer", layer), ("first_item", first_item)):
            if not 0 <= operator.index(v) < 2 ** 32:
                raise ValueError(f"{name} must be in [0, 2^32), got {v}")
        self.layer, self.per_channel, self.first_item = operator.index(layer), bool(per_channel), operator.index(first_item)

    @property
    def probability(self) -> float:
        return self.threshold / 65536

    def for_layer(self, layer: int) -> "DropoutMask":
        """The same draw for another place of the model."""
        return DropoutMask(self.probability, self.rng if self.rng is not None else (self.seed, self.step), layer, self.per_channel,
                           self.first_item)

    def _args(self):
        return (self.rng, self.seed, self.step, self.layer, self.first_item, self.threshold, self.per_channel)


_NO_MASK = (None, 0, 0, 0, 0, 0, False)


def _ctypes_mask(mask):
    if mask is None:
        return _NO_MASK
    rng, *rest = mask._args()
    return (ptr(rng), *rest)


def _check_mask(mask, x: Tensor) -> None:
    if not isinstance(mask, DropoutMask):
        raise TypeError(f"a DropoutMask is needed, got {type(mask).__name__}")
    if mask.rng is not None and mask.rng.device != x.device:
        raise TypeError(f"the mask's rng is on {mask.rng.device}, the activations on {x.device}")
    if mask.first_item + x.shape[0] > 2 ** 32:
        raise ValueError("first_item plus the batch size must not pass 2^32")


# ----------------------------------------------------------------------------- group norm
class _Plan:
    """what is known of a shape: sizes, and the floats of the statistics (2 B G) and of the workspace of either direction"""

    __slots__ = ("B", "N", "C", "G", "dt", "stats", "fwd", "bwd")

    def __init__(self, shape, dtype, groups):
        C = shape[-1]
        if groups < 1 or C < 1 or C % groups:
            raise ValueError(f"groups must divide the {C} channels, got {groups}")
        rows = 1
        for n in shape[:-1]:
            rows *= n
        self.B, self.C, self.G, self.dt = shape[0], C, groups, _DTYPES[dtype]
        self.N = rows // shape[0] if shape[0] else 0
        self.stats = self.fwd = self.bwd = 0
        if rows:
            n = [_lib.load().sfm_group_norm_workspace_floats(self.B, self.N, C, groups, self.dt, back) for back in (0, 1)]
            if min(n) < 0:
                raise ValueError(f"unsupported group-norm shape {tuple(shape)} with {groups} groups (rc {min(n)})")
            self.stats = 2 * self.B * groups                 # even: the workspace behind it stays aligned to 8 bytes
            self.fwd, self.bwd = n


@functools.lru_cache(maxsize=1024)
def _plan(shape, dtype, groups) -> _Plan:
    return _Plan(shape, dtype, groups)


def _raw_gn(plan, x, ld_x, gamma, beta, epsilon, act, mask, y, ld_y, keep):
    """-> the buffer of (keep: the statistics, for the backward, and) the workspace.  y: a tensor of its own or a channel slice (row
    stride ld_y)"""
    p = plan
    buf = torch.empty(p.stats + p.fwd if keep else p.fwd, dtype=torch.float32, device=x.device)
    at = buf.data_ptr()
    call("sfm_group_norm_act_fwd", ptr(x), ld_x, p.dt, ptr(gamma), ptr(beta), p.B, p.N, p.C, p.G, epsilon, act, *_ctypes_mask(mask),
         ptr(y), ld_y, at if keep else None, at + 2 * p.stats if keep else None, at + 4 * p.stats if keep else at, stream_of(x))
    return buf


def _raw_gn_bwd(plan, x, ld_x, srcs, gamma, beta, buf, act, mask, need_x=True, need_params=True):
    """srcs: [(tensor whose data pointer is the slice's first channel at row 0, row stride)], summed while loading.  buf: the forward's; it is
    read only, and the workspace is this pass's own: a graph may be run again while a captured pass of it replays"""
    p, n = plan, len(srcs)
    ws = torch.empty(p.bwd, dtype=torch.float32, device=x.device)
    gx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
    gg, gb = (_grad_out(gamma), _grad_out(beta)) if need_params else (None, None)
    at = buf.data_ptr()
    call("sfm_group_norm_act_bwd", ptr(x), ld_x, p.dt, (ctypes.c_void_p * n)(*[t.data_ptr() for t, _ in srcs]),
         (ctypes.c_longlong * n)(*[ld for _, ld in srcs]), n, ptr(gamma), ptr(beta), at, at + 2 * p.stats, p.B, p.N, p.C, p.G, act,
         *_ctypes_mask(mask), ptr(gx), ptr(gg), ptr(gb), ptr(ws), stream_of(x))
    return gx, gg, gb


class _GroupNormActInBuckets(torch.autograd.Function):
    """the same node as sfm_amd._autograd's, in Python, for parameters whose gradients are born inside a ``GradBuckets``"""

    @staticmethod
    def forward(ctx, x, gamma, beta, plan, epsilon, act, mask):
        x, ld = _nodes().rows_of(x)  # itself, if it is dense or a channel slice
        with torch.cuda.device(x.device):
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            buf = _raw_gn(plan, x, ld, gamma, beta, epsilon, act, mask, y, plan.C, any(ctx.needs_input_grad)) if plan.fwd else None
        ctx.save_for_backward(x, gamma, beta, buf, None if mask is None else mask.rng)
        ctx.cfg = (plan, act, mask)
        return y

    @staticmethod
    def backward(ctx, gy):
        if torch.is_grad_enabled():  # a backward runs with gradients on under create_graph=True alone
            raise RuntimeError("group_norm_act is differentiable once: its backward was called with create_graph=True")
        x, gamma, beta, buf, _ = ctx.saved_tensors  # (unpacking checks that the mask's rng is what the forward read)
        plan, act, mask = ctx.cfg
        if buf is None:
            return torch.zeros_like(x), torch.zeros_like(gamma), torch.zeros_like(beta), None, None, None, None
        need_x, need_g, need_b = ctx.needs_input_grad[:3]
        with torch.cuda.device(x.device):
            x, ld = _nodes().rows_of(x)
            return (*_raw_gn_bwd(plan, x, ld, (_nodes().rows_of(gy),), gamma, beta, buf, act, mask, need_x, need_g or need_b),
                    None, None, None, None)


def group_norm_act(x: Tensor, gamma: Tensor, beta: Tensor, groups: int, epsilon: float = GN_EPSILON,
                   activation: Optional[str] = "elu", dropout: Optional[DropoutMask] = None) -> Tensor:
    """``dropout(activation(group_norm(x)))`` with the parameters ``gamma``, ``beta`` [C] (fp32), channels last.

    x [B, ..., C] (fp32, bf16 or fp16; a channel slice of a dense buffer is read in place): for every item and group of C / groups
    adjacent channels the mean and the population variance over all rows, z = gamma (x - mean) / sqrt(var + epsilon) + beta, the
    activation ("elu", "relu", "silu" or None), and, with a ``DropoutMask``, the mask.  Statistics and parameter gradients are
    fp32 for every type.  Differentiable once, in x, gamma and beta; the backward reads x and forms z and the mask again."""
    _check_activation(x, "x")
    shape, device = x.shape, x.device
    C = shape[-1]
    for name, t in (("gamma", gamma), ("beta", beta)):
        if not (isinstance(t, Tensor) and t.dtype is torch.float32 and t.dim() == 1 and t.shape[0] == C and t.device == device):
            _check(t, name, 1, C)
            _same_device(x, t)
    if not gamma.is_contiguous():
        gamma = gamma.contiguous()
    if not beta.is_contiguous():
        beta = beta.contiguous()
    epsilon = float(epsilon)
    if not _FP32.tiny <= epsilon <= _FP32.max:
        raise ValueError(f"epsilon must be positive and finite in float32, got {epsilon}")
    act = ACTIVATIONS.get(activation, -1) if activation is None or isinstance(activation, str) else -1
    if act < 0:
        raise ValueError(f"activation must be one of {[a for a in ACTIVATIONS if a]} or None, got {activation!r}")
    if dropout is not None:
        _check_mask(dropout, x)
        if dropout.threshold == 0:
            dropout = None
    groups = operator.index(groups)
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"groups must divide the {C} channels, got {groups}")
    if torch.is_grad_enabled() and (_sink_of(gamma) is not None or _sink_of(beta) is not None):
        _nodes().refuse_tracing("group_norm_act")
        _nodes().refuse_foreign_leaves("group_norm_act", [x, gamma, beta], x)
        return _GroupNormActInBuckets.apply(x, gamma, beta, _plan(shape, x.dtype, groups), epsilon, act, dropout)
    return _nodes().group_norm_act(x, gamma, beta, groups, epsilon, act, *(_NO_MASK if dropout is None else dropout._args()))


# ----------------------------------------------------------------------------- dropout
def dropout(x: Tensor, mask: DropoutMask) -> Tensor:
    """``x`` [B, ..., C] (fp32, bf16 or fp16) with the elements, or the channels, that ``mask`` drops set to 0 and the others
    multiplied by 1 / (1 - mask.probability).  What is dropped is 0 even where x is infinite or NaN.  Differentiable once: the backward
    draws the same mask again, nothing is kept for it."""
    _check_activation(x, "x")
    _check_mask(mask, x)
    return _nodes().dropout(x, *mask._args())
