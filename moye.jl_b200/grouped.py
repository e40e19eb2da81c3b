"""Rows that choose their own weights: the operators around mixture-of-experts layers and low-rank adapters.

    group_rows(ids, groups)                       ->  moye_b200_group_rows          a RowGroups plan
    gather_rows_(dst, src, plan)                  ->  moye_b200_gather_rows         rows to their groups' positions
    combine_rows_(dst, src, plan, weights)        ->  moye_b200_combine_rows        and back, weighted and summed
    combine_rows_grad_(dsrc, dweights, ...)       ->  moye_b200_combine_rows_grad
    gemm_grouped_(D, A, B, offsets)               ->  moye_b200_gemm_grouped        every group times its weight
    gemm_grouped_grad_(dB, dD, A, offsets)        ->  moye_b200_gemm_grouped_grad   gradient of the weights
    gemm_lora_(D, X, A, B, adapters, offsets)     ->  moye_b200_gemm_lora           adapters beside a projection

They stand beside `gemm_`, `copyto_` and `axpby_` and follow their conventions: names ending in `_` write their first
argument (and return it), operands are torch CUDA tensors or MoYeArrays, calls are asynchronous on the current stream of
the operands' device or on `stream`, a violation raises `MoyeError`, nothing falls back to another implementation.  Group
borders, choices and adapter numbers stay on the device: no call waits for the GPU, and a captured call follows new
values in the same arrays.  The reference has no counterpart.

Every call is offered to the compiled module of csrc/calls.cpp first (`_lib.calls`), which takes plain tensors on the
current device into the same entry points; what it does not take is checked, explained and launched here.
"""
import struct
import threading

import torch

from . import _lib
from .array import TORCH_TO_MOYE, MoYeArray
from .layout import coalesce

__all__ = ["RowGroups", "group_rows", "group_rows_", "gather_rows_", "combine_rows_", "combine_rows_grad_", "gemm_grouped_",
           "gemm_grouped_grad_", "gemm_lora_"]


# the stream's handle alone: a torch Stream object costs 2 us a call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_thread = threading.get_ident
_PACK = _lib.TENSOR_PACKERS
_INT32, _FLOAT32 = torch.int32, torch.float32


class RowGroups:
    """The result of sorting (tokens, choices) group numbers: int32 tensors on one device.

    `order[p]` is the entry (token * choices + choice) at sorted position p, -1 behind the last kept one;
    `offsets[g]` the first position of group g, `offsets[groups]` the number of kept entries; `inverse[t, j]` the
    position of a choice, -1 if it was dropped.  A plan made once can be filled again by `group_rows_` (a captured
    step needs that: the tensors keep their addresses)."""

    __slots__ = ("tokens", "choices", "groups", "_buf", "_at")

    def __init__(self, tokens, choices, groups, device, buf=None):
        self.tokens, self.choices, self.groups = tokens, choices, groups
        # order, inverse, offsets
        self._buf = torch.empty(2 * tokens * choices + groups + 1, dtype=_INT32, device=device) if buf is None else buf
        self._at = self._buf.get_device()

    @property
    def order(self):
        return self._buf[:self.tokens * self.choices]

    @property
    def inverse(self):
        n = self.tokens * self.choices
        return self._buf[n:2 * n].view(self.tokens, self.choices)

    @property
    def offsets(self):
        return self._buf[2 * self.tokens * self.choices:]

    def _pointers(self):
        """Addresses of order, inverse and offsets."""
        p, n = self._buf.data_ptr(), 4 * self.tokens * self.choices
        return p, p + n, p + 2 * n


def _arg(x, rank, what):
    """(descriptor bytes, device index) of a rank-`rank` device array."""
    if isinstance(x, torch.Tensor):
        dev = x.get_device()
        if dev >= 0:
            try:
                return _PACK[rank].pack(x.data_ptr(), TORCH_TO_MOYE[x.dtype], rank, *x.shape, *x.stride()), dev
            except (KeyError, struct.error):  # a type that has no counterpart, another rank: said below
                pass
        shape, where, dtype = tuple(x.shape), x.device, TORCH_TO_MOYE.get(x.dtype)
    elif isinstance(x, MoYeArray):
        l = x.layout
        modes = [coalesce(l[i]) for i in range(len(l))] if len(l) > 1 else [coalesce(l)]
        if any(isinstance(m.shape, tuple) for m in modes):
            raise _lib.MoyeError(-3, f"{what} must have one stride per mode, got layout {l}")
        shape, dtype, where = tuple(int(m.shape) for m in modes), x.dtype, x.device
        if where.type == "cuda" and len(shape) == rank:
            return _lib.pack_tensor(x.ptr, dtype, shape, [int(m.stride) for m in modes]), where.index
    else:
        raise TypeError(f"{what} must be a torch.Tensor or a MoYeArray, got {type(x).__name__}")
    if where.type != "cuda":
        raise RuntimeError(f"libmoye_b200 runs on device global memory only; {what} is on {where} (there is no CPU fallback)")
    if dtype is None:
        raise _lib.MoyeError(-2, f"{what}: unsupported element type {x.dtype}")
    raise _lib.MoyeError(-4, f"{what} must be rank {rank}, got shape {shape}")


def _vector(x, what, dev, numel=None, dtype=_INT32):
    """Address of a contiguous device vector of `dtype` on device `dev`."""
    if not isinstance(x, torch.Tensor) or x.dtype != dtype or not x.is_contiguous():
        raise _lib.MoyeError(-1, f"{what} must be a contiguous {dtype} tensor")
    if x.get_device() != dev:
        raise RuntimeError("operands live on different devices")
    if numel is not None and x.numel() != numel:
        raise _lib.MoyeError(-4, f"{what} must hold {numel} values, got {x.numel()}")
    return x.data_ptr()


def _differ():
    raise RuntimeError("operands live on different devices")


def _fits(plan, x, what):
    """The kernels index the plan by the tokens of `x`: an array of another length would reach outside it."""
    if x.shape[0] != plan.tokens:
        raise _lib.MoyeError(-4, f"the plan is for {plan.tokens} tokens, {what} has {x.shape[0]} rows")


def _call(fn, dev, stream, *args):
    """fn(handle, *args, stream) with device number `dev`, the operands', current."""
    if stream is None:
        stream = _raw_stream(dev)
    handle = _lib._handles.get((_thread(), dev)) or _lib.handle(dev)
    if _current_device() == dev:
        rc = fn(handle, *args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(handle, *args, stream)
    if rc:
        _lib.check(rc)


def _taken(rc):
    """What the compiled call said: True if it launched, False if it leaves the call to this module; raises its errors."""
    if rc < 0:
        _lib.check(rc)
    return rc == 0


def group_rows(ids, groups):
    """Sort the group numbers `ids` ((tokens,) or (tokens, choices), int32 or int64) by group: a new `RowGroups`.
    Equal numbers keep their order; numbers outside 0..groups-1 are dropped (a capacity that ran out, a masked token).
    At most 1024 groups.  Runs on the current stream, which also owns the new tensors."""
    if _lib.calls is not None:
        buf = _lib.calls.new_plan(ids, groups)
        if type(buf) is torch.Tensor:
            shape = ids.shape
            return RowGroups(shape[0], shape[1] if len(shape) == 2 else 1, groups, None, buf)
        if buf < 0:
            _lib.check(buf)
    if not torch.is_tensor(ids):
        raise TypeError("ids must be a torch.Tensor")
    if ids.dim() not in (1, 2):
        raise _lib.MoyeError(-4, f"ids must be (tokens,) or (tokens, choices), got shape {tuple(ids.shape)}")
    if not ids.is_cuda:
        raise RuntimeError(f"libmoye_b200 runs on device global memory only; ids is on {ids.device} (there is no CPU fallback)")
    if not 1 <= groups <= 1024:
        raise _lib.MoyeError(-4, f"group_rows: 1 to 1024 groups (got {groups})")
    return group_rows_(RowGroups(ids.shape[0], ids.shape[1] if ids.dim() == 2 else 1, groups, ids.device), ids)


def group_rows_(plan, ids, stream=None):
    """`group_rows` into the tensors of an existing plan of the same tokens, choices and groups."""
    if _lib.calls is not None:
        rc = _lib.calls.group_rows(ids, plan._buf, plan.tokens, plan.choices, plan.groups, stream)
        if _taken(rc):
            return plan
    rank = len(ids.shape)
    t, dev = _arg(ids, 1 if rank == 1 else 2, "ids")
    if ids.shape[0] != plan.tokens or (ids.shape[1] if rank == 2 else 1) != plan.choices:
        raise _lib.MoyeError(-4, f"the plan is for ({plan.tokens}, {plan.choices}) choices, ids are {tuple(ids.shape)}")
    if dev != plan._at:
        _differ()
    order, inverse, offsets = plan._pointers()
    _call(_lib.load().moye_b200_group_rows, dev, stream, t, plan.groups, order, offsets, inverse)
    return plan


def gather_rows_(dst, src, plan, stream=None):
    """dst[p] = src[plan.order[p] // choices] for the kept positions; rows of dst behind them are left as they were.
    src (tokens, width), dst (tokens * choices, width); any element type a MoYeArray takes, contiguous rows.  Its gradient is
    `combine_rows_(dsrc, ddst, plan)`."""
    if _lib.calls is not None and _taken(_lib.calls.gather_rows(dst, src, plan._buf, plan.tokens, plan.choices, stream)):
        return dst
    td, dev = _arg(dst, 2, "dst")
    ts, d1 = _arg(src, 2, "src")
    _fits(plan, src, "src")
    if not dev == d1 == plan._at:
        _differ()
    _call(_lib.load().moye_b200_gather_rows, dev, stream, td, ts, plan._pointers()[1], plan.choices)
    return dst


def combine_rows_(dst, src, plan, weights=None, stream=None):
    """dst[t] = sum_j weights[t, j] * src[plan.inverse[t, j]] over the choices that were kept (none: zeros), in fp32 in
    the order of j with one rounding.  `weights` (tokens, choices) in f32, f16 or bf16; None counts every choice once."""
    if _lib.calls is not None and _taken(_lib.calls.combine_rows(dst, src, plan._buf, plan.tokens, plan.choices, weights, stream)):
        return dst
    td, dev = _arg(dst, 2, "dst")
    ts, d1 = _arg(src, 2, "src")
    tw, d2 = (None, dev) if weights is None else _arg(weights, 2, "weights")
    _fits(plan, dst, "dst")
    if not dev == d1 == d2 == plan._at:
        _differ()
    _call(_lib.load().moye_b200_combine_rows, dev, stream, td, ts, tw, plan._pointers()[1], plan.choices)
    return dst


def combine_rows_grad_(dsrc, dweights, ddst, src, plan, weights, stream=None):
    """The gradient of `combine_rows_(dst, src, plan, weights)`: dsrc[inverse[t, j]] = weights[t, j] * ddst[t] (rows
    behind the kept positions are left as they were), dweights[t, j] = <ddst[t], src[inverse[t, j]]>, 0 where the choice
    was dropped.  Returns (dsrc, dweights)."""
    if _lib.calls is not None and _taken(_lib.calls.combine_rows_grad(dsrc, dweights, ddst, src, plan._buf, plan.tokens, plan.choices,
                                                                      weights, stream)):
        return dsrc, dweights
    t0, dev = _arg(dsrc, 2, "dsrc")
    t1, d1 = _arg(dweights, 2, "dweights")
    t2, d2 = _arg(ddst, 2, "ddst")
    t3, d3 = _arg(src, 2, "src")
    t4, d4 = _arg(weights, 2, "weights")
    _fits(plan, ddst, "ddst")
    if not dev == d1 == d2 == d3 == d4 == plan._at:
        _differ()
    _call(_lib.load().moye_b200_combine_rows_grad, dev, stream, t0, t1, t2, t3, t4, plan._pointers()[1], plan.choices)
    return dsrc, dweights


def _borders_plain(offsets):
    """The tensor that holds the borders and the index of the first."""
    if isinstance(offsets, RowGroups):
        return offsets._buf, 2 * offsets.tokens * offsets.choices
    return offsets, 0


def _borders(offsets, groups, dev):
    if isinstance(offsets, RowGroups):
        if offsets._at != dev:
            _differ()
        if offsets.groups != groups:
            raise _lib.MoyeError(-4, f"the plan has {offsets.groups} groups, the weights {groups}")
        return offsets._pointers()[2]
    return _vector(offsets, "offsets", dev, groups + 1)


def gemm_grouped_(D, A, B, offsets, alpha=1.0, beta=0.0, stream=None):
    """D[i] = alpha * A[i] . B[g]^T + beta * D[i] for the rows i of every group g, offsets[g] <= i < offsets[g + 1].

    A (rows, K), B (groups, N, K), D (rows, N); f16 or bf16, D also f32.  `offsets` is an int32 device tensor of
    groups + 1 borders or the RowGroups they come from.  B may be the swapped view of a (groups, K, N) array:
    `gemm_grouped_(dA, dD, B.transpose(1, 2), offsets)` is the gradient of A.  Rows outside the groups are left as they
    were; D is not read when beta == 0."""
    if _lib.calls is not None and _taken(_lib.calls.gemm_grouped(D, A, B, *_borders_plain(offsets), alpha, beta, stream)):
        return D
    td, dev = _arg(D, 2, "D")
    ta, d1 = _arg(A, 2, "A")
    tb, d2 = _arg(B, 3, "B")
    if not dev == d1 == d2:
        _differ()
    _call(_lib.load().moye_b200_gemm_grouped, dev, stream, td, ta, tb, _borders(offsets, int(B.shape[0]), dev), float(alpha), float(beta))
    return D


def gemm_grouped_grad_(dB, dD, A, offsets, alpha=1.0, beta=0.0, stream=None):
    """dB[g] = alpha * sum of dD[i]^T A[i] over the rows of group g + beta * dB[g]: the gradient of `gemm_grouped_` with
    respect to B.  Every group is written (an empty one becomes beta * dB[g]); beta = 1 accumulates over micro-batches."""
    if _lib.calls is not None and _taken(_lib.calls.gemm_grouped_grad(dB, dD, A, *_borders_plain(offsets), alpha, beta, stream)):
        return dB
    tb, dev = _arg(dB, 3, "dB")
    td, d1 = _arg(dD, 2, "dD")
    ta, d2 = _arg(A, 2, "A")
    if not dev == d1 == d2:
        _differ()
    _call(_lib.load().moye_b200_gemm_grouped_grad, dev, stream, tb, td, ta, _borders(offsets, int(dB.shape[0]), dev), float(alpha), float(beta))
    return dB


def gemm_lora_(D, X, A, B, adapters, offsets=None, scales=None, C=None, stream=None):
    """D[i] = C[i] + scales[a] * (X[i] . A[a]^T) . B[a]^T: the low-rank adapters of many requests beside a shared
    projection whose output is C (None: D itself, in place).

    X (rows, K), A (count, R, K), B (count, N, R), f16 or bf16; C and D (rows, N) in that type or f32.  `adapters` holds
    one int32 per request, a number outside 0..count-1 means none.  `offsets` (requests + 1 borders, int32) says which
    rows are a request's; without it every row is one.  Rows outside every request are left as they were.  R is a
    multiple of 8 up to 128: pad adapters of smaller rank with zeros."""
    if _lib.calls is not None and _taken(_lib.calls.gemm_lora(D, X, A, B, adapters, offsets, scales, C, stream)):
        return D
    td, dev = _arg(D, 2, "D")
    tx, d1 = _arg(X, 2, "X")
    ta, d2 = _arg(A, 3, "A")
    tb, d3 = _arg(B, 3, "B")
    tc, d4 = (None, dev) if C is None else _arg(C, 2, "C")
    if not dev == d1 == d2 == d3 == d4:
        _differ()
    which, requests = _vector(adapters, "adapters", dev), adapters.numel()
    edges = None if offsets is None else _vector(offsets, "offsets", dev, requests + 1)
    s = None if scales is None else _vector(scales, "scales", dev, int(A.shape[0]), _FLOAT32)
    _call(_lib.load().moye_b200_gemm_lora, dev, stream, td, tx, ta, tb, tc, which, edges, requests, s)
    return D
