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
"""
import ctypes

import torch

from . import _lib
from .array import TORCH_TO_MOYE, MoYeArray
from .layout import coalesce

__all__ = ["RowGroups", "group_rows", "group_rows_", "gather_rows_", "combine_rows_", "combine_rows_grad_", "gemm_grouped_",
           "gemm_grouped_grad_", "gemm_lora_"]


class RowGroups:
    """The result of sorting (tokens, choices) group numbers: int32 tensors on one device.

    `order[p]` is the entry (token * choices + choice) at sorted position p, -1 behind the last kept one;
    `offsets[g]` the first position of group g, `offsets[groups]` the number of kept entries; `inverse[t, j]` the
    position of a choice, -1 if it was dropped.  A plan made once can be filled again by `group_rows_` (a captured
    step needs that: the tensors keep their addresses)."""

    __slots__ = ("order", "offsets", "inverse", "tokens", "choices", "groups")

    def __init__(self, tokens, choices, groups, device):
        n = tokens * choices
        buf = torch.empty(2 * n + groups + 1, dtype=torch.int32, device=device)
        self.order, self.offsets = buf[:n], buf[2 * n:]
        self.inverse = buf[n:2 * n].view(tokens, choices)
        self.tokens, self.choices, self.groups = tokens, choices, groups


def _arg(x, rank, what):
    """(descriptor bytes, device) of a rank-`rank` device array."""
    if isinstance(x, torch.Tensor):
        shape, stride, dtype, ptr, dev = x.shape, x.stride(), TORCH_TO_MOYE.get(x.dtype), x.data_ptr(), x.device
    elif isinstance(x, MoYeArray):
        l = x.layout
        modes = [coalesce(l[i]) for i in range(len(l))] if len(l) > 1 else [coalesce(l)]
        if any(isinstance(m.shape, tuple) for m in modes):
            raise _lib.MoyeError(-3, f"{what} must have one stride per mode, got layout {l}")
        shape, stride = [int(m.shape) for m in modes], [int(m.stride) for m in modes]
        dtype, ptr, dev = x.dtype, x.ptr, x.device
    else:
        raise TypeError(f"{what} must be a torch.Tensor or a MoYeArray, got {type(x).__name__}")
    if dev.type != "cuda":
        raise RuntimeError(f"libmoye_b200 runs on device global memory only; {what} is on {dev} (there is no CPU fallback)")
    if dtype is None:
        raise _lib.MoyeError(-2, f"{what}: unsupported element type")
    if len(shape) != rank:
        raise _lib.MoyeError(-4, f"{what} must be rank {rank}, got shape {tuple(shape)}")
    return _lib.pack_tensor(ptr, dtype, shape, stride), dev


def _ints(x, what, dev, numel=None, dtype=torch.int32):
    """Address of a contiguous device vector of whole numbers (or scales) on `dev`."""
    if not torch.is_tensor(x) or x.dtype != dtype or not x.is_contiguous():
        raise _lib.MoyeError(-1, f"{what} must be a contiguous {dtype} tensor")
    if x.device != dev:
        raise RuntimeError("operands live on different devices")
    if numel is not None and x.numel() != numel:
        raise _lib.MoyeError(-4, f"{what} must hold {numel} values, got {x.numel()}")
    return x.data_ptr()


def _same_device(dev, *others):
    for d in others:
        if d != dev:
            raise RuntimeError("operands live on different devices")


def _call(fn, dev, stream, *args):
    """fn(handle, *args, stream) with the operands' device current."""
    if stream is None:
        stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
    if torch.cuda.current_device() == dev.index:
        _lib.check(fn(_lib.handle(dev.index), *args, stream))
    else:
        with torch.cuda.device(dev):
            _lib.check(fn(_lib.handle(dev.index), *args, stream))


def group_rows(ids, groups):
    """Sort the group numbers `ids` ((tokens,) or (tokens, choices), int32 or int64) by group: a new `RowGroups`.
    Equal numbers keep their order; numbers outside 0..groups-1 are dropped (a capacity that ran out, a masked token).
    At most 1024 groups.  Runs on the current stream, which also owns the new tensors."""
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
    t, dev = _arg(ids, 1 if len(ids.shape) == 1 else 2, "ids")
    if ids.shape[0] != plan.tokens or (ids.shape[1] if len(ids.shape) == 2 else 1) != plan.choices:
        raise _lib.MoyeError(-4, f"the plan is for ({plan.tokens}, {plan.choices}) choices, ids are {tuple(ids.shape)}")
    _same_device(dev, plan.order.device)
    _call(_lib.load().moye_b200_group_rows, dev, stream, t, plan.groups, plan.order.data_ptr(), plan.offsets.data_ptr(),
          plan.inverse.data_ptr())
    return plan


def gather_rows_(dst, src, plan, stream=None):
    """dst[p] = src[plan.order[p] // choices] for the kept positions; rows of dst behind them are left as they were.
    src (tokens, width), dst (tokens * choices, width); any element type, contiguous rows.  Its gradient is
    `combine_rows_(dsrc, ddst, plan)`."""
    (td, dev), (ts, d1) = _arg(dst, 2, "dst"), _arg(src, 2, "src")
    _same_device(dev, d1, plan.inverse.device)
    _call(_lib.load().moye_b200_gather_rows, dev, stream, td, ts, plan.inverse.data_ptr(), plan.choices)
    return dst


def combine_rows_(dst, src, plan, weights=None, stream=None):
    """dst[t] = sum_j weights[t, j] * src[plan.inverse[t, j]] over the choices that were kept (none: zeros), in fp32 in
    the order of j with one rounding.  `weights` (tokens, choices) in f32, f16 or bf16; None counts every choice once."""
    (td, dev), (ts, d1) = _arg(dst, 2, "dst"), _arg(src, 2, "src")
    _same_device(dev, d1, plan.inverse.device)
    tw = None
    if weights is not None:
        tw, d2 = _arg(weights, 2, "weights")
        _same_device(dev, d2)
    _call(_lib.load().moye_b200_combine_rows, dev, stream, td, ts, tw, plan.inverse.data_ptr(), plan.choices)
    return dst


def combine_rows_grad_(dsrc, dweights, ddst, src, plan, weights, stream=None):
    """The gradient of `combine_rows_(dst, src, plan, weights)`: dsrc[inverse[t, j]] = weights[t, j] * ddst[t] (rows
    behind the kept positions are left as they were), dweights[t, j] = <ddst[t], src[inverse[t, j]]>, 0 where the choice
    was dropped.  Returns (dsrc, dweights)."""
    args = [_arg(x, 2, n) for x, n in ((dsrc, "dsrc"), (dweights, "dweights"), (ddst, "ddst"), (src, "src"), (weights, "weights"))]
    dev = args[0][1]
    _same_device(dev, plan.inverse.device, *(d for _, d in args[1:]))
    _call(_lib.load().moye_b200_combine_rows_grad, dev, stream, *(t for t, _ in args), plan.inverse.data_ptr(), plan.choices)
    return dsrc, dweights


def _borders(offsets, groups, dev):
    if isinstance(offsets, RowGroups):
        offsets = offsets.offsets
    return _ints(offsets, "offsets", dev, groups + 1)


def gemm_grouped_(D, A, B, offsets, alpha=1.0, beta=0.0, stream=None):
    """D[i] = alpha * A[i] . B[g]^T + beta * D[i] for the rows i of every group g, offsets[g] <= i < offsets[g + 1].

    A (rows, K), B (groups, N, K), D (rows, N); f16 or bf16, D also f32.  `offsets` is an int32 device tensor of
    groups + 1 borders or the RowGroups they come from.  B may be the swapped view of a (groups, K, N) array:
    `gemm_grouped_(dA, dD, B.transpose(1, 2), offsets)` is the gradient of A.  Rows outside the groups are left as they
    were; D is not read when beta == 0."""
    (td, dev), (ta, d1), (tb, d2) = _arg(D, 2, "D"), _arg(A, 2, "A"), _arg(B, 3, "B")
    _same_device(dev, d1, d2)
    _call(_lib.load().moye_b200_gemm_grouped, dev, stream, td, ta, tb, _borders(offsets, int(B.shape[0]), dev), alpha, beta)
    return D


def gemm_grouped_grad_(dB, dD, A, offsets, alpha=1.0, beta=0.0, stream=None):
    """dB[g] = alpha * sum of dD[i]^T A[i] over the rows of group g + beta * dB[g]: the gradient of `gemm_grouped_` with
    respect to B.  Every group is written (an empty one becomes beta * dB[g]); beta = 1 accumulates over micro-batches."""
    (tb, dev), (td, d1), (ta, d2) = _arg(dB, 3, "dB"), _arg(dD, 2, "dD"), _arg(A, 2, "A")
    _same_device(dev, d1, d2)
    _call(_lib.load().moye_b200_gemm_grouped_grad, dev, stream, tb, td, ta, _borders(offsets, int(dB.shape[0]), dev), alpha, beta)
    return dB


def gemm_lora_(D, X, A, B, adapters, offsets=None, scales=None, C=None, stream=None):
    """D[i] = C[i] + scales[a] * (X[i] . A[a]^T) . B[a]^T: the low-rank adapters of many requests beside a shared
    projection whose output is C (None: D itself, in place).

    X (rows, K), A (count, R, K), B (count, N, R), f16 or bf16; C and D (rows, N) in that type or f32.  `adapters` holds
    one int32 per request, a number outside 0..count-1 means none.  `offsets` (requests + 1 borders, int32) says which
    rows are a request's; without it every row is one.  Rows outside every request are left as they were.  R is a
    multiple of 8 up to 128: pad adapters of smaller rank with zeros."""
    (td, dev), (tx, d1), (ta, d2), (tb, d3) = _arg(D, 2, "D"), _arg(X, 2, "X"), _arg(A, 3, "A"), _arg(B, 3, "B")
    _same_device(dev, d1, d2, d3)
    tc = None
    if C is not None:
        tc, d4 = _arg(C, 2, "C")
        _same_device(dev, d4)
    which = _ints(adapters, "adapters", dev)
    requests = adapters.numel()
    edges = None if offsets is None else _ints(offsets, "offsets", dev, requests + 1)
    s = None if scales is None else _ints(scales, "scales", dev, int(A.shape[0]), torch.float32)
    _call(_lib.load().moye_b200_gemm_lora, dev, stream, td, tx, ta, tb, tc, which, edges, requests, s)
    return D
