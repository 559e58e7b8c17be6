"""Rows grouped by inverted list, on the GPU through qinco_group_* (csrc/group_kernel.hpp).

`group_rows` sorts the entries of (n, k) list ids by list: the IVF column of a code matrix (k = 1, filling an index, reference
qinco/search/search_utils.py:121-162) or the k nearest centroids of `KnnSearcher.search` (multi-probe, a router).  `RowGroups.gather`
carries rows into that order, `RowGroups.combine` brings them back with weights; both have gradients.  All of it can be captured into a graph
(`check=False`); a captured backward pass wants leaves that no eager graph holds at the same time, as torch's own operators do.  Forward-mode
and second derivatives are refused.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .sample import _TYPES, as_stored, being_traced, on_device, on_its_device, recording, refuse_trace, row_type, unit_rows

MAX_LISTS = 1 << 24
_IDS = {torch.int64: _lib.CODE_I64, torch.int32: _lib.CODE_I32, torch.uint8: _lib.CODE_U8}


def group_rows(lists, n_lists: int, check: bool = True) -> "RowGroups":
    """lists: torch CUDA tensor (n,) or (n, k) of int64 / int32 / uint8 ids in [0, n_lists), any row stride (`codes[:, 0]` is taken as it
    is); an id < 0 has no list.  Returns the entries (row * k + slot) in list order, stable: RowGroups.  Asynchronous on the current
    stream, except for check: wait and raise IndexError if an id is >= n_lists; check=False leaves such an entry without a list."""
    lib = _lib.load()
    if being_traced() or recording() is not None:
        refuse_trace("group_rows")
    on_device(lists, "lists")
    if lists.dim() not in (1, 2):
        raise ValueError(f"lists must be (n,) or (n, k), got {tuple(lists.shape)}")
    if not 1 <= int(n_lists) <= MAX_LISTS:
        raise ValueError(f"n_lists must be in [1, 2^24], got {n_lists}")
    code = _IDS.get(lists.dtype)
    if code is None:
        raise ValueError(f"lists must be int64, int32 or uint8, got {lists.dtype}")
    n, k = lists.shape if lists.dim() == 2 else (lists.shape[0], 1)
    if k < 1 or n * k >= 1 << 31:
        raise ValueError(f"need k >= 1 and n k < 2^31, got {tuple(lists.shape)}")
    if k > 1:
        lists = unit_rows(lists)
    dev = lists.device
    N, E = n * k, int(n_lists)
    need = lib.qinco_group_workspace(N, E)
    if need <= 1 << 16:   # few entries: the call is all that counts, and one allocation is 2 us less of it than four
        ws, order, place, offsets = torch.empty(need // 4 + 2 * N + E + 1, dtype=torch.int32, device=dev).split_with_sizes((need // 4, N, N, E + 1))
        place = place.view(n, k)
    else:
        order, place, offsets = (torch.empty(s, dtype=torch.int32, device=dev) for s in (N, (n, k), E + 1))
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    bad = torch.zeros(1, dtype=torch.int32, device=dev) if check else None
    on_its_device(dev.index, lib.qinco_group_rows, lists.data_ptr(), code, lists.stride(0), n, k, E, order.data_ptr(), place.data_ptr(),
                  offsets.data_ptr(), bad.data_ptr() if check else None, ws.data_ptr(), need)
    if check and int(bad):
        raise IndexError(f"a list id is >= n_lists = {n_lists}")
    groups = RowGroups.__new__(RowGroups)
    groups._set(order, place, offsets)
    return groups


def _no_tangents(*tensors):
    """Forward-mode derivatives are refused: a library call would answer its values without them."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("gather and combine have no forward-mode derivatives")


class RowGroups:
    """Entries in list order (int32 CUDA tensors):
      order   (n k,)         entry row * k + slot in each place; -1 behind the last place in use
      place   (n, k)         place of each entry; -1 without a list
      offsets (n_lists + 1,) first place of each list; the last value = places in use
    They are not to change while a backward pass may still use them."""

    def __init__(self, order, place, offsets):
        for t, what, dim in ((order, "order", 1), (place, "place", 2), (offsets, "offsets", 1)):
            if on_device(t, what).dtype != torch.int32 or t.dim() != dim or not t.is_contiguous() or t.device != place.device:
                raise ValueError(f"{what} must be a contiguous int32 tensor of {dim} dimension(s) on one device with the others")
        if order.numel() != place.numel() or place.shape[1] < 1 or offsets.numel() < 2:
            raise ValueError(f"order {tuple(order.shape)}, place {tuple(place.shape)}, offsets {tuple(offsets.shape)} do not belong together")
        self._set(order, place, offsets)

    def _set(self, order, place, offsets):
        self._tensors = order, place, offsets
        self.n, self.k = place.shape
        self.n_lists = offsets.numel() - 1
        # what the library calls take (a call's time in Python counts: autograd runs backward passes on a thread of its own, with cold caches)
        self._lib, self._index = _lib.load(), place.device.index
        self._order, self._place, self._end = order.data_ptr(), place.data_ptr(), offsets.data_ptr() + 4 * self.n_lists   # (the places in use)

    order = property(lambda self: self._tensors[0])
    place = property(lambda self: self._tensors[1])
    offsets = property(lambda self: self._tensors[2])

    def counts(self):
        """Entries of every list (n_lists,)."""
        return self.offsets.diff()

    def _rows(self, t, rows: int, what: str):
        shape = on_device(t, what).shape
        if len(shape) != 2 or shape[0] != rows or not 1 <= shape[1] < 1 << 31 or t.device.index != self._index:
            raise ValueError(f"{what} must be ({rows}, D) with 1 <= D < 2^31 on {self.place.device}, got {tuple(t.shape)} on {t.device}")
        return unit_rows(t)

    def gather(self, x):
        """x (n, D) of any type, also code rows -> (n k, D): row order[s] // k at place s, zeros behind the last place in use.
        The gradient is the sum over a row's places, in 32 bits, rounded once (float32, float16, bfloat16)."""
        x = self._rows(x, self.n, "x")
        if recording() is not None:
            refuse_trace("gather")
        if forward_ad._current_level >= 0:             # (between dual levels there are no tangents)
            _no_tangents(x)
        traced = being_traced()                        # (a trace holds the function, with these groups)
        if x.requires_grad and torch.is_grad_enabled():
            row_type(x, "x that requires a gradient")
            return _Gather.apply(x, self, traced)
        return _Gather.apply(x, self, True) if traced else self._gather(x)

    def combine(self, y, weights=None):
        """y (n k, D) float32 / float16 / bfloat16 in list order -> (n, D): sum_j weights[r, j] y[place[r, j]] over the entries that have
        a list (zeros for a row without one), in 32 bits in the order of j, rounded once.  weights (n, k) float32 or y's type; None: ones.
        Rows of y behind the last place in use and weights of entries without a list are not read; their gradients are zeros."""
        y, weights = self._combine_args(y, weights)
        if recording() is not None:
            refuse_trace("combine")
        if forward_ad._current_level >= 0:
            _no_tangents(y, weights)
        traced = being_traced()
        if traced or torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
            return _Combine.apply(y, weights, self, traced)
        return self._combine(y, weights)

    def _combine_args(self, y, weights):
        y = self._rows(y, self.n * self.k, "y")
        row_type(y, "y")
        if weights is not None:
            if on_device(weights, "weights").shape != (self.n, self.k) or weights.dtype not in (torch.float32, y.dtype) or weights.device != y.device:
                raise ValueError(f"weights must be ({self.n}, {self.k}) float32 or {y.dtype} on {y.device}, got {tuple(weights.shape)} {weights.dtype}")
            weights = as_stored(weights).contiguous()
        return y, weights

    # -- the library calls; arguments are checked already, rows in unit_rows' form
    def _gather(self, x):
        D, size = x.shape[1], x.element_size()
        out = x.new_empty((self.n * self.k, D))
        on_its_device(self._index, self._lib.qinco_group_gather, x.data_ptr(), x.stride(0) * size, D * size, self._order, self._place,
                      self._end, self.n, self.k, out.data_ptr())
        return out

    def _combine(self, y, weights):
        D, wt, w_type = y.shape[1], None, 0
        out = y.new_empty((self.n, D))
        if weights is not None:
            wt, w_type = weights.data_ptr(), _TYPES[weights.dtype]
        on_its_device(self._index, self._lib.qinco_group_combine, y.data_ptr(), _TYPES[y.dtype], y.stride(0), D, wt, w_type, self._place,
                      self.n, self.k, out.data_ptr())
        return out

    def _combine_grad(self, dout, y, weights, need_dy, need_dw):
        D = y.shape[1]
        dy = y.new_empty((self.n * self.k, D)) if need_dy else None
        dw = weights.new_empty((self.n, self.k)) if need_dw else None
        on_its_device(self._index, self._lib.qinco_group_combine_grad, dout.data_ptr(), dout.stride(0), y.data_ptr(), y.stride(0),
                      _TYPES[y.dtype], D, weights.data_ptr(), _TYPES[weights.dtype], self._place, self._end, self.n, self.k,
                      dy.data_ptr() if need_dy else None, dw.data_ptr() if need_dw else None)
        return dy, dw


def _gather_grad(ctx, dout):
    if forward_ad._current_level >= 0:
        _no_tangents(dout)
    return ctx.groups._combine(unit_rows(dout), None), None, None


def _combine_grad(ctx, dout):
    if forward_ad._current_level >= 0:
        _no_tangents(dout)
    dout = unit_rows(dout)
    if not ctx.weighted:
        return ctx.groups._gather(dout), None, None, None
    y, weights = ctx.saved_tensors
    need_dy, need_dw = ctx.needs_input_grad[:2]
    return (*ctx.groups._combine_grad(dout, y, weights, need_dy, need_dw), None, None)


# Second derivatives are refused.  once_differentiable() costs as much as the rest of a small backward call, and without create_graph (the
# gradient mode is off then) there is nothing to refuse.
_gather_grad_once, _combine_grad_once = once_differentiable(_gather_grad), once_differentiable(_combine_grad)


# traced: a trace goes on from here, with tensors that nothing has looked at
class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups, traced):
        ctx.groups = groups
        return groups._gather(groups._rows(x, groups.n, "x") if traced else x)

    @staticmethod
    def backward(ctx, dout):
        return _gather_grad_once(ctx, dout) if torch.is_grad_enabled() else _gather_grad(ctx, dout)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, groups, traced):
        if traced:
            y, weights = groups._combine_args(y, weights)
        ctx.groups, ctx.weighted = groups, weights is not None
        if weights is not None:
            ctx.save_for_backward(y, weights)
        return groups._combine(y, weights)

    @staticmethod
    def backward(ctx, dout):
        return _combine_grad_once(ctx, dout) if torch.is_grad_enabled() else _combine_grad(ctx, dout)
