"""Rows of a mixture of experts: tokens sorted by expert, and the experts' rows weighted and summed back to tokens, both differentiable.  (The reference has no such operators.)

A place p = t * k + j is the j-th expert of token t.  The functions enqueue on the current stream and check shapes, types and devices on the host; nothing is copied to the host, so the routing may
change between the replays of a graph.  What they compute is in include/fp6mi.h.  They go through the torch extension where it is built, else through ctypes."""
import sys

import torch

from . import _lib, ops

_package = sys.modules[__package__]

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MAX_CHOSEN, MAX_EXPERTS = 64, 1024


class ExpertPlan:
    """Where an index [tokens, k] sends every place, int32 on the GPU: place[tokens * k], the row of a place among the sorted ones (a permutation); order[tokens * k], its inverse, -1 for
    rows behind the last one with an expert; offsets[experts + 1], the first row of every expert, and in the end the number of places that have one.  (One tensor, `table`, holds all three.)"""
    __slots__ = ("table", "tokens", "k", "experts")

    def __init__(self, table, tokens, k, experts):
        self.table, self.tokens, self.k, self.experts = table, tokens, k, experts

    @property
    def places(self):
        return self.tokens * self.k

    @property
    def offsets(self):
        return self.table[:self.experts + 1]

    @property
    def order(self):
        return self.table[self.experts + 1:self.experts + 1 + self.places]

    @property
    def place(self):
        return self.table[self.experts + 1 + self.places:]

    def _addresses(self):
        """Of offsets, order, place and the number of places that have an expert."""
        t = self.table
        if t.dtype != torch.int32 or t.shape != (self.experts + 1 + 2 * self.places,) or self.experts < 1 or not t.is_contiguous() or t.device.type != "cuda":
            raise ValueError("the plan must be that of expert_sort or expert_plan")
        p = t.data_ptr()
        return p, p + 4 * (self.experts + 1), p + 4 * (self.experts + 1 + self.places), p + 4 * self.experts

    def __repr__(self):
        return "ExpertPlan(tokens=%d, k=%d, experts=%d)" % (self.tokens, self.k, self.experts)


# ---------------------------------------------------------------------------------------------------------------- through ctypes (the extension makes the same checks, and its own autograd functions)
def _sorted(x, index, experts):
    """(rows or None, plan) of x (or None) by index."""
    dev = index.device
    if index.dtype not in (torch.int32, torch.int64) or index.dim() != 2 or dev.type != "cuda":
        raise ValueError("index must be a 2-D int32 or int64 tensor [tokens, k] on the GPU")
    T, k = index.shape
    if not 1 <= k <= MAX_CHOSEN or not 1 <= experts <= MAX_EXPERTS or T * k > 1 << 30:
        raise ValueError("need 1 to %d experts of a token, 1 to %d in all, and up to 2^30 places" % (MAX_CHOSEN, MAX_EXPERTS))
    rows = None
    if x is not None:
        if x.dtype not in TYPES or x.dim() != 2 or x.shape[0] != T or x.shape[1] < 1 or x.shape[1] > 1 << 24 or x.device != dev:
            raise ValueError("x must be float16, bfloat16 or float32 [tokens=%d, features], on the index's GPU" % T)
        x = x.resolve_neg()
        if x.stride(1) != 1 or (T > 1 and x.stride(0) < x.shape[1]):
            x = x.contiguous()
        rows = torch.empty(T * k, x.shape[1], dtype=x.dtype, device=dev)
    index = index.contiguous()
    plan = ExpertPlan(torch.empty(experts + 1 + 2 * T * k, dtype=torch.int32, device=dev), T, k, experts)
    offsets, order, place, _ = plan._addresses()
    L = _lib.lib()
    ops._launch("fp6mi_expert_sort", dev, L.fp6mi_expert_sort_workspace_bytes(T, k, experts), None, lambda stream, ws: L.fp6mi_expert_sort(
        stream, index.data_ptr(), index.dtype == torch.int64, offsets, order, place, ops._ptr(x), 0 if x is None else x.stride(0), ops._ptr(rows), T, k, experts,
        0 if x is None else x.shape[1], 0 if x is None else TYPES[x.dtype], ws))
    return rows, plan


def _check_rows(rows, plan, out_dtype):
    if rows.dtype not in TYPES or rows.dim() != 2 or rows.shape[0] != plan.places or not 1 <= rows.shape[1] <= 1 << 24 or rows.device != plan.table.device:
        raise ValueError("rows must be float16, bfloat16 or float32 [tokens * k = %d, features], on the plan's GPU" % plan.places)
    if out_dtype not in TYPES or (out_dtype != rows.dtype and rows.dtype != torch.float32):
        raise ValueError("sums have the rows' type, those of float32 rows any")


def _combined(rows, plan, weights, out_dtype):
    _check_rows(rows, plan, out_dtype)
    _, _, place, valid = plan._addresses()
    rows = rows.resolve_neg().contiguous()
    out = torch.empty(plan.tokens, rows.shape[1], dtype=out_dtype, device=rows.device)
    L = _lib.lib()
    ops._launch("fp6mi_expert_combine", rows.device, 0, None, lambda stream, ws: L.fp6mi_expert_combine(
        stream, rows.data_ptr(), place, valid, ops._ptr(weights), out.data_ptr(), plan.tokens, plan.k, rows.shape[1], TYPES[rows.dtype], TYPES[out_dtype]))
    return out


def _combined_backward(grad, rows, plan, weights, row_dtype, want_rows, want_weights):
    """(grad_rows, grad_weights), None where it is not wanted; rows only for those of the weights."""
    grad = grad.resolve_neg().contiguous()
    dev, H = grad.device, grad.shape[1]
    _, _, place, valid = plan._addresses()
    grad_rows = torch.empty(plan.places, H, dtype=row_dtype, device=dev) if want_rows else None
    grad_weights = torch.empty(plan.tokens, plan.k, dtype=torch.float32, device=dev) if want_weights else None
    L = _lib.lib()
    ops._launch("fp6mi_expert_combine_backward", dev, 0, None, lambda stream, ws: L.fp6mi_expert_combine_backward(
        stream, grad.data_ptr(), ops._ptr(rows), place, valid, ops._ptr(weights), ops._ptr(grad_rows), ops._ptr(grad_weights), plan.tokens, plan.k, H, TYPES[row_dtype], TYPES[grad.dtype]))
    return grad_rows, grad_weights


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, index, experts, plans):
        rows, plan = _sorted(x, index, experts)
        plans.append(plan)
        ctx.plan = plan
        return rows

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _combined(grad, ctx.plan, None, grad.dtype), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan, out_dtype):
        rows = rows.resolve_neg().contiguous()
        ctx.plan, ctx.row_dtype = plan, rows.dtype
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weights)
        return _combined(rows, plan, weights, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        rows, weights = ctx.saved_tensors
        want_rows, want_weights = ctx.needs_input_grad[:2]
        return _combined_backward(grad, rows, ctx.plan, weights, ctx.row_dtype, want_rows, want_weights) + (None, None)


# ---------------------------------------------------------------------------------------------------------------- the operators
def expert_plan(index, experts):
    """The ExpertPlan of index, int32 or int64 [tokens, k] on the GPU: the experts of every token, numbers outside 0..experts-1 (-1, say) for none."""
    _ext = _package._ext
    if _ext is not None:
        return ExpertPlan(_ext.expert_sort(None, index, experts)[1], *index.shape, experts)
    return _sorted(None, index, experts)[1]


def expert_sort(x, index, experts):
    """(rows, plan): rows[tokens * k, features] holds row t of x for each of token t's experts, sorted by expert, ties in the order of tokens and of their places; rows behind the last one that
    has an expert are zeros.  Differentiable in x (float16, bfloat16 or float32): the gradients of a token's rows are summed in float32."""
    _ext = _package._ext
    _refuse_unseen(x)
    differentiates = _differentiates(x)
    if _ext is not None:
        rows, table = _ext.expert_sort(x, index, experts)
        return rows, ExpertPlan(table, index.shape[0], index.shape[1], experts)
    if not differentiates:
        return _sorted(x, index, experts)
    plans = []
    rows = _Sort.apply(x, index, experts, plans)
    return rows, plans[0]


def expert_combine(rows, plan, weights=None, dtype=None):
    """out[t] = sum over token t's experts of weights[t, j] * (its row among the sorted ones), in float32, rounded once; without weights all are 1.  weights: [tokens, k], float32 (other float types
    are converted).  dtype: of out, the rows' type by default; float32 rows may be summed to float16 or bfloat16.  Differentiable in rows and weights."""
    _ext = _package._ext
    differentiates = _differentiates(rows)
    if weights is None:
        _refuse_unseen(rows)
    else:
        _refuse_unseen(rows, weights)
        differentiates |= _differentiates(weights)
    if _ext is not None:
        return _ext.expert_combine(rows, plan.table, plan.tokens, plan.k, plan.experts, weights, dtype)
    if weights is not None:
        if weights.shape != (plan.tokens, plan.k) or not weights.is_floating_point() or weights.device != plan.table.device:
            raise ValueError("weights must be float [tokens=%d, k=%d] on the plan's GPU, got %s" % (plan.tokens, plan.k, list(weights.shape)))
        weights = weights.float().resolve_neg().contiguous()
    dtype = rows.dtype if dtype is None else dtype
    if differentiates:
        _check_rows(rows, plan, dtype)
        return _Combine.apply(rows, weights, plan, dtype)
    return _combined(rows, plan, weights, dtype)


from .module import _differentiates, _refuse_unseen  # noqa: E402  (it imports the package's functions)
