"""Rows of a table by integer ids, scaled, and the gradient of that: `tf.nn.embedding_lookup` / `tf.gather` as they
appear inside a likelihood or a surrogate's network, on gfx950 kernels (include/bvi.h: bvi_lookup, bvi_lookup_plan,
bvi_lookup_grad).  `symbolic.gather` is the spelling for likelihood callables.

Tables are [rows, width] (or [rows]) in float32, bfloat16 or float16 with any row stride; ids int32 or int64 of any shape.
An id outside [0, rows) is padding: it reads zeros and takes no part in the gradient.  Products and sums are in float32,
rounded once to the table's type.  Derivatives go backwards and forwards (torch.autograd, forward_ad); torch.func
transforms raise.  Everything runs on the current stream of the table's device; nothing synchronises, and
every call can be recorded into a graph.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _native


def _check_ids(ids, device):
    if not isinstance(ids, torch.Tensor) or ids.dtype not in _native.ID_TYPES:
        raise TypeError('ids must be an int32 or int64 tensor, got %s'
                        % (ids.dtype if isinstance(ids, torch.Tensor) else type(ids).__name__))
    if ids.device != device:
        raise ValueError('ids are on %s, the other operand on %s' % (ids.device, device))


def _rows_view(t, what):
    """t[rows, width] as (tensor, row stride) with unit stride inside a row; a copy only where the layout has none."""
    if not t.is_cuda:
        raise _native.BviError('%s must be on the GPU (there is no CPU fallback); got %s' % (what, t.device))
    if t.dtype not in _native.ELEMENT_TYPES:
        raise TypeError('%s must be float32, bfloat16 or float16, got %s' % (what, t.dtype))
    rows, width = t.shape
    if width > 1 and t.stride(1) != 1 or rows > 1 and t.stride(0) < width:
        t = t.contiguous()
    return t, (t.stride(0) if rows > 1 else width)


def _differentiated(t):
    """Whether autograd follows t: backwards, or forwards by a tangent (which `requires_grad` says nothing about)."""
    return (t.requires_grad and torch.is_grad_enabled()
            or _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None)


class LookupPlan:
    """The sorted order of `ids` over a table of `num_rows`: what the gradient needs of the ids alone.  A program whose
    ids stay the same (a fixed dataset) makes one and hands it to every `lookup` / `lookup_grad`; without one each
    gradient sorts anew.  The plan describes the ids as they were when it was made."""

    def __init__(self, ids, num_rows):
        _check_ids(ids, ids.device if isinstance(ids, torch.Tensor) else None)
        if not ids.is_cuda:
            raise _native.BviError('ids must be on the GPU (there is no CPU fallback); got %s' % ids.device)
        self.num_rows, self.n, self.device = int(num_rows), ids.numel(), ids.device
        if self.num_rows < 1:
            raise ValueError('num_rows must be at least 1, got %d' % self.num_rows)
        self.buffer = _native.lookup_plan(ids.contiguous(), self.num_rows)

    def check(self, n, num_rows, device):
        if (self.n, self.num_rows, self.device) != (n, num_rows, device):
            raise ValueError('this plan is for %d ids over %d rows on %s; the call has %d ids over %d rows on %s'
                             % (self.n, self.num_rows, self.device, n, num_rows, device))


def lookup_grad(grad_out, ids, num_rows, scale=1.0, plan=None):
    """The table's gradient [num_rows, width] (or [num_rows] for grad_out of the ids' own shape): row r is `scale` times
    the sum of grad_out's rows whose id is r.  Rows that no id asks for are zero.  The sum's order is fixed by the
    ids, the sizes and the operands' alignment: the same call gives the same bits.  Linear in grad_out, and differentiable
    in it (the derivative is the lookup)."""
    if not isinstance(grad_out, torch.Tensor):
        raise TypeError('grad_out must be a tensor, got %s' % type(grad_out).__name__)
    _check_ids(ids, grad_out.device)
    num_rows = int(num_rows)
    if num_rows < 1:
        raise ValueError('num_rows must be at least 1, got %d' % num_rows)
    flat = grad_out.shape == ids.shape
    if not flat and (grad_out.dim() != ids.dim() + 1 or grad_out.shape[:-1] != ids.shape or grad_out.shape[-1] < 1):
        raise ValueError('grad_out must have shape %s or %s + (width,), got %s'
                         % (tuple(ids.shape), tuple(ids.shape), tuple(grad_out.shape)))
    if plan is not None:
        plan.check(ids.numel(), num_rows, grad_out.device)
    if _differentiated(grad_out):
        return _LookupGrad.apply(grad_out, ids, num_rows, float(scale), plan)
    return _gradient(grad_out, ids, num_rows, float(scale), plan, flat)


def _gradient(grad_out, ids, num_rows, scale, plan, flat):
    n, width = ids.numel(), 1 if flat else grad_out.shape[-1]
    g, stride = _rows_view(grad_out.reshape(n, width), 'grad_out')
    ids = ids.contiguous()
    out = torch.empty((num_rows,) if flat else (num_rows, width), dtype=g.dtype, device=g.device)
    _native.lookup_grad(g, n, width, stride, ids, None if plan is None else plan.buffer, num_rows, scale, out)
    return out


def _forward(table, ids, scale):
    t, stride = _rows_view(table[:, None] if table.dim() == 1 else table, 'table')
    ids = ids.contiguous()
    out = torch.empty(tuple(ids.shape) + tuple(table.shape[1:]), dtype=t.dtype, device=t.device)
    _native.lookup(t, t.shape[0], t.shape[1], stride, ids, scale, out)
    return out


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, plan):
        ctx.scale, ctx.plan, ctx.rows = scale, plan, table.shape[0]
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        return _forward(table, ids, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        ids, = ctx.saved_tensors
        return lookup_grad(grad_out, ids, ctx.rows, ctx.scale, ctx.plan), None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):                           # the map is linear in the table
        ids, = ctx.saved_tensors
        return lookup(tangent, ids, ctx.scale, ctx.plan)


class _LookupGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad_out, ids, num_rows, scale, plan):
        ctx.rows, ctx.scale, ctx.plan = num_rows, scale, plan
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        return _gradient(grad_out, ids, num_rows, scale, plan, grad_out.dim() == ids.dim())

    @staticmethod
    def backward(ctx, grad_table):
        ids, = ctx.saved_tensors
        return lookup(grad_table, ids, ctx.scale, ctx.plan), None, None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        ids, = ctx.saved_tensors
        return lookup_grad(tangent, ids, ctx.rows, ctx.scale, ctx.plan)


def lookup(table, ids, scale=1.0, plan=None):
    """scale * table[ids]: shape ids.shape + (width,), or ids.shape for a one-dimensional table.  Differentiable once in
    the table, backwards and in forward mode; `plan` (see `LookupPlan`) is used by the gradient only."""
    if not isinstance(table, torch.Tensor) or table.dim() not in (1, 2):
        raise ValueError('table must be a tensor [rows, width] or [rows]')
    if table.shape[0] < 1 or table.shape[-1] < 1:
        raise ValueError('table has no entries: shape %s' % (tuple(table.shape),))
    _check_ids(ids, table.device)
    if plan is not None:
        plan.check(ids.numel(), table.shape[0], table.device)
    if _differentiated(table):
        return _Lookup.apply(table, ids, float(scale), plan)
    return _forward(table, ids, float(scale))
