"""Token plans and scaled table lookups (csrc/tokens.hip).

    p = plan(ids, n_groups)                 # stable sort of tokens by id
    y = lookup(table, ids)                  # table[ids], differentiable
    y = lookup(table, ids, weights)         # sum_k weights[.., k] table[ids[.., k]]

The map tables of the reference are read this way: eight trilinear corner
weights of a voxel (slam/model_components/voxel_helpers_voxfusion.py:72-123),
eight inverse-distance neighbours of a point
(slam/model_components/decoder_pointslam.py:135-160).  The gradient of the
table is summed over the tokens sorted by row, in token order and in f32: no
atomics, so equal inputs give equal bits.  Ids outside the table (the -1 of a
missing neighbour) read as a row of zeros and get no gradient.

CUDA tensors only (no CPU fallback).  Nothing is kept between calls: the
workspaces come from torch's allocator on the caller's stream, so calls may be
captured into graphs and run on several streams."""
from __future__ import annotations

import contextlib

import torch

from .. import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # XRD_F32 ..
_HERE = contextlib.nullcontext()


def refuse(message):
    raise _lib.XrdError(message)


def on_device(dev):
    """makes ``dev`` the current device for a block, at no cost if it is"""
    return _HERE if dev.index == torch.cuda.current_device() else \
        torch.cuda.device(dev)


def raw_stream(dev):
    """the caller's current stream on ``dev`` as an address"""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def dense_rows(t):
    """a 2-D tensor whose rows are contiguous (columns side by side, any
    distance between rows), copied only if it is not one"""
    if t.is_contiguous():
        return t
    s = t.stride()
    return t if s[0] >= 0 and (s[1] == 1 or t.shape[1] == 1) else \
        t.contiguous()


def _check_ids(ids, what):
    if not ids.is_cuda:
        refuse(f'{what}: CUDA tensors only (no CPU fallback)')
    if ids.dtype not in (torch.int32, torch.int64):
        refuse(f'{what}: ids must be int32 or int64, got {ids.dtype}')


class TokenPlan:
    """``order`` [n] i32: token numbers sorted by id (equal ids in token
    order, ids outside the groups last); ``starts`` [n_groups + 1] i32: group g
    is ``order[starts[g]:starts[g + 1]]``; ``rank`` [n] i32 or None:
    ``rank[order[i]] == i``"""

    def __init__(self, order, starts, rank, n_groups):
        self.order, self.starts, self.rank = order, starts, rank
        self.n_groups = n_groups


def plan(ids, n_groups, rank=False):
    """sort the tokens ``ids`` (any shape, i32 / i64) into ``n_groups``"""
    _check_ids(ids, 'plan')
    n_groups = int(n_groups)
    if n_groups < 1:
        refuse('plan: n_groups must be at least 1')
    if ids.numel() > _lib.MAX_TOKENS or n_groups > _lib.MAX_TOKENS:
        refuse(f'plan: {ids.numel()} tokens in {n_groups} groups: too many')
    order, starts, where = _plan(ids.contiguous(), n_groups, rank)
    return TokenPlan(order, starts, where, n_groups)


def _plan(ids, n_groups, rank=False):
    lib = _lib.lib()
    dev, n = ids.device, ids.numel()
    with on_device(dev):
        sizes = (n, n_groups + 1, n if rank else 0,
                 lib.xrd_token_plan_ws_ints(n, n_groups))
        if sizes[3] < 0:
            refuse(f'plan: {n} tokens in {n_groups} groups: not supported')
        order, starts, where, ws = (
            torch.empty(v, dtype=torch.int32, device=dev) for v in sizes)
        _lib.check(lib.xrd_token_plan(
            n, n_groups, ids.data_ptr(), ids.element_size(), order.data_ptr(),
            starts.data_ptr(), where.data_ptr() if rank else None,
            ws.data_ptr(), raw_stream(dev)), 'xrd_token_plan')
    return order, starts, where if rank else None


def _lookup(table, ids, weights, k, scale):
    lib = _lib.lib()
    dev, n = table.device, ids.numel() // k
    rows, dim = table.shape
    with on_device(dev):
        table = dense_rows(table)
        out = torch.empty(n, dim, dtype=table.dtype, device=dev)
        _lib.check(lib.xrd_lookup_fwd(
            DTYPES[table.dtype], n, k, rows, dim, table.data_ptr(),
            table.stride(0), ids.data_ptr(), ids.element_size(),
            None if weights is None else weights.data_ptr(), scale,
            out.data_ptr(), raw_stream(dev)), 'xrd_lookup_fwd')
    return out


class _LookupFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, weights, k, scale, token_plan):
        need_w = ctx.needs_input_grad[2]
        ctx.k, ctx.scale, ctx.plan = k, scale, token_plan
        ctx.shape, ctx.dtype = table.shape, table.dtype
        # the table is needed for the weights' gradient alone
        ctx.save_for_backward(table if need_w else None, ids, weights)
        return _lookup(table, ids, weights, k, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        lib = _lib.lib()
        table, ids, weights = ctx.saved_tensors
        (rows, dim), k, scale = ctx.shape, ctx.k, ctx.scale
        dev, dtype = dout.device, DTYPES[ctx.dtype]
        n = ids.numel() // k
        need_table, _, need_w = ctx.needs_input_grad[:3]
        dtable = dw = None
        wp = None if weights is None else weights.data_ptr()
        with on_device(dev):
            dout = dense_rows(dout)
            st = raw_stream(dev)
            if need_table:
                p = ctx.plan
                order, starts = (p.order, p.starts) if p is not None else \
                    _plan(ids, max(rows, 1))[:2]
                dtable = torch.empty(rows, dim, dtype=ctx.dtype, device=dev)
                ws = torch.empty(lib.xrd_lookup_bwd_ws_floats(n, k, dim),
                                 dtype=torch.float32, device=dev)
                _lib.check(lib.xrd_lookup_bwd_table(
                    dtype, n, k, rows, dim, dout.data_ptr(), dout.stride(0),
                    ids.data_ptr(), ids.element_size(), order.data_ptr(),
                    starts.data_ptr(), wp, scale, dtable.data_ptr(),
                    ws.data_ptr(), st), 'xrd_lookup_bwd_table')
            if need_w:
                table = dense_rows(table)
                dw = torch.empty(weights.shape, dtype=torch.float32,
                                 device=dev)
                _lib.check(lib.xrd_lookup_bwd_weights(
                    dtype, n, k, rows, dim, table.data_ptr(), table.stride(0),
                    ids.data_ptr(), ids.element_size(), dout.data_ptr(),
                    dout.stride(0), scale, dw.data_ptr(), st),
                    'xrd_lookup_bwd_weights')
        return dtable, None, dw, None, None, None


def lookup(table, ids, weights=None, scale=1.0, plan=None):
    """table [rows, dim] (f32 / bf16 / f16), ids i32 / i64.

    Without ``weights``: ``scale * table[ids]``, shape ids.shape + (dim,).
    With ``weights`` (ids' shape [..., k], taken as f32):
    ``scale * sum_k weights[..., k] * table[ids[..., k]]``, shape [..., dim].

    Differentiable in table and weights (once).  ``plan``: a TokenPlan of these
    ids over the table's rows, to be used by the backward pass instead of
    sorting them there."""
    if not table.is_cuda:
        refuse('lookup: CUDA tensors only (no CPU fallback)')
    _check_ids(ids, 'lookup')
    dev, shape, lead = table.device, table.shape, ids.shape
    if len(shape) != 2 or shape[1] < 1:
        refuse('lookup: table must be [rows, dim]')
    if table.dtype not in DTYPES:
        refuse(f'lookup: table of {table.dtype}: float32, bfloat16 or float16')
    if ids.device != dev:
        refuse('lookup: ids on another device')
    k = 1
    if weights is not None:
        if weights.shape != lead or not lead or lead[-1] < 1:
            refuse('lookup: weights must have the shape of ids, [..., k]')
        if weights.device != dev:
            refuse('lookup: weights on another device')
        if not weights.is_floating_point():
            refuse('lookup: weights must be floats')
        k, lead = lead[-1], lead[:-1]
        weights = weights.float().contiguous()
    if plan is not None and (plan.n_groups != shape[0] or
                             plan.order.numel() != ids.numel() or
                             plan.order.device != dev):
        refuse('lookup: the plan is not one of these ids over the rows')
    ids = ids.contiguous()
    if torch.is_grad_enabled() and (table.requires_grad or (
            weights is not None and weights.requires_grad)):
        out = _LookupFn.apply(table, ids, weights, k, float(scale), plan)
    else:
        out = _lookup(table, ids, weights, k, float(scale))
    return out if len(lead) == 1 else out.view(*lead, shape[1])
