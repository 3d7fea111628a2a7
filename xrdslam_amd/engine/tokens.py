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

import torch

from .. import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # XRD_F32 ..


def require(ok, message):
    if not ok:
        raise _lib.XrdError(message)


def dense_rows(t):
    """a 2-D tensor whose rows are contiguous (columns side by side, any
    distance between rows), copied only if it is not one"""
    if t.dim() == 2 and t.stride(0) >= 0 and (t.stride(1) == 1 or
                                               t.shape[1] == 1):
        return t
    return t.contiguous()


def address(t):
    """device pointer of a tensor with strides of its own (``_lib.ptr`` takes
    dense ones)"""
    return None if t is None else t.data_ptr()


def _check_ids(ids, what):
    require(ids.is_cuda, f'{what}: CUDA tensors only (no CPU fallback)')
    require(ids.dtype in (torch.int32, torch.int64),
            f'{what}: ids must be int32 or int64, got {ids.dtype}')


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
    n_groups, n = int(n_groups), ids.numel()
    require(n_groups >= 1, 'plan: n_groups must be at least 1')
    lib = _lib.lib()
    words = lib.xrd_token_plan_ws_ints(n, n_groups)
    require(words >= 0, f'plan: {n} tokens in {n_groups} groups: too many')
    dev = ids.device
    with torch.cuda.device(dev):
        ids = ids.detach().contiguous()
        i = dict(dtype=torch.int32, device=dev)
        order = torch.empty(n, **i)
        starts = torch.empty(n_groups + 1, **i)
        where = torch.empty(n, **i) if rank else None
        ws = torch.empty(words, **i)
        _lib.check(lib.xrd_token_plan(
            n, n_groups, _lib.ptr(ids), ids.element_size(), _lib.ptr(order),
            _lib.ptr(starts), _lib.ptr(where), _lib.ptr(ws),
            _lib.stream_ptr(dev)), 'xrd_token_plan')
    return TokenPlan(order, starts, where, n_groups)


class _LookupFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, weights, k, scale, token_plan):
        lib = _lib.lib()
        dev = table.device
        n = ids.numel() // k
        rows, dim = table.shape
        with torch.cuda.device(dev):
            tab = dense_rows(table.detach())
            out = torch.empty(n, dim, dtype=table.dtype, device=dev)
            _lib.check(lib.xrd_lookup_fwd(
                DTYPES[table.dtype], n, k, rows, dim, address(tab),
                tab.stride(0), _lib.ptr(ids), ids.element_size(),
                _lib.ptr(weights), scale, _lib.ptr(out),
                _lib.stream_ptr(dev)), 'xrd_lookup_fwd')
        ctx.k, ctx.scale, ctx.plan = k, scale, token_plan
        # the table is needed for the weights' gradient alone
        ctx.shape, ctx.dtype = (rows, dim), table.dtype
        ctx.save_for_backward(
            table if ctx.needs_input_grad[2] else None, ids, weights)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        lib = _lib.lib()
        table, ids, weights = ctx.saved_tensors
        (rows, dim), k = ctx.shape, ctx.k
        dev, dtype = dout.device, DTYPES[ctx.dtype]
        n = ids.numel() // k
        dtable = dw = None
        with torch.cuda.device(dev):
            dout = dense_rows(dout)
            st = _lib.stream_ptr(dev)
            if ctx.needs_input_grad[0]:
                p = ctx.plan if ctx.plan is not None else \
                    plan(ids, max(rows, 1))
                dtable = torch.empty(rows, dim, dtype=ctx.dtype, device=dev)
                _lib.check(lib.xrd_lookup_bwd_table(
                    dtype, n, k, rows, dim, address(dout), dout.stride(0),
                    _lib.ptr(p.order), _lib.ptr(p.starts), _lib.ptr(weights),
                    ctx.scale, _lib.ptr(dtable), st), 'xrd_lookup_bwd_table')
            if ctx.needs_input_grad[2]:
                tab = dense_rows(table.detach())
                dw = torch.empty(n, k, dtype=torch.float32, device=dev)
                _lib.check(lib.xrd_lookup_bwd_weights(
                    dtype, n, k, rows, dim, address(tab), tab.stride(0),
                    _lib.ptr(ids), ids.element_size(), address(dout),
                    dout.stride(0), ctx.scale, _lib.ptr(dw), st),
                    'xrd_lookup_bwd_weights')
                dw = dw.view(weights.shape)
        return dtable, None, dw, None, None, None


def lookup(table, ids, weights=None, scale=1.0, plan=None):
    """table [rows, dim] (f32 / bf16 / f16), ids i32 / i64.

    Without ``weights``: ``scale * table[ids]``, shape ids.shape + (dim,).
    With ``weights`` (ids' shape [..., k], taken as f32):
    ``scale * sum_k weights[..., k] * table[ids[..., k]]``, shape [..., dim].

    Differentiable in table and weights (once).  ``plan``: a TokenPlan of these
    ids over the table's rows, to be used by the backward pass instead of
    sorting them there."""
    require(table.is_cuda, 'lookup: CUDA tensors only (no CPU fallback)')
    _check_ids(ids, 'lookup')
    require(table.dim() == 2 and table.shape[1] >= 1,
            'lookup: table must be [rows, dim]')
    require(table.dtype in DTYPES,
            f'lookup: table of {table.dtype}: float32, bfloat16 or float16')
    require(ids.device == table.device, 'lookup: ids on another device')
    k, lead = 1, ids.shape
    if weights is not None:
        require(weights.shape == ids.shape and ids.dim() >= 1 and
                ids.shape[-1] >= 1,
                'lookup: weights must have the shape of ids, [..., k]')
        require(weights.device == table.device,
                'lookup: weights on another device')
        require(weights.is_floating_point(), 'lookup: weights must be floats')
        k, lead = int(ids.shape[-1]), ids.shape[:-1]
        weights = weights.float().contiguous()
    if plan is not None:
        require(plan.n_groups == table.shape[0] and
                plan.order.numel() == ids.numel() and
                plan.order.device == table.device,
                'lookup: the plan is not one of these ids over the rows')
    out = _LookupFn.apply(table, ids.detach().contiguous(), weights, k,
                          float(scale), plan)
    return out.view(*lead, table.shape[1])
