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
captured into graphs (after one call outside, which loads the kernels; a
backward pass with no older autograd graph of its leaves alive) and run on
several streams.  The autograd nodes are host
C++ (csrc_torch/token_ops.cpp) over the C ABI."""
from __future__ import annotations

import os

import torch

from .. import _lib

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_ops = None


def refuse(message):
    raise _lib.XrdError(message)


def ops():
    """torch.ops.xrdslam, loaded (and built, if nothing is) on first use"""
    global _ops
    if _ops is None:
        from .. import build_torch_ext as ext
        if not os.path.exists(ext.TOKEN_LIB):
            ext.build()
        torch.ops.load_library(ext.TOKEN_LIB)
        _ops = torch.ops.xrdslam
    return _ops


def call(op, *args):
    """an operator, its refusals raised as XrdError"""
    try:
        return op(*args)
    except RuntimeError as e:
        if str(e).startswith('xrd_'):
            raise _lib.XrdError(str(e).splitlines()[0]) from e
        raise


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
    order, starts, where = call(ops().plan.default, ids, n_groups, bool(rank))
    return TokenPlan(order, starts, where if rank else None, n_groups)


def lookup(table, ids, weights=None, scale=1.0, plan=None):
    """table [rows, dim] (f32 / bf16 / f16), ids i32 / i64.

    Without ``weights``: ``scale * table[ids]``, shape ids.shape + (dim,).
    With ``weights`` (ids' shape [..., k], taken as f32):
    ``scale * sum_k weights[..., k] * table[ids[..., k]]``, shape [..., dim].

    Differentiable in table and weights (once, backward).  ``plan``: a TokenPlan of these
    ids over the table's rows, to be used by the backward pass instead of
    sorting them there."""
    if not table.is_cuda:
        refuse('lookup: CUDA tensors only (no CPU fallback)')
    _check_ids(ids, 'lookup')
    dev, shape = table.device, table.shape
    if len(shape) != 2 or shape[1] < 1:
        refuse('lookup: table must be [rows, dim]')
    if table.dtype not in DTYPES:
        refuse(f'lookup: table of {table.dtype}: float32, bfloat16 or float16')
    if ids.device != dev:
        refuse('lookup: ids on another device')
    if weights is not None:
        if weights.shape != ids.shape or not ids.dim() or ids.shape[-1] < 1:
            refuse('lookup: weights must have the shape of ids, [..., k]')
        if weights.device != dev:
            refuse('lookup: weights on another device')
        if not weights.is_floating_point():
            refuse('lookup: weights must be floats')
    if isinstance(scale, torch.Tensor) and scale.requires_grad and \
            torch.is_grad_enabled():
        refuse('lookup: scale is a number, a tensor gets no gradient here')
    order = starts = None
    if plan is not None:
        order, starts = plan.order, plan.starts
        if plan.n_groups != shape[0] or order.numel() != ids.numel() or \
                starts.numel() != shape[0] + 1 or order.device != dev or \
                starts.device != dev or order.dtype != torch.int32 or \
                starts.dtype != torch.int32 or \
                not (order.is_contiguous() and starts.is_contiguous()):
            refuse('lookup: the plan is not one of these ids over the rows')
    return call(ops().lookup.default, table, ids, weights, float(scale), order,
                starts)
