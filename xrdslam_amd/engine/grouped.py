"""The linear layer of several decoders at once (csrc/grouped.hip).

    p = tokens.plan(which_decoder, n_decoders, rank=True)
    x = tokens.lookup(points, p.order)                  # rows sorted by decoder
    h = linear(x, weight, p.starts, bias, relu=True)    # weight [e, out, in]
    y = tokens.lookup(h, p.rank)                        # back in point order

A point set that several local decoders share (one per room or sub-map) is a
ragged batch: decoder e owns rows starts[e] .. starts[e + 1].  ``starts`` stays
on the device; no size is read back.  CUDA tensors only (no CPU fallback)."""
from __future__ import annotations

import torch

from .tokens import DTYPES, call, ops, refuse


def linear(x, weight, starts, bias=None, relu=False):
    """y[r] = act(weight[e] @ x[r] + bias[e]), e the group of row r.

    x [m, in], weight [groups, out, in], bias [groups, out] or None, all of
    one type (f32 / bf16 / f16); starts [groups + 1] i32 on the device,
    ascending: group e owns rows starts[e] .. starts[e + 1] - 1.  Rows of no
    group (behind starts[-1], before starts[0]) come back as zeros and get a
    zero gradient.  ``relu`` applies max(., 0) to the result.  Differentiable
    in x, weight and bias (once, backward).  At most 65536 groups."""
    if not x.is_cuda:
        refuse('linear: CUDA tensors only (no CPU fallback)')
    dev, ty, ws = x.device, x.dtype, weight.shape
    if x.dim() != 2 or len(ws) != 3 or ws[2] != x.shape[1] or min(ws) < 1:
        refuse('linear: x [m, in] and weight [groups, out, in] expected')
    if ty not in DTYPES or weight.dtype != ty:
        refuse('linear: x and weight must share float32, bfloat16 or float16')
    if starts.dtype != torch.int32 or starts.shape != (ws[0] + 1, ) or \
            not starts.is_contiguous():
        refuse('linear: starts must be i32 [groups + 1], contiguous')
    if weight.device != dev or starts.device != dev:
        refuse('linear: tensors on different devices')
    if bias is not None and (bias.shape != ws[:2] or bias.dtype != ty or
                             bias.device != dev):
        refuse('linear: bias must be [groups, out] of x\'s type and device')
    return call(ops().linear.default, x, weight, starts, bias, bool(relu))
