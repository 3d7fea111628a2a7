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

from .. import _lib
from .tokens import DTYPES, dense_rows, on_device, raw_stream, refuse


def _linear(x, weight, starts, bias, relu):
    lib = _lib.lib()
    dev = x.device
    m, n_in = x.shape
    e, n_out, _ = weight.shape
    with on_device(dev):
        x, weight = dense_rows(x), weight.contiguous()
        if bias is not None:
            bias = bias.contiguous()
        y = torch.empty(m, n_out, dtype=x.dtype, device=dev)
        _lib.check(lib.xrd_grouped_fwd(
            DTYPES[x.dtype], m, e, n_in, n_out, x.data_ptr(), x.stride(0),
            weight.data_ptr(), None if bias is None else bias.data_ptr(),
            starts.data_ptr(), relu, y.data_ptr(), raw_stream(dev)),
            'xrd_grouped_fwd')
    return y


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, starts, bias, relu):
        y = _linear(x, weight, starts, bias, relu)
        need_x, need_w, _, need_b, _ = ctx.needs_input_grad
        ctx.relu, ctx.sizes = relu, (*x.shape, *weight.shape[:2])
        ctx.save_for_backward(x if need_w or need_b else None,
                              weight if need_x else None, starts,
                              y if relu else None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib = _lib.lib()
        x, weight, starts, y = ctx.saved_tensors
        m, n_in, e, n_out = ctx.sizes
        dev, ty = dy.device, dy.dtype
        dtype = DTYPES[ty]
        dx = dw = db = None
        need_x, need_w, _, need_b, _ = ctx.needs_input_grad
        with on_device(dev):
            st = raw_stream(dev)
            dz = dense_rows(dy)
            if ctx.relu:
                masked = torch.empty(m, n_out, dtype=ty, device=dev)
                _lib.check(lib.xrd_grouped_relu_grad(
                    dtype, m, n_out, y.data_ptr(), dz.data_ptr(),
                    dz.stride(0), masked.data_ptr(), st),
                    'xrd_grouped_relu_grad')
                dz = masked
            dzp, dzs, sp = dz.data_ptr(), dz.stride(0), starts.data_ptr()
            if need_x:
                weight = weight.contiguous()
                dx = torch.empty(m, n_in, dtype=ty, device=dev)
                _lib.check(lib.xrd_grouped_bwd_x(
                    dtype, m, e, n_in, n_out, dzp, dzs, weight.data_ptr(), sp,
                    dx.data_ptr(), st), 'xrd_grouped_bwd_x')
            if need_w or need_b:
                x = dense_rows(x)
                dw = torch.empty(e, n_out, n_in, dtype=ty, device=dev)
                if need_b:
                    db = torch.empty(e, n_out, dtype=ty, device=dev)
                words = lib.xrd_grouped_ws_floats(dtype, m, e, n_in, n_out)
                ws = torch.empty(words, device=dev) if words > 0 else None
                _lib.check(lib.xrd_grouped_bwd_w(
                    dtype, m, e, n_in, n_out, x.data_ptr(), x.stride(0), dzp,
                    dzs, sp, dw.data_ptr(),
                    db.data_ptr() if need_b else None,
                    None if ws is None else ws.data_ptr(), st),
                    'xrd_grouped_bwd_w')
                if not need_w:
                    dw = None
        return dx, dw, None, db, None


def linear(x, weight, starts, bias=None, relu=False):
    """y[r] = act(weight[e] @ x[r] + bias[e]), e the group of row r.

    x [m, in], weight [groups, out, in], bias [groups, out] or None, all of
    one type (f32 / bf16 / f16); starts [groups + 1] i32 on the device,
    ascending: group e owns rows starts[e] .. starts[e + 1] - 1.  Rows of no
    group (behind starts[-1], before starts[0]) come back as zeros and get a
    zero gradient.  ``relu`` applies max(., 0) to the result.  Differentiable
    in x, weight and bias (once)."""
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
    if torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad or
            (bias is not None and bias.requires_grad)):
        return _LinearFn.apply(x, weight, starts, bias, bool(relu))
    return _linear(x, weight, starts, bias, bool(relu))
