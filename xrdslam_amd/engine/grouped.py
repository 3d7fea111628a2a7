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
from .tokens import DTYPES, address, dense_rows, require


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, starts, bias, relu):
        lib = _lib.lib()
        dev = x.device
        m, n_in = x.shape
        e, n_out, _ = weight.shape
        with torch.cuda.device(dev):
            xr, w = dense_rows(x.detach()), weight.detach().contiguous()
            b = None if bias is None else bias.detach().contiguous()
            y = torch.empty(m, n_out, dtype=x.dtype, device=dev)
            _lib.check(lib.xrd_grouped_fwd(
                DTYPES[x.dtype], m, e, n_in, n_out, address(xr), xr.stride(0),
                _lib.ptr(w), _lib.ptr(b), _lib.ptr(starts), int(relu),
                _lib.ptr(y), _lib.stream_ptr(dev)), 'xrd_grouped_fwd')
        ctx.relu, ctx.sizes = relu, (m, e, n_in, n_out)
        need = ctx.needs_input_grad
        ctx.save_for_backward(x if need[1] or need[3] else None,
                              weight if need[0] else None, starts,
                              y if relu else None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib = _lib.lib()
        x, weight, starts, y = ctx.saved_tensors
        m, e, n_in, n_out = ctx.sizes
        dev, dtype = dy.device, DTYPES[dy.dtype]
        dx = dw = db = None
        need_x, need_w, _, need_b, _ = ctx.needs_input_grad
        with torch.cuda.device(dev):
            st = _lib.stream_ptr(dev)
            dz = dense_rows(dy)
            if ctx.relu:
                masked = torch.empty(m, n_out, dtype=dy.dtype, device=dev)
                _lib.check(lib.xrd_grouped_relu_grad(
                    dtype, m, n_out, _lib.ptr(y), address(dz), dz.stride(0),
                    _lib.ptr(masked), st), 'xrd_grouped_relu_grad')
                dz = masked
            if need_x:
                w = weight.detach().contiguous()
                dx = torch.empty(m, n_in, dtype=dy.dtype, device=dev)
                _lib.check(lib.xrd_grouped_bwd_x(
                    dtype, m, e, n_in, n_out, address(dz), dz.stride(0),
                    _lib.ptr(w), _lib.ptr(starts), _lib.ptr(dx), st),
                    'xrd_grouped_bwd_x')
            if need_w or need_b:
                xr = dense_rows(x.detach())
                dw = torch.empty(e, n_out, n_in, dtype=dy.dtype, device=dev)
                if need_b:
                    db = torch.empty(e, n_out, dtype=dy.dtype, device=dev)
                ws = torch.empty(lib.xrd_grouped_ws_floats(
                    dtype, m, e, n_in, n_out), dtype=torch.float32, device=dev)
                _lib.check(lib.xrd_grouped_bwd_w(
                    dtype, m, e, n_in, n_out, address(xr), xr.stride(0),
                    address(dz), dz.stride(0), _lib.ptr(starts), _lib.ptr(dw),
                    _lib.ptr(db), _lib.ptr(ws), st), 'xrd_grouped_bwd_w')
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
    require(x.is_cuda, 'linear: CUDA tensors only (no CPU fallback)')
    require(x.dim() == 2 and weight.dim() == 3 and
            weight.shape[2] == x.shape[1] and min(weight.shape) >= 1,
            'linear: x [m, in] and weight [groups, out, in] expected')
    require(x.dtype in DTYPES and weight.dtype == x.dtype,
            'linear: x and weight must share float32, bfloat16 or float16')
    require(starts.dtype == torch.int32 and starts.dim() == 1 and
            starts.numel() == weight.shape[0] + 1 and starts.is_contiguous(),
            'linear: starts must be i32 [groups + 1], contiguous')
    require(weight.device == x.device and starts.device == x.device,
            'linear: tensors on different devices')
    if bias is not None:
        require(bias.shape == weight.shape[:2] and bias.dtype == x.dtype and
                bias.device == x.device,
                'linear: bias must be [groups, out] of x\'s type and device')
    return _LinearFn.apply(x, weight, starts, bias, bool(relu))
