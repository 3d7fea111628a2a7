"""Refusals of the token and grouped-product operators (no GPU needed): the C
entry points report bad arguments before any HIP call, the Python ones refuse
host tensors, and the plain forms the GPU tests compare against agree with
torch's own autograd."""
import ctypes

import numpy as np
import pytest
import torch

import token_util as tu
from xrdslam_amd import _lib
from xrdslam_amd.engine import grouped, tokens

BUF = (ctypes.c_double * 64)()
P = ctypes.cast(BUF, ctypes.c_void_p)


def test_plan_refusals():
    f = _lib.lib().xrd_token_plan
    assert f(-1, 4, P, 4, P, P, None, P, None) == 1
    assert f(4, 0, P, 4, P, P, None, P, None) == 1
    assert f(4, 4, P, 2, P, P, None, P, None) == 1
    assert f(4, 4, None, 4, P, P, None, P, None) == 1
    assert f(4, 4, P, 4, None, P, None, P, None) == 1
    assert f(4, 4, P, 4, P, None, None, P, None) == 1
    assert f(4, 4, P, 4, P, P, None, None, None) == 1
    assert f(1 << 31, 4, P, 4, P, P, None, P, None) == 3
    assert f(4, 1 << 31, P, 4, P, P, None, P, None) == 3
    ws = _lib.lib().xrd_token_plan_ws_ints
    assert ws(-1, 4) == -1 and ws(4, 0) == -1 and ws(1 << 31, 4) == -1
    assert ws(0, 1) >= 1 and ws(1000, 16) >= 1


def test_lookup_refusals():
    lib = _lib.lib()

    def fwd(dtype=0, n=4, k=1, rows=4, dim=2, table=P, stride=2, ids=P, ib=4,
            out=P):
        return lib.xrd_lookup_fwd(dtype, n, k, rows, dim, table, stride, ids,
                                  ib, None, 1.0, out, None)
    assert fwd(dtype=3) == 1 and fwd(dtype=-1) == 1 and fwd(n=-1) == 1
    assert fwd(k=0) == 1 and fwd(rows=-1) == 1 and fwd(dim=0) == 1
    assert fwd(stride=-2) == 1 and fwd(ib=3) == 1 and fwd(table=None) == 1
    assert fwd(ids=None) == 1 and fwd(out=None) == 1
    assert fwd(n=0, table=None, ids=None, out=None) == 0

    def bwd(dtype=0, n=4, k=1, rows=4, dim=2, table=P, stride=2, ids=P, ib=4,
            dout=P, ds=2, order=P, starts=P, dtable=P, dw=P, ws=P):
        return lib.xrd_lookup_bwd(dtype, n, k, rows, dim, table, stride, ids,
                                  ib, None, dout, ds, order, starts, 1.0,
                                  dtable, dw, ws, None)
    assert bwd(dtype=7) == 1 and bwd(n=-1) == 1 and bwd(k=0) == 1
    assert bwd(rows=-1) == 1 and bwd(dim=0) == 1 and bwd(stride=-1) == 1
    assert bwd(ds=-1) == 1 and bwd(ib=5) == 1 and bwd(ids=None) == 1
    assert bwd(dout=None) == 1 and bwd(order=None) == 1
    assert bwd(starts=None) == 1 and bwd(ws=None) == 1
    assert bwd(table=None) == 1 and bwd(dtable=None, dw=None) == 1
    assert bwd(n=1 << 31) == 3
    assert bwd(n=0, rows=0, table=None, ids=None, dout=None, order=None,
               starts=None, ws=None) == 0
    assert lib.xrd_lookup_bwd_ws_floats(1 << 31, 1, 4) == -1


def test_grouped_refusals():
    lib = _lib.lib()

    def fwd(dtype=0, m=4, e=2, i=2, o=2, x=P, s=2, w=P, starts=P, y=P):
        return lib.xrd_grouped_fwd(dtype, m, e, i, o, x, s, w, None, starts, 0,
                                   y, None)

    def bwd_x(dtype=0, m=4, e=2, i=2, o=2, x=P, s=2, w=P, starts=P, y=P):
        return lib.xrd_grouped_bwd_x(dtype, m, e, i, o, x, s, w, starts, y,
                                     None)
    for f in (fwd, bwd_x):
        assert f(dtype=3) == 1 and f(m=-1) == 1 and f(e=0) == 1
        assert f(i=0) == 1 and f(o=0) == 1 and f(x=None) == 1
        assert f(s=-1) == 1 and f(w=None) == 1 and f(starts=None) == 1
        assert f(y=None) == 1 and f(m=1 << 31) == 3 and f(i=1 << 21) == 3
        assert f(e=(1 << 20) + 1) == 3 and f(o=1 << 21) == 3
        assert f(e=(1 << 16) + 1) == 3
        assert f(s=(1 << 20) + 1) == 3
        assert f(m=0, x=None, y=None) == 0
    assert lib.xrd_grouped_relu_grad(0, 4, 2, None, P, 2, P, None) == 1
    assert lib.xrd_grouped_relu_grad(0, 4, 0, P, P, 2, P, None) == 1
    assert lib.xrd_grouped_relu_grad(0, 4, 2, P, P, -2, P, None) == 1
    assert lib.xrd_grouped_relu_grad(0, 0, 2, None, None, 2, None, None) == 0


def test_host_tensors_are_refused():
    ids = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(_lib.XrdError):
        tokens.plan(ids, 4)
    with pytest.raises(_lib.XrdError):
        tokens.lookup(torch.zeros(4, 8), ids)
    with pytest.raises(_lib.XrdError):
        grouped.linear(torch.zeros(4, 8), torch.zeros(2, 3, 8),
                       torch.zeros(3, dtype=torch.int32))


def test_plain_forms_agree_with_autograd():
    """the 64-bit forms of tests/token_util.py against torch's gradients"""
    g = torch.Generator().manual_seed(0)
    table = torch.randn(7, 5, generator=g, dtype=torch.float64,
                        requires_grad=True)
    ids = torch.randint(-1, 8, (6, 3), generator=g)
    w = torch.rand(6, 3, generator=g, dtype=torch.float64, requires_grad=True)
    ok = (ids >= 0) & (ids < 7)
    y = 0.5 * (torch.where(ok, w, 0.0)[..., None] *
               table[torch.where(ok, ids, 0)]).sum(1)
    dout = torch.randn(6, 5, generator=g, dtype=torch.float64)
    dt, dw = torch.autograd.grad(y, (table, w), dout)
    assert np.allclose(tu.lookup64(table, ids, w, 0.5)[0], y.detach())
    got = tu.lookup_grads64(table, ids, w, 0.5, dout)
    assert np.allclose(got[0], dt) and np.allclose(got[3], dw)
    x = torch.randn(9, 4, generator=g, dtype=torch.float64, requires_grad=True)
    wt = torch.randn(3, 2, 4, generator=g, dtype=torch.float64,
                     requires_grad=True)
    b = torch.randn(3, 2, generator=g, dtype=torch.float64, requires_grad=True)
    starts = [1, 4, 4, 8]
    z = torch.cat([x[:1, :2] * 0, x[1:4] @ wt[0].T + b[0],
                   x[4:8] @ wt[2].T + b[2], x[8:, :2] * 0])
    dz = torch.randn(9, 2, generator=g, dtype=torch.float64)
    want = torch.autograd.grad(z, (x, wt, b), dz)
    assert np.allclose(tu.linear64(x, wt, starts, b)[0], z.detach())
    got = tu.linear_grads64(x, wt, starts, dz.numpy())
    for k, t in zip('xwb', want):
        assert np.allclose(got[k][0], t), k
