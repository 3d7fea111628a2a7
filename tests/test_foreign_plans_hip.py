"""The table's gradient over a plan of any content: nothing outside the arrays
is read or written (csrc/tokens.hip cuts every token number and start to the
list; the guard values around the outputs show the writes)."""
import pytest
import torch

from xrdslam_amd import _lib
from xrdslam_amd.engine import tokens

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TOP, LOW = 2**31 - 1, -2**31


def contents(n, rows, seed):
    """(order, starts) that no plan of the ids has"""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(n, generator=g).int()
    starts = torch.linspace(0, n, rows + 1).int()
    wild = torch.randint(LOW, TOP, (n, ), generator=g).int()
    any_starts = torch.randint(LOW, TOP, (rows + 1, ), generator=g).int()
    yield order, starts                                # of other ids
    yield wild, starts
    yield torch.full((n, ), -1, dtype=torch.int32), starts
    yield torch.full((n, ), TOP, dtype=torch.int32), starts
    yield torch.full((n, ), n, dtype=torch.int32), starts
    yield order, any_starts
    yield order, starts.flip(0)
    yield order, torch.full_like(starts, TOP)
    yield order, torch.full_like(starts, LOW)
    yield order, starts + n
    yield order, starts - n // 2
    high = starts.clone()
    high[-1] = TOP
    yield order, high
    yield wild, any_starts


@pytest.mark.parametrize('dtype,code,dim', [(torch.float32, 0, 16),
                                            (torch.float32, 0, 5),
                                            (torch.bfloat16, 1, 264),
                                            (torch.float16, 2, 3)])
@pytest.mark.parametrize('n,k,rows', [(300, 3, 40), (1, 1, 1), (700, 1, 3),
                                      (64, 8, 5000)])
def test_stays_inside(n, k, rows, dtype, code, dim):
    lib = _lib.lib()
    g = torch.Generator().manual_seed(n + rows)
    ids = torch.randint(-1, rows + 1, (n, k), generator=g).to(DEV)
    w = torch.randn(n, k, generator=g).to(DEV)
    dout = torch.randn(n, dim, generator=g).to(dtype).to(DEV)
    words = lib.xrd_lookup_bwd_ws_floats(n, k, dim)
    pad = 4096
    for order, starts in contents(n * k, rows, n):
        order, starts = order.to(DEV), starts.to(DEV)
        ws = torch.full((words + 2 * pad, ), 7.0, device=DEV)
        dt = torch.full((rows * dim + 2 * pad, ), 7.0, dtype=dtype, device=DEV)
        _lib.check(lib.xrd_lookup_bwd(
            code, n, k, rows, dim, None, 0, ids.data_ptr(), 8, w.data_ptr(),
            dout.data_ptr(), dim, order.data_ptr(), starts.data_ptr(), 1.0,
            dt[pad:].data_ptr(), None, ws[pad:].data_ptr(),
            _lib.stream_ptr(ids.device)))
        torch.cuda.synchronize()
        for t, size in ((ws, words), (dt, rows * dim)):
            assert (t[:pad] == 7).all() and (t[pad + size:] == 7).all()


def test_a_plan_of_the_ids_is_unchanged():
    ids = torch.randint(-1, 41, (300, 3), device=DEV)
    table = torch.randn(40, 16, device=DEV, requires_grad=True)
    dout = torch.randn(300, 16, device=DEV)
    w = torch.rand(300, 3, device=DEV)
    a, = torch.autograd.grad(tokens.lookup(table, ids, w), table, dout)
    b, = torch.autograd.grad(tokens.lookup(
        table, ids, w, plan=tokens.plan(ids, 40)), table, dout)
    assert torch.equal(a, b)
