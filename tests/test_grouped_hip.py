"""The grouped linear against plain forms in 64 bits (tests/token_util.py).

Bounds: a sum of c products is taken to be off by 2 c U sum|terms|: the matrix
unit's adds may round in either direction, a whole step instead of half a one."""
import numpy as np
import pytest
import torch

import token_util as tu
from xrdslam_amd import _lib
from xrdslam_amd.engine import grouped, tokens

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def gen(seed):
    return torch.Generator().manual_seed(seed)


LAYOUTS = {
    'one': ([0, 77], 77),
    'one_row': ([0, 1], 1),
    'empty_groups': ([0, 0, 1, 1, 64, 64, 129, 259, 259], 259),
    'tail_and_lead': ([3, 20, 20, 85], 90),
    'no_rows_used': ([0, 0, 0, 0], 40),
    'no_rows': ([0, 0, 0], 0),
    'many': (list(np.minimum(np.arange(131) // 2 * 3, 190)), 192),
    'long': ([0, 5, 900, 901, 1300], 1300),
}
SIZES = [(1, 1), (3, 5), (16, 8), (24, 40), (128, 128), (144, 129), (96, 260),
         (260, 72), (33, 64)]


def make(layout, n_in, n_out, dtype, bias, seed=0):
    starts, m = LAYOUTS[layout]
    g = gen(seed + n_in * 31 + n_out)
    e = len(starts) - 1
    x = torch.randn(m, n_in, generator=g).to(dtype).to(DEV)
    w = (torch.randn(e, n_out, n_in, generator=g) / n_in**0.5).to(dtype)
    b = torch.randn(e, n_out, generator=g).to(dtype).to(DEV) if bias else None
    dy = torch.randn(m, n_out, generator=g).to(dtype).to(DEV)
    return x, w.to(DEV), starts, b, dy


def check(x, w, starts, b, dy, relu):
    st = torch.tensor(starts, dtype=torch.int32, device=DEV)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)
              if t is not None]
    y = grouped.linear(leaves[0], leaves[1], st,
                       leaves[2] if b is not None else None, relu)
    grads = torch.autograd.grad(y, leaves, dy)
    z, za = tu.linear64(x, w, starts, b)
    n_in = x.shape[1]
    tu.within(y, np.maximum(z, 0) if relu else z, za, 2 * (n_in + 2), 'y')
    dz = tu.host(dy)
    if relu:            # the mask is the result's own
        dz = np.where(tu.host(y) > 0, dz, 0.0)
    want = tu.linear_grads64(x, w, starts, dz)
    for k, got in zip('xwb', grads):
        v, t, c = want[k]
        tu.within(got, v, t, 2 * (c + 2), 'd' + k)
    return (y, *grads)


@pytest.mark.parametrize('dtype', tu.DTYPES)
@pytest.mark.parametrize('n_in,n_out', SIZES)
def test_linear(n_in, n_out, dtype):
    for j, layout in enumerate(LAYOUTS):
        bias, relu = j % 2 == 0, j % 3 == 0
        check(*make(layout, n_in, n_out, dtype, bias), relu)


@pytest.mark.parametrize('dtype', tu.DTYPES)
@pytest.mark.parametrize('layout', list(LAYOUTS))
def test_linear_bias_relu(layout, dtype):
    for bias in (False, True):
        for relu in (False, True):
            check(*make(layout, 40, 48, dtype, bias, 5), relu)


@pytest.mark.parametrize('dtype', tu.DTYPES)
@pytest.mark.parametrize('n_in,n_out', [(512, 640), (1000, 264), (777, 300)])
def test_linear_wide(n_in, n_out, dtype):
    check(*make('long', n_in, n_out, dtype, True), False)
    check(*make('empty_groups', n_in, n_out, dtype, False), False)


@pytest.mark.parametrize('dtype', tu.DTYPES)
def test_few_rows(dtype):
    """single tokens of many groups"""
    g = gen(2)
    for m, e, n_in, n_out in ((1, 4, 256, 512), (8, 16, 1024, 136),
                              (5, 70, 64, 1000), (16, 2, 520, 33)):
        at = torch.randint(0, e, (m, ), generator=g).sort().values
        starts = torch.searchsorted(at, torch.arange(e + 1)).tolist()
        x = torch.randn(m, n_in, generator=g).to(dtype).to(DEV)
        w = torch.randn(e, n_out, n_in, generator=g).to(dtype).to(DEV)
        b = torch.randn(e, n_out, generator=g).to(dtype).to(DEV)
        dy = torch.randn(m, n_out, generator=g).to(dtype).to(DEV)
        check(x, w, starts, b, dy, False)
        check(x, w, starts, None, dy, True)


@pytest.mark.parametrize('dtype', tu.DTYPES)
def test_many_rows_of_few_groups(dtype):
    """weight gradients over many rows: the contraction is cut and joined"""
    g = gen(4)
    for m, starts, n_in, n_out in ((9001, [0, 8000, 8001, 9001], 32, 48),
                                   (12000, [0, 0, 11990], 17, 128)):
        x = torch.randn(m, n_in, generator=g).to(dtype).to(DEV)
        w = torch.randn(len(starts) - 1, n_out, n_in, generator=g).to(dtype)
        dy = torch.randn(m, n_out, generator=g).to(dtype).to(DEV)
        b = torch.randn(len(starts) - 1, n_out, generator=g).to(dtype).to(DEV)
        check(x, w.to(DEV), starts, b, dy, False)


def test_linear_strides():
    x, w, starts, b, dy = make('empty_groups', 24, 40, torch.float32, True)
    m = x.shape[0]
    big = torch.randn(m, 100, device=DEV)
    check(big[:, 3:27], w, starts, b, dy, False)
    check(big[:, 4:28], w, starts, b, big[:, 56:96], True)
    check(torch.randn(24, m, device=DEV).t(), w, starts, b, dy, False)
    check(x, w, starts, b, torch.randn(1, 40, device=DEV).expand(m, 40), False)
    check(x, w, starts, b, torch.randn(1, 1, device=DEV).expand(m, 40), False)
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)     # [e, in, out] held
    check(x, wt, starts, b, dy, False)
    check(x.bfloat16()[:, 1:18], w.bfloat16()[:, :, :17], starts,
          b.bfloat16(), dy.bfloat16(), False)


@pytest.mark.parametrize('dtype', tu.DTYPES)
@pytest.mark.parametrize('n_in,n_out', [(128, 128), (40, 33)])
def test_rows_of_no_group_do_not_leak(n_in, n_out, dtype):
    """NaN in rows outside every group, in the gradient there and in the
    weights of groups without rows"""
    starts, m = [10, 30, 30, 75], 90
    g = gen(8)
    x = torch.randn(m, n_in, generator=g).to(dtype).to(DEV)
    w = torch.randn(3, n_out, n_in, generator=g).to(dtype).to(DEV)
    dy = torch.randn(m, n_out, generator=g).to(dtype).to(DEV)
    for t in (x, dy):
        t[:10], t[75:] = float('nan'), float('inf')
    w[1] = float('nan')
    for t in (x, w):
        t.requires_grad_(True)
    st = torch.tensor(starts, dtype=torch.int32, device=DEV)
    y = grouped.linear(x, w, st)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for t in (y, dx):
        assert torch.isfinite(t).all()
        assert not t[:10].any() and not t[75:].any()
    assert torch.isfinite(dw).all() and not dw[1].any()
    # a NaN inside one group stays there
    with torch.no_grad():
        x[30, 0] = float('nan')
    y = grouped.linear(x, w, st)
    assert torch.isfinite(y[10:30]).all() and torch.isnan(y[30]).all()
    assert torch.isfinite(y[31:75]).all()


def test_offsets_past_32_bits():
    """rows behind element 2^31 of the result and of its gradient, two groups
    whose border lies there; rows of ones and twos, so sums are exact"""
    m, n_out, n_in = 1100000, 2048, 8
    assert m * n_out > 1 << 31
    st = torch.tensor([0, 1080003, m], dtype=torch.int32, device=DEV)
    x = torch.ones(m, n_in, dtype=torch.float16, device=DEV)
    x[-5:] = 2
    w = torch.ones(2, n_out, n_in, dtype=torch.float16, device=DEV)
    w[1] = 3
    for t in (x, w):
        t.requires_grad_(True)
    y = grouped.linear(x, w, st)
    want = torch.full((m, ), 8.0, device=DEV)
    want[1080003:], want[-5:] = 24, 48
    for c in (0, 1000, n_out - 1):
        assert torch.equal(y[:, c].float(), want)
    dy = torch.zeros_like(y)
    dy[-3:], dy[1080002] = 1, 1
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wx = torch.zeros(m, device=DEV)
    wx[-3:], wx[1080002] = 3 * n_out, n_out
    assert torch.equal(dx[:, 0].float(), wx)
    assert (dw[0] == 1).all() and (dw[1] == 6).all()


def test_relu_keeps_nan():
    x = torch.tensor([[float('nan'), 1.0], [1.0, -2.0]], device=DEV,
                     requires_grad=True)
    w = torch.ones(1, 3, 2, device=DEV)
    st = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    y = grouped.linear(x, w, st, relu=True)
    assert torch.isnan(y[0]).all() and not y[1].any()
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx, torch.tensor([[3.0, 3.0], [0.0, 0.0]], device=DEV))


def test_starts_of_any_content_stay_in_bounds():
    """starts that are not ascending or leave the rows: nothing outside is
    read or written (the guard rows keep their value)"""
    x = torch.randn(100, 16, device=DEV)
    w = torch.randn(4, 8, 16, device=DEV)
    lib = _lib.lib()
    for starts in ([5, 1000, -7, 3, 1 << 30], [100, 0, 100, 0, 100],
                   [-1, -1, -1, -1, -1], [0, 1 << 31 - 1, 0, 50, 20]):
        st = torch.tensor([max(min(v, 2**31 - 1), -2**31) for v in starts],
                          dtype=torch.int32, device=DEV)
        guard = torch.full((300, 8), 7.0, device=DEV)
        _lib.check(lib.xrd_grouped_fwd(
            0, 100, 4, 16, 8, x.data_ptr(), 16, w.data_ptr(), None,
            st.data_ptr(), 0, guard[100:].data_ptr(),
            _lib.stream_ptr(x.device)))
        torch.cuda.synchronize()
        assert (guard[:100] == 7).all() and (guard[200:] == 7).all()
        # the weight gradient's partial sums stay in their workspace as well
        x2 = torch.randn(3000, 16, device=DEV)
        dz = torch.randn(3000, 8, device=DEV)
        words = lib.xrd_grouped_ws_floats(0, 3000, 4, 16, 8)
        ws = torch.full((words + 2000, ), 7.0, device=DEV)
        dw = torch.full((4 * 16 * 8 + 2000, ), 7.0, device=DEV)
        _lib.check(lib.xrd_grouped_bwd_w(
            0, 3000, 4, 16, 8, x2.data_ptr(), 16, dz.data_ptr(), 8,
            st.data_ptr(), dw[1000:].data_ptr(), None, ws[1000:].data_ptr(),
            _lib.stream_ptr(x.device)))
        torch.cuda.synchronize()
        for t, n in ((ws, words), (dw, 4 * 16 * 8)):
            assert (t[:1000] == 7).all() and (t[1000 + n:] == 7).all()


def test_gradient_against_differences():
    """the layer is linear in x and in the weight: a central difference over
    any step equals <gradient, direction>"""
    x, w, starts, b, dy = make('empty_groups', 24, 40, torch.float32, True)
    st = torch.tensor(starts, dtype=torch.int32, device=DEV)
    _, dx, dw, _ = check(x, w, starts, b, dy, False)
    for leaf, grad, f, count in (
            (x, dx, lambda t: grouped.linear(t, w, st), 40),
            (w, dw, lambda t: grouped.linear(x, t, st), 259)):
        d = torch.randn(leaf.shape, generator=gen(9)).to(DEV)
        diff = float((0.5 * (f(leaf + d).double() - f(leaf - d).double()) *
                      dy.double()).sum())
        ana = float((grad.double() * d.double()).sum())
        ax, aw = (leaf.abs() + d.abs(), w.abs()) if leaf is x else \
            (x.abs(), leaf.abs() + d.abs())
        terms = tu.linear64(ax, aw, starts, None)[1]
        total = float((terms * dy.abs().double().cpu().numpy()).sum())
        # forward sums over 24 (+1 for leaf +- d), gradient sums over `count`
        assert abs(diff - ana) <= 2 * (24 + 3 + count + 2) * tu.U * total


@pytest.mark.parametrize('dtype', tu.DTYPES)
def test_equal_inputs_give_equal_bits(dtype):
    args = make('long', 128, 144, dtype, True)
    a = check(*args, False)
    for _ in range(3):
        b = check(*args, False)
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def bank(points, gates, which, w1, b1, w2, b2, n):
    """k decoders a point: dispatch, two layers, combination"""
    t, k = which.shape
    p = tokens.plan(which, n, rank=True)
    x = tokens.lookup(points, p.order // k)
    h = grouped.linear(x, w1, p.starts, b1, relu=True)
    y = grouped.linear(h, w2, p.starts, b2)
    return tokens.lookup(y, p.rank.view(t, k), gates)


def bank_inputs(seed, t=700, k=2, n=6, d=16, hidden=128, out=4):
    """points, the first layer and its bias on coarse binary grids: the
    pre-activations are exact in f32, so the ReLU masks of any two right
    computations agree"""
    g = gen(seed)

    def grid(step, *shape):
        return (torch.randn(*shape, generator=g) / step).round().clamp(
            -3 / step, 3 / step) * step
    which = torch.rand(t, n, generator=g).argsort(1)[:, :k]
    which[::50, 0] = -1                       # a point with one decoder only
    r = [grid(1 / 8, t, d), torch.rand(t, k, generator=g), which,
         grid(1 / 16, n, hidden, d) / 4, grid(1 / 16, n, hidden) / 4,
         torch.randn(n, out, hidden, generator=g) / 11,
         torch.randn(n, out, generator=g) / 4,
         torch.randn(t, out, generator=g)]
    return [v.to(DEV) for v in r]


def bank64(leaves, which, masks=None):
    points, gates, w1, b1, w2, b2 = leaves
    y, kept = 0, []
    for j in range(which.shape[1]):
        e = which[:, j].clamp(min=0)
        pre = (w1[e] * points[:, None]).sum(-1) + b1[e]
        kept.append(pre > 0 if masks is None else masks[j])
        h = torch.where(kept[j], pre, 0.0)
        o = (w2[e] * h[:, None]).sum(-1) + b2[e]
        y = y + torch.where(which[:, j:j + 1] >= 0, o, 0.0) * gates[:, j:j + 1]
    return y, kept


def test_decoder_bank_together():
    """plan, dispatch lookup, two grouped layers and the weighted combination:
    values and every gradient against the dense formula in f64.  The same
    formula on magnitudes (with the masks of the first) bounds the terms of
    every result; each passes at most 16 + 1 + 128 + 1 + 4 + 2 + 1400 + 10
    roundings (both layers, the combination, the rows of a weight gradient)."""
    points, gates, which, w1, b1, w2, b2, dout = bank_inputs(1)
    leaves = [points, gates, w1, b1, w2, b2]
    for v in leaves:
        v.requires_grad_(True)
    y = bank(points, gates, which, w1, b1, w2, b2, 6)
    got = torch.autograd.grad(y, leaves, dout)

    def reference(sign, masks):
        ls = [(v.detach().double().cpu().abs() if sign else
               v.detach().double().cpu()).requires_grad_(True) for v in leaves]
        d = dout.double().cpu()
        y, kept = bank64(ls, which.cpu(), masks)
        return (y, *torch.autograd.grad(y, ls, d.abs() if sign else d)), kept
    want, masks = reference(False, None)
    terms, _ = reference(True, masks)
    for a, b, t in zip((y, *got), want, terms):
        off = (a.detach().double().cpu() - b.detach()).abs()
        assert (off <= 2 * 1562 * tu.U * t.detach()).all()


def test_decoder_bank_graph():
    """the whole run captured and replayed on new inputs"""
    args = bank_inputs(2)
    dout, which = args[-1], args[2]
    leaves = [args[0], args[1], *args[3:7]]
    for v in leaves:
        v.requires_grad_(True)

    def step():
        y = bank(leaves[0], leaves[1], which, *leaves[2:], 6)
        return (y, *torch.autograd.grad(y, leaves, dout))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(4):
        with torch.no_grad():
            for old, fresh in zip(args, bank_inputs(10 + r)):
                old.copy_(fresh)
        graph.replay()
        got = [t.detach().clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_refusals():
    x = torch.zeros(6, 8, device=DEV)
    w = torch.zeros(2, 4, 8, device=DEV)
    st = torch.tensor([0, 3, 6], dtype=torch.int32, device=DEV)
    b = torch.zeros(2, 4, device=DEV)
    bad = [
        lambda: grouped.linear(x[0], w, st),
        lambda: grouped.linear(x, w[0], st),
        lambda: grouped.linear(x[:, :7], w, st),
        lambda: grouped.linear(x.double(), w.double(), st),
        lambda: grouped.linear(x.bfloat16(), w, st),
        lambda: grouped.linear(x, w, st.long()),
        lambda: grouped.linear(x, w, st[:2]),
        lambda: grouped.linear(x, w, st.cpu()),
        lambda: grouped.linear(x, w.cpu(), st),
        lambda: grouped.linear(x, w, st, b[:1]),
        lambda: grouped.linear(x, w, st, b.bfloat16()),
    ]
    for f in bad:
        with pytest.raises(_lib.XrdError):
            f()
    x.requires_grad_(True)
    y = grouped.linear(x, w, st)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize('dtype,m,n_in,n_out', [
    (torch.float32, 70, 1200, 2500), (torch.bfloat16, 260, 2400, 2600),
    (torch.float16, 6000, 40, 3000), (torch.float32, 9000, 1000, 24)])
def test_results_larger_than_the_caches(dtype, m, n_in, n_out):
    """dW (the first two), y and dx of more than 32 MB are stored another way"""
    g = gen(m)
    starts = [0, m // 3, m // 3, m - 2]
    x = torch.randn(m, n_in, generator=g).to(dtype).to(DEV)
    w = (torch.randn(3, n_out, n_in, generator=g) / n_in**0.5).to(dtype)
    b = torch.randn(3, n_out, generator=g).to(dtype).to(DEV)
    dy = torch.randn(m, n_out, generator=g).to(dtype).to(DEV)
    big = max(m * n_out, m * n_in, w.numel()) * w.element_size()
    assert big > 32 << 20
    check(x, w.to(DEV), starts, b, dy, False)
