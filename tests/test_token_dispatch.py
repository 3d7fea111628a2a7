"""The token operators under torch's dispatcher: a kernel under the device's key
and a node under the autograd key, so that what works by dispatch (forward-mode
derivatives, traces, negated views, function transforms) gets the operators or
a refusal, never a wrong value."""
import itertools

import pytest
import torch
import torch.autograd.forward_ad as fwad

from xrdslam_amd import _lib
from xrdslam_amd.engine import grouped, tokens

DEV = 'cuda:0'
KERNELS = ('plan', 'lookup', 'lookup_grads', 'linear', 'linear_grads')


def has(name, key):
    return torch._C._dispatch_has_kernel_for_dispatch_key('xrdslam::' + name,
                                                          key)


def test_operators_have_their_keys():
    tokens.ops()
    for name in KERNELS:
        assert has(name, 'CUDA'), name
        # (such a kernel would hide the operator from every mode)
        assert not has(name, 'CompositeImplicitAutograd'), name
    for name in ('lookup', 'linear'):
        assert has(name, 'Autograd'), name


def duals(f, *args):
    """f with each floating argument in turn as a dual tensor"""
    for i, t in enumerate(args):
        if t is None or not t.is_floating_point():
            continue
        with fwad.dual_level():
            a = list(args)
            a[i] = fwad.make_dual(t, torch.ones_like(t))
            yield lambda: f(*a)


def test_tangents_are_refused_before_any_launch():
    """(host tensors: the refusal comes from the autograd key, in front of the
    device's kernel)"""
    ops = tokens.ops()
    table, w = torch.ones(4, 8), torch.ones(5, 2)
    ids = torch.zeros(5, 2, dtype=torch.int64)
    for f in duals(lambda t, v: ops.lookup(t, ids, v, 1.0, None, None), table,
                   w):
        with pytest.raises(RuntimeError, match='xrd_lookup.*forward-mode'):
            f()
    st = torch.tensor([0, 2, 5], dtype=torch.int32)
    for f in duals(lambda x, v, b: ops.linear(x, v, st, b, False),
                   torch.ones(5, 8), torch.ones(2, 3, 8), torch.ones(2, 3)):
        with pytest.raises(RuntimeError, match='xrd_grouped.*forward-mode'):
            f()


def test_sizes_past_32_bits_are_refused_before_any_copy():
    """(expanded tensors: one element each; 2^32 + 2 columns used to arrive as
    2 in the C entry points)"""
    ops = tokens.ops()
    wide = (1 << 32) + 2
    ids = torch.zeros(1, dtype=torch.int64)
    one = torch.zeros(1)
    st = torch.zeros(2, dtype=torch.int32)
    for f in (lambda: ops.lookup(one.expand(1, wide), ids, None, 1.0, None,
                                 None),
              lambda: ops.lookup(torch.zeros(1, 2), ids.expand(1, wide),
                                 one.expand(1, wide), 1.0, None, None),
              lambda: ops.linear(one.expand(1, wide), one.expand(1, 2, wide),
                                 st, None, False),
              lambda: ops.linear(torch.zeros(1, 2), one.expand(1, wide, 2), st,
                                 None, False)):
        with pytest.raises(RuntimeError, match='xrd_.*unsupported'):
            f()


def test_a_fake_tensor_gets_no_answer():
    """(there is no rule for shapes alone, so a compiler stops here)"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = tokens.ops()
    with FakeTensorMode():
        table = torch.empty(4, 8, device='cuda')
        ids = torch.empty(5, dtype=torch.int64, device='cuda')
        st = torch.empty(3, dtype=torch.int32, device='cuda')
        for f in (lambda: ops.plan(ids, 4, False),
                  lambda: ops.lookup(table, ids, None, 1.0, None, None),
                  lambda: ops.linear(table, torch.empty(2, 3, 8, device='cuda'),
                                     st, None, False)):
            with pytest.raises(Exception):
                f()


def inputs(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(30, 16, generator=g).to(dtype)
    ids = torch.randint(-1, 31, (70, 3), generator=g)
    w = torch.randn(70, 3, generator=g)
    weight = torch.randn(4, 24, 16, generator=g).to(dtype)
    bias = torch.randn(4, 24, generator=g).to(dtype)
    starts = torch.tensor([0, 11, 11, 40, 65], dtype=torch.int32)
    return [t.to(DEV) for t in (table, ids, w, weight, bias, starts)]


def run(table, ids, w, weight, bias, starts):
    x = tokens.lookup(table, ids, w, scale=0.5)
    return grouped.linear(x, weight, starts, bias, relu=True)


@pytest.mark.gpu
def test_tangents_are_refused():
    table, ids, w, weight, bias, starts = inputs(0)
    x = tokens.lookup(table, ids, w)
    for f in itertools.chain(
            duals(lambda t, v: tokens.lookup(t, ids, v), table, w),
            duals(lambda t: tokens.lookup(t, ids), table),
            duals(lambda a, v, b: grouped.linear(a, v, starts, b), x, weight,
                  bias)):
        with pytest.raises(_lib.XrdError):
            f()
    for f, t in ((lambda t: tokens.lookup(t, ids, w), table),
                 (lambda v: grouped.linear(x, v, starts), weight)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (t, ), (torch.ones_like(t), ))
        # forward over reverse: a tangent that reaches the backward pass
        t = t.detach().requires_grad_(True)
        y = f(t)
        with fwad.dual_level(), pytest.raises(RuntimeError):
            torch.autograd.grad(y, t, fwad.make_dual(torch.ones_like(y),
                                                     torch.ones_like(y)))


@pytest.mark.gpu
@pytest.mark.parametrize('leaves', [(), (0, 2, 3, 4), (0, ), (3, ), (4, )])
def test_traced_graph_computes(leaves):
    """a trace records the operators, of the backward pass too, and gives the
    eager bits on other inputs"""
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(*args):
        args = [t.detach().requires_grad_(True) if i in leaves else t
                for i, t in enumerate(args)]
        y = run(*args)
        if not leaves:
            return (y, )
        return (y.detach(), *torch.autograd.grad(
            y, [args[i] for i in leaves], torch.ones_like(y)))
    graph = make_fx(step)(*inputs(1))
    seen = {str(n.target) for n in graph.graph.nodes}
    want = {'xrdslam.lookup.default', 'xrdslam.linear.default'}
    if leaves:
        want.add('xrdslam.linear_grads.default')
    if 0 in leaves:
        want.add('xrdslam.lookup_grads.default')
    assert want <= seen
    for seed in (1, 2, 3):
        args = inputs(seed)
        # (what a freed buffer would hold)
        for t in (torch.full((1 << 16, ), float('nan'), device=DEV)
                  for _ in range(8)):
            del t
        for a, b in zip(graph(*args), step(*args)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_traced_plan_computes():
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(ids):
        p = tokens.plan(ids, 31, rank=True)
        return p.order, p.starts, p.rank
    graph = make_fx(step)(inputs(1)[1])
    for seed in (2, 3):
        ids = inputs(seed)[1]
        assert all(torch.equal(a, b) for a, b in zip(graph(ids), step(ids)))


@pytest.mark.gpu
def test_negated_views_are_read_with_their_sign():
    table, ids, w, weight, bias, starts = inputs(4)
    neg = torch._neg_view
    want = run(-table, ids, -w, -weight, -bias, starts)
    got = run(neg(table), ids, neg(w), neg(weight), neg(bias), starts)
    assert torch.equal(got, want)
    table.requires_grad_(True)
    y = tokens.lookup(table, ids, w)
    d = torch.randn_like(y)
    a, = torch.autograd.grad(y, table, neg(d), retain_graph=True)
    b, = torch.autograd.grad(y, table, -d)
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_function_transforms_are_right_or_refused():
    table, ids, w, weight, bias, starts = inputs(5)
    for f, t in ((lambda t: tokens.lookup(t, ids, w).square().sum(), table),
                 (lambda v: tokens.lookup(table, ids, v).square().sum(), w),
                 (lambda v: grouped.linear(table, v, starts).square().sum(),
                  weight)):
        leaf = t.detach().requires_grad_(True)
        want, = torch.autograd.grad(f(leaf), leaf)
        try:
            got = torch.func.grad(f)(t)
        except RuntimeError:
            continue
        assert torch.equal(got, want)
    many = torch.stack([table, table * 2, table - 1])
    try:
        got = torch.vmap(lambda t: tokens.lookup(t, ids, w))(many)
    except RuntimeError:
        return
    assert torch.equal(got, torch.stack([tokens.lookup(t, ids, w)
                                         for t in many]))


@pytest.mark.gpu
def test_shapes_of_gradients():
    """ids of several axes: the gradient arrives in the result's shape"""
    table = inputs(6)[0].requires_grad_(True)
    for shape in ((), (3, ), (2, 5), (2, 0, 4), (3, 2, 4)):
        ids = torch.randint(0, 30, shape, device=DEV)
        y = tokens.lookup(table, ids, scale=2.0)
        assert y.shape == (*shape, 16)
        d = torch.randn(16, *shape[::-1], device=DEV).permute(
            *range(len(shape), -1, -1))
        got, = torch.autograd.grad(y, table, d)
        want = torch.zeros(30, 16, dtype=torch.float64, device=DEV)
        want.index_add_(0, ids.reshape(-1), d.reshape(-1, 16).double())
        # at most 24 f32 sums of values below 6
        assert (got - 2 * want).abs().max() <= 24 * 2.0**-24 * 2 * 24 * 6
        if shape and shape[-1]:
            w = torch.rand(shape, device=DEV, requires_grad=True)
            y = tokens.lookup(table, ids, w)
            assert y.shape == (*shape[:-1], 16)
            gt, gw = torch.autograd.grad(y, (table, w), torch.ones_like(y))
            assert gt.shape == table.shape and gw.shape == w.shape
