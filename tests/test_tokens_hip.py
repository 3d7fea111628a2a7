"""Token plans and scaled lookups against plain forms in 64 bits
(tests/token_util.py, bounds derived there)."""
import numpy as np
import pytest
import torch

import token_util as tu
from xrdslam_amd import _lib
from xrdslam_amd.engine import tokens

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check_plan(ids, groups):
    p = tokens.plan(ids.to(DEV), groups, rank=True)
    i = ids.reshape(-1).numpy().astype(np.int64)
    key = np.where((i >= 0) & (i < groups), i, groups)
    order = np.argsort(key, kind='stable')
    starts = np.searchsorted(key[order], np.arange(groups + 1))
    assert p.order.dtype == p.starts.dtype == p.rank.dtype == torch.int32
    assert np.array_equal(p.order.cpu().numpy(), order)
    assert np.array_equal(p.starts.cpu().numpy(), starts)
    rank = np.empty_like(order)
    rank[order] = np.arange(order.size)
    assert np.array_equal(p.rank.cpu().numpy(), rank)


@pytest.mark.parametrize('n', [0, 1, 63, 64, 65, 1023, 4095, 4096, 4097, 8193,
                               70001])
@pytest.mark.parametrize('groups', [1, 2, 16, 255, 256, 257, 20000, 70000])
def test_plan(n, groups):
    g = gen(n * 7 + groups)
    ids = torch.randint(-2, groups + 2, (n, ), generator=g)
    check_plan(ids, groups)
    check_plan(ids.int(), groups)


@pytest.mark.parametrize('groups', [1, 3, 300, 1 << 17, (1 << 24) + 5])
def test_plan_corners(groups):
    check_plan(torch.full((9001, ), groups - 1), groups)          # one group
    check_plan(torch.full((5000, ), -1), groups)                  # none
    check_plan(torch.full((130, ), 1 << 40), groups)              # far ids
    check_plan(torch.full((130, ), -(1 << 31)).int(), groups)
    check_plan(torch.arange(6000).flip(0) % (groups + 1), groups)
    check_plan(torch.tensor([[groups - 1, 0], [0, groups]]), groups)


def test_plan_large():
    g = gen(5)
    check_plan((torch.rand(1 << 20, generator=g)**3 * 100000).long(), 100000)
    check_plan((torch.rand(2500001, generator=g)**2 * 37).int(), 37)


@pytest.mark.parametrize('n', [524287, 524288, 524289, 1048576, 1048577])
def test_plan_between_tile_sizes(n):
    g = gen(n)
    check_plan(torch.randint(-1, 700, (n, ), generator=g).int(), 699)
    check_plan(torch.randint(0, 3, (n, ), generator=g), 2)


SHAPES = [(1, 1), (5, 3), (40, 8), (33, 16), (17, 33), (9, 256), (6, 520),
          (300, 32)]


def make(rows, n, k, dim, dtype, seed, low=-1):
    g = gen(seed)
    table = torch.randn(rows, dim, generator=g).to(dtype)
    shape = (n, ) if k is None else (n, k)
    ids = torch.randint(low, rows + 1, shape, generator=g)
    w = None if k is None else torch.randn(n, k, generator=g)
    dout = torch.randn(n, dim, generator=g).to(dtype)
    return table, ids, w, dout


def check_lookup(table, ids, w, dout, scale, plan=False):
    """forward and every gradient; the arguments live on the device"""
    table = table.detach().requires_grad_(True)
    wl = None if w is None else w.detach().requires_grad_(True)
    p = tokens.plan(ids, table.shape[0]) if plan else None
    y = tokens.lookup(table, ids, wl, scale=scale, plan=p)
    leaves = [table] if w is None else [table, wl]
    grads = torch.autograd.grad(y, leaves, dout)
    i2 = ids.reshape(-1, 1 if w is None else ids.shape[-1])
    k, dim = i2.shape[1], table.shape[1]
    s32 = float(np.float32(scale))
    want, terms = tu.lookup64(table, i2, w, s32)
    tu.within(y, want, terms, k + 2, 'y')
    d, da, cnt, dw, dwa = tu.lookup_grads64(table, i2, w, s32, dout)
    assert grads[0].dtype == table.dtype
    tu.within(grads[0], d, da, cnt + 2, 'dtable')
    if w is not None:
        tu.within(grads[1], dw, dwa, dim + 2, 'dweights')
    return (y, *grads)


@pytest.mark.parametrize('dtype', tu.DTYPES)
@pytest.mark.parametrize('k', [None, 1, 3, 8])
@pytest.mark.parametrize('rows,dim', SHAPES)
def test_lookup(rows, dim, k, dtype):
    for n in (1, 67):
        table, ids, w, dout = make(rows, n, k, dim, dtype, rows + n)
        args = [t if t is None else t.to(DEV) for t in (table, ids, w, dout)]
        check_lookup(*args, 0.75)
        args[1] = args[1].int()
        check_lookup(*args, 3.0, plan=True)


@pytest.mark.parametrize('dtype', tu.DTYPES)
def test_one_row_owns_the_tokens(dtype):
    """rows with thousands of tokens beside rows with a few and with none"""
    g = gen(11)
    for n, k, dim, rows in ((6000, 1, 16, 50), (2500, 8, 32, 9),
                            (5000, 1, 129, 3), (700, 3, 1024, 1000)):
        table, ids, w, dout = make(rows, n, k, dim, dtype, n)
        hot = torch.rand(n, k, generator=g) < 0.8
        ids = torch.where(hot, rows // 2, ids)
        check_lookup(table.to(DEV), ids.to(DEV), w.to(DEV), dout.to(DEV), 1.0)


def test_lookup_shapes_and_empty():
    table = torch.randn(10, 4, device=DEV, requires_grad=True)
    ids = torch.randint(0, 10, (2, 3, 5), device=DEV)
    y = tokens.lookup(table, ids)
    assert y.shape == (2, 3, 5, 4) and torch.equal(y, table[ids])
    w = torch.rand(2, 3, 5, device=DEV)
    assert tokens.lookup(table, ids, w).shape == (2, 3, 4)
    assert tokens.lookup(table, torch.tensor(3, device=DEV)).shape == (4, )
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    y = tokens.lookup(table, none)
    assert y.shape == (0, 4)
    assert torch.equal(torch.autograd.grad(y.sum(), table)[0],
                       torch.zeros(10, 4, device=DEV))
    empty = torch.zeros(0, 4, device=DEV, requires_grad=True)
    y = tokens.lookup(empty, ids)                   # no row: zeros
    assert torch.equal(y, torch.zeros_like(y))
    assert torch.autograd.grad(y.sum(), empty)[0].shape == (0, 4)


def test_lookup_strides():
    """rows of a wider table, an expanded and a transposed gradient,
    misaligned views, non-contiguous ids and weights"""
    big = torch.randn(40, 50, device=DEV)
    ids = torch.randint(-1, 40, (3, 30), device=DEV).t()
    w = torch.randn(3, 30, device=DEV).t()
    for cols in (slice(0, 16), slice(1, 17), slice(2, 35)):
        table = big[:, cols]
        d = table.shape[1]
        for dout in (torch.randn(30, d, device=DEV),
                     torch.randn(1, d, device=DEV).expand(30, d),
                     torch.randn(1, 1, device=DEV).expand(30, d),
                     torch.randn(d, 30, device=DEV).t(),
                     torch.randn(30, 2 * d + 1, device=DEV)[:, 1:1 + d]):
            check_lookup(table, ids, w, dout, 0.5)
    check_lookup(big.t()[:9], ids % 9, w, torch.randn(30, 40, device=DEV), 1.0)


def test_missing_rows_do_not_leak():
    """NaN and infinity in rows, weights and gradients that no token uses"""
    table = torch.randn(6, 8, device=DEV)
    table[2], table[3] = float('nan'), float('inf')
    ids = torch.tensor([[0, -1], [5, 6], [-1, -1]], device=DEV)
    w = torch.tensor([[1.0, float('nan')], [2.0, float('inf')],
                      [float('nan')] * 2], device=DEV)
    table.requires_grad_(True)
    w.requires_grad_(True)
    y = tokens.lookup(table, ids, w)
    dout = torch.ones(3, 8, device=DEV)
    dout[2] = float('nan')
    dt, dw = torch.autograd.grad(y, (table, w), dout)
    assert torch.isfinite(y).all() and torch.isfinite(dt).all()
    assert torch.equal(y[2], torch.zeros(8, device=DEV))
    assert torch.equal(dt[1:5], torch.zeros(4, 8, device=DEV))
    assert torch.isfinite(dw).all() and torch.equal(
        dw[2], torch.zeros(2, device=DEV))


def test_gradient_against_differences():
    """the lookup is linear in the table and in the weights: a central
    difference over any step equals <gradient, direction>"""
    table, ids, w, dout = (t.to(DEV) for t in make(
        50, 200, 4, 24, torch.float32, 3, low=0))
    ids = ids.clamp(max=49)
    _, dt, dw = check_lookup(table, ids, w, dout, 2.0)
    for leaf, grad, f in (
            (table, dt, lambda t: tokens.lookup(t, ids, w, scale=2.0)),
            (w, dw, lambda t: tokens.lookup(table, ids, t, scale=2.0))):
        d = torch.randn(leaf.shape, generator=gen(9)).to(DEV)
        hi, lo = f(leaf + d).double(), f(leaf - d).double()
        diff = float((0.5 * (hi - lo) * dout.double()).sum())
        # every y is off by (k + 2) U of its terms (and leaf +- d by U): bound
        # it by the sum over all outputs of |terms| at |leaf| + |d|
        i2 = ids
        if leaf is table:
            terms = tu.lookup64(leaf.abs() + d.abs(), i2, w.abs(), 2.0)[1]
        else:
            terms = tu.lookup64(table.abs(), i2, leaf.abs() + d.abs(), 2.0)[1]
        lim = 9 * tu.U * float((terms * dout.abs().double().cpu().numpy()
                                ).sum())
        ana = float((grad.double() * d.double()).sum())
        count = 200 * 4 + 2 if leaf is table else 24 + 2
        lim += count * tu.U * float(
            (terms * dout.abs().double().cpu().numpy()).sum())
        assert abs(diff - ana) <= lim


@pytest.mark.parametrize('dtype', tu.DTYPES)
def test_equal_inputs_give_equal_bits(dtype):
    table, ids, w, dout = (t.to(DEV) for t in make(
        100, 3000, 8, 32, dtype, 21))
    a = check_lookup(table, ids, w, dout, 1.0)
    for _ in range(3):
        b = check_lookup(table, ids, w, dout, 1.0)
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_another_stream():
    table, ids, w, dout = (t.to(DEV) for t in make(
        100, 500, 8, 32, torch.float32, 5))
    want = check_lookup(table, ids, w, dout, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = check_lookup(table, ids, w, dout, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(want, got))


def test_graph_replays():
    """forward and backward captured together; every replay on new inputs
    equals the eager call, with eager work between the replays"""
    table, ids, w, dout = (t.to(DEV) for t in make(
        300, 1000, 8, 16, torch.float32, 6))
    table.requires_grad_(True)
    w.requires_grad_(True)

    def step():
        y = tokens.lookup(table, ids, w, scale=0.5)
        return (y, *torch.autograd.grad(y, (table, w), dout))
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
            new = make(300, 1000, 8, 16, torch.float32, 100 + r)
            for old, fresh in zip((table, ids, w, dout), new):
                old.copy_(fresh.to(DEV))
        graph.replay()
        got = [t.detach().clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_offsets_past_32_bits():
    """rows behind element 2^31 of a table and of its gradient (8.6 GB each)"""
    rows, dim = 2100000, 2048
    table = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    far = torch.tensor([rows - 1, 0, rows - 2, rows - 1, 1050000], device=DEV)
    assert rows * dim > 1 << 32
    table[far] = torch.randn(5, dim, generator=gen(1)).bfloat16().to(DEV)
    table.requires_grad_(True)
    y = tokens.lookup(table, far)
    assert torch.equal(y, table.detach()[far])
    dout = torch.randn(5, dim, generator=gen(2)).bfloat16().to(DEV)
    d, = torch.autograd.grad(y, table, dout)
    used = far.unique()
    want = torch.stack([dout[far == r].float().sum(0) for r in used])
    assert torch.equal(d[used], want.bfloat16())
    d[used] = 0
    assert not any(bool(c.any()) for c in d.split(300000))


def voxel_batch(seed, n=900, voxels=40, rows=150, dim=16):
    g = gen(seed)
    samples = {
        'sampled_point_voxel_idx': torch.randint(0, voxels, (n, ), generator=g),
        'sampled_point_xyz': torch.rand(n, 3, generator=g),
        'sampled_point_distance': torch.rand(n, generator=g)}
    states = {
        'voxel_vertex_idx': torch.randint(0, rows, (voxels, 8), generator=g
                                          ).int(),
        'voxel_center_xyz': torch.rand(voxels, 3, generator=g),
        'voxel_vertex_emb': torch.randn(rows, dim, generator=g)}
    dout = torch.randn(n, dim, generator=g)
    return samples, states, dout


def voxel_features(samples, states, dout, device, dtype, sorted_lookup):
    """Vox-Fusion's modular features -> (features, dxyz, dembeddings)"""
    from xrdslam_amd.slam.model_components import voxel_helpers_voxfusion as vh

    def put(t):
        t = t.to(device)
        return t.to(dtype) if t.is_floating_point() else t
    s, m = ({k: put(v) for k, v in d.items()} for d in (samples, states))
    m['voxel_vertex_emb'].requires_grad_(True)
    y = vh.get_features(s, m, 0.2, sorted_lookup)['emb']
    return (y, *torch.autograd.grad(
        y, (s['sampled_point_xyz'], m['voxel_vertex_emb']), put(dout).float()))


def test_voxel_features_through_the_lookup():
    """the modular Vox-Fusion features with sorted_lookup: values and both
    gradients against the f64 run of the plain path on the CPU, and equal bits
    from equal batches.  Bounds: eight products of magnitudes up to |w| max|e|
    with |w| <= (1 + |p|)^3, p the local coordinate; 40 roundings a value cover
    the weight's own 12, the eight products and sums and the sums of a gradient
    in f32 of at most 900 * 8 / 150 expected, 200 at most, tokens a row."""
    samples, states, dout = voxel_batch(3)
    want = voxel_features(samples, states, dout, 'cpu', torch.float64, False)
    got = voxel_features(samples, states, dout, DEV, torch.float32, True)
    p = ((samples['sampled_point_xyz'] - states['voxel_center_xyz'][
        samples['sampled_point_voxel_idx']]) / 0.2).abs().max()
    e = float(states['voxel_vertex_emb'].abs().max())
    d = float(dout.abs().max())
    w = float((1.5 + p)**3)
    rows = torch.bincount(states['voxel_vertex_idx'][
        samples['sampled_point_voxel_idx']].reshape(-1).long()).max()
    assert int(rows) <= 200
    for a, b, terms in zip(got, want, (8 * w * e, 8 * 16 * w * e * d / 0.2 * 3,
                                       200 * w * d)):
        off = (a.detach().double().cpu() - b.detach().double()).abs().max()
        assert float(off) <= 240 * tu.U * terms
    again = voxel_features(samples, states, dout, DEV, torch.float32, True)
    assert all(torch.equal(u, v) for u, v in zip(got, again))


def test_refusals():
    table = torch.zeros(4, 8, device=DEV)
    ids = torch.zeros(5, dtype=torch.int64, device=DEV)
    bad = [
        lambda: tokens.plan(ids.float(), 4),
        lambda: tokens.plan(ids, 0),
        lambda: tokens.plan(ids, 1 << 31),
        lambda: tokens.lookup(table, ids.float()),
        lambda: tokens.lookup(table.double(), ids),
        lambda: tokens.lookup(table[0], ids),
        lambda: tokens.lookup(table, ids.cpu()),
        lambda: tokens.lookup(table, ids, torch.ones(4, device=DEV)),
        lambda: tokens.lookup(table, ids, torch.ones(5)),
        lambda: tokens.lookup(table, ids, torch.ones(
            5, dtype=torch.int64, device=DEV)),
        lambda: tokens.lookup(table, ids, plan=tokens.plan(ids, 5)),
        lambda: tokens.lookup(table, ids, plan=tokens.plan(ids[:3], 4)),
    ]
    for f in bad:
        with pytest.raises(_lib.XrdError):
            f()
    table.requires_grad_(True)
    y = tokens.lookup(table, ids)
    g, = torch.autograd.grad(y.square().sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):       # differentiable once
        torch.autograd.grad(g.sum(), table)


def test_a_plan_that_was_taken_apart_is_refused():
    table = torch.zeros(4, 8, device=DEV)
    ids = torch.zeros(5, dtype=torch.int64, device=DEV)
    p = tokens.plan(ids, 4)
    for order, starts in ((p.order.long(), p.starts),
                          (p.order, p.starts.float()),
                          (p.order, p.starts[:4]), (p.order.cpu(), p.starts),
                          (p.order, p.starts.cpu()),
                          (p.order.repeat(2)[::2], p.starts)):
        with pytest.raises(_lib.XrdError):
            tokens.lookup(table, ids,
                          plan=tokens.TokenPlan(order, starts, None, 4))
    tokens.lookup(table, ids, plan=p)


@pytest.mark.parametrize('dtype,rows,dim', [(torch.float32, 9001, 1024),
                                            (torch.bfloat16, 70000, 248),
                                            (torch.float16, 120001, 144)])
def test_table_gradient_larger_than_the_caches(dtype, rows, dim):
    """more than 32 MB: stored another way"""
    assert rows * dim * torch.finfo(dtype).bits // 8 > 32 << 20
    for k in (None, 2):
        table, ids, w, dout = make(rows, 500, k, dim, dtype, 3)
        ids[::3] = 7                           # a row of many tokens
        args = [t if t is None else t.to(DEV) for t in (table, ids, w, dout)]
        check_lookup(*args, 0.75)
