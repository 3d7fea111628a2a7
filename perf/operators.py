"""What is measured of the token and grouped-product operators
(``xrdslam_amd.engine.tokens``, ``xrdslam_amd.engine.grouped``): cases, their
inputs, one pass through each, and the same in plain torch.

    plan    tokens sorted stably by id: order, group starts
    lookup  y_i = scale * sum_k w_ik table[id_ik], with its gradients
    linear  y_r = act(W_e x_r + b_e) over the ragged groups e, with its gradients

``run`` goes through the plain form unless ``own`` is set.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPE = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
_SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}


def listed():
    return [
        # a router's choice of two of sixteen local decoders for 1000 rays: the
        # plan's launch latency is all there is
        dict(name='plan_router', op='plan', n=2000, groups=16, ids='router',
             bits=64),
        # the eight corner ids of 49152 samples of a mapping batch, sorted for
        # the gradient of a 20000-row voxel table
        dict(name='plan_voxels', op='plan', n=393216, groups=20000,
             ids='voxels', bits=32),
        # rows of four tokens of a wide table, one step of a running program
        dict(name='lookup_step', op='lookup', n=4, k=0, rows=32768, dim=1024,
             dtype='bf16', ids='zipf', scale=32.0, train=False, missing=0.0),
        # trilinear features of a voxel-map mapping iteration: eight weighted
        # corners, 16 columns, gradients to the table and to the weights
        dict(name='lookup_voxels', op='lookup', n=49152, k=8, rows=20000,
             dim=16, dtype='f32', ids='voxels', scale=1.0, train=True,
             missing=0.0),
        # inverse-distance features of a point map: eight neighbours of which
        # some are missing, 32 columns, an odd number of points
        dict(name='lookup_points', op='lookup', n=25000, k=8, rows=100003,
             dim=32, dtype='f32', ids='points', scale=1.0, train=True,
             missing=0.2),
        # a wide 16-bit table with word-like frequencies: a few rows own much
        # of the batch
        dict(name='lookup_wide', op='lookup', n=8192, k=0, rows=32000,
             dim=2048, dtype='bf16', ids='zipf', scale=math.sqrt(2048.0),
             train=True, missing=0.0),
        # eight rows spread over six of sixteen decoders: weights are read for
        # a handful of rows
        dict(name='linear_few', op='linear', m=8, groups=16, active=6, tail=0,
             inp=1024, out=2048, dtype='bf16', bias=False, relu=False,
             train=False),
        # a hidden layer of eight local decoders over a mapping batch
        dict(name='linear_bank', op='linear', m=49152, groups=8, active=8,
             tail=0, inp=128, out=128, dtype='f32', bias=True, relu=False,
             train=True),
        # the colour head's odd widths, an odd number of rows, some of them
        # outside every decoder
        dict(name='linear_odd', op='linear', m=20011, groups=5, active=5,
             tail=37, inp=144, out=129, dtype='f32', bias=True, relu=False,
             train=True),
        # a wide first layer in half precision, its ReLU included, answers only
        dict(name='linear_relu', op='linear', m=5000, groups=32, active=27,
             tail=0, inp=1024, out=4096, dtype='f16', bias=True, relu=True,
             train=False),
        # a training step of sixteen wide experts
        dict(name='linear_wide', op='linear', m=16384, groups=16, active=16,
             tail=0, inp=2048, out=2048, dtype='bf16', bias=False, relu=False,
             train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(
        rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['plan', 'lookup', 'lookup', 'linear', 'linear', 'linear'])
    if op == 'plan':
        ids = rng.choice(['router', 'voxels', 'zipf'])
        return dict(op=op, n=_log(rng, 1, 1 << 20),
                    groups=_log(rng, 1, 256) if ids == 'router'
                    else _log(rng, 100, 200000), ids=ids,
                    bits=rng.choice([32, 64]))
    if op == 'lookup':
        k = rng.choice([0, 0, 1, 2, 3, 8, 8])
        n = _log(rng, 1, 65536)
        dim = rng.choice([rng.randint(1, 64), 16, 32, _log(rng, 64, 2048),
                          8 * _log(rng, 8, 256)])
        while n * max(k, 1) * dim > 1 << 24:
            n = max(1, n // 2 - rng.randint(0, 1))
        rows = _log(rng, 2, 100000)
        while rows * dim > 1 << 26:
            rows = rows // 2 + rng.randint(0, 1)
        return dict(op=op, n=n, k=k, rows=rows, dim=dim,
                    dtype=rng.choice(['f32', 'f32', 'bf16', 'f16']),
                    ids=rng.choice(['voxels', 'points', 'zipf']) if k
                    else 'zipf',
                    scale=rng.choice([1.0, 0.5, math.sqrt(dim)]),
                    train=rng.random() < 0.7,
                    missing=rng.choice([0.0, 0.2]) if k else 0.0)
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    top = 512 if dtype == 'f32' else 2048
    inp, out = (rng.choice([_log(rng, 3, top), 8 * _log(rng, 4, top // 8)])
                for _ in range(2))
    m = _log(rng, 1, 32768)
    while m * inp * out > 1 << 35:
        m = m // 2 - rng.randint(0, 1)
    groups = _log(rng, 1, 64)
    return dict(op='linear', m=m, groups=groups,
                active=min(m, rng.randint(1, groups)),
                tail=rng.choice([0, 0, rng.randint(1, 40)]), inp=inp, out=out,
                dtype=dtype, bias=rng.random() < 0.5,
                relu=(relu := rng.random() < 0.3),
                train=not relu and rng.random() < 0.7)


# ------------------------------------------------------------------- inputs
def _bounds(case, seed):
    """group starts on the host: ``active`` groups of uneven sizes, the others
    empty"""
    rng = random.Random(seed * 7919 + 17)
    free = case['m'] - case['active']
    cuts = sorted(rng.randint(0, free) for _ in range(case['active'] - 1))
    sizes = [1 + b - a for a, b in zip([0] + cuts, cuts + [free])]
    at = set(rng.sample(range(case['groups']), case['active']))
    b = [0]
    for e in range(case['groups']):
        b.append(b[-1] + (sizes.pop() if e in at else 0))
    return b


def _ids(kind, n, k, rows, missing, gen, dev):
    """[n, k] ids: 'voxels' - runs of samples inside one voxel, whose corners
    are k rows of the table; 'points' - k different rows near each other;
    'zipf' - word-like frequencies; 'router' - k experts, unevenly loved"""
    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=dev)
    if kind == 'voxels':
        runs = n // 6 + 1
        corner = (rand(max(rows // 2, 1), k) * rows).long()
        voxel = (rand(runs) * corner.shape[0]).long()
        ids = corner[voxel.repeat_interleave(6)[:n]]
    elif kind == 'points':
        ids = ((rand(n, 1) * rows).long() +
               torch.arange(k, device=dev) * 7) % rows
    elif kind == 'router':
        ids = (rand(n, k)**2 * rows).long()
    else:
        ids = torch.exp(rand(n, k) * math.log(rows)).long() - 1
    ids = ids.clamp(0, rows - 1)
    if missing:
        ids = torch.where(rand(n, k) < missing, -1, ids)
    return ids


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)
    s = dict(case=case)
    if case['op'] == 'plan':
        k = 8 if case['ids'] == 'voxels' and case['n'] % 8 == 0 else 1
        ids = _ids(case['ids'], case['n'] // k, k, case['groups'], 0.0, gen,
                   dev).reshape(-1)
        s['ids'] = ids if case['bits'] == 64 else ids.int()
        return s
    dt = _DTYPE[case['dtype']]
    if case['op'] == 'lookup':
        n, k, rows, dim = case['n'], case['k'], case['rows'], case['dim']
        ids = _ids(case['ids'], n, max(k, 1), rows, case['missing'], gen, dev)
        s['ids'] = ids if k else ids.reshape(-1)
        s['table'] = (normal(rows, dim) * 0.1).to(dt)
        s['weights'] = None
        if k:
            w = torch.rand(n, k, generator=gen, device=dev) + 0.01
            w = torch.where(ids < 0, torch.zeros_like(w), w)
            s['weights'] = w / w.sum(1, keepdim=True).clamp(min=1e-6)
        if case['train']:
            s['table'].requires_grad_(True)
            if k:
                s['weights'].requires_grad_(True)
            s['dout'] = (normal(n, dim) * 0.1).to(dt)
        return s
    m, inp, out = case['m'] + case['tail'], case['inp'], case['out']
    s['bounds'] = _bounds(case, seed)
    s['starts'] = torch.tensor(s['bounds'], dtype=torch.int32, device=dev)
    s['x'] = normal(m, inp).to(dt)
    s['weight'] = ((torch.rand(case['groups'], out, inp, generator=gen,
                               device=dev) * 2 - 1) / math.sqrt(inp)).to(dt)
    s['bias'] = (normal(case['groups'], out) * 0.1).to(dt) \
        if case['bias'] else None
    if case['train']:
        for key in ('x', 'weight', 'bias'):
            if s[key] is not None:
                s[key].requires_grad_(True)
        s['dout'] = (normal(m, out) * 0.1).to(dt)
    return s


# --------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {'plan': _plain_plan, 'lookup': _plain_lookup,
                'linear': _plain_linear}[state['case']['op']](state)


def _run_own(s):
    from xrdslam_amd.engine import grouped, tokens
    case = s['case']
    if case['op'] == 'plan':
        p = tokens.plan(s['ids'], case['groups'])
        return p.order, p.starts
    if case['op'] == 'lookup':
        y = tokens.lookup(s['table'], s['ids'], s['weights'],
                          scale=case['scale'])
        leaves = [s['table'], s['weights']]
    else:
        y = grouped.linear(s['x'], s['weight'], s['starts'], bias=s['bias'],
                           relu=case['relu'])
        leaves = [s['x'], s['weight'], s['bias']]
    if not case['train']:
        return y
    leaves = [t for t in leaves if t is not None]
    return (y.detach(), *torch.autograd.grad(y, leaves, s['dout']))


def _plain_plan(s):
    ids, groups = s['ids'], s['case']['groups']
    key = torch.where((ids >= 0) & (ids < groups), ids, groups)
    key, order = torch.sort(key, stable=True)
    at = torch.arange(groups + 1, device=ids.device, dtype=ids.dtype)
    return order.int(), torch.searchsorted(key, at).int()


def _plain_lookup(s):
    case, table, ids = s['case'], s['table'], s['ids']
    dt, scale = table.dtype, case['scale']
    if s['weights'] is None:
        y = table[ids].float() * scale
    else:
        hit = ids >= 0
        idc = ids.clamp(min=0)
        w = torch.where(hit, s['weights'], 0.0)
        rows = table[idc].float()
        y = (w[..., None] * rows).sum(1) * scale
    if not case['train']:
        return y.to(dt)
    g = s['dout'].float() * scale
    dtable = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
    if s['weights'] is None:
        dtable.index_add_(0, ids, g)
        return y.to(dt), dtable.to(dt)
    dtable.index_add_(0, idc.reshape(-1),
                      (w[..., None] * g[:, None]).reshape(-1, case['dim']))
    dw = torch.where(hit, (rows * g[:, None]).sum(-1), 0.0)
    return y.to(dt), dtable.to(dt), dw


def _plain_linear(s):
    case, x, w, b = s['case'], s['x'].float(), s['weight'], s['bias']
    dt = w.dtype
    y = torch.zeros(x.shape[0], case['out'], device=x.device)
    spans = [(e, lo, hi) for e, (lo, hi) in enumerate(
        zip(s['bounds'], s['bounds'][1:])) if hi > lo]
    for e, lo, hi in spans:
        y[lo:hi] = x[lo:hi] @ w[e].float().T
        if b is not None:
            y[lo:hi] += b[e].float()
    if case['relu']:
        y = y.clamp(min=0.0)
    if not case['train']:
        return y.to(dt)
    g = s['dout'].float()
    dx = torch.zeros_like(x)
    dw = torch.zeros(w.shape, device=x.device)
    db = torch.zeros(w.shape[:2], device=x.device)
    for e, lo, hi in spans:
        dx[lo:hi] = g[lo:hi] @ w[e].float()
        dw[e] = g[lo:hi].T @ x[lo:hi]
        db[e] = g[lo:hi].sum(0)
    grads = (dx.to(dt), dw.to(dt)) + (() if b is None else (db.to(dt), ))
    return (y.to(dt), *grads)


# -------------------------------------------------------------------- work
def work(case):
    """each input read once, each output written once"""
    if case['op'] == 'plan':
        return dict(bytes=case['n'] * (case['bits'] // 8 + 4) +
                    4 * (case['groups'] + 1), flops=0)
    b = _SIZE[case['dtype']]
    if case['op'] == 'lookup':
        n, k, dim = case['n'], max(case['k'], 1), case['dim']
        touched = min(case['rows'], n * k)
        w = 4 * n * case['k']
        byt = 8 * n * k + w + (touched + n) * dim * b
        if case['train']:
            byt += (n + case['rows']) * dim * b + w
        passes = 1 + (1 + (case['k'] > 0)) * case['train']
        return dict(bytes=byt, flops=2 * n * k * dim * passes)
    m, inp, out = case['m'], case['inp'], case['out']
    wb = inp * out * b
    byt = m * (inp + out) * b + case['active'] * wb
    if case['train']:
        byt += m * (out + inp) * b + case['groups'] * wb
    return dict(bytes=byt + case['tail'] * out * b,
                flops=2 * m * inp * out * (3 if case['train'] else 1))


# -------------------------------------------------------------------- exact
def exact(case, seed):
    """the definitions in 64 bits: numpy for the sort and the lookup, a float64
    product per group for the linear"""
    s = prepare(case, seed)
    if case['op'] == 'plan':
        ids = s['ids'].cpu().numpy().astype(np.int64)
        order = np.lexsort((np.arange(ids.size), ids))
        counts = np.bincount(ids, minlength=case['groups'])
        starts = np.concatenate([[0], np.cumsum(counts)])
        return order.astype(np.int32), starts.astype(np.int32)
    if case['op'] == 'lookup':
        return _exact_lookup(case, s)
    return _exact_linear(case, s)


def _exact_lookup(case, s):
    def host(t):
        return t.detach().double().cpu().numpy()
    n, k, scale = case['n'], max(case['k'], 1), case['scale']
    ids = s['ids'].cpu().numpy().reshape(n, k)
    table = host(s['table'])
    w = np.ones((n, k)) if s['weights'] is None else host(s['weights'])
    hit = ids >= 0
    padded = np.concatenate([table, np.zeros((1, case['dim']))])
    y = np.zeros((n, case['dim']))
    for j in range(k):
        y += (scale * w[:, j])[:, None] * padded[ids[:, j]]
    if not case['train']:
        return y
    g = scale * host(s['dout'])
    flat = np.flatnonzero(hit.reshape(-1))
    flat = flat[np.argsort(ids.reshape(-1)[flat], kind='stable')]
    dtable = np.zeros_like(table)
    if flat.size:
        who = ids.reshape(-1)[flat]
        first = np.flatnonzero(np.concatenate([[True], who[1:] != who[:-1]]))
        dtable[who[first]] = np.add.reduceat(
            g[flat // k] * w.reshape(-1)[flat][:, None], first, axis=0)
    if s['weights'] is None:
        return y, dtable
    dw = np.zeros((n, k))
    for j in range(k):
        dw[:, j] = np.einsum('nd,nd->n', padded[ids[:, j]], g) * hit[:, j]
    return y, dtable, dw


def _exact_linear(case, s):
    x, w = s['x'].detach().double(), s['weight'].detach()
    y = x.new_zeros(x.shape[0], case['out'])
    group = np.repeat(np.arange(case['groups']), np.diff(s['bounds']))
    train = case['train']
    if train:
        g = s['dout'].double()
        dx, dw = torch.zeros_like(x), x.new_zeros(w.shape)
        db = x.new_zeros(w.shape[:2])
    for e in np.unique(group):
        r = torch.from_numpy(np.flatnonzero(group == e)).to(x.device)
        we, xe = w[e].double(), x[r]
        ye = torch.mm(we, xe.t()).t()
        if s['bias'] is not None:
            ye = ye + s['bias'][e].detach().double()
        y[r] = torch.relu(ye) if case['relu'] else ye
        if train:
            ge = g[r]
            dx[r] = torch.mm(ge, we)
            dw[e] = torch.mm(xe.t(), ge).t()
            db[e] = torch.ones(1, len(r), device=x.device,
                               dtype=torch.float64).mm(ge)[0]
    if not train:
        return y
    return (y, dx, dw) if s['bias'] is None else (y, dx, dw, db)
