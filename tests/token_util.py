"""Plain 64-bit forms of the token and grouped-product operators, and the
error bounds their f32 sums have to stay within.

U is half a step of f32.  A sum of c products in f32, in any order, is off by at
most c U sum|terms| (first order); the scale and the weight are two more
roundings.  The result's own rounding is half a step of its type."""
import numpy as np
import torch

U = 2.0**-24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, terms, count, what=''):
    """|got - want| <= count U terms + half a step of got's type (plus its
    smallest subnormal, for results that round below it).  The 1.01 covers the
    second-order terms: count U stays under 0.01 in every test."""
    assert float(np.max(count, initial=0)) * U < 0.01
    g = got.detach().double().cpu().numpy()
    f = torch.finfo(got.dtype)
    lim = 1.01 * (count * U * terms + half_step(got.dtype) * np.abs(want)) + \
        half_step(got.dtype) * count * U * terms + f.tiny * f.eps
    bad = ~(np.abs(g - want) <= lim)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(),
                           g[bad][:4], want[bad][:4], lim[bad][:4])


def host(t):
    return t.detach().double().cpu().numpy()


def lookup64(table, ids, weights, scale):
    """-> (y, sum of |terms|) for ids [n, k]"""
    e, w = host(table), np.ones(ids.shape) if weights is None else host(weights)
    i = ids.cpu().numpy().astype(np.int64)
    ok = (i >= 0) & (i < e.shape[0])
    rows = np.where(ok[..., None], e[np.where(ok, i, 0)], 0.0) if e.size else \
        np.zeros(i.shape + (e.shape[1], ))
    w = np.where(ok, w, 0.0)
    t = scale * w[..., None] * rows
    return t.sum(1), np.abs(t).sum(1)


def lookup_grads64(table, ids, weights, scale, dout):
    """-> (dtable, its |terms|, tokens a row, dweights, its |terms|)"""
    e, g = host(table), host(dout)
    n, k = ids.shape
    i = ids.cpu().numpy().astype(np.int64)
    ok = (i >= 0) & (i < e.shape[0])
    w = np.ones((n, k)) if weights is None else host(weights)
    d, da = np.zeros_like(e), np.zeros_like(e)
    cnt = np.zeros((e.shape[0], 1))
    t = scale * np.where(ok, w, 0.0)[..., None] * g[:, None]
    np.add.at(d, i[ok], t[ok])
    np.add.at(da, i[ok], np.abs(t[ok]))
    np.add.at(cnt, i[ok], 1.0)
    dw, dwa = np.zeros((n, k)), np.zeros((n, k))
    if e.size:
        p = scale * e[np.where(ok, i, 0)] * g[:, None]
        dw, dwa = np.where(ok, p.sum(-1), 0), np.where(ok, np.abs(p).sum(-1), 0)
    return d, da, cnt, dw, dwa


def spans(starts, m):
    s = np.clip(np.asarray(starts, np.int64), 0, m)
    return [(e, int(a), int(max(a, b)))
            for e, (a, b) in enumerate(zip(s, s[1:]))]


def linear64(x, w, starts, bias):
    """-> (pre-activation z, sum of |terms|)"""
    x, w = host(x), host(w)
    z = np.zeros((x.shape[0], w.shape[1]))
    za = np.zeros_like(z)
    for e, a, b in spans(starts, x.shape[0]):
        if a == b:
            continue
        z[a:b] = x[a:b] @ w[e].T
        za[a:b] = np.abs(x[a:b]) @ np.abs(w[e]).T
        if bias is not None:
            z[a:b] += host(bias)[e]
            za[a:b] += np.abs(host(bias)[e])
    return z, za


def linear_grads64(x, w, starts, dz):
    """dz: numpy f64, already masked -> {name: (value, |terms|, count)}"""
    x, w = host(x), host(w)
    out = {k: (np.zeros(s), np.zeros(s), np.zeros(c)) for k, s, c in (
        ('x', x.shape, (1, 1)), ('w', w.shape, (w.shape[0], 1, 1)),
        ('b', w.shape[:2], (w.shape[0], 1)))}
    out['x'][2][...] = w.shape[1]
    for e, a, b in spans(starts, x.shape[0]):
        if a == b:
            continue
        out['x'][0][a:b] = dz[a:b] @ w[e]
        out['x'][1][a:b] = np.abs(dz[a:b]) @ np.abs(w[e])
        out['w'][0][e] = dz[a:b].T @ x[a:b]
        out['w'][1][e] = np.abs(dz[a:b]).T @ np.abs(x[a:b])
        out['b'][0][e] = dz[a:b].sum(0)
        out['b'][1][e] = np.abs(dz[a:b]).sum(0)
        out['w'][2][e] = out['b'][2][e] = b - a
    return out
