"""The device sine and cosine (csrc/common.h sincos_cw), emulated in numpy with
the header's own parts of pi/2 and coefficients in its fma order: against
float64 up to 1e5 rad."""
import os
import re

import numpy as np

HEADER = os.path.join(os.path.dirname(__file__), '..', 'xrdslam_amd', 'csrc',
                      'common.h')
f = np.float32


def fma(a, b, c):
    # (a product of two floats is exact in 64 bits)
    return (a.astype(np.float64) * np.float64(f(b)) if np.isscalar(b) else
            a.astype(np.float64) * b.astype(np.float64)) + \
        (np.float64(f(c)) if np.isscalar(c) else c.astype(np.float64))


def test_parts_of_half_pi():
    text = open(HEADER).read()
    parts = [float(re.search(r'kHalfPi%d = ([-+.e0-9]+)f' % i, text)[1])
             for i in range(3)]
    # pi/2 to 40 digits, in two doubles
    hi, lo = 1.5707963267948966, 6.123233995736766e-17
    want = []
    for _ in range(3):
        p = f(hi + lo)
        want.append(p)
        hi, lo = hi - np.float64(p), lo
    assert [f(p) for p in parts] == want


def test_accuracy():
    text = open(HEADER).read()
    p0, p1, p2 = (float(re.search(r'kHalfPi%d = ([-+.e0-9]+)f' % i, text)[1])
                  for i in range(3))
    body = text[text.index('void sincos_cw'):text.index('struct SinStages')]
    s1, s2, s3 = [float(v) for v in re.search(
        r'ps = fmaf\(s, ([-.e0-9]+)f, ([-.e0-9]+)f\);\s*ps = fmaf\(s, ps, '
        r'([-.e0-9]+)f\)', body).groups()]
    c1, c2, c3 = [float(v) for v in re.search(
        r'pc = fmaf\(s, ([-.e0-9]+)f, ([-.e0-9]+)f\);\s*pc = fmaf\(s, pc, '
        r'([-.e0-9]+)f\)', body).groups()]
    g = np.random.default_rng(0)
    x = np.concatenate([g.uniform(-1e5, 1e5, 400000), g.uniform(-8, 8, 100000),
                        [0.0]]).astype(f)
    k = np.rint(x * f(0.636619772367581)).astype(f)
    r = fma(k, -p0, x).astype(f)
    r = fma(k, -p1, r).astype(f)
    r = fma(k, -p2, r).astype(f)
    s = (r * r).astype(f)
    ps = fma(s, s1, s2).astype(f)
    ps = fma(s, ps, s3).astype(f)
    sn = fma((r * s).astype(f), ps, r).astype(f)
    pc = fma(s, c1, c2).astype(f)
    pc = fma(s, pc, c3).astype(f)
    cs = fma((s * s).astype(f), pc, fma(s, -0.5, 1.0).astype(f)).astype(f)
    n = k.astype(np.int64) & 3
    S = np.where(n == 0, sn, np.where(n == 1, cs, np.where(n == 2, -sn, -cs)))
    C = np.where(n == 0, cs, np.where(n == 1, -sn, np.where(n == 2, -cs, sn)))
    x = x.astype(np.float64)
    # half an ulp of 1 at the result, one of the reduced argument (below pi/4),
    # half of each polynomial's last term, and the polynomials' own 3e-9
    assert np.abs(S - np.sin(x)).max() < 1.5e-7
    assert np.abs(C - np.cos(x)).max() < 1.5e-7
