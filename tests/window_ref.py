"""Attention with a sliding window and sinks in 64 bits, written from its definition, and the error an
f32-accurate kernel may have against it."""
import numpy as np


def visible(p, n, window, sinks):
    """Positions below the cache length n that a query at position p sees, ascending."""
    return [j for j in range(min(p + 1, n)) if p - j < window or j < sinks]


def attend(q, k, v, pos, scale, group):
    """q [heads, D] over the cache rows k, v [n, kv, D] (any dtype) it sees; (out, bound), both [heads, D].
    bound is how far an f32 result may be off, per element:

      a score is a sum of D products of operands held to 2^-22 (two 11-bit halves; f32 holds more), in f32:
          ds <= (D + 8) 2^-23 sum |q k| scale             (every partial sum truncated: an ulp, not half)
      a weight is off by ds relative, the exponential and the joining of parts by a few ulp more:
          dp / p <= 2 max ds + 2^-20
      and the sum over n positions adds n ulp in the worst order:  n 2^-23.
    All of it multiplies sum p |v|; the division by the sum of the weights repeats it once."""
    heads, D = q.shape
    if len(pos) == 0:
        return np.full((heads, D), np.nan), np.zeros((heads, D))
    out, bound = np.zeros((heads, D)), np.zeros((heads, D))
    for h in range(heads):
        kk, vv, qq = k[pos, h // group].astype(np.float64), v[pos, h // group].astype(np.float64), q[h].astype(np.float64)
        s = kk @ qq * scale
        ds = ((D + 8) * 2.0**-23 * (np.abs(kk) @ np.abs(qq)) * abs(scale)).max()
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h] = w @ vv
        bound[h] = 2 * (2 * ds + 2.0**-20 + len(pos) * 2.0**-23) * (w @ np.abs(vv)) + 2.0**-126
    return out, bound


# A kernel may also not be off by more than this in the 2-norm of a whole output.  The four operands of the
# two products are held to 2^-22 or better, which is 2^-20 together, and unlike the bound above the
# roundings of a sum of n random signs grow as sqrt(n), not n: 2^-18 leaves four times that for them.
NORM = 2.0**-18


def check(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: rows that see nothing, and only they, are NaN"
    m = ~np.isnan(want)
    if not m.any():
        return
    d = np.abs(got[m] - want[m])
    worst = float(np.max(d / bound[m]))
    assert worst <= 1, f"{what}: {worst:.2f} of the bound"
    assert np.linalg.norm(d) <= NORM * np.linalg.norm(want[m]), f"{what}: {np.linalg.norm(d) / np.linalg.norm(want[m]):.2e}"
