"""Windowed attention over queries, keys and values whose elements are far apart in size, on a B200.  The products are taken of
parts of fewer bits; what a large element of a row may cost its small ones is what these tests look for.  Tolerances are
window_ref's: every operand is held as f32 holds it, but for two bits."""
import numpy as np
import pytest
import torch

from accel_b200 import runtime as rt
from accel_b200 import tensor as T
from util import attn_scale
from window_ref import attend, check, visible

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).to(DEV)


def spread(rng, kind, tokens, n, qH, kv, D):
    """Scores of ordinary size out of channels that are not: (q, k)."""
    q, k = rng.standard_normal((tokens, qH, D)), rng.standard_normal((n, kv, D))
    if kind == "one channel":                       # a query channel at 60 over keys of a thousandth there, one key channel at 300
        q *= 0.07
        q[..., 3] = 60
        k[..., 3] *= 1e-3
        k[..., 9] *= 300
    else:                                           # half the channels small in q and as large in k
        q[..., ::2] *= 1e-4
        k[..., ::2] *= 1e4
    return q.astype(np.float32), k


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("kind", ["one channel", "half"])
@pytest.mark.parametrize("tokens,qH,kv,D", [(1, 4, 1, 128), (1, 8, 1, 128), (1, 6, 2, 40), (300, 4, 2, 128), (300, 4, 1, 64), (300, 3, 3, 40)])
def test_queries_whose_channels_differ_in_size(tokens, qH, kv, D, kind, f16):
    n, window, sinks = 700, 400, 3
    rng = np.random.default_rng(tokens + D)
    q, k = spread(rng, kind, tokens, n, qH, kv, D)
    k = k.astype(np.float16 if f16 else np.float32)
    assert np.isfinite(k).all()
    v = rng.standard_normal((n, kv, D)).astype(k.dtype)
    got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
        lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D), base=n - tokens, window=window, sinks=sinks)).cpu().numpy()
    assert ("tcgen05 tiles" in rt.last_selection()) == (tokens > 1)
    rows = range(0, tokens, 11)
    ref = [attend(q[i], k, v, visible(n - tokens + i, n, window, sinks), attn_scale(D), qH // kv) for i in rows]
    check(got[list(rows)], np.stack([r[0] for r in ref]), np.stack([r[1] for r in ref]), kind)
