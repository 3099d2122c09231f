"""Windowed attention over queries, keys and values whose elements are far apart in size, on a B200.  The products are taken of
parts of fewer bits; what a large element of a row may cost its small ones is what these tests look for.  Tolerances are
window_ref's: every operand is held as f32 holds it, but for two bits."""
import numpy as np
import pytest
import torch

from accel_b200 import runtime as rt
from accel_b200 import tensor as T
from accel_b200.blockpool import BlockPool
from test_window_attention_gpu import Cache
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


def prefill(q, k, v, n, base, window, sinks, scale=None):
    D = q.shape[-1]
    got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
        lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D) if scale is None else scale, base=base, window=window,
        sinks=sinks)).cpu().numpy()
    assert "tcgen05 tiles" in rt.last_selection()
    rt.attention_error()
    return got


@pytest.mark.parametrize("qH,kv,D", [(4, 2, 128), (8, 1, 64), (3, 3, 40)])
@pytest.mark.parametrize("where,size", [("key", 1e8), ("key element", 1e15), ("value", 1e8), ("value element", 1e20), ("value", 1e5), ("key", -1e36)])
def test_a_large_key_or_value_stays_with_the_rows_that_see_it(where, size, qH, kv, D):
    # a tile holds 128 positions: the large one lies among others that earlier and later rows see without it
    tokens, window, sinks, j = 300, 60, 2, 140
    rng = np.random.default_rng(7)
    k, v = (rng.standard_normal((tokens, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
    x = k if where.startswith("key") else v
    if where.endswith("element"):
        x[j, 0, 5] = size
    else:
        x[j] = size * rng.uniform(0.5, 1, (kv, D))
    got = prefill(q, k, v, tokens, 0, window, sinks)
    for i in [*range(j - 30, j + 3), j + window - 1, *range(j + window, j + window + 40), 299]:
        check(got[i], *attend(q[i], k, v, visible(i, tokens, window, sinks), attn_scale(D), qH // kv), f"row {i}")


@pytest.mark.parametrize("size", [1e5, 1e10, 1e30])
@pytest.mark.parametrize("qH,kv,D", [(4, 2, 128), (4, 1, 64)])
def test_a_large_channel_of_the_values_costs_the_others_nothing(qH, kv, D, size):
    tokens, n, window = 260, 400, 150
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((n, kv, D)).astype(np.float32) for _ in range(2))
    v[..., 7] *= size
    v[..., 9] /= size
    q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
    got = prefill(q, k, v, n, n - tokens, window, 0)
    for i in range(0, tokens, 13):
        want, bound = attend(q[i], k, v, visible(n - tokens + i, n, window, 0), attn_scale(D), qH // kv)
        for part in ([7], [9], [d for d in range(D) if d not in (7, 9)]):
            check(got[i][:, part], want[:, part], bound[:, part], f"row {i} channel(s) {part[:3]}")


@pytest.mark.parametrize("order", [1, -1])
def test_large_values_under_small_weights(order):
    # tiles of 128 positions at values of 1e8 and scores 31 below the others', before and behind them
    qH, kv, D, n, tokens = 4, 2, 128, 1024, 256
    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((n, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
    q[..., 0], k[..., 0] = 1, 0
    low = (np.arange(n) // 128 >= 3)[::order]
    k[low, :, 0], v[low] = -31 / attn_scale(D), v[low] * 1e8
    got = prefill(q, k, v, n, n - tokens, n, 0)
    for i in range(0, tokens, 17):
        check(got[i], *attend(q[i], k, v, visible(n - tokens + i, n, n, 0), attn_scale(D), qH // kv), f"row {i}")


def test_values_near_the_end_of_f32():
    qH, kv, D, tokens, window = 4, 2, 128, 300, 90
    rng = np.random.default_rng(6)
    k, v = (rng.standard_normal((tokens, kv, D)).astype(np.float32) for _ in range(2))
    v *= np.float32(2e35)                                          # sums of 90 of them with weights up to 1 fit
    q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
    got = prefill(q, k, v, tokens, 0, window, 1)
    for i in range(0, tokens, 13):
        check(got[i], *attend(q[i], k, v, visible(i, tokens, window, 1), attn_scale(D), 2), f"row {i}")


FAR = np.float32(2.0**22)


@pytest.mark.parametrize("qH,kv,D,block", [(8, 2, 128, 16), (6, 2, 40, 5), (4, 4, 64, 8), (5, 1, 96, 7)])
def test_channels_further_apart_than_two_parts_hold(qH, kv, D, block):
    # every tile goes to the CUDA cores: paged prefills over windows, sinks and missing pages, split and whole
    for tokens, base, window, sinks in ((256, 0, 300, 0), (260, 77, 200, 9), (256, 500, 128, 4), (300, 40, 1, 0), (256, 3000, 2900, 30)):
        n = base + tokens
        c = Cache(tokens, kv, D, block, [n], [base], window, sinks, False)
        c.pk[..., ::2] *= FAR
        c.k[0][..., ::2] *= FAR
        q = np.random.default_rng(3).standard_normal((tokens, qH, D)).astype(np.float32)
        q[..., ::2] /= FAR
        lost = None
        if tokens == 260:                                          # a visible page that is not in the cache: its positions are masked
            lost = (base + 100) // block
            c.pages[0, lost] = BlockPool.NONE
        got = T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
            lengths=dev(np.array([n], np.uint32)), pages=dev(c.pages[0]), block=block, scale=attn_scale(D), base=base, window=window,
            sinks=sinks)).cpu().numpy()
        assert "tcgen05 tiles" in rt.last_selection()
        for i in range(0, tokens, 9):
            seen = [j for j in visible(base + i, n, window, sinks) if j // block != lost]
            check(got[i], *attend(q[i], c.k[0], c.v[0], seen, attn_scale(D), qH // kv), f"{tokens} behind {base}, row {i}")
    rt.attention_error()


def test_ragged_chunks_with_channels_far_apart_beside_ordinary_ones():
    qH, kv, D, block, window, sinks = 8, 2, 128, 16, 90, 3
    lengths, counts = [300, 41, 200, 150], [70, 1, 200, 130]
    c = Cache(5, kv, D, block, lengths, [n - m for n, m in zip(lengths, counts)], window, sinks, False)
    q = np.random.default_rng(8).standard_normal((sum(counts), qH, D)).astype(np.float32)
    for page in c.pages[2]:                                        # the third sequence alone
        if page != BlockPool.NONE:
            c.pk[int(page) * block:(int(page) + 1) * block, :, ::2] *= FAR
    c.k[2][..., ::2] *= FAR
    q[71:271, :, ::2] /= FAR
    got = T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
        lengths=dev(np.array(lengths, np.uint32)), pages=dev(c.pages), block=block, scale=attn_scale(D),
        query_extents=dev(np.array(counts, np.uint32)), window=window, sinks=sinks)).cpu().numpy()
    assert "tcgen05 tiles" in rt.last_selection()
    r = 0
    for b, (n, m) in enumerate(zip(lengths, counts)):
        for i in range(m):
            if i % 7 == 0:
                check(got[r], *attend(q[r], c.k[b], c.v[b], visible(n - m + i, n, window, sinks), attn_scale(D), qH // kv), f"{b} {i}")
            r += 1
    rt.attention_error()


def test_values_that_are_not_finite_beside_large_ones():
    qH, kv, D, tokens, window = 4, 2, 128, 300, 20
    rng = np.random.default_rng(6)
    k, v = (rng.standard_normal((tokens, kv, D)).astype(np.float32) for _ in range(2))
    v[150, 0, 5], v[151, 1, 7], k[160, 0, 3], v[140] = np.inf, np.nan, np.nan, 1e9
    k[170] *= 1e6
    q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
    got = prefill(q, k, v, tokens, 0, window, 2)
    for i in range(120, 200):
        for h in range(qH):
            seen, kvh = visible(i, tokens, window, 2), h // 2
            if kvh == 0 and 160 in seen:
                assert np.isnan(got[i, h]).all(), i
            elif (150 if kvh == 0 else 151) in seen:
                d = 5 if kvh == 0 else 7
                assert not np.isfinite(got[i, h, d]) and np.isfinite(np.delete(got[i, h], d)).all(), i
            else:
                o, b = attend(q[i, h:h + 1], k[:, kvh:kvh + 1], v[:, kvh:kvh + 1], seen, attn_scale(D), 1)
                check(got[i, h:h + 1], o, b, f"row {i} head {h}")


@pytest.mark.parametrize("qH,kv,D", [(4, 4, 128), (4, 1, 64), (8, 1, 128), (20, 2, 40)])
def test_single_tokens_over_channels_and_positions_far_apart(qH, kv, D):
    # the row kernels' parts have f32's exponents: the same inputs without tiles
    n, window, sinks = 900, 700, 4
    rng = np.random.default_rng(D)
    k, v = (rng.standard_normal((n, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((3, qH, D)).astype(np.float32)
    k[..., ::2] *= FAR
    q[..., ::2] /= FAR
    v[..., 7] *= np.float32(1e12)
    v[50], v[190] = 1e9, -1e30                                     # positions that no row sees
    base = n - 3
    got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
        lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D), base=base, window=window, sinks=sinks)).cpu().numpy()
    assert "tcgen05 tiles" not in rt.last_selection()
    rest = [d for d in range(D) if d != 7]
    for i in range(3):
        want, bound = attend(q[i], k, v, visible(base + i, n, window, sinks), attn_scale(D), qH // kv)
        for part in ([7], rest):
            check(got[i][:, part], want[:, part], bound[:, part], f"row {i}")


def test_tiles_far_apart_repeat_their_bits_on_any_stream_and_in_graphs():
    def job(seed):
        rng = np.random.default_rng(seed)
        k, v = (rng.standard_normal((400, 2, 128)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((300, 8, 128)).astype(np.float32)
        v[150:160] *= np.float32(1e8)
        k[300:, :, ::2] *= FAR
        k, v, q = dev(k), dev(v), dev(q)
        o = T.AttentionOptions(lengths=dev(np.array([400], np.uint32)), scale=0.09, base=100, window=90, sinks=4)
        return lambda: T.attention(q, k, v, o)

    jobs = [job(1), job(2)]
    want = [j().cpu() for j in jobs]
    graphs, outs = [], []
    for j in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(j())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in jobs]
    eager = []
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s, j in zip(graphs, streams, jobs):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(j())
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), w) for o, w in zip(outs, want))
    assert all(torch.equal(e.cpu(), want[i % 2]) for i, e in enumerate(eager))
