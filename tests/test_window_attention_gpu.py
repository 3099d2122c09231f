"""Attention with a sliding window and sink positions against its definition in 64 bits, on a B200."""
import numpy as np
import pytest
import torch

from accel_b200 import runtime as rt
from accel_b200 import tensor as T
from accel_b200.blockpool import BlockPool
from util import attn_scale
from window_ref import attend, check, visible

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).to(DEV)


class Cache:
    """Sequences over one paged cache: every position that nobody may read is NaN, and the table entries of
    pages without a visible position are BlockPool.NONE."""

    def __init__(self, seed, kv, D, block, lengths, first, window, sinks, f16, max_pages=None):
        """first[b]: the lowest position of the sequence's queries."""
        rng = np.random.default_rng(seed)
        self.rows, live = [], []
        for n, p in zip(lengths, first):
            see = set()
            for j in range(n):
                if j < sinks or j > p - window:
                    see.add(j // block)
            live.append(see)
            self.rows.append((n + block - 1) // block)
        pool = sum(len(s) for s in live) + 2
        self.capacity = pool * block
        perm = rng.permutation(pool)
        mp = max_pages if max_pages is not None else max(max(self.rows), 1)
        self.pages = np.full((len(lengths), mp), BlockPool.NONE, np.uint32)
        dt = np.float16 if f16 else np.float32
        self.pk, self.pv = (np.full((self.capacity, kv, D), np.nan, dt) for _ in range(2))
        self.k, self.v = [], []
        at = 0
        for b, n in enumerate(lengths):
            k, v = (rng.standard_normal((n, kv, D)).astype(dt) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            for pg in sorted(live[b]):
                if pg < mp:
                    self.pages[b, pg] = perm[at]
                at += 1
                for j in range(pg * block, min((pg + 1) * block, n)):
                    if j < sinks or j > first[b] - window:
                        r = int(perm[at - 1]) * block + j % block
                        self.pk[r], self.pv[r] = k[j], v[j]


HEADS = [(32, 8, 128, 16), (4, 4, 128, 16), (6, 2, 40, 4), (15, 5, 64, 13), (8, 1, 96, 1), (20, 1, 128, 32), (3, 3, 8, 16)]
WINDOWS = [(1, 0), (1, 3), (17, 0), (64, 4), (100, 40), (300, 1), (5000, 7)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("qH,kv,D,block", HEADS)
def test_batched_over_lengths_and_windows(qH, kv, D, block, f16):
    lengths = [1, 2, 16, 63, 64, 65, 256, 301, 517]
    for window, sinks in WINDOWS:
        c = Cache(window * 31 + D, kv, D, block, lengths, [n - 1 for n in lengths], window, sinks, f16)
        q = np.random.default_rng(5).standard_normal((len(lengths), 1, qH, D)).astype(np.float32)
        got = T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
            lengths=dev(np.array(lengths, np.uint32)), pages=dev(c.pages), block=block, scale=attn_scale(D),
            window=window, sinks=sinks)).cpu().numpy()
        ref = [attend(q[b, 0], c.k[b], c.v[b], visible(n - 1, n, window, sinks), attn_scale(D), qH // kv)
               for b, n in enumerate(lengths)]
        check(got, np.stack([r[0] for r in ref]), np.stack([r[1] for r in ref]), f"window {window} sinks {sinks}")


@pytest.mark.parametrize("f16", [False, True])
def test_long_windows_are_split_and_joined(f16):
    # one sequence, so that every part of the list falls to another block of the grid
    for qH, kv, D, n, window, sinks in ((8, 2, 128, 9001, 8000, 5), (2, 1, 64, 5000, 4999, 0), (4, 1, 128, 4096, 2047, 64)):
        c = Cache(9, kv, D, 16, [n], [n - 1], window, sinks, f16)
        q = 3 * np.random.default_rng(5).standard_normal((qH, D)).astype(np.float32)
        got = T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
            lengths=dev(np.array([n], np.uint32)), pages=dev(c.pages[0]), block=16, scale=attn_scale(D), window=window,
            sinks=sinks)).cpu().numpy()
        check(got, *attend(q, c.k[0], c.v[0], visible(n - 1, n, window, sinks), attn_scale(D), qH // kv), f"n {n}")


def test_empty_lengths_past_the_table_and_pages_outside_the_cache():
    kv, D, block, window, sinks = 2, 64, 4, 6, 3
    lengths = [0, 9, 30]
    c = Cache(2, kv, D, block, [0, 9, 30], [0, 8, 20], window, sinks, False, max_pages=8)
    q = np.random.default_rng(1).standard_normal((3, 1, 4, D)).astype(np.float32)

    def run(pages, lens):
        return T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
            lengths=dev(np.array(lens, np.uint32)), pages=dev(pages), block=block, scale=0.1, window=window,
            sinks=sinks)).cpu().numpy()

    got = run(c.pages, lengths)
    assert np.isnan(got[0]).all()                               # nothing to see: 0 / 0
    ref = [attend(q[b, 0], c.k[b], c.v[b], visible(n - 1, n, window, sinks), 0.1, 2) for b, n in enumerate(lengths)]
    check(got, np.stack([r[0] for r in ref]), np.stack([r[1] for r in ref]))
    # a length past the table: the positions beyond it are not there, the window is where the length says
    cut = c.pages[:, :6].copy()
    got = run(cut, lengths)
    seen = [j for j in visible(29, 30, window, sinks) if j < 24]
    check(got[2], *attend(q[2, 0], c.k[2], c.v[2], seen, 0.1, 2), "past the table")
    # a visible position on a page outside the cache counts as masked
    for bad in (c.capacity // block, 0x7fffffff, 0xffffffff):
        pages = c.pages.copy()
        pages[2, 7] = bad                                       # positions 28 and 29
        got = run(pages, lengths)
        check(got[2], *attend(q[2, 0], c.k[2], c.v[2], [j for j in visible(29, 30, window, sinks) if j < 28], 0.1, 2), "bad page")
    assert np.isnan(run(np.full((3, 8), 0xfffffff0, np.uint32), lengths)).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("qH,kv,D,block", [(8, 2, 128, 16), (6, 2, 40, 5), (4, 4, 64, 8)])
def test_ragged_steps(qH, kv, D, block, f16):
    # one token, a prompt's first chunk, a sequence with no token in this step, a chunk behind a context;
    # two padding rows behind the last sequence
    lengths, counts = [200, 37, 50, 333, 1], [1, 37, 0, 61, 1]
    for window, sinks in ((32, 4), (1, 0), (1000, 2)):
        first = [n - m if m else n for n, m in zip(lengths, counts)]
        c = Cache(7, kv, D, block, lengths, first, window, sinks, f16)
        tokens = sum(counts) + 2
        q = np.random.default_rng(8).standard_normal((tokens, qH, D)).astype(np.float32)
        got = T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
            lengths=dev(np.array(lengths, np.uint32)), pages=dev(c.pages), block=block, scale=attn_scale(D),
            query_extents=dev(np.array(counts, np.uint32)), window=window, sinks=sinks)).cpu().numpy()
        assert not got[-2:].any()
        r = 0
        for b, (n, m) in enumerate(zip(lengths, counts)):
            for i in range(m):
                check(got[r], *attend(q[r], c.k[b], c.v[b], visible(n - m + i, n, window, sinks), attn_scale(D), qH // kv),
                      f"sequence {b} token {i} window {window}")
                r += 1


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("qH,kv,D,block", [(8, 2, 128, 16), (6, 2, 40, 5), (4, 4, 64, 8), (3, 1, 128, 16), (2, 2, 96, 7)])
def test_prefill(qH, kv, D, block, paged, f16):
    for tokens, base, window, sinks in ((1, 0, 5, 0), (1, 300, 64, 4), (3, 5, 2, 1), (70, 0, 16, 2), (130, 77, 200, 9),
                                        (257, 500, 128, 4), (200, 1000, 1, 0)):
        n = base + tokens
        c = Cache(tokens, kv, D, block if paged else 1, [n], [base], window, sinks, f16)
        if not paged:                                            # NaN where nobody looks, as in the paged cache
            see = sorted({j for p in range(base, n) for j in visible(p, n, window, sinks)})
            c.pk, c.pv = np.full_like(c.k[0], np.nan), np.full_like(c.v[0], np.nan)
            c.pk[see], c.pv[see] = c.k[0][see], c.v[0][see]
        q = np.random.default_rng(3).standard_normal((tokens, qH, D)).astype(np.float32)
        got = T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
            lengths=dev(np.array([n], np.uint32)), pages=dev(c.pages[0]) if paged else None, block=block if paged else 0,
            scale=attn_scale(D), base=base, window=window, sinks=sinks)).cpu().numpy()
        ref = [attend(q[i], c.k[0], c.v[0], visible(base + i, n, window, sinks), attn_scale(D), qH // kv) for i in range(tokens)]
        check(got, np.stack([r[0] for r in ref]), np.stack([r[1] for r in ref]), f"{tokens} tokens behind {base}, window {window}")


@pytest.mark.parametrize("f16", [False, True])
def test_a_prefill_past_the_cache_length_and_rows_that_see_nothing(f16):
    # the cache holds 40 positions and the queries stand at 30 ..: the window slides off its end
    qH, kv, D, n, base, tokens = 4, 2, 128, 40, 30, 100
    rng = np.random.default_rng(4)
    k, v = (rng.standard_normal((64, kv, D)).astype(np.float16 if f16 else np.float32) for _ in range(2))
    k[n:], v[n:] = np.nan, np.nan
    q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
    for window, sinks in ((8, 0), (8, 3)):
        got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
            lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D), base=base, window=window, sinks=sinks)).cpu().numpy()
        for i in range(tokens):
            seen = visible(base + i, n, window, sinks)
            check(got[i], *attend(q[i], k, v, seen, attn_scale(D), 2), f"row {i}")
            assert len(seen) or np.isnan(got[i]).all()


@pytest.mark.parametrize("f16", [False, True])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(f16):
    qH, kv, D, tokens = 4, 2, 128, 300
    rng = np.random.default_rng(6)
    k, v = (rng.standard_normal((tokens, kv, D)).astype(np.float16 if f16 else np.float32) for _ in range(2))
    v[150, 0, 5], v[151, 1, 7], k[160, 0, 3] = np.inf, np.nan, np.nan
    q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
    window = 20
    got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
        lengths=dev(np.array([tokens], np.uint32)), scale=attn_scale(D), base=0, window=window, sinks=2)).cpu().numpy()
    for i in range(tokens):
        for h in range(qH):
            seen = visible(i, tokens, window, 2)
            kvh = h // 2
            if kvh == 0 and 160 in seen:
                assert np.isnan(got[i, h]).all(), i
            elif (150 if kvh == 0 else 151) in seen:
                d = 5 if kvh == 0 else 7
                assert not np.isfinite(got[i, h, d]) and np.isfinite(np.delete(got[i, h], d)).all(), i
            else:
                o, b = attend(q[i, h:h + 1], k[:, kvh:kvh + 1], v[:, kvh:kvh + 1], seen, attn_scale(D), 1)
                check(got[i, h:h + 1], o, b, f"row {i} head {h}")


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("tokens", [1, 200])
def test_magnitudes_far_from_one(tokens, f16):
    # scores of ordinary size from keys and queries that are not, values of any size
    qH, kv, D, n = 4, 1, 128, 700
    rng = np.random.default_rng(12)
    for qs, ks, vs in ((1e-9, 1e9, 1e12), (1e12, 1e-12, 1e-20), (3e4, 3e-5, 6e4)):
        if f16:
            ks, vs = min(max(ks, 1e-4), 1e4), min(max(vs, 1e-4), 1e4)
            qs = 1 / ks
        k, v = ((rng.standard_normal((n, kv, D)) * x).astype(np.float16 if f16 else np.float32) for x in (ks, vs))
        q = (rng.standard_normal((tokens, qH, D)) * qs).astype(np.float32)
        base = n - tokens
        got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
            lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D), base=base, window=400, sinks=3)).cpu().numpy()
        ref = [attend(q[i], k, v, visible(base + i, n, 400, 3), attn_scale(D), qH) for i in range(tokens)]
        check(got, np.stack([r[0] for r in ref]), np.stack([r[1] for r in ref]), f"{qs} {ks} {vs}")


def test_a_wide_window_gives_what_no_window_gives():
    # every position visible: the unwindowed forms, within the sum of both kernels' tolerances (theirs: 2e-3)
    qH, kv, D, n = 8, 2, 128, 400
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((n, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((qH, D)).astype(np.float32)
    o = T.AttentionOptions(lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D))
    plain = T.attention(dev(q), dev(k), dev(v), o).cpu().numpy()
    o.window = n
    wide = T.attention(dev(q), dev(k), dev(v), o).cpu().numpy()
    assert np.abs(wide - plain).max() <= (2e-3 + 2e-3) * np.abs(plain).max()
    o.window = 0xffffffff
    assert np.array_equal(T.attention(dev(q), dev(k), dev(v), o).cpu().numpy(), wide)


def test_offsets_past_32_bits():
    # a cache of 2^32 + elements; the sequence's pages lie at its end
    kv, D, block = 32, 128, 16
    capacity = ((1 << 32) // (kv * D) // block + 40) * block
    pages = capacity // block
    k, v = (torch.zeros((capacity, kv, D), dtype=torch.float16, device=DEV) for _ in range(2))
    rng = np.random.default_rng(2)
    n, tokens = 500, 200
    lk, lv = (rng.standard_normal((n, kv, D)).astype(np.float16) for _ in range(2))
    row = np.array([pages - 1 - i for i in range((n + block - 1) // block)], np.uint32)
    for j in range(n):
        r = int(row[j // block]) * block + j % block
        k[r], v[r] = dev(lk[j]), dev(lv[j])
    for rows in (1, tokens):
        q = rng.standard_normal((rows, kv, D)).astype(np.float32)
        got = T.attention(dev(q), k, v, T.AttentionOptions(lengths=dev(np.array([n], np.uint32)), pages=dev(row), block=block,
                                                           scale=attn_scale(D), base=n - rows, window=150, sinks=4)).cpu().numpy()
        for i in (0, rows - 1):
            check(got[i], *attend(q[i], lk, lv, visible(n - rows + i, n, 150, 4), attn_scale(D), 1), f"row {i}")


def _job(seed, tokens, f16=False):
    """A prefill and its arguments; a closure that runs it."""
    rng = np.random.default_rng(seed)
    n = tokens + 100
    k, v = (dev(rng.standard_normal((n, 2, 128)).astype(np.float16 if f16 else np.float32)) for _ in range(2))
    q = dev(rng.standard_normal((tokens, 8, 128)).astype(np.float32))
    o = T.AttentionOptions(lengths=dev(np.array([n], np.uint32)), scale=0.09, base=100, window=90, sinks=4)
    return lambda: T.attention(q, k, v, o)


def test_a_call_repeats_its_bits_on_any_stream_and_in_graphs():
    jobs = [_job(1, 300), _job(2, 150), _job(3, 1)]
    want = [j().cpu() for j in jobs]
    for _ in range(3):
        assert all(torch.equal(j().cpu(), w) for j, w in zip(jobs, want))
    graphs, outs = [], []
    for j in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(j())
        graphs.append(g)
    # all three on streams of their own, several times over, beside the same calls made eagerly
    streams = [torch.cuda.Stream() for _ in jobs]
    eager = []
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s, j in zip(graphs, streams, jobs):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(j())
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o.cpu(), w)
    for i, e in enumerate(eager):
        assert torch.equal(e.cpu(), want[i % 3])


def test_views_and_unaligned_tables():
    # a table row and lengths that start anywhere, caches that are slices of one tensor of both
    qH, kv, D, block, n = 4, 2, 64, 8, 50
    rng = np.random.default_rng(3)
    both = dev(rng.standard_normal((64, 2, kv, D)).astype(np.float32))
    k, v = both[:, 0], both[:, 1]                                 # strided: a row of k, a row of v, ...
    table = torch.arange(24, dtype=torch.int32, device=DEV).view(3, 8)[:, 1:].contiguous()[1]   # pages 9 .. 15: out of the cache
    table = torch.arange(21, dtype=torch.int32, device=DEV).view(3, 7).remainder(8)[1]
    lens = torch.tensor([1, n, 3], dtype=torch.int32, device=DEV)[1:2]
    q = rng.standard_normal((qH, D)).astype(np.float32)
    got = T.attention(dev(q), k, v, T.AttentionOptions(lengths=lens, pages=table, block=block, scale=0.2, window=30, sinks=5)).cpu().numpy()
    tab = table.cpu().numpy()
    phys = [int(tab[j // block]) * block + j % block for j in visible(n - 1, n, 30, 5)]
    check(got, *attend(q, k.cpu().numpy(), v.cpu().numpy(), phys, 0.2, 2), "views")


def test_no_wait_ran_out():
    _job(9, 300)()
    assert "tcgen05 tiles" in rt.last_selection()
    rt.attention_error()
    _job(9, 3)()
    assert "tcgen05 tiles" not in rt.last_selection()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("qH,kv,D,block", [(8, 2, 128, 16), (6, 2, 40, 5), (2, 2, 64, 8), (30, 1, 128, 16)])
def test_ragged_steps_of_chunks_and_tokens(qH, kv, D, block, f16):
    # prompts' chunks (on tiles) between single tokens (row by row), in more than one block of the plan; sequences without
    # tokens, with one position, with fewer positions than tokens; padding rows behind the last
    rng = np.random.default_rng(11)
    batch = 300
    counts = np.where(rng.random(batch) < 0.05, rng.integers(64, 200, batch), rng.integers(0, 3, batch))
    counts[[0, 255, 256, 299]] = (130, 64, 70, 129)
    lengths = counts + rng.integers(0, 300, batch) * (rng.random(batch) < 0.8)
    lengths[7], counts[7] = 3, 5                                  # two rows have no position: zeros
    lengths[8], counts[8] = 60, 100
    lengths = np.maximum(lengths, 1)
    for window, sinks in ((90, 5), (1, 0), (5000, 3)):
        first = np.maximum(lengths - np.maximum(counts, 1), 0)
        c = Cache(window, kv, D, block, lengths.tolist(), first.tolist(), window, sinks, f16)
        tokens = int(counts.sum()) + 3
        q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
        got = T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
            lengths=dev(lengths.astype(np.uint32)), pages=dev(c.pages), block=block, scale=attn_scale(D),
            query_extents=dev(counts.astype(np.uint32)), window=window, sinks=sinks)).cpu().numpy()
        assert not got[-3:].any()
        r = 0
        for b, (n, m) in enumerate(zip(lengths.tolist(), counts.tolist())):
            if b not in (0, 1, 7, 8, 255, 256, 299) and m < 64 and b % 9:
                r += m
                continue
            for i in range(m):
                if n - m + i < 0:
                    assert not got[r].any()
                elif i % 7 == 0 or i == m - 1:
                    check(got[r], *attend(q[r], c.k[b], c.v[b], visible(n - m + i, n, window, sinks), attn_scale(D), qH // kv),
                          f"sequence {b} token {i} window {window}")
                r += 1


def test_ragged_chunks_in_graphs_on_two_streams():
    def job(seed):
        rng = np.random.default_rng(seed)
        counts, lengths = [70, 1, 200, 3], [300, 41, 200, 9]
        c = Cache(seed, 2, 128, 16, lengths, [n - m for n, m in zip(lengths, counts)], 100, 4, False)
        q, k, v = dev(rng.standard_normal((sum(counts), 8, 128)).astype(np.float32)), dev(c.pk), dev(c.pv)
        o = T.AttentionOptions(lengths=dev(np.array(lengths, np.uint32)), pages=dev(c.pages), block=16, scale=0.1,
                               query_extents=dev(np.array(counts, np.uint32)), window=100, sinks=4)
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
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), w) for o, w in zip(outs, want))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("tokens,n,tiles", [(31, 4200, False), (127, 2112, False), (128, 2048, True), (128, 2047, False), (255, 255, False), (256, 256, True)])
def test_prefill_on_either_side_of_the_choice_of_kernel(tokens, n, tiles, f16):
    kv, D, window, sinks = 2, 64, 2044, 4                         # 128 rows x 2048 positions x 2 KV heads, or 256 rows
    rng = np.random.default_rng(tokens)
    k, v = (rng.standard_normal((n, kv, D)).astype(np.float16 if f16 else np.float32) for _ in range(2))
    q = rng.standard_normal((tokens, kv, D)).astype(np.float32)
    got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
        lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D), base=n - tokens, window=window, sinks=sinks)).cpu().numpy()
    assert ("tcgen05 tiles" in rt.last_selection()) == tiles
    for i in range(0, tokens, 5):
        check(got[i], *attend(q[i], k, v, visible(n - tokens + i, n, window, sinks), attn_scale(D), 1), f"row {i}")


def test_ragged_steps_of_single_tokens_take_one_launch():
    qH, kv, D, block, batch = 8, 2, 64, 8, 40
    rng = np.random.default_rng(1)
    lengths = rng.integers(1, 100, batch)
    c = Cache(4, kv, D, block, lengths.tolist(), (lengths - 1).tolist(), 50, 2, False)
    for counts in (np.ones(batch, np.int64), np.where(np.arange(batch) == 11, 30, np.arange(batch) % 4 == 0)):
        q = rng.standard_normal((int(counts.sum()), qH, D)).astype(np.float32)
        lens = np.maximum(lengths, counts)
        c = Cache(4, kv, D, block, lens.tolist(), (lens - counts).tolist(), 50, 2, False)
        got = T.attention(dev(q), dev(c.pk), dev(c.pv), T.AttentionOptions(
            lengths=dev(lens.astype(np.uint32)), pages=dev(c.pages), block=block, scale=attn_scale(D),
            query_extents=dev(counts.astype(np.uint32)), window=50, sinks=2)).cpu().numpy()
        r = 0
        for b, (n, m) in enumerate(zip(lens.tolist(), counts.tolist())):
            for i in range(m):
                check(got[r], *attend(q[r], c.k[b], c.v[b], visible(n - m + i, n, 50, 2), attn_scale(D), qH // kv), f"{b} {i}")
                r += 1


def test_ragged_lists_longer_than_the_tiles_there_is_room_for():
    # twelve sequences over one shared cache: 12 x 100000 positions are more than the 8192 tiles of 128 a pass packs
    # (f32, head dimension 128), so that the last chunks go row by row
    qH, D, block, batch, n, m = 8, 128, 16, 12, 100000, 40
    gen = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn((n, 1, D), device=DEV, generator=gen) for _ in range(2))
    q = torch.randn((batch * m, qH, D), device=DEV, generator=gen)
    table = torch.arange(n // block, dtype=torch.int32, device=DEV).expand(batch, -1).contiguous()
    lengths = np.arange(n - batch + 1, n + 1).astype(np.uint32)
    got = T.attention(q, k, v, T.AttentionOptions(
        lengths=dev(lengths), pages=table, block=block, scale=attn_scale(D), query_extents=dev(np.full(batch, m, np.uint32)),
        window=n, sinks=0)).cpu().numpy()
    hq, hk, hv = q.cpu().numpy(), k.cpu().numpy(), v.cpu().numpy()
    for b in (0, 5, 9, 10, 11):
        for i in (0, m - 1):
            r = b * m + i
            check(got[r], *attend(hq[r], hk, hv, visible(int(lengths[b]) - m + i, int(lengths[b]), n, 0), attn_scale(D), qH), f"{b} {i}")
    rt.attention_error()


@pytest.mark.parametrize("f16", [False, True])
def test_more_sequences_than_a_grid_has_rows(f16):
    # every query sees one position: its value is the answer
    batch, kv, D = 70000, 2, 8
    gen = torch.Generator(device=DEV).manual_seed(5)
    k, v = (torch.randn((batch, kv, D), device=DEV, generator=gen).to(torch.float16 if f16 else torch.float32) for _ in range(2))
    q = torch.randn((batch, 1, kv, D), device=DEV, generator=gen)
    pages = torch.randperm(batch, device=DEV, generator=gen).to(torch.int32)[:, None]
    got = T.attention(q, k, v, T.AttentionOptions(lengths=torch.ones(batch, dtype=torch.int32, device=DEV), pages=pages, block=1,
                                                  scale=0.3, window=3))
    want = v[pages[:, 0].long()].float()
    assert ((got - want).abs() <= 2.0**-22 * want.abs()).all()      # a weight of 1: a quotient and two products of one value


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("tokens,qH,kv", [(1, 4, 2), (1, 12, 1), (200, 4, 2)])
def test_scales_of_any_sign_and_size(tokens, qH, kv, f16):
    D, n = 64, 300
    rng = np.random.default_rng(9)
    k, v = (rng.standard_normal((n, kv, D)).astype(np.float16 if f16 else np.float32) for _ in range(2))
    q = rng.standard_normal((tokens, qH, D)).astype(np.float32)
    q[0, 0] = 0                                                   # and a query of zeros: every weight the same
    for scale in (0.0, -0.3, 1e-30, 1e-40):
        got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
            lengths=dev(np.array([n], np.uint32)), scale=scale, base=n - tokens, window=100, sinks=2)).cpu().numpy()
        for i in range(0, tokens, 9):
            check(got[i], *attend(q[i], k, v, visible(n - tokens + i, n, 100, 2), scale, qH // kv), f"scale {scale} row {i}")
