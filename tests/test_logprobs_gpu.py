"""Log probabilities, entropy and alternatives against 64 bits, on a B200."""
import numpy as np
import pytest
import torch

from accel_b200 import tensor as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference(x, targets, top):
    """In 64 bits: (logprobs, entropy, ids, logprobs of the ids, and the means of |x - m| and its square under the
    distribution)."""
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        z = e.sum(1, keepdims=True)
        lp = x - m - np.log(z)
        p = e / z
        lost = ~np.isfinite(z[:, 0]) | (z[:, 0] == 0) | ~np.isfinite(m[:, 0])
        mean = np.where(e > 0, p * (x - m), 0.0).sum(1)
        h = np.log(z[:, 0]) - mean
        square = np.where(e > 0, p * np.where(e > 0, x - m, 0.0) ** 2, 0.0).sum(1)
    lp[lost], h[lost] = np.nan, np.nan
    mean, square = np.where(lost, 0.0, mean), np.where(lost, 0.0, square)
    key = np.where(np.isnan(x), np.inf, x)
    first = np.isnan(x)
    ids = np.stack([np.lexsort((np.arange(x.shape[1]), -key[r], ~first[r]))[:top] for r in range(x.shape[0])])
    t = targets.astype(np.int64)
    t2 = t.reshape(x.shape[0], -1)
    got = np.take_along_axis(lp, np.minimum(t2, x.shape[1] - 1), 1)
    got = np.where((t2 < 0) | (t2 >= x.shape[1]), np.nan, got).reshape(t.shape)
    return got, h, ids, np.take_along_axis(lp, ids, 1), np.abs(mean), square


def run(x, targets, top):
    u = None if targets is None else torch.from_numpy(targets.astype(np.uint32).view(np.int32)).to(DEV)
    return T.token_logprobs(torch.from_numpy(x).to(DEV), u, top)


def check(x, targets, top):
    """With ulp = 2^-24 of one: a log probability is (x - m) - log s.  x - m is rounded once; e^d is off by |d| + 2 ulp
    of itself; s by those (on average over the distribution) and by its f32 sum, in which no term passes through
    more than 1024 additions; log s by 2 ulp of itself.  The entropy is log s - sum d e^d / s: the same errors, each
    times its |d|.  What multiplies the parts is doubled for the joining of partial maxima."""
    lp, h, ids, top_lp, mean, square = reference(x, targets, top)
    r = run(x, targets, top)
    ulp = 2.0**-24

    def near(got, want, tol):
        got = got.cpu().numpy().astype(np.float64)
        assert got.shape == want.shape
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fin = np.isfinite(want)
        assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
        d = np.abs(got - np.where(fin, want, 0))[fin]
        assert (d <= tol[fin]).all(), float((d / tol[fin]).max())

    s_off = ulp * (1024 + 2 * mean + 4)
    per_row = lambda a: s_off if a.ndim == 1 else s_off[:, None]
    near(r.logprobs, lp, 4 * ulp * np.abs(lp) + per_row(lp))
    near(r.top_logprobs, top_lp, 4 * ulp * np.abs(top_lp) + per_row(top_lp))
    near(r.entropy, h, 4 * ulp * np.abs(h) + s_off * (1 + mean) + 2 * ulp * (square + 4 * mean))
    assert np.array_equal(r.top_ids.cpu().numpy().view(np.uint32), ids)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 33), (1, 257), (7, 1000), (16, 32000), (3, 32001), (1, 131072),
                                        (2, 50003), (300, 515), (149, 4099)])
def test_matches_64_bits(rows, vocab, f16):
    rng = np.random.default_rng(rows * 7 + vocab)
    x = (rng.standard_normal((rows, vocab)) * 4).astype(np.float16 if f16 else np.float32)
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}):
        check(x, rng.integers(0, vocab, rows), top)
    check(x, rng.integers(0, vocab, (rows, 3)), min(2, vocab))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("vocab", [5, 300, 40000])
def test_ties_go_to_the_lowest_index(vocab, f16):
    dt = np.float16 if f16 else np.float32
    top = min(32, vocab)
    rng = np.random.default_rng(2)
    rows = [np.zeros(vocab), np.where(np.arange(vocab) % 2, -0.0, 0.0), rng.integers(0, 3, vocab), rng.integers(0, max(2, vocab // 40), vocab),
            np.arange(vocab) // 2, -np.arange(vocab) // 2, np.full(vocab, -1e4), np.arange(vocab)[::-1] % 7]
    check(np.stack(rows).astype(dt), rng.integers(0, vocab, len(rows)), top)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("vocab", [40, 5000, 70000])
def test_masks_infinities_and_nan(vocab, f16):
    dt = np.float16 if f16 else np.float32
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((12, vocab)) * 3).astype(dt)
    x[0, 3:] = -np.inf                                     # fewer tokens than alternatives
    x[1] = -np.inf                                         # nothing
    x[2, ::3] = -np.inf
    x[3, vocab // 2] = np.nan
    x[4, 7] = np.inf
    x[5, 7], x[5, vocab - 1], x[5, 2] = np.nan, np.nan, -np.inf
    x[6] = np.finfo(dt).min                                # a mask of the type's lowest value, everywhere
    x[7, 1:] = np.finfo(dt).min
    x[8, :-1] = -np.inf                                    # all the mass on the last token
    x[9] = np.finfo(dt).max
    x[10] = -np.inf
    x[10, 9] = np.inf
    t = rng.integers(0, vocab, 12)
    t[2] = 3
    check(x, t, 32)
    check(x, np.stack([t, np.arange(12)], 1), 5)


def test_sums_of_many_small_terms():
    # one token of a probability near one, and a long tail that holds the rest
    x = np.full((3, 131072), -8.0, np.float32)
    x[:, 100] = 8.0
    x[1, 100] = -8.0
    x[2] = np.linspace(-80, 0, 131072)
    check(x, np.array([100, 5, 131071]), 20)


def test_targets_outside_the_vocabulary_and_none():
    x = np.random.default_rng(1).standard_normal((4, 50)).astype(np.float32)
    r = run(x, np.array([0, 50, 0xffffffff, 49], np.uint64), 2)
    assert np.isnan(r.logprobs.cpu().numpy()).tolist() == [False, True, True, False]
    r = run(x, None, 3)
    assert r.logprobs is None and r.top_ids.shape == (4, 3) and torch.isfinite(r.entropy).all()
    r = run(x, np.zeros((4, 0)), 0)
    assert r.logprobs.shape == (4, 0) and r.top_ids.shape == (4, 0)
    r = run(np.zeros((0, 50), np.float32), np.zeros(0), 3)
    assert r.logprobs.shape == (0,) and r.entropy.shape == (0,)


def test_views_streams_and_graphs():
    g = torch.Generator(device=DEV).manual_seed(4)
    big = torch.randn(9, 1003, generator=g, device=DEV)
    view = big[2:7, 1:]                                    # rows of another stride, from an odd address
    t = torch.arange(7, dtype=torch.int32, device=DEV)[2:]
    want = T.token_logprobs(view.contiguous().clone(), t.clone(), 4)
    got = T.token_logprobs(view, t, 4)
    same = lambda a, b: all(torch.equal(getattr(a, f), getattr(b, f)) for f in ("logprobs", "entropy", "top_ids", "top_logprobs"))
    assert same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = T.token_logprobs(view, t, 4)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            graph.replay()
            again = T.token_logprobs(view, t, 4)
    torch.cuda.synchronize()
    assert same(held, want) and same(again, want)


def test_more_logits_than_32_bits_count():
    # 33000 rows of 131072 are more than 2^32 logits: the last rows are read where they are
    rows, vocab = 33000, 131072
    x = torch.zeros(rows, vocab, dtype=torch.float16, device=DEV)
    x[-1, 77], x[32768, 5] = 3.0, 2.0
    r = T.token_logprobs(x, torch.full((rows,), 77, dtype=torch.int32, device=DEV), 1)
    z = vocab - 1 + np.exp(3.0)
    assert abs(float(r.logprobs[-1]) - (3 - np.log(z))) < 1e-5 and int(r.top_ids[-1]) == 77
    assert int(r.top_ids[32768]) == 5 and int(r.top_ids[0]) == 0
    assert abs(float(r.logprobs[0]) + np.log(vocab)) < 1e-5
