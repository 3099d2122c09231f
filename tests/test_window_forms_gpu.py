"""Forms and paths of the windowed attention that no other test launches, on a B200: one token over a contiguous cache, lists too
long for one pass over the KV heads; and which kernels a ragged step takes."""
import numpy as np
import pytest
import torch

from accel_b200 import runtime as rt
from accel_b200 import tensor as T
from test_window_attention_gpu import Cache, dev
from util import attn_scale
from window_ref import attend, check, visible

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("qH,kv,D", [(4, 4, 128), (4, 2, 64), (6, 2, 40), (8, 2, 128), (15, 3, 96), (8, 1, 128), (20, 1, 72), (2, 2, 8)])
def test_one_token_over_a_contiguous_cache(qH, kv, D, f16):
    for n, window, sinks in ((1, 1, 0), (1, 50, 4), (2, 1, 1), (65, 64, 0), (300, 17, 3), (300, 299, 40), (1000, 5000, 2), (5000, 4000, 9)):
        rng = np.random.default_rng(n + D)
        k, v = (np.full((n + 3, kv, D), np.nan, np.float16 if f16 else np.float32) for _ in range(2))
        seen = visible(n - 1, n, window, sinks)
        k[seen], v[seen] = (rng.standard_normal((len(seen), kv, D)).astype(k.dtype) for _ in range(2))
        q = rng.standard_normal((qH, D)).astype(np.float32)
        got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
            lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D), window=window, sinks=sinks))
        assert rt.last_selection().startswith("AttentionWindow" + ("F16" if f16 else "") + ":")
        check(got.cpu().numpy(), *attend(q, k, v, seen, attn_scale(D), qH // kv), f"length {n}, window {window}")
    got = T.attention(dev(q), dev(k), dev(v), T.AttentionOptions(
        lengths=dev(np.array([0], np.uint32)), scale=attn_scale(D), window=window, sinks=sinks))
    assert torch.isnan(got).all()                                  # nothing to see: 0 / 0


@pytest.mark.parametrize("f16,kv", [(False, 4), (True, 8)])
@pytest.mark.parametrize("ragged", [False, True])
def test_lists_that_take_several_passes_over_the_kv_heads(f16, kv, ragged):
    # 300000 positions are 2344 tiles of 128 KB (f32) or 64 KB: a pass holds three heads of them, or six
    D, n, tokens, group = 128, 300000, 70, 1
    gen = torch.Generator(device=DEV).manual_seed(4)
    k, v = (torch.randn((n, kv, D), device=DEV, generator=gen).to(torch.float16 if f16 else torch.float32) for _ in range(2))
    q = torch.randn((tokens, kv * group, D), device=DEV, generator=gen)
    o = T.AttentionOptions(lengths=dev(np.array([n], np.uint32)), scale=attn_scale(D), window=n - 1000, sinks=5)
    if ragged:
        o.query_extents, o.block = dev(np.array([tokens], np.uint32)), 16
        o.pages = torch.arange(n // 16, dtype=torch.int32, device=DEV).view(1, -1)
    else:
        o.base = n - tokens
    got = T.attention(q, k, v, o).cpu().numpy()
    assert "2 pass(es)" in rt.last_selection()
    rt.attention_error()
    hq, hk, hv = q.cpu().numpy(), k.cpu().numpy(), v.cpu().numpy()
    for i in (0, 33, tokens - 1):
        check(got[i], *attend(hq[i], hk, hv, visible(n - tokens + i, n, n - 1000, 5), attn_scale(D), group), f"row {i}")


@pytest.mark.parametrize("f16,kernel", [(False, "a row a group of lanes"), (True, "up to 8 heads a CTA on the tensor cores")])
def test_ragged_steps_of_single_tokens_are_one_kernel_behind_their_offsets(f16, kernel):
    qH, kv, D, block, window, sinks = 8, 2, 64, 8, 50, 2

    def launches(counts, lengths):
        c = Cache(4, kv, D, block, lengths, [n - m for n, m in zip(lengths, counts)], window, sinks, f16)
        q = dev(np.random.default_rng(1).standard_normal((sum(counts), qH, D)).astype(np.float32))
        o = T.AttentionOptions(lengths=dev(np.array(lengths, np.uint32)), pages=dev(c.pages), block=block, scale=attn_scale(D),
                               query_extents=dev(np.array(counts, np.uint32)), window=window, sinks=sinks)
        T.attention(q, dev(c.pk), dev(c.pv), o)
        before = rt.launch_count()
        T.attention(q, dev(c.pk), dev(c.pv), o)
        return rt.launch_count() - before, rt.last_selection()

    n, how = launches([1] * 40, list(range(20, 60)))
    assert n == 2 and kernel in how                                # the offsets' prefix sums, the rows
    n, how = launches([1, 130, 1], [20, 200, 40])
    assert n == 5 and "tcgen05 tiles" in how                       # and the plan, the packing, the tiles
