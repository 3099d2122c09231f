"""Copies of cache pages, on a B200: bit for bit, nothing else touched."""
import numpy as np
import pytest
import torch

from accel_b200 import tensor as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.uint8])
@pytest.mark.parametrize("caches,capacity,width,block,pairs", [
    (1, 8, (1, 8), 1, 1), (2, 40, (2, 3), 4, 5), (4, 640, (8, 128), 16, 20), (3, 333, (5, 7), 13, 12), (130, 64, (2, 8), 4, 7),
    (2, 9000, (1, 8), 8, 500), (2, 9, (4, 128), 2, 2), (1, 64, (32, 128), 32, 1), (5, 100, (3,), 7, 3)])
def test_copies(caches, capacity, width, block, pairs, dtype):
    g = torch.Generator(device=DEV).manual_seed(capacity)
    held = [torch.randint(0, 256, (capacity * int(np.prod(width)) * dtype.itemsize,), generator=g, device=DEV, dtype=torch.uint8)
            .view(dtype).view(capacity, *width) for _ in range(caches)]
    want = [c.clone() for c in held]
    order = np.random.default_rng(1).permutation(capacity // block)
    src, dst = order[:pairs].tolist(), order[pairs:2 * pairs].tolist()
    more = order[2 * pairs:2 * pairs + 2].tolist()                  # one page to several places
    src, dst = src + src[:1] * len(more), dst + more
    for w in want:
        for a, b in zip(src, dst):
            w[b * block:(b + 1) * block] = w[a * block:(a + 1) * block]
    T.copy_pages(held, src, dst, block)
    for c, w in zip(held, want):
        assert torch.equal(c.view(torch.uint8), w.view(torch.uint8))    # NaN patterns and the rest behind the last page too
    T.copy_pages(held, [], [], block)


def test_caches_that_start_anywhere():
    flat = torch.arange(4000, device=DEV, dtype=torch.float16)
    for off in (1, 2, 4, 8):
        c = flat.clone()[off:off + 320].view(40, 8)
        w = c.clone()
        w[8:12] = w[20:24]
        T.copy_pages([c], [5], [2], 4)
        assert torch.equal(c, w)


def test_streams_and_graphs():
    c = [torch.randn(64, 4, 32, device=DEV) for _ in range(3)]
    w = [x.clone() for x in c]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        T.copy_pages(c, [0], [1], 16)
        T.copy_pages(c, [1], [2], 16)                       # in order on its stream
    side.synchronize()
    for x, y in zip(c, w):
        y[16:32] = y[:16]
        y[32:48] = y[:16]
        assert torch.equal(x, y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        T.copy_pages(c, [3], [0], 16)
    for x, y in zip(c, w):
        assert torch.equal(x, y)
        x[48:] = 7
        y[48:] = 7
        y[:16] = 7
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(c, w))


def test_offsets_past_32_bits():
    c = torch.zeros(1 << 17, 32, 1024, dtype=torch.uint8, device=DEV)      # 4 GiB
    c[16:32], c[-16:] = 3, 5
    T.copy_pages([c], [1, (1 << 13) - 1], [(1 << 13) - 2, 0], 16)
    assert bool((c[-32:-16] == 3).all()) and bool((c[:16] == 5).all()) and not bool(c[32:48].any())
