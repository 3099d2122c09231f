"""Pages trimmed and moved between captured steps that feed themselves, on a B200."""
import numpy as np
import pytest
import torch

from test_window_engine_gpu import BLOCK, config, model

from accel_b200 import decode as dec

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_trim_and_compact_between_captured_steps_that_feed_themselves(dtype):
    m = model(config(dtype))
    a, b = (dec.DecodeEngine(m, 3, max_context=112) for _ in range(2))
    for e in (a, b):
        other = e.pool.grow(None, 20 * BLOCK)
        for s in range(3):
            e.reserve(s, 80)
        e.upload_pages()
        e.pool.free(other)
        e.set_inputs(np.array([3, 50, 400]))
        e.capture(warmup=1)
        e.set_inputs(np.array([3, 50, 400]))
    moved = 0
    for t in range(60):
        for e in (a, b):
            e.run_step()
        assert torch.equal(a.full_logits(), b.full_logits()), t
        for e in (a, b):
            e.advance_on_device()
        if t % 7 == 3:
            a.trim()
            moved += a.compact()
    assert moved > 20


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_pool_of_a_few_windows_holds_a_conversation_many_times_its_size(dtype):
    m = model(config(dtype))
    rng = np.random.default_rng(3)
    a = dec.DecodeEngine(m, 3, max_context=400, pool_pages=3 * 14)         # windows of 20, pieces of 24 positions, the sinks
    b = dec.DecodeEngine(m, 3, max_context=400)
    assert a.k_cache[0].shape[0] == 3 * 14 * BLOCK and b.k_cache[0].shape[0] == 3 * 400
    prompts = rng.integers(0, 1024, (3, 120))
    for at in range(0, 120, 24):
        for e in (a, b):
            e.prepare()
            e.prefill(prompts[:, at:at + 24], chunk=8)
        a.trim()
    ta = tb = prompts[:, -1]
    for t in range(200):
        for e in (a, b):
            for s in range(3):
                e.reserve(s, int(e.lengths_host[s]) + 1)
            e.upload_pages()
        ta, tb = a.step(ta), b.step(tb)
        assert torch.equal(a.full_logits(), b.full_logits()), t
        a.trim()
        if t == 100:
            a.fork(0, 2), b.fork(0, 2)
            ta[2] = tb[2] = 5
            a.compact()
    assert np.array_equal(ta, tb)
    with pytest.raises(Exception, match="does not evict"):
        a.prefill(prompts)
