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
