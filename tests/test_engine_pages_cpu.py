"""The decode engine's page bookkeeping on the CPU, the oracle standing in for the kernels: what moves pages also moves the
slots that the next step writes to."""
import numpy as np
import pytest
import torch

import oracle_ops
from accel_b200 import decode as dec


def cfg(**kw):
    return dec.ModelConfig(layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=640, block=4, **kw)


def engine(c, batch=3, **kw):
    model = dec.DecodeModel(c, dec.Shard.plan(c, 1, 0), "cpu", seed=5, quantize=oracle_ops.quantize, std=0.08)
    e = dec.DecodeEngine(model, batch, max_context=32, ops=oracle_ops, **kw)
    e.prepare()

    def copy(src, dst):
        for cache in (*e.k_cache, *e.v_cache):
            pages = cache.view(-1, c.block, *cache.shape[1:])
            pages[dst] = pages[src].clone()
    e._copy_pages = copy
    return e


def scattered(e, held):
    """Rows of 16 positions on the pool's last pages: the first ones are taken, and then given back, by somebody else."""
    other = e.pool.grow(None, held * 4)
    for s in range(e.batch):
        e.reserve(s, 16)
    e.upload_pages()
    e.pool.free(other)


@pytest.mark.parametrize("steps", [1, 4, 6])
def test_compaction_between_steps_that_feed_themselves(steps):
    # (after 4 steps the next token is the first of a page)
    a, b = engine(cfg()), engine(cfg())
    for e in (a, b):
        scattered(e, 7)
        e.set_inputs(np.array([3, 50, 400]))
        for _ in range(steps):
            e.run_step()
            e.advance_on_device()
    assert a.compact() > 0
    for t in range(5):
        for e in (a, b):
            e.run_step()
        assert torch.equal(a.full_logits(), b.full_logits()), t
        for e in (a, b):
            e.advance_on_device()
        if t == 2:
            assert a.compact() == 0
    held = {p for row in a.page_rows for p in row}
    assert held == set(range(len(held)))


def test_compaction_leaves_slots_of_pages_that_stay():
    e = engine(cfg())
    for s in range(e.batch):
        e.reserve(s, 16)
    e.upload_pages()
    e.pool.free(e.page_rows[1])
    e.page_rows[1] = []
    e.upload_pages()
    e.slots[:] = torch.tensor([e.page_rows[0][0] * 4 + 3, -1, e.page_rows[2][3] * 4 + 2], dtype=torch.int32)
    before = e.page_rows[2][3]
    assert e.compact() > 0 and e.page_rows[2][3] != before
    assert e.slots.tolist() == [e.page_rows[0][0] * 4 + 3, -1, e.page_rows[2][3] * 4 + 2]
