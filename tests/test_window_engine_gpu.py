"""The decode engine over an attention window: prefill, steps, pages freed behind the window, forks, compaction and
scored tokens together, as a serving loop uses them.  On a B200."""
import numpy as np
import pytest
import torch

from accel_b200 import decode as dec
from accel_b200 import runtime as rt
from accel_b200.blockpool import BlockPool
from util import assert_close
from window_ref import visible

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WINDOW, SINKS, BLOCK = 20, 3, 4


def config(dtype=torch.float32, window=WINDOW):
    return dec.ModelConfig(layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=1024, block=BLOCK,
                           cache_dtype=dtype, window=window, sinks=SINKS if window else 0)


def model(cfg):
    return dec.DecodeModel(cfg, dec.Shard.plan(cfg, 1, 0), DEV, seed=3, std=0.08)


class PlainAttention:
    """The library's dispatch with the windowed attention kernels replaced by their definition in 64 bits."""
    calls = 0

    @staticmethod
    def launch_count():
        return 0

    @classmethod
    def launch(cls, name, bindings, uniform=None):
        if not name.startswith("AttentionWindow"):
            return rt.launch(name, bindings, uniform)
        cls.calls += 1
        q, k, v, pages, lengths, out = bindings
        d = np.frombuffer(uniform, np.uint32)
        batch, heads, kv, D, block, window, sinks, q_seq, base = (int(d[i]) for i in (0, 1, 2, 3, 4, 7, 8, 10, 11))
        scale = float(np.frombuffer(uniform, np.float32)[6])
        prefill = "Prefill" in name
        table = pages.view(1 if prefill else batch, -1).long()
        rows = [(0, base + i, int(lengths[0])) for i in range(q_seq)] if prefill else [(b, int(n) - 1, int(n)) for b, n in enumerate(lengths)]
        qs, o = q.view(len(rows), heads, D).double(), out.view(len(rows), heads, D)
        for r, (b, p, n) in enumerate(rows):
            j = torch.tensor(visible(p, n, window, sinks), device=DEV)
            at = table[b][j // block] * block + j % block
            kk, vv = (x[at].double().repeat_interleave(heads // kv, 1) for x in (k, v))
            w = torch.softmax(torch.einsum("hd,nhd->hn", qs[r], kk) * scale, 1)
            o[r] = torch.einsum("hn,nhd->hd", w, vv).float()


def engine(m, batch, context=96):
    e = dec.DecodeEngine(m, batch, max_context=context)
    e.prepare()
    return e


def steps(e, tok, n, trim=False):
    logits = []
    for _ in range(n):
        for s in range(e.batch):
            e.reserve(s, int(e.lengths_host[s]) + 1)
        e.upload_pages()
        tok = e.step(tok)
        logits.append(e.full_logits().clone())
        if trim:
            e.trim()
    return tok, torch.stack(logits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_prefill_and_steps_against_plain_attention(dtype):
    m = model(config(dtype))
    rng = np.random.default_rng(1)
    prompts = rng.integers(0, 1024, (3, 41))
    a, b = engine(m, 3), engine(m, 3)
    b.ops = PlainAttention
    PlainAttention.calls = 0
    for e in (a, b):
        e.prefill(prompts, chunk=16)
    tok = prompts[:, -1]
    for t in range(30):
        for e in (a, b):
            for s in range(3):
                e.reserve(s, 41 + t + 1)
            e.upload_pages()
            e.set_inputs(tok)
            e.run_step()
            e.lengths_host += 1
        assert_close(a.full_logits().cpu().numpy(), b.full_logits().cpu().numpy(), 5e-3, f"logits at step {t}")
        tok = rng.integers(0, 1024, 3)
        if t % 4 == 0:
            a.trim(), b.trim()
    assert PlainAttention.calls == 3 * 3 * 2 + 30 * 2
    assert any(x == BlockPool.NONE for x in a.page_rows[0])


def test_freeing_forking_and_compaction_change_no_bit():
    m = model(config())
    rng = np.random.default_rng(2)
    prompts = rng.integers(0, 1024, (4, 33))
    a, b = engine(m, 4), engine(m, 4)
    for e in (a, b):
        e.prefill(prompts, chunk=16)
    free0 = a.pool.available()
    tok = prompts[:, -1]
    ta, la = steps(a, tok, 12, trim=True)
    tb, lb = steps(b, tok, 12)
    assert np.array_equal(ta, tb) and torch.equal(la, lb)                # freed pages are never read
    assert a.pool.available() > b.pool.available() and free0 >= 0
    # sequence 2 becomes a copy of 0; both go on with the same token: the same bits, and 0's are untouched
    a.fork(0, 2)
    assert a.lengths_host[2] == a.lengths_host[0] and a.lengths_host[0] % BLOCK
    last = int(a.lengths_host[0]) // BLOCK
    assert a.page_rows[2][last] != a.page_rows[0][last]                  # the partly filled page is its own
    assert all(x == y for x, y in zip(a.page_rows[2][:last], a.page_rows[0][:last]))
    tok = np.array([7, 8, 7, 9])
    ta, la = steps(a, tok, 3, trim=True)
    tb, lb = steps(b, np.array([7, 8, 1, 9]), 3)
    assert torch.equal(la[:, 0], la[:, 2]) and torch.equal(la[:, 0], lb[:, 0]) and torch.equal(la[:, 1], lb[:, 1])
    # then they part: what one writes the other does not see
    ta, la = steps(a, np.array([5, 6, 900, 6]), 4)
    tb, lb = steps(b, np.array([5, 6, 1, 6]), 4)
    assert torch.equal(la[:, 0], lb[:, 0]) and torch.equal(la[:, 3], lb[:, 3]) and not torch.equal(la[:, 0], la[:, 2])
    # the pages in use move to the front of the pool
    a.trim()
    held = {x for r in a.page_rows for x in r if x != BlockPool.NONE}
    moved = a.compact()
    assert moved == len([x for x in held if x >= len(held)]) and moved > 0
    assert {x for r in a.page_rows for x in r if x != BlockPool.NONE} == set(range(len(held)))
    for c in (*a.k_cache, *a.v_cache):
        c[len(held) * BLOCK:] = float("nan")                             # nothing lives there any more
    ta, la = steps(a, np.array([5, 6, 900, 6]), 2)
    tb, lb = steps(b, np.array([5, 6, 1, 6]), 2)
    assert torch.equal(la[:, 0], lb[:, 0]) and torch.equal(la[:, 1], lb[:, 1]) and torch.isfinite(la).all()
    for s in range(4):
        a.pool.free(a.page_rows[s])
    assert a.pool.available() == a.batch * a.max_pages


def test_fork_refuses_and_survives_a_full_pool():
    e = engine(model(config()), 2, context=16)
    for bad in ((0, 0), (0, 2), (-1, 0)):
        with pytest.raises(ValueError, match="fork of sequence"):
            e.fork(*bad)
    with pytest.raises(ValueError, match="no attention window"):
        engine(model(config(window=0)), 1).trim()
    e.reserve(0, 6)
    e.lengths_host[0] = 6
    extra = e.pool.grow(None, e.pool.available() * BLOCK)                 # somebody holds the rest
    with pytest.raises(Exception, match="does not evict"):
        e.fork(0, 1)
    assert e.page_rows[1] == [] and e.lengths_host[1] == 0 and all(e.pool.refs(p) == 1 for p in e.page_rows[0])
    e.pool.free(extra)
    e.fork(0, 1)
    assert e.lengths_host[1] == 6 and len(e.page_rows[1]) == len(e.page_rows[0])


def test_captured_steps_and_the_plan_seam_run_the_windowed_kernels():
    m = model(config())
    a, b, c = (engine(m, 2) for _ in range(3))
    for e in (a, b, c):
        e.fill_context(30, seed=2)
        for s in range(2):
            e.reserve(s, 60)
        e.upload_pages()
    tok = np.array([3, 4])
    b.set_inputs(tok)
    b.capture(warmup=1)
    seam = dec.SeamStep(c)
    t1 = t2 = t3 = tok
    for _ in range(10):
        t1, t2, t3 = a.step(t1), b.step(t2), seam.step(t3)
        assert np.array_equal(t1, t2) and np.array_equal(t1, t3)
        assert torch.equal(a.full_logits(), b.full_logits()) and torch.equal(a.full_logits(), c.full_logits())
    seam.close()


def test_scored_tokens_are_those_of_the_logits():
    e = engine(model(config()), 3)
    e.fill_context(25, seed=4)
    nxt, logits = steps(e, np.array([1, 2, 3]), 1)
    r = e.score(e.next_tokens, top=4)
    x = logits[0].double()
    lp = torch.log_softmax(x, 1)
    want = lp.gather(1, e.next_tokens.long()[:, None])[:, 0]
    # (the sum over 1024 tokens and the difference x - m: 1024 + |lp| ulp at most)
    assert (r.logprobs.double() - want).abs().max() <= 2.0**-24 * (1024 + 4 * want.abs().max())
    assert torch.equal(r.top_ids[:, 0], e.next_tokens) and torch.equal(r.top_logprobs[:, 0], r.logprobs)
    assert torch.equal(r.top_ids, torch.sort(logits[0], dim=1, descending=True, stable=True).indices[:, :4].int())
    assert ((r.entropy.double() + (lp.exp() * lp).sum(1)).abs() <= 2.0**-24 * 1024 * 20).all()


def test_a_fork_without_room_leaves_both_sequences_as_they_were():
    e = engine(model(config()), 3, context=16)
    for s, n in ((0, 10), (1, 9)):
        e.reserve(s, n)
        e.lengths_host[s] = n
    e.fork(0, 2)
    before = [list(r) for r in e.page_rows]
    extra = e.pool.grow(None, e.pool.available() * BLOCK)
    e.reserve(1, 9)
    e.fork(2, 1)                                     # 1 gives back three pages of its own, and one is needed
    assert e.lengths_host[1] == 10 and e.page_rows[1][:2] == before[2][:2]
    taken = e.pool.grow(None, e.pool.available() * BLOCK)
    before = [list(r) for r in e.page_rows]
    e.pool.free([taken[0]])
    e.fork(0, 1)                                     # its own last page and the free one: room for one
    refs = [e.pool.refs(x) for r in e.page_rows for x in r]
    before = [list(r) for r in e.page_rows]
    more = e.pool.grow(None, e.pool.available() * BLOCK)
    e.lengths_host[0] = 1                            # the source now shares one page and wants three new ones
    with pytest.raises(Exception, match="does not evict"):
        e.fork(0, 1)
    assert [list(r) for r in e.page_rows] == before and e.lengths_host[1] == 10
    assert [e.pool.refs(x) for r in e.page_rows for x in r] == refs and len(extra) and more is not None


def test_a_context_is_not_written_over_shared_or_missing_pages():
    e = engine(model(config()), 2, context=64)
    for s in range(2):
        e.reserve(s, 50)
    e.lengths_host[:] = 50
    e.trim()
    with pytest.raises(ValueError, match="given pages back or shares"):
        e.fill_context(60)
    f = engine(model(config()), 2, context=64)
    f.reserve(0, 50)
    f.lengths_host[0] = 50
    f.fork(0, 1)
    with pytest.raises(ValueError, match="given pages back or shares"):
        f.fill_context(60)


@pytest.mark.parametrize("graphs", [False, True])
def test_chunks_tokens_and_scores_through_the_plan_seam(graphs):
    # a prefill on tiles, a ragged step of chunks and tokens, and log probabilities of f16 logits as one plan, two submissions of
    # it in flight: the bits of the calls
    from accel_b200 import driver as D
    from accel_b200 import tensor as T
    qH, kv, Dh, block, window, sinks = 8, 2, 64, 16, 60, 3
    rng = np.random.default_rng(8)
    counts, lengths = np.array([70, 1, 90, 2], np.uint32), np.array([200, 33, 90, 400], np.uint32)
    pages = rng.permutation(4 * 25).astype(np.uint32).reshape(4, 25)
    k, v = (rng.standard_normal((100 * block, kv, Dh)).astype(np.float16) for _ in range(2))
    q1, q2 = rng.standard_normal((300, qH, Dh)).astype(np.float32), rng.standard_normal((163, qH, Dh)).astype(np.float32)
    n1 = np.array([400], np.uint32)
    x, t = rng.standard_normal((5, 1000)).astype(np.float16), rng.integers(0, 1000, 5).astype(np.uint32)
    gpu = lambda a: torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).to(DEV)
    kd, vd = gpu(k), gpu(v)
    o = dict(scale=0.2, window=window, sinks=sinks)
    want1 = T.attention(gpu(q1), kd, vd, T.AttentionOptions(lengths=gpu(n1), pages=gpu(pages[3]), block=block, base=100, **o)).cpu().numpy()
    want2 = T.attention(gpu(q2), kd, vd, T.AttentionOptions(lengths=gpu(lengths), pages=gpu(pages), block=block,
                                                            query_extents=gpu(counts), **o)).cpu().numpy()
    r = T.token_logprobs(gpu(x), gpu(t), top=3)
    dev = D.Device(0, use_graphs=graphs)
    op = lambda b, n=None: D.Operand(block=b, offset=0, size=b.size if n is None else n)
    up = lambda a: dev.upload(np.ascontiguousarray(a))
    blocks = [up(a) for a in (k, v, q1, n1, pages[3], q2, lengths, pages, np.r_[0, np.cumsum(counts)].astype(np.uint32), x, t)]
    bk, bv, bq1, bn1, bp3, bq2, bl, bp, boff, bx, bt = blocks
    outs = [dev.alloc(n) for n in (q1.nbytes, q2.nbytes, 20, 20, 60, 60)]
    dims = lambda batch, mp, q_seq, base: rt.window_dims(batch, qH, kv, Dh, block, mp, 0.2, window, sinks, 100 * block, q_seq, base)
    exe = dev.compile([
        D.Dispatch("AttentionWindowPrefillPagedF16", [op(bq1, q1.nbytes), op(bk, k.nbytes), op(bv, k.nbytes), op(bp3, 100), op(bn1, 4),
                                                      op(outs[0], q1.nbytes)], dims(1, 25, 300, 100)),
        D.Dispatch("AttentionWindowRaggedF16", [op(bq2, q2.nbytes), op(bk, k.nbytes), op(bv, k.nbytes), op(bp, 400), op(bl, 16), op(boff, 20),
                                                op(outs[1], q2.nbytes)], dims(4, 25, 0, 0)),
        D.Dispatch("TokenLogprobsF16", [op(bx, x.nbytes), op(bt, 20), op(outs[2], 20), op(outs[3], 20), op(outs[4], 60), op(outs[5], 60)],
                   rt.logprob_dims(1000, 5, 1, 3)),
    ], max_in_flight=2)
    for _ in range(2):
        fences = [exe.submit(), exe.submit()]
        for f in fences:
            f.wait()
        assert np.array_equal(outs[0].read(0, np.zeros_like(q1)), want1) and np.array_equal(outs[1].read(0, np.zeros_like(q2)), want2)
        for b, w in zip(outs[2:], (r.logprobs, r.entropy, r.top_ids, r.top_logprobs)):
            w = w.cpu().numpy()
            assert np.array_equal(b.read(0, np.zeros_like(w)), w)
    exe.close()
    for b in blocks + outs:
        b.free()
    dev.close()
    rt.attention_error()
