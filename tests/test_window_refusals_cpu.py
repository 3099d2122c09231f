"""What the windowed attention, the page copies and the log probabilities refuse, without a GPU."""
import struct

import pytest
import torch

from accel_b200 import _lib, runtime as rt
from accel_b200 import tensor as T

Q, K = torch.zeros(4, 64), torch.zeros(32, 2, 64)
LEN = torch.ones(1, dtype=torch.int32)


def opts(**kw):
    return T.AttentionOptions(lengths=LEN, scale=0.1, **kw)


@pytest.mark.parametrize("kw,why", [
    (dict(window=-1), "Window is -1"), (dict(window=1 << 32), "number of positions"), (dict(window=2.5), "number of positions"),
    (dict(window=True), "number of positions"), (dict(window=4, sinks=-2), "Sinks is -2"), (dict(sinks=4), "Window is 0"),
    (dict(window=4, pages=torch.zeros(2, 3, dtype=torch.int32), block=4), "one row of block ids"),
    (dict(window=4, pages=torch.zeros(3), block=4), "page table is u32"),
    (dict(window=4, pages=torch.zeros(3, dtype=torch.int32)), "Block is 0"),
])
def test_attention_refuses(kw, why):
    with pytest.raises(T.Refused, match=why):
        T.attention(Q, K, K, opts(**kw))


def test_prefill_refuses_positions_past_32_bits_and_tables_of_two_axes():
    q = torch.zeros(3, 4, 64)
    for base in (-1, 0xffffffff - 2):
        with pytest.raises(T.Refused, match="positions are u32"):
            T.attention(q, K, K, opts(window=4, base=base))
    with pytest.raises(T.Refused, match="one row of block ids"):
        T.attention(q, K, K, opts(window=4, base=0, pages=torch.zeros(1, 3, dtype=torch.int32), block=4))
    with pytest.raises(T.Refused, match="BaseName"):
        T.attention(q, K, K, opts(window=4))


def test_there_is_no_cpu_path():
    for call in (lambda: T.attention(Q, K, K, opts(window=4)), lambda: T.token_logprobs(torch.zeros(2, 8)),
                 lambda: T.copy_pages([K], [0], [1], 4)):
        with pytest.raises(_lib.AccelError, match="no CPU path"):
            call()


def window(batch=2, qh=4, kv=2, d=64, block=4, mp=8, win=8, sinks=0, cap=32, q_seq=2, base=0):
    return rt.window_dims(batch, qh, kv, d, block, mp, 0.1, win, sinks, cap, q_seq, base)


def test_the_launcher_refuses():
    lens = [2 * 4 * 64, 32 * 2 * 64, 32 * 2 * 64, 16, 2, 2 * 4 * 64]
    ws = lambda u, le=lens: rt.workspace_bytes("AttentionWindowBatched", le, u)
    ws(window())
    for u, why in ((window(win=0), "window of 0"), (window(d=60), "multiple of eight"), (window(d=136), "at most 128"),
                   (window(kv=3), "query heads over 3"), (window(kv=0), "query heads over 0"), (window(block=0), "Block is 0"),
                   (window(cap=33), "Capacity=33"), (window(batch=3), "Batch=3"), (window(mp=9), "MaxPages=9")):
        with pytest.raises(_lib.AccelError, match=why):
            ws(u)
    ws(window(cap=1 << 26, kv=4, qh=8, d=32), [2 * 4 * 64, 0xffffffff, 0xffffffff, 16, 2, 2 * 4 * 64])
    with pytest.raises(_lib.AccelError, match="takes 6 bindings"):
        ws(window(), lens[:5])
    with pytest.raises(_lib.AccelError, match="48-byte uniform"):
        ws(window()[:32])
    with pytest.raises(_lib.AccelError, match="pass 32 bits"):
        rt.workspace_bytes("AttentionWindowPrefill", [2 * 4 * 64, lens[1], lens[2], 1, 2 * 4 * 64], window(base=0xffffffff))


@pytest.mark.parametrize("kw,why", [
    (dict(top=33), "at most 32"), (dict(top=-1), "at most 32"), (dict(top=9), "vocabulary of 8"), (dict(top=True), "at most 32"),
    (dict(targets=torch.zeros(3, dtype=torch.int32)), "hold 2 rows"), (dict(targets=torch.zeros(2, dtype=torch.int64)), "u32"),
    (dict(targets=torch.zeros(2, 1, 1, dtype=torch.int32)), r"\[rows\] or"),
])
def test_logprobs_refuse(kw, why):
    with pytest.raises(T.Refused, match=why):
        T.token_logprobs(torch.zeros(2, 8), **kw)


def test_logprobs_refuse_other_logits():
    for x in (torch.zeros(2, 8, dtype=torch.float64), torch.zeros(8), torch.zeros(2, 0)):
        with pytest.raises(T.Refused, match="f32 or f16"):
            T.token_logprobs(x)
    dims = lambda *a: struct.pack("<IIII", *a)
    good = [16, 2, 2, 2, 6, 6]
    rt.workspace_bytes("TokenLogprobs", good, dims(8, 2, 1, 3))
    for lens, u in ((good, dims(8, 3, 1, 3)), (good, dims(9, 2, 1, 3)), (good, dims(8, 2, 2, 3)), (good, dims(8, 2, 1, 4)),
                    (good, dims(0, 2, 1, 0))):
        with pytest.raises(_lib.AccelError, match="lengths block"):
            rt.workspace_bytes("TokenLogprobs", lens, u)
    with pytest.raises(_lib.AccelError, match="at most 32"):
        rt.workspace_bytes("TokenLogprobs", [99, 1, 1, 1, 33, 33], dims(99, 1, 1, 33))


def test_page_copies_refuse():
    c = torch.zeros(32, 2, 8)
    for args, why in ((([c], [0], [1, 2], 4), "1 source"), (([c], [0], [1], 0), "Block is 0"), (([c, c], [0], [1], 4), "named twice"),
                      (([c, torch.zeros(32, 2, 4)], [0], [1], 4), "one form"), (([c, c.half()], [0], [1], 4), "one form"),
                      (([c[:, :1]], [0], [1], 4), "strided")):
        with pytest.raises(T.Refused, match=why):
            T.copy_pages(*args)
    assert T.copy_pages([], [0], [1], 4) is None
    # what the entry point itself refuses, before anything is launched: the pointers are never followed
    import ctypes as C
    L = _lib.lib()
    ptr = (C.c_void_p * 1)(1 << 20)
    call = lambda src, dst, pages=8, size=64, n=1: _lib.check(L.ab_cache_copy_pages(
        None, ptr, n, size, pages, (C.c_uint32 * len(src))(*src), (C.c_uint32 * len(dst))(*dst), len(src)))
    for src, dst, why in (([0, 1], [2, 2], "written twice"), ([0, 2], [2, 3], "both read and written"), ([4], [4], "both read"),
                          ([8], [0], "of 8 pages"), ([0], [8], "of 8 pages")):
        with pytest.raises(_lib.AccelError, match=why):
            call(src, dst)
    with pytest.raises(_lib.AccelError, match="bad argument"):
        call([0], [1], size=0)
    assert call([], []) == 0


def test_page_copies_refuse_caches_that_overlap():
    import ctypes as C
    L = _lib.lib()
    for starts in ((1 << 20, (1 << 20) + 8 * 64 - 64), ((1 << 20) + 64, 1 << 20), (1 << 20, 1 << 20)):
        ptrs = (C.c_void_p * 2)(*starts)
        with pytest.raises(_lib.AccelError, match="overlap"):
            _lib.check(L.ab_cache_copy_pages(None, ptrs, 2, 64, 8, (C.c_uint32 * 1)(0), (C.c_uint32 * 1)(1), 1))


def test_positions_are_u32():
    q, lens = torch.zeros(4, 8, device="meta"), torch.ones(1, dtype=torch.int32, device="meta")
    k = torch.empty(1 << 32, 1, 8, dtype=torch.float16, device="meta")
    with pytest.raises(T.Refused, match="capacity is 4294967296"):
        T.attention(q, k, k, T.AttentionOptions(lengths=lens, window=4))
    with pytest.raises(T.Refused, match="Block is 4294967296"):
        T.attention(q, k[:64], k[:64], T.AttentionOptions(lengths=lens, window=4, block=1 << 32,
                                                          pages=torch.zeros(3, dtype=torch.int32, device="meta")))


def test_query_rows_are_counted_in_32_bits():
    q = torch.empty(1 << 24, 32, 8, device="meta")                # 2^32 elements
    k = torch.empty(64, 32, 8, device="meta")
    one = torch.ones(1, dtype=torch.int32, device="meta")
    with pytest.raises(T.Refused, match="counts them in 32 bits"):
        T.attention(q, k, k, T.AttentionOptions(lengths=one, window=4, base=0))
    with pytest.raises(_lib.AccelError, match="does not fit 32 bits"):
        rt.workspace_bytes("AttentionWindowRagged", [0xffffffff, 64 * 256, 64 * 256, 4, 1, 2, 0xffffffff],
                           window(batch=1, qh=32, kv=32, d=8, block=16, mp=4, cap=64))
