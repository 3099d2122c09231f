"""The block pool's sharing, copy on write, freeing behind a window and compaction, against a model of it."""
import numpy as np
import pytest

from accel_b200 import _lib
from accel_b200.blockpool import BlockPool

NONE = BlockPool.NONE


def test_share_own_and_free():
    p = BlockPool(6, 4)
    a = p.grow(None, 10)                       # three pages
    b = p.share(a)
    assert b == a and p.available() == 3 and all(p.refs(x) == 2 for x in a)
    c, src, dst = p.own(b, 9, 10)              # the last page is partly filled and both write on
    assert c[:2] == a[:2] and c[2] not in a and (src, dst) == ([a[2]], [c[2]])
    assert p.refs(a[2]) == 1 and p.refs(c[2]) == 1 and p.available() == 2
    assert p.own(c, 9, 10) == (c, [], [])      # already its own
    assert p.own(c, 12, 16) == (c, [], [])     # no page there yet
    p.free(a)
    assert p.available() == 3 and p.refs(a[0]) == 1
    p.free(c)
    assert p.available() == 6
    with pytest.raises(_lib.AccelError, match="already free"):
        p.free([c[0]])
    with pytest.raises(_lib.AccelError, match="only a held block can be shared"):
        p.share([c[0]])
    with pytest.raises(_lib.AccelError, match="only a held block can be written"):
        p.own([c[0]], 0, 4)
    with pytest.raises(_lib.AccelError):
        p.refs(6)


def test_own_and_share_change_nothing_when_they_refuse():
    p = BlockPool(3, 4)
    a = p.grow(None, 8)
    b = p.share(a)
    with pytest.raises(_lib.AccelError, match="does not evict"):
        p.own(b, 0, 8)                         # two shared pages and one free
    assert [p.refs(x) for x in a] == [2, 2] and p.available() == 1
    free = next(x for x in range(3) if x not in a)
    with pytest.raises(_lib.AccelError):
        p.share([a[0], free])
    assert p.refs(a[0]) == 2
    with pytest.raises(_lib.AccelError):
        p.own(b, 5, 4)


@pytest.mark.parametrize("block", [1, 4, 16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 0), (8, 3), (16, 16), (40, 1), (3, 50)])
def test_trim_frees_exactly_what_no_later_query_sees(block, window, sinks):
    for n in (0, 1, 7, 16, 33, 100):
        p = BlockPool(128, block)
        row = p.grow(None, n)
        kept = p.trim(row, n, window, sinks)
        seen = {j // block for q in range(n, n + 60) for j in range(n) if q - j < window or j < sinks}
        # a page is kept if a later query sees a position of it, and the reserved rest of the row too
        assert [x != NONE for x in kept] == [i in seen or (i + 1) * block > n + 1 - window for i in range(len(row))], (n, kept)
        assert all(a in (b, NONE) for a, b in zip(kept, row))
        assert p.available() == 128 - sum(x != NONE for x in kept)
        assert p.trim(kept, n, window, sinks) == kept
        again = p.grow(kept, n + 10)           # a trimmed row goes on growing
        assert again[:len(kept)] == kept
        p.free(again)
        assert p.available() == 128
    for bad in ((-1, 4, 0), (4, 0, 0), (4, 4, -1)):
        with pytest.raises(_lib.AccelError):
            BlockPool(4, 4).trim([], *bad)


def test_a_random_script_against_a_model():
    """Contents follow the rows through growing, sharing, writing, trimming, freeing and compaction."""
    rng = np.random.default_rng(4)
    blocks, block, window, sinks = 96, 4, 24, 5
    p, mem = BlockPool(blocks, block), np.full(blocks, -1)
    rows, want, length = {}, {}, {}
    tag = 0

    def copy(src, dst):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        mem[dst] = mem[src]

    for step in range(1500):
        op, s = rng.integers(0, 7), int(rng.integers(0, 6))
        if op <= 1:                            # write some positions
            n0 = length.get(s, 0)
            n = n0 + int(rng.integers(1, 12))
            try:
                row = p.grow(rows.get(s), n)
                rows[s] = row
                row, src, dst = p.own(row, n0, n)
            except _lib.AccelError:
                rows.setdefault(s, []), want.setdefault(s, []), length.setdefault(s, 0)
                want[s] += [-1] * (len(rows[s]) - len(want[s]))
                for i in range(len(want[s])):
                    if rows[s][i] != NONE and (i * block >= n0):
                        want[s][i] = mem[rows[s][i]]
                continue
            copy(src, dst)
            rows[s], length[s] = row, n
            w = want.setdefault(s, [])
            w += [-1] * (len(row) - len(w))
            for i in range(n0 // block, len(row)):
                assert p.refs(row[i]) == 1
                tag += 1
                mem[row[i]] = w[i] = tag
        elif op == 2 and rows:                 # fork
            a = sorted(rows)[int(rng.integers(0, len(rows)))]
            if a != s:
                if s in rows:
                    p.free(rows[s])
                rows[s], want[s], length[s] = p.share(rows[a]), list(want[a]), length[a]
        elif op == 3 and s in rows:
            p.free(rows.pop(s))
            want.pop(s), length.pop(s)
        elif op == 4 and s in rows:
            rows[s] = p.trim(rows[s], length[s], window, sinks)
        elif op == 5:
            names = sorted(rows)
            out, src, dst = p.compact([rows[n] for n in names])
            copy(src, dst)
            rows = dict(zip(names, out))
            live = {x for r in rows.values() for x in r if x != NONE}
            assert live == set(range(len(live)))
        held = {}
        for r in rows.values():
            for x in r:
                if x != NONE:
                    held[x] = held.get(x, 0) + 1
        assert p.available() == blocks - len(held)
        assert all(p.refs(x) == held.get(x, 0) for x in range(blocks))
        for n in rows:
            for x, w in zip(rows[n], want[n]):
                assert x == NONE or mem[x] == w, (step, n)


def test_compaction_wants_every_row():
    p = BlockPool(8, 4)
    a, b = p.grow(None, 8), p.grow(None, 12)
    p.free(a[:1])
    with pytest.raises(_lib.AccelError, match="every row in use"):
        p.compact([b])
    assert p.available() == 4
    rows, src, dst = p.compact([[NONE, a[1]], b])
    assert len(src) == len(dst) and {x for r in rows for x in r} == {NONE, 0, 1, 2, 3}


def test_compaction_refuses_rows_that_name_pages_nobody_holds():
    p = BlockPool(8, 4)
    other = p.grow(None, 8)
    a = p.grow(None, 8)
    p.free([other[0]])
    for rows in ([[*a, other[0]]], [[a[0]], [a[1], 7 if 7 not in a + other else 6]], [[*a, 8]]):
        free = p.available()
        with pytest.raises(_lib.AccelError):            # as many as are held, and not those: other[1] would move unseen
            p.compact(rows)
        assert p.available() == free and all(p.refs(x) == 1 for x in (*a, other[1]))
    rows, src, dst = p.compact([a, [other[1], NONE]])
    assert sorted(x for r in rows for x in r if x != NONE) == [0, 1, 2] and len(src) == len(dst)
