"""The list statement of the cache's pages keeps its own promises (CPU), and the entry points refuse what they must before
any device work."""
import ctypes as C
import random

import pytest
import torch

from oracle.pages import Pool


@pytest.mark.parametrize("seed", range(5))
def test_model_counts_pages_and_keeps_data(seed):
    r = random.Random(seed)
    size, rows, most = r.choice([1, 4, 16]), 8, 12
    pool = Pool(60, size, rows, most)
    cache = torch.zeros(60, size, dtype=torch.long)
    text = {i: [] for i in range(rows)}  # what each row's positions should hold
    stamp = 0
    for _ in range(120):
        op = r.choice(["extend", "extend", "fork", "free", "compact"])
        if op == "extend":
            row, n = r.randrange(rows), r.randrange(0, 2 * size + 1)
            loc, bad = pool.extend([row], [n])
            if not bad:
                for at in loc:
                    stamp += 1
                    cache.view(-1)[at] = stamp
                    text[row].append(stamp)
                pool.seq[row] += n
        elif op == "fork":
            p, c = r.sample(range(rows), 2)
            bad = pool.fork([p], [c], [cache])
            text[c] = [] if bad else list(text[p])
        elif op == "free":
            row = r.randrange(rows)
            pool.free([row, row])
            text[row] = []
        else:
            n, _ = pool.compact([cache])
            assert all(x > 0 for x in pool.refs[:n]) and not any(pool.refs[n:])
        assert pool.consistent()
        for row in range(rows):
            got = [int(cache[pool.table[row][i // size], i % size]) for i in range(pool.seq[row])]
            assert got == text[row]


def test_refusals():
    from muse_spark_open_b200 import abi, build, pages
    build.build()
    lib = abi.lib()
    n = C.c_size_t()
    q = abi.Pages(16, 16, 16, 4, 4, 10, 16)  # addresses that a refused call never touches
    assert lib.msk_pages_scratch_bytes(C.byref(q), 4, C.byref(n)) == 0 and n.value > 0
    ws = C.c_void_p(256)
    assert lib.msk_pages_free(None, None, 0, None, None) == -1
    assert lib.msk_pages_free(C.byref(q), None, 3, None, None) == -1
    assert lib.msk_pages_free(C.byref(abi.Pages(16, 16, 16, 4, 4, 10, 12)), None, 0, None, None) == -3  # page size 12
    assert lib.msk_pages_trim(C.byref(q), C.c_void_p(16), 1, -1, 0, None, None) == -1
    assert lib.msk_pages_trim(C.byref(q), C.c_void_p(16), 1, 8, -2, None, None) == -1
    assert lib.msk_pages_trim(C.byref(q), C.c_void_p(16), 1, 0, 0, None, None) == 0  # nothing to do, nothing launched
    assert lib.msk_pages_extend(C.byref(q), C.c_void_p(16), 1, 1, None, 0, None, ws, 5, None, None) == -1      # workspace too small
    assert lib.msk_pages_extend(C.byref(q), C.c_void_p(16), 1, -1, None, 0, None, ws, n.value, None, None) == -1
    one = (C.c_void_p * 1)(256)
    assert lib.msk_pages_fork(C.byref(q), C.c_void_p(16), C.c_void_p(16), 1, one, 1, 24, ws, n.value, None, None) == -3  # 24 bytes per token
    assert lib.msk_pages_fork(C.byref(q), C.c_void_p(16), C.c_void_p(16), 1, one, 129, 16, ws, n.value, None, None) == -1
    assert lib.msk_pages_compact(C.byref(q), one, 1, 16, None, C.c_void_p(8), n.value, None, None) == -1      # workspace alignment
    pool = pages.prepare(10, 16, 4, 4, device="cpu")
    rows = torch.zeros(1, dtype=torch.int32)
    for bad in (lambda: pages.free(pool, rows), lambda: pages.extend(pool, rows), lambda: pages.free(pool, rows.long()),
                lambda: pages.free(dict(pool, refs=pool["refs"].long()), rows), lambda: pages.prepare(10, 12, 4, 4, device="cpu")):
        with pytest.raises(abi.MskError):
            bad()


def test_model_refuses_tokens_in_shared_pages():
    pool = Pool(20, 8, 3, 6)
    pool.extend([0], [20])
    pool.seq[0] = 20
    assert not pool.fork([0], [1], [])
    pool.seq[0] = 12                           # back into the second page, which row 1 holds too
    assert pool.extend([0], [4]) == ([-1] * 4, {"bounds"})
    pool.seq[0] = 16                           # behind the shared pages: its own page
    assert pool.extend([0], [4])[1] == set()
    pool.free([1])
    pool.seq[0] = 12
    assert pool.extend([0], [4])[1] == set()
