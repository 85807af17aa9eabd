"""Pages of a paged cache on the GPU against the list statement: whole numbers and bytes have to be equal."""
import random

import pytest
import torch

from oracle.pages import Pool

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def status():
    """The kinds of problems reported since the last look."""
    from muse_spark_open_b200 import abi
    torch.cuda.synchronize()
    t = abi.status_for("cuda").t
    code = int(t[0])
    t.zero_()
    return {0: set(), 2: {"bounds"}, 3: {"capacity"}}[code]


def upload(model, shapes):
    """A device pool in the model's state, and caches of random bytes."""
    g = torch.Generator().manual_seed(len(model.refs))
    pool = {"page_table": i32(model.table), "seq_lens": i32(model.seq), "refs": i32(model.refs), "page_size": model.size}
    caches = [torch.randint(0, 256, (len(model.refs), model.size, *s), generator=g, dtype=torch.uint8) for s in shapes]
    return pool, caches, [c.cuda() for c in caches]


def same(model, pool, caches=(), dev=()):
    assert pool["page_table"].tolist() == model.table
    assert pool["seq_lens"].tolist() == model.seq
    assert pool["refs"].tolist() == model.refs
    for a, b in zip(caches, dev):
        assert torch.equal(a, b.cpu())


@pytest.mark.parametrize("seed,num_pages,size,rows,most", [(0, 40, 16, 6, 9), (1, 7, 1, 3, 20), (2, 300, 4, 70, 8), (3, 9000, 64, 40, 300), (4, 4099, 2, 300, 33),
                                                           (5, 33000, 16, 20, 1500)])
def test_random_sequences(seed, num_pages, size, rows, most):
    """Calls in any order with lists of rows, some of them out of range or listed twice, until pages run out and after."""
    from muse_spark_open_b200 import pages
    r = random.Random(seed)
    model = Pool(num_pages, size, rows, most)
    pool, caches, dev = upload(model, [(1, 16), (1, 16)])
    for step in range(60):
        op = r.choice(["extend", "extend", "ragged", "fork", "free", "trim", "compact"])
        n = r.randrange(1, min(rows, 40) + 1)
        listed = [r.randrange(rows) for _ in range(n)] if r.random() < 0.3 else r.sample(range(rows), n)
        if r.random() < 0.1:
            listed[r.randrange(n)] = r.choice([-1, rows, 1 << 30])
        what = (seed, step, op, listed)
        if op == "extend":
            q = r.choice([1, 8, r.randrange(0, max(1, most * size // 3))])
            loc = pages.extend(pool, i32(listed), q)
            want, bad = model.extend(listed, [q] * n)
        elif op == "ragged":
            counts = [r.randrange(0, max(1, most * size // 2)) for _ in range(n)]
            cu = [0] + list(torch.tensor(counts).cumsum(0).tolist())
            loc = pages.extend(pool, i32(listed), cu_seqlens=i32(cu), tokens=cu[-1] + 3)
            want, bad = model.extend(listed, counts)
            want += [-1] * 3
        elif op == "fork":
            parents = [r.randrange(rows) for _ in range(n)]
            if r.random() < 0.7:  # mostly: no child is a parent
                some = r.sample(range(rows), rows)
                parents, listed = [r.choice(some[:max(1, rows // 3)]) for _ in range(n)], [r.choice(some[rows // 3:]) for _ in range(n)]
            pages.fork(pool, i32(parents), i32(listed), dev)
            bad = model.fork(parents, listed, caches)
        elif op == "free":
            pages.free(pool, i32(listed))
            bad = model.free(listed)
        elif op == "trim":
            window, sinks = r.randrange(0, most * size), r.choice([0, 1, size, 2 * size + 1])
            pages.trim(pool, i32(listed), window, sinks)
            bad = model.trim(listed, window, sinks) if window else set()
        else:
            result, bad = pages.compact(pool, dev), set()
            assert tuple(result.tolist()) == model.compact(caches), what
        said = status()
        assert said <= bad and bool(said) == bool(bad), (what, said, bad)
        if op in ("extend", "ragged"):
            assert loc.tolist() == want, what
            for j, row in enumerate(listed):  # the tokens arrive, where there was room for all of them
                count = q if op == "extend" else counts[j]
                if 0 <= row < rows and listed.index(row) == j and model.seq[row] + count <= most * size and \
                        all(x >= 0 for x in model.table[row][model.seq[row] // size:(model.seq[row] + count + size - 1) // size]):
                    model.seq[row] += count
            pool["seq_lens"].copy_(i32(model.seq))
        assert model.consistent(), what
        same(model, pool, caches, dev)


@pytest.mark.parametrize("shape,dtype", [((4, 128), torch.float8_e4m3fn), ((1, 128), torch.bfloat16), ((3, 112), torch.uint8), ((8, 128), torch.float32)])
def test_fork_and_compact_move_every_type(shape, dtype):
    """Pages of 1 to 256 KB in several caches, forks at every fill of the last page."""
    from muse_spark_open_b200 import pages
    size = 64
    model = Pool(90, size, 9, 6)
    for row, n in enumerate([0, 1, 63, 64, 65, 200]):
        model.seq[row] = 0
        model.extend([row], [n])
        model.seq[row] = n
    model.free([3])
    pool, caches, dev = upload(model, [(*shape, torch.empty(0, dtype=dtype).element_size())] * 5)
    typed = [d.flatten(2).view(dtype).view(90, size, *shape) for d in dev]
    assert typed[0].data_ptr() == dev[0].data_ptr()
    pages.fork(pool, i32([5, 4, 2, 0]), i32([6, 7, 8, 3]), typed)
    assert not model.fork([5, 4, 2, 0], [6, 7, 8, 3], caches) and not status()
    same(model, pool, caches, dev)
    pages.free(pool, i32([1, 5, 1]))
    model.free([1, 5])
    pages.compact(pool, typed)
    model.compact(caches)
    assert not status()
    same(model, pool, caches, dev)


def test_calls_in_a_graph_and_on_another_stream():
    """Extend, fork, trim, free and compact captured into one graph and replayed twice, on a stream of their own; the pool
    in between is put back, so both replays give what the model gives."""
    from muse_spark_open_b200 import pages
    model = Pool(64, 16, 6, 8)
    for row, n in enumerate([100, 17, 64]):
        model.extend([row], [n])
        model.seq[row] = n
    pool, caches, dev = upload(model, [(2, 128)])
    keep = {k: v.clone() for k, v in pool.items() if k != "page_size"}
    data = dev[0].clone()
    lists = {k: i32(v) for k, v in {"p": [0, 1, 0], "c": [3, 4, 5], "gone": [1], "all": [0, 2, 3, 4, 5]}.items()}

    def loop():
        pages.fork(pool, lists["p"], lists["c"], dev)
        loc = pages.extend(pool, lists["all"], 8)
        pages.trim(pool, lists["all"], 40, 3)
        pages.free(pool, lists["gone"])
        return loc, pages.compact(pool, dev)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loop()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            loc, result = loop()
    model.fork([0, 1, 0], [3, 4, 5], caches)
    want, _ = model.extend([0, 2, 3, 4, 5], [8] * 5)
    model.trim([0, 2, 3, 4, 5], 40, 3)
    model.free([1])
    moved = model.compact(caches)
    for _ in range(2):
        for k, v in keep.items():
            pool[k].copy_(v)
        dev[0].copy_(data)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert loc.tolist() == want and tuple(result.tolist()) == moved
        same(model, pool, caches, dev)
    assert not status()


def test_lists_longer_than_the_pool_and_the_kept_workspace():
    """More list entries than rows (all but the first of a row are refused), before and after the workspace is kept."""
    from muse_spark_open_b200 import pages
    model = Pool(64, 16, 4, 8)
    pool, _, _ = upload(model, [])
    for listed in ([0, 1, 0, 2, 3, 3, 1, 0, 2], [2, 0], [3, 2, 1, 0, 0, 1, 2, 3]):
        loc = pages.extend(pool, i32(listed), 20)
        want, bad = model.extend(listed, [20] * len(listed))
        assert loc.tolist() == want and status() == bad
        same(model, pool)
    first = pool["scratch"][1]
    pages.compact(pool, [])
    assert pool["scratch"][1] == first and not status()


def test_nothing_to_do():
    from muse_spark_open_b200 import pages
    pool = pages.prepare(8, 16, 4, 4)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    cache = torch.zeros(8, 16, 16, dtype=torch.uint8, device="cuda")
    assert pages.extend(pool, none, 5).numel() == 0
    pages.fork(pool, none, none, [cache])
    pages.free(pool, none)
    pages.trim(pool, i32([0, 1, 2, 3]), 5, 0)
    assert pages.compact(pool, [cache]).tolist() == [0, 0]
    pages.fork(pool, i32([0]), i32([1]), [])  # an empty parent, no caches
    assert not status() and not pool["refs"].any() and (pool["page_table"] == -1).all()


@pytest.mark.parametrize("num_pages", [40, 20000])
@pytest.mark.parametrize("ragged", [False, True])
def test_tokens_do_not_go_into_a_page_that_a_fork_shares(num_pages, ragged):
    """seq_lens set back behind a fork: the rows that would write into a shared page are refused, the others get theirs;
    once the other holder is gone, the same call goes through."""
    from muse_spark_open_b200 import pages
    model = Pool(num_pages, 16, 5, 40)
    for row, n in enumerate([40, 64, 10]):
        model.extend([row], [n])
        model.seq[row] = n
    pool, caches, dev = upload(model, [(2, 16)])
    pages.fork(pool, i32([0, 1]), i32([3, 4]), dev)
    model.fork([0, 1], [3, 4], caches)
    # row 0: into the second of two shared pages; row 4: ends in front of its shared ones; row 3: behind them, in its own page
    for row, n in ((0, 20), (4, 64), (1, 0)):
        model.seq[row] = n
        pool["seq_lens"][row] = n
    counts = [8, 8, 8, 8, 8] if not ragged else [8, 300, 0, 5, 3]
    cu = i32([0, *torch.tensor(counts).cumsum(0).tolist()]) if ragged else None
    for gone in (None, 3, 4):
        if gone is not None:
            pages.free(pool, i32([gone]))
            model.free([gone])
        rows = [0, 1, 2, 3, 4]
        loc = pages.extend(pool, i32(rows), 8) if not ragged else pages.extend(pool, i32(rows), 1, cu, sum(counts))
        want, bad = model.extend(rows, counts)
        assert loc.tolist() == want and status() == bad and ("bounds" in bad) == (gone != 4)
        same(model, pool, caches, dev)


def test_a_copied_pool_has_a_workspace_of_its_own():
    from muse_spark_open_b200 import pages
    pool = pages.prepare(64, 16, 4, 8)
    pages.extend(pool, i32([0, 1]), 20)
    twin = dict(pool, **{k: pool[k].clone() for k in ("page_table", "seq_lens", "refs")})
    pages.extend(twin, i32([2]), 20)
    assert twin["scratch"][1] != pool["scratch"][1]
    first = pool["scratch"][1], twin["scratch"][1]
    pages.extend(twin, i32([3]), 20)
    pages.extend(pool, i32([3]), 20)
    assert first == (pool["scratch"][1], twin["scratch"][1]) and not status()
