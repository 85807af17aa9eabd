"""What the page calls find wrong in their lists is reported, and the entries concerned are skipped."""
import pytest
import torch

from oracle.pages import Pool
from test_gpu_pages import i32, same, status, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("num_pages", [50, 20000])  # one CTA plans, or a cluster
@pytest.mark.parametrize("cu,tokens,bad", [([0, 5, 25, 30], 24, [1, 2]), ([0, 5, 25, 30], 29, [2]), ([0, 5, 25, 30], 0, [0, 1, 2]), ([0, 9, 5, 5], 9, [1]),
                                           ([-3, 2, 4, 6], 6, [0]), ([0, 3, 3, 2 ** 31 - 1], 3, [2])])
def test_ragged_extend_reports_tokens_that_have_no_entry(num_pages, cu, tokens, bad):
    from muse_spark_open_b200 import pages
    model = Pool(num_pages, 4, 5, 12)
    for row, n in enumerate([3, 0, 8, 1]):
        model.extend([row], [n])
        model.seq[row] = n
    pool, _, _ = upload(model, [])
    rows = [2, 0, 3]
    loc = pages.extend(pool, i32(rows), cu_seqlens=i32(cu), tokens=tokens)
    assert status() == {"bounds"}
    want = [-1] * tokens
    for j in range(3):
        if j not in bad:
            want[cu[j]:cu[j + 1]] = model.extend([rows[j]], [cu[j + 1] - cu[j]])[0]
    assert loc.tolist() == want
    same(model, pool)
    assert model.consistent()


@pytest.mark.parametrize("num_pages", [50, 20000])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("seq", [-1, -4, -2 ** 31])
def test_extend_reports_a_negative_length(num_pages, ragged, seq):
    from muse_spark_open_b200 import pages
    model = Pool(num_pages, 4, 3, 12)
    model.extend([0], [7])
    model.seq[0] = 7
    pool, _, _ = upload(model, [])
    pool["seq_lens"][1] = seq
    loc = pages.extend(pool, i32([2, 1, 0]), cu_seqlens=i32([0, 5, 10, 15]), tokens=15) if ragged else pages.extend(pool, i32([2, 1, 0]), 5)
    assert status() == {"bounds"}
    want = model.extend([2, 0], [5, 5])[0]
    assert loc.tolist() == want[:5] + [-1] * 5 + want[5:]
    pool["seq_lens"][1] = 0
    same(model, pool)


@pytest.mark.parametrize("seq", [-1, -4, -2 ** 31])
def test_fork_reports_a_parent_of_negative_length(seq):
    """The child stays what it was, the other forks go through."""
    from muse_spark_open_b200 import pages
    model = Pool(30, 4, 5, 6)
    for row, n in enumerate([7, 5, 3]):
        model.extend([row], [n])
        model.seq[row] = n
    pool, caches, dev = upload(model, [(1, 16)])
    pool["seq_lens"][1] = seq
    pages.fork(pool, i32([1, 0]), i32([2, 3]), dev)
    assert status() == {"bounds"}
    assert not model.fork([0], [3], caches)
    pool["seq_lens"][1] = 5
    same(model, pool, caches, dev)


@pytest.mark.parametrize("at", [0, 1])  # a page that is shared, and the last one, which is copied
def test_fork_reports_a_page_that_does_not_exist(at):
    """The child gets no page there, the rest of the fork goes through."""
    from muse_spark_open_b200 import pages
    model = Pool(30, 4, 5, 6)
    for row, n in enumerate([7, 5]):
        model.extend([row], [n])
        model.seq[row] = n
    model.refs[model.table[0][at]] = 0
    model.table[0][at] = -1
    pool, caches, dev = upload(model, [(1, 16)])
    pool["page_table"][0, at] = 10 ** 6
    pages.fork(pool, i32([0, 1]), i32([2, 3]), dev)
    assert status() == {"bounds"}
    assert not model.fork([0, 1], [2, 3], caches)
    pool["page_table"][0, at] = -1
    same(model, pool, caches, dev)
