"""What pages.py makes of its arguments, without a GPU: the pool's kept workspace, the caches' layout, lists and counts."""
import copy

import pytest
import torch

from muse_spark_open_b200 import abi, build, pages


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return abi.lib()


def packed(pool):
    table, seq, refs = pool["page_table"], pool["seq_lens"], pool["refs"]
    return pages._pages_args.pack(table.data_ptr(), seq.data_ptr(), refs.data_ptr(), *table.shape, refs.shape[0], pool["page_size"]), (table.shape[0], refs.shape[0])


def test_a_deep_copy_does_not_write_into_the_first_pools_workspace(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    pool = pages.prepare(64, 16, 4, 8, device="cpu")
    first = pages._scratch(pool, *packed(pool), 2)
    again = pages._scratch(pool, *packed(pool), 2)
    assert again[0] == first[0] and again[1] == first[1]
    twin = copy.deepcopy(pool)
    mine = pages._scratch(twin, *packed(twin), 2)
    assert mine[0] == twin["scratch"][3].data_ptr() and mine[0] != first[0]
    assert pages._scratch(twin, *packed(twin), 2)[0] == mine[0]
    assert pages._scratch(pool, *packed(pool), 2)[0] == first[0]
