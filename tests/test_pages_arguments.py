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


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("num_pages", [1, 6])
def test_bytes_per_token_of_caches_whose_sizes_are_one(page, num_pages):
    """Strides of axes of length one may be anything in a contiguous tensor; the bytes per token follow from the shape."""
    pool = {"refs": torch.zeros(num_pages, dtype=torch.int32), "page_size": page}
    cache = torch.empty((num_pages, page, 2, 16), dtype=torch.uint8)
    odd = cache.as_strided(cache.shape, (cache.stride(0) if num_pages > 1 else 7, cache.stride(1) if page > 1 else 4096, 16, 1))
    assert odd.is_contiguous()
    for c in (cache, odd, odd.view(torch.int8)):
        assert pages._caches([c], pool, -1)[2] == 32


def test_caches_of_other_layouts_are_refused():
    pool = {"refs": torch.zeros(6, dtype=torch.int32), "page_size": 4}
    good = torch.empty((6, 4, 2, 16), dtype=torch.uint8)
    for bad in (torch.empty((6, 4), dtype=torch.uint8), torch.empty((7, 4, 32), dtype=torch.uint8), torch.empty((6, 8, 32), dtype=torch.uint8),
                torch.empty((6, 2, 4, 16), dtype=torch.uint8).transpose(1, 2), torch.empty((6, 4, 2, 16), dtype=torch.int16)):
        with pytest.raises(abi.MskError):
            pages._caches([good, bad], pool, -1)


@pytest.mark.parametrize("more", [{}, {"tokens": None}, {"tokens": -1}])
def test_ragged_extend_wants_to_know_how_many_tokens(more):
    pool = pages.prepare(8, 4, 2, 3, device="cpu")
    with pytest.raises(abi.MskError, match="tokens"):
        pages.extend(pool, torch.zeros(1, dtype=torch.int32), cu_seqlens=torch.tensor([0, 3], dtype=torch.int32), **more)
