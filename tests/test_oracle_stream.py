"""The 64-bit statement of attention with sinks and any number of new tokens agrees with the statement pinned to the
reference's outputs, where both apply (CPU)."""
import pytest
import torch

from oracle import attention as oattn


@pytest.mark.parametrize("q_len,window,sinks", [(1, 0, 0), (1, 40, 0), (8, 40, 0), (8, 5, 3), (1, 40, 7), (8, 64, 100)])
def test_stream_statement_is_the_pinned_one(q_len, window, sinks):
    data = oattn.make_input(3, [70, 5, 130], seed=q_len + window, q_len=q_len, hq=8, hkv=1, page=16, window=window)
    data["config"]["sinks"] = sinks
    ref, k, v = oattn.ref_kernel(data)
    out, k64, v64 = oattn.ref_stream(data)
    assert (k64.view(torch.uint8).view(-1) != k.view(torch.uint8).view(-1)).float().mean() < 2e-3
    assert torch.equal(v64.view(torch.uint8).view(-1), v.view(torch.uint8).view(-1))
    out = oattn.ref_stream(data, new_kv=(k, v))[0]
    # FP32 against FP64 (angles: 5e-4 at most at these positions); a query that rounds to BF16 the other way moves one row
    assert float((out - ref.double().view(out.shape)).norm() / out.norm()) < 2e-3


def test_sinks_beyond_the_window_change_what_is_seen():
    data = oattn.make_input(1, [100], seed=1, hq=8, hkv=1, page=16, window=20)
    base = oattn.ref_stream(data)[0]
    data["config"]["sinks"] = 81  # positions 0 .. 80 and 81 .. 100: everything
    full = oattn.ref_stream(dict(data, config=dict(data["config"], window=0)))[0]
    assert torch.equal(oattn.ref_stream(data)[0], full) and not torch.allclose(base, full)
