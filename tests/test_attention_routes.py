"""Which kernels attention.kernel_fn takes, without a GPU: the entry points are replaced by markers."""
import pytest
import torch

from muse_spark_open_b200 import attention


@pytest.mark.parametrize("q_len,window,sinks,took", [
    (1, 0, 0, "step"), (1, 64, 4, "step"), (8, 0, 0, "step"), (8, 64, 0, "step"), (8, 64, 4, "prompt"), (7, 0, 0, "prompt"), (9, 64, 4, "prompt"),
    (8, 0, 4, "step"),  # without a window sinks are nothing: the block runs as it does when they are not named, cache_loc and all
])
def test_which_kernels_a_block_takes(monkeypatch, q_len, window, sinks, took):
    calls = []
    monkeypatch.setattr(attention, "_run_step", lambda *a: calls.append("step"))
    monkeypatch.setattr(attention, "_run_prompt", lambda *a: calls.append("prompt"))
    cfg = {"batch": 2, "q_len": q_len, "num_q_heads": 8, "head_dim": 128, "window": window, "sinks": sinks}
    data = {"config": cfg, "qkv": torch.empty(2, q_len, 18 * 128, dtype=torch.bfloat16), "k_cache": torch.zeros(1).to(torch.float8_e4m3fn),
            "seq_lens": torch.zeros(2, dtype=torch.int32), "page_table": torch.zeros(2, 1, dtype=torch.int32),
            "cache_loc": torch.zeros(2 * q_len, dtype=torch.int64)}
    monkeypatch.setattr(attention.abi, "ptr", lambda t: t.data_ptr())
    attention.kernel_fn(data)
    assert calls == [took]
