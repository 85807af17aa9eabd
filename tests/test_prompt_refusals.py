"""What the prompt attention's entry point refuses, without a GPU: shapes, types and layouts are checked before any device
work, and the C function turns its own arguments down before it touches CUDA."""
import ctypes as C

import pytest
import torch

from muse_spark_open_b200 import abi, attention, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.lib()


def _data(**kw):
    cfg = {"batch": 2, "num_q_heads": 8, "num_kv_heads": 1, "head_dim": 128, "page_size": 64, "window": 0, "rope_theta": 0.0, "qk_scale_factor": 1.0,
           "sm_scale": 0.1}
    cfg.update(kw.pop("config", {}))
    d = {"qkv": torch.zeros(5, 18 * 128, dtype=torch.bfloat16), "k_cache": torch.zeros(4, 64, 1, 128).to(torch.float8_e4m3fn),
         "v_cache": torch.zeros(4, 64, 1, 128).to(torch.float8_e4m3fn), "k_scale": torch.ones(()), "v_scale": torch.ones(()),
         "seq_lens": torch.zeros(2, dtype=torch.int32), "page_table": torch.zeros(2, 2, dtype=torch.int32),
         "cu_seqlens_q": torch.tensor([0, 2, 5], dtype=torch.int32), "config": cfg}
    d.update(kw)
    return d


@pytest.mark.parametrize("bad,words", [
    ({"qkv": torch.zeros(5, 18 * 128)}, "bfloat16"),
    ({"qkv": torch.zeros(5, 17 * 128, dtype=torch.bfloat16)}, "qkv must be"),
    ({"qkv": torch.zeros(18 * 128, 5, dtype=torch.bfloat16).t()}, "qkv must be"),
    ({"k_cache": torch.zeros(4, 64, 1, 128)}, "float8_e4m3fn"),
    ({"v_cache": torch.zeros(4, 32, 1, 128).to(torch.float8_e4m3fn)}, "k_cache / v_cache"),
    ({"seq_lens": torch.zeros(2, dtype=torch.int64)}, "int32"),
    ({"seq_lens": torch.zeros(3, dtype=torch.int32)}, "contiguous"),
    ({"page_table": torch.zeros(2, 4, dtype=torch.int32)[:, ::2]}, "contiguous"),
    ({"cu_seqlens_q": torch.zeros(2, dtype=torch.int32)}, "contiguous"),
    ({}, "CUDA"),
])
def test_python_refusals(lib, bad, words):
    with pytest.raises(abi.MskError, match=words):
        attention.prompt_fn(_data(**bad))


def test_c_refusals(lib):
    ok = dict(B=2, T=5, Hq=8, Hkv=1, d=128, page_size=64, num_pages=4, max_pages=2, sm_scale=0.1, qk_scale_factor=1.0)
    n = C.c_size_t()

    def size(**kw):
        p = abi.PromptParams(**{**ok, **kw})
        return lib.msk_attn_prompt_scratch_bytes(C.byref(p), C.byref(n))
    assert size() == 0 and n.value >= 5 * 8 * 256
    assert [size(d=64), size(Hq=4), size(page_size=48), size(page_size=256), size(B=0), size(T=0)] == [-3] * 6
    assert [size(window=-1), size(sinks=-1), size(splits=65)] == [-1] * 3
    p = abi.PromptParams(**ok)
    assert lib.msk_attn_prompt(C.byref(p), None, None) == -1  # null pointers
    assert lib.msk_attn_prompt(None, None, None) == -1 and lib.msk_attn_prompt_scratch_bytes(None, C.byref(n)) == -1
