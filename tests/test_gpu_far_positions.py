"""Prompts and steps on one cache at far positions, without sinks.  Prompts turn by the exact angle, tokens and verify blocks
without sinks by the reference's product in 32 bits, which is off by up to 2^-10 rad between positions 16384 and 32768.  A step
over keys that a prompt has cached is the reference's formula on those keys, and no further from the exact one than its other
roundings put it.

Bounds.  Against the reference's angle: those of tests/test_gpu_sinks.py (rounding of queries to two E4M3 terms, 0.0033 of a
score; 6e-3 of the relative L2 norm).  Against the exact angle: queries of elements around 5.5 move by 5.6e-4 x 5.5 = 3e-3 rms
in the six fastest pairs and by half as much every three pairs, a tenth of BF16's step of 2^-5, so 2.4 of 128 elements round the
other way, each 2^-5 x |k| / 11.3 = 0.0028 of a score: 0.0043 rms, with the 0.0033 that makes 0.0054, so 1e-2 of the norm."""
import pytest
import torch

from oracle import attention as oattn
from test_gpu_prompt import check, make_prompt, new_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len", [1, 8])
def test_steps_over_keys_that_a_prompt_cached(q_len):
    from muse_spark_open_b200 import abi, attention
    n, hkv = 600, 2
    data = make_prompt([16500], [n + q_len], 31, hkv=hkv, window=500)
    dev = oattn.to_device(data, "cuda")
    first = dict(dev, qkv=dev["qkv"][:n], cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    out = attention.prompt_fn(first)
    torch.cuda.synchronize()
    rows = new_rows(data)
    k_new, v_new = (dev[x].view(-1, hkv, 128)[rows[:n].cuda()].cpu() for x in ("k_cache", "v_cache"))
    check(dict(data, qkv=data["qkv"][:n], cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32)), out.cpu(), k_new, v_new, "prompt")
    # the step sees only keys that the prompt wrote
    step = {"qkv": data["qkv"][n:].view(1, q_len, -1).contiguous(), "k_cache": dev["k_cache"].cpu(), "v_cache": dev["v_cache"].cpu(),
            "k_scale": data["k_scale"], "v_scale": data["v_scale"], "page_table": data["page_table"], "seq_lens": data["seq_lens"] + n,
            "cache_loc": rows[n:], "config": dict(data["config"], q_len=q_len)}
    run = oattn.to_device(step, "cuda")
    out = attention.kernel_fn(run).cpu().double().view(q_len, -1)
    abi.status_for("cuda").raise_if_set("attention")
    new = [run[x].view(-1, hkv, 128)[rows[n:].cuda()].cpu() for x in ("k_cache", "v_cache")]
    ref = oattn.ref_kernel(step, new_kv=[x.view(1, q_len, hkv, 128) for x in new])[0].double().view(q_len, -1)
    assert float((out - ref).norm() / ref.norm()) < 6e-3
    exact = oattn.ref_stream(dict(step, cu_seqlens_q=torch.tensor([0, q_len], dtype=torch.int32)), new_kv=new)[0]
    assert float((out - exact).norm() / exact.norm()) < 1e-2
