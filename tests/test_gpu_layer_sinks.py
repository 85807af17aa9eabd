"""First tokens that stay visible, through the whole layer against its oracle, for single tokens and for blocks of 8 (which the
layer keeps on the verify kernel), and that kernel by itself with its own choice of chunks."""
import pytest
import torch

from oracle import attention as oattn
from oracle import layer as olayer
from test_gpu_layer import _run_and_check
from test_gpu_sinks import close, streaming

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len", [1, 8])
@pytest.mark.parametrize("sinks", [1, 4, 200])
def test_layer_with_sinks_matches_the_oracle(q_len, sinks):
    """Pages that no token sees are gone, positions that none sees hold NaN."""
    weights = olayer.make_weights(3, hidden=1024, hq=8, hkv=1, d=128, n_experts=16, inner=128)
    data = olayer.make_input(3, [700, 1300, 5], 7, q_len=q_len, hidden=1024, hq=8, hkv=1, d=128, window=128, rope_theta=1e6)
    _run_and_check(weights, streaming(data, sinks), f"sinks {sinks}, {q_len} tokens")


@pytest.mark.parametrize("seqs,window,sinks,hkv", [([1500, 3000], 1024, 4, 2), ([6000], 4096, 300, 1), ([i * 37 % 900 for i in range(60)], 100, 5, 4),
                                                   ([130, 2, 4000, 0], 64, 1, 8)])
def test_verify_kernel_picks_its_chunks(seqs, window, sinks, hkv):
    from muse_spark_open_b200 import abi, attention
    b = len(seqs)
    data = streaming(oattn.make_input(b, seqs, seed=b + sinks, q_len=8, hq=8 * hkv, hkv=hkv, page=64, window=window), sinks)
    dev = oattn.to_device(data, "cuda")
    out = torch.empty((8 * b, 8 * hkv * 128), dtype=torch.bfloat16, device="cuda")
    attention.launch(dev["qkv"].view(8 * b, -1), out, dev, dev["config"])
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    k_new, v_new = (dev[n].view(-1, hkv, 128).view(torch.uint8)[dev["cache_loc"]].cpu().view(torch.float8_e4m3fn) for n in ("k_cache", "v_cache"))
    # the largest error of up to 2e6 elements: the bound of tests/test_gpu_sinks.py beyond one wave
    close(out.cpu(), oattn.ref_stream(data, new_kv=(k_new, v_new))[0], f"{b} requests", atol=4e-2)
