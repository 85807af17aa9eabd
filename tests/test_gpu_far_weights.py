"""Attention rows in which one key draws almost all of the weight and has a small value, as a first token often does: the
output is carried by thousands of keys whose weights lie 2^-14 to 2^-26 below the largest, and RMSNorm brings it back to size.

Every query head is a vector of equal magnitudes, s with its first m entries' signs flipped, so q . k0 for k0 along s falls
linearly with m: eight heads see key 0 from 16 down to 8 nats above the others.  New keys alternate against s in pairs, their
scores are zero for every head.  Queries are 5.4730 x (+-1), 0.004 from BF16's 5.46875 and 0.011 from the border of its step, so
no rounding falls the other way than in 64 bits.

Tolerances: those of tests/test_gpu_prompt.py without the allowance for queries (none differs): probabilities are off by 2^-12 of
their value, independently, or by half of FP16's smallest step, which for all keys together is 2^-20 (9.5e-7) of the largest
weight; a row is at least 0.002 of it (key 0's own value), so that is 5e-4 of the row.  The rest is the
output's rounding to BF16, 2^-8 of an element at most and 1.6e-3 rms: a row is off by 3e-3 of its norm at most, an element by
2^-7 of itself and 2e-3 (rows have elements of 0.7)."""
import pytest
import torch

from oracle import attention as oattn

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
K_SCALE, V_SCALE, D = 1.0 / 256, 1.0 / 64, 128


def far_weights(ctx, new, seed, window=0, sinks=0, nats=16.0, page=64):
    """One request per entry of ctx, `new` tokens each, one KV head; key 0 lies `nats` above the others for the first query head."""
    g = torch.Generator().manual_seed(seed)
    b = len(ctx)
    sign = torch.where(torch.rand(D, generator=g) < 0.5, -1.0, 1.0)
    heads = sign.repeat(8, 1)
    for h in range(8):
        heads[h, :4 * h] *= -1  # q_h . k0 = (1 - 8 h / 128) of head 0's
    alternate = sign * torch.tensor([1.0, -1.0]).repeat(D // 2)
    columns = (max(ctx) + new + page - 1) // page
    pages = b * columns
    table = torch.randperm(pages, generator=g).to(torch.int32).view(b, columns)
    k = 0.055 * torch.randn((pages, page, 1, D), generator=g)  # scores of 0.3 nats
    v = 0.5 + torch.randn((pages, page, 1, D), generator=g)
    unit = oattn.QK_SCALE_FACTOR * D * D ** -0.5  # q . s in units of the softmax's exponent
    for r in range(b):
        k[table[r, 0].long(), 0, 0] = nats / unit * sign
        v[table[r, 0].long(), 0, 0] *= 0.002
    qkv = torch.empty((b * new, 18 * D))
    qkv[:, :8 * D] = heads.reshape(-1)
    qkv[:, 8 * D:9 * D] = alternate
    qkv[:, 9 * D:10 * D] = 0.5 + torch.randn((b * new, D), generator=g)
    qkv[:, 10 * D:] = torch.randn((b * new, 8 * D), generator=g)
    pos = torch.tensor(ctx)[:, None] + torch.arange(new)
    cfg = {"batch": b, "q_len": new, "num_q_heads": 8, "num_kv_heads": 1, "head_dim": D, "page_size": page, "window": window, "sinks": sinks,
           "rope_theta": 0.0, "qk_scale_factor": oattn.QK_SCALE_FACTOR, "sm_scale": D ** -0.5}
    return {"qkv": qkv.to(torch.bfloat16), "k_cache": (k / K_SCALE).clamp(-448, 448).to(FP8), "v_cache": (v / V_SCALE).clamp(-448, 448).to(FP8),
            "k_scale": torch.tensor(K_SCALE), "v_scale": torch.tensor(V_SCALE), "page_table": table, "seq_lens": torch.tensor(ctx, dtype=torch.int32),
            "cu_seqlens_q": torch.arange(0, b * new + 1, new, dtype=torch.int32),
            "cache_loc": (torch.gather(table.long(), 1, pos // page) * page + pos % page).reshape(-1), "config": cfg}


def off(out, data):
    """(relative L2 of the worst row, largest excess over 2^-7 of an element) against the 64-bit statement."""
    ref = oattn.ref_stream(data)[0].view(-1, D)
    out = out.cpu().double().view(-1, D)
    assert torch.isfinite(out).all()
    return float(((out - ref).norm(dim=1) / ref.norm(dim=1)).max()), float(((out - ref).abs() - 2 ** -7 * ref.abs()).max())


@pytest.mark.parametrize("nats", [12.0, 16.0, 20.0])
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("new", [20, 40])  # single CTAs, and pairs
def test_prompt_keeps_the_weights_far_below_the_largest(new, splits, nats):
    from muse_spark_open_b200 import abi, attention
    data = far_weights([8192], new, 5, nats=nats)
    out = attention.prompt_fn(oattn.to_device(data, "cuda"), splits=splits)
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    row, element = off(out, data)
    assert row < 3e-3 and element < 2e-3, (row, element)


def test_prompt_with_a_first_token_that_stays_visible():
    """The same under a window, the first token a sink: its tile is the last one that is read."""
    from muse_spark_open_b200 import abi, attention
    for new, splits in ((20, 1), (40, 0)):
        data = far_weights([9000, 6000], new, 6, window=4096, sinks=4)
        out = attention.prompt_fn(oattn.to_device(data, "cuda"), splits=splits)
        torch.cuda.synchronize()
        abi.status_for("cuda").raise_if_set("attention")
        row, element = off(out, data)
        assert row < 3e-3 and element < 2e-3, (new, row, element)


@pytest.mark.parametrize("nats", [12.0, 16.0, 20.0])
@pytest.mark.parametrize("sinks", [4, 64, 300])
@pytest.mark.parametrize("q_len,chunks", [(1, 0), (1, 1), (8, 1), (8, 2)])
def test_steps_with_a_first_token_that_stays_visible(q_len, chunks, sinks, nats):
    """Single tokens and blocks on the verify kernel.  Their probabilities are two E4M3 terms, off by 2^-8 of their value at most and
    independently, so by nothing over thousands of keys, down to 2^-22 of the tile's largest.  Keys in the tile of key 0 may be
    lost: at most 127 of 4400, which carry at most a tenth of the output where they are (from 15 nats on), so 3e-3 of a row;
    with the rounding to BF16 5e-3.  An element of 0.7 may miss as much of itself, 3.5e-3, and that rounding."""
    from muse_spark_open_b200 import abi, attention
    data = far_weights([9000, 6000], q_len, 6, window=4096, sinks=sinks, nats=nats)
    out = attention.kernel_fn(oattn.to_device(data, "cuda"), chunks=chunks)
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    row, element = off(out, data)
    assert row < 5e-3 and element < 3.5e-3, (row, element)


@pytest.mark.parametrize("ctx,new", [(100, 5), (600, 40), (2000, 20), (66000, 20), (66000, 40)])
def test_prompt_keeps_them_at_any_length(ctx, new):
    """The rounding of the smallest probabilities, times the keys there are, is 2^-20 of the largest weight."""
    from muse_spark_open_b200 import abi, attention
    for nats in (12.0, 15.0, 18.0):
        data = far_weights([ctx], new, 7, nats=nats)
        for splits in (0, 1):
            out = attention.prompt_fn(oattn.to_device(data, "cuda"), splits=splits)
            torch.cuda.synchronize()
            abi.status_for("cuda").raise_if_set("attention")
            row, element = off(out, data)
            assert row < 3e-3 and element < 2e-3, (nats, splits, row, element)
