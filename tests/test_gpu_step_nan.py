"""Single tokens and verify blocks: a NaN reaches every row that sees it and no other, whether it lies in a cached key or value,
in a query, or in a new token's key or value; the other rows keep their bits."""
import pytest
import torch

from oracle import attention as oattn

pytestmark = pytest.mark.gpu
SEQ, WINDOW = 200, 100


def make(q_len, sinks, window=WINDOW):
    data = oattn.make_input(2, [SEQ, 30], seed=q_len + sinks, q_len=q_len, hq=16, hkv=2, page=64, window=window)
    data["config"]["sinks"] = sinks
    return data


def run(data, chunks):
    """bf16 [2, q_len, 16 heads, 128] of the decode and verify kernels (a given number of chunks keeps blocks on them)."""
    from muse_spark_open_b200 import abi, attention
    out = attention.kernel_fn(oattn.to_device(data, "cuda"), chunks=chunks)
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    return out.cpu().view(2, data["config"]["q_len"], 16, 128)


def check(clean, out, bad):
    """`bad` bool [2, q_len, 16]: whole rows are NaN there, and nothing differs elsewhere."""
    assert torch.isfinite(clean.float()).all()
    assert torch.equal(torch.isnan(out.float()).all(-1), bad) and torch.equal(torch.isnan(out.float()).any(-1), bad)
    assert torch.equal(out[~bad].view(torch.int16), clean[~bad].view(torch.int16))


@pytest.mark.parametrize("what", ["k_cache", "v_cache"])
@pytest.mark.parametrize("q_len,sinks,chunks", [(1, 0, 1), (1, 3, 2), (1, 0, 4), (8, 0, 1), (8, 3, 1), (8, 3, 4), (8, 0, 2)])
def test_nan_in_the_cache(q_len, sinks, chunks, what):
    data = make(q_len, sinks)
    clean = run(data, chunks)
    for at in (0, 2, 3, 100, 101, 102, 104, 107, 108, 127, 128, 199):
        for channel in (0, 93):
            d = dict(data)
            d[what] = data[what].clone()
            d[what].view(torch.uint8)[int(data["page_table"][0, at // 64]), at % 64, 1, channel] = 0xFF
            bad = torch.zeros(2, q_len, 16, dtype=torch.bool)
            for j in range(q_len):
                bad[0, j, 8:] = at > SEQ + j - WINDOW or at < sinks
            check(clean, run(d, chunks), bad)


@pytest.mark.parametrize("q_len,window,sinks,chunks", [(1, 100, 0, 1), (1, 100, 3, 2), (8, 100, 0, 1), (8, 0, 0, 2), (8, 3, 0, 1), (8, 3, 201, 2), (8, 100, 3, 4)])
def test_nan_in_a_new_token(q_len, window, sinks, chunks):
    data = make(q_len, sinks, window)
    clean = run(data, chunks)
    for at in {0, q_len // 2, q_len - 1}:
        for column, own in ((5 * 128 + 7, True), (17 * 128 + 7, False), (19 * 128 + 7, False)):  # a query head, a key, a value
            d = dict(data, qkv=data["qkv"].clone())
            d["qkv"].view(2, q_len, -1)[0, at, column] = float("nan")
            bad = torch.zeros(2, q_len, 16, dtype=torch.bool)
            if own:
                bad[0, at, 5] = True
            else:
                for j in range(at, q_len):
                    bad[0, j, 8:] = not window or j - at < window or SEQ + at < sinks
            check(clean, run(d, chunks), bad)
