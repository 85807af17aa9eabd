"""cu_seqlens_q that names rows which are not there is reported; the requests in front of them are what they were."""
import pytest
import torch

from oracle import attention as oattn
from test_gpu_prompt import make_prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[30, 55, 8], [3, 9, 8]])  # pairs of CTAs, and single ones
@pytest.mark.parametrize("splits", [0, 1])
@pytest.mark.parametrize("what", ["beyond", "falls", "negative", "far beyond"])
def test_lists_that_do_not_fit_are_reported(new, splits, what):
    from muse_spark_open_b200 import abi, attention
    data = make_prompt([10, 200, 64], new, 5, window=100, sinks=4)
    good = attention.prompt_fn(oattn.to_device(data, "cuda"), splits=splits)
    a, b, c = (int(x) for x in data["cu_seqlens_q"][1:])
    cu = {"beyond": [0, a, b, c + 5], "falls": [0, a, b, b - 1], "negative": [-4, a, b, c], "far beyond": [0, a, b, 2 ** 31 - 1]}[what]
    out = torch.zeros_like(good)
    dev = oattn.to_device(dict(data, cu_seqlens_q=torch.tensor(cu, dtype=torch.int32)), "cuda")
    attention.prompt_fn(dev, out=out, splits=splits)
    torch.cuda.synchronize()
    with pytest.raises(abi.MskError, match="out of range in attn_prompt"):
        abi.status_for("cuda").raise_if_set("lists")
    same = {"negative": slice(a, b), "falls": slice(0, a)}.get(what, slice(0, b))
    assert torch.equal(out[same], good[same])


def test_many_requests_are_all_looked_at():
    from muse_spark_open_b200 import abi, attention
    data = make_prompt([5] * 70, [2] * 70, 3, hkv=1)
    for at in (0, 1, 33, 69):
        cu = data["cu_seqlens_q"].clone()
        cu[at + 1:] -= 3  # request `at` ends before it begins
        attention.prompt_fn(oattn.to_device(dict(data, cu_seqlens_q=cu), "cuda"))
        torch.cuda.synchronize()
        with pytest.raises(abi.MskError, match="out of range in attn_prompt"):
            abi.status_for("cuda").raise_if_set("lists")
    attention.prompt_fn(oattn.to_device(data, "cuda"))
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("lists")
