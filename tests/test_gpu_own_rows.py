"""A request's outputs depend on nothing but the request: not on its neighbours in the batch, nor on what the workspace held in
the rows of a padded batch.  Bit for bit."""
import pytest
import torch

from oracle import attention as oattn
from test_gpu_prompt import make_prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ctx,new,pad", [([10, 200], [30, 55], 40), ([300], [5], 3), ([0, 77], [1, 70], 64)])
def test_a_padded_batch_does_not_feel_the_workspace(monkeypatch, ctx, new, pad):
    """The same call with a workspace of zeros, of large FP16 numbers, of NaN, and of small ones."""
    from muse_spark_open_b200 import abi, attention
    data = oattn.to_device(make_prompt(ctx, new, 5, window=100, sinks=4, pad=pad), "cuda")
    out = torch.empty((sum(new) + pad, 2048), dtype=torch.bfloat16, device="cuda")
    empty, seen, filled = torch.empty, [], []

    def with_bytes(*args, **kw):
        t = empty(*args, **kw)
        if t.dtype == torch.uint8:
            filled.append(t.fill_(byte).numel())
        return t

    monkeypatch.setattr(torch, "empty", with_bytes)
    for byte in (0x00, 0x7B, 0xFF, 0x5A):
        out.zero_()
        attention.prompt_fn(data, out=out)
        seen.append(out.clone())
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    assert len(filled) == 4 and all(torch.equal(seen[0], x) for x in seen[1:])


@pytest.mark.parametrize("window,sinks,splits", [(0, 0, 0), (64, 4, 0), (100, 9, 3)])
@pytest.mark.parametrize("ctx,new", [([300, 40, 0, 129], [70, 33, 5, 100]), ([300, 40, 0, 129], [7, 3, 5, 18])])
def test_a_request_at_every_place_of_the_batch(ctx, new, window, sinks, splits):
    from muse_spark_open_b200 import abi, attention
    data = make_prompt(ctx, new, 9, window=window, sinks=sinks)
    cu = data["cu_seqlens_q"].tolist()
    first = None
    for order in ([0, 1, 2, 3], [3, 2, 1, 0], [1, 3, 0, 2], [2, 0, 3, 1]):
        rows = torch.cat([torch.arange(cu[b], cu[b + 1]) for b in order])
        moved = dict(data, qkv=data["qkv"][rows], seq_lens=data["seq_lens"][order], page_table=data["page_table"][order].contiguous(),
                     cu_seqlens_q=torch.tensor([0, *torch.tensor([new[b] for b in order]).cumsum(0)], dtype=torch.int32))
        out = torch.empty((cu[-1], 2048), dtype=torch.bfloat16)
        out[rows] = attention.prompt_fn(oattn.to_device(moved, "cuda"), splits=splits).cpu()
        first = out if first is None else first
        assert torch.equal(out.view(torch.int16), first.view(torch.int16)), order
    abi.status_for("cuda").raise_if_set("attention")
