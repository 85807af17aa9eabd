"""The streaming operators where calls go wrong: graphs, streams, caches past 2^31 bytes, page ids and positions that do not
exist, blocks of every length."""
import pytest
import torch

from oracle import attention as oattn
from test_gpu_prompt import check, make_prompt, new_rows
from test_gpu_sinks import close, run_step, streaming

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("q_len", [2, 3, 7, 9, 16, 33, 70])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5)])
def test_blocks_of_every_length(q_len, window, sinks):
    data = oattn.make_input(3, [90, 0, 301], seed=q_len, q_len=q_len, hq=16, hkv=2, page=32, window=window)
    if sinks:
        data = streaming(data, sinks)
    out, k_new, v_new = run_step(data)
    close(out, oattn.ref_stream(data, new_kv=(k_new, v_new))[0], f"{q_len} tokens")


@pytest.mark.parametrize("batch,q_len", [(50, 8), (20, 40), (13, 2), (33, 3)])
@pytest.mark.parametrize("page", [8, 128])
def test_blocks_of_many_requests(batch, q_len, page):
    """Blocks in more units than the GPU has SMs (the prep kernel lists them) and in fewer (every CTA finds its own), alone and
    in pairs of CTAs."""
    seqs = [(37 * i) % 311 for i in range(batch)]
    data = streaming(oattn.make_input(batch, seqs, seed=batch, q_len=q_len, hq=32, hkv=4, page=page, window=60), 3)
    out, k_new, v_new = run_step(data)
    close(out, oattn.ref_stream(data, new_kv=(k_new, v_new))[0], f"{batch} x {q_len} tokens")


def test_prompt_in_a_graph_with_fresh_inputs():
    """Captured once, replayed with new inputs in the same buffers: bit for bit the eager call; two graphs do not share
    memory."""
    from muse_spark_open_b200 import abi, attention
    data = make_prompt([300, 0, 40], [70, 33, 5], 2, window=100, sinks=3)
    dev = oattn.to_device(data, "cuda")
    outs = [torch.empty((108, 2048), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        attention.prompt_fn(dev, out=outs[0])
        side.synchronize()
        for out in outs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                attention.prompt_fn(dev, out=out)
            graphs.append(g)
    torch.cuda.synchronize()
    gen = torch.Generator(device="cuda").manual_seed(5)
    for _ in range(3):
        dev["qkv"].copy_(2 * torch.randn(dev["qkv"].shape, generator=gen, device="cuda"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = attention.prompt_fn(dev)
        torch.cuda.synchronize()
        abi.status_for("cuda").raise_if_set("graph")
        assert torch.equal(got[0], want) and torch.equal(got[1], want)


def test_prompts_on_two_streams_at_once():
    from muse_spark_open_b200 import abi, attention
    cases = [oattn.to_device(make_prompt([200 * i, 0], [150, 60], i, window=64 * i, sinks=i), "cuda") for i in range(3)]
    want = [attention.prompt_fn(c).clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(attention.prompt_fn(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    abi.status_for("cuda").raise_if_set("streams")


def test_caches_past_two_gigabytes():
    """Pages beyond byte 2^31 of the cache: prompt, tokens, fork and compact."""
    from muse_spark_open_b200 import abi, attention, pages
    n, page, hkv = 70000, 64, 4
    kc, vc = (torch.zeros((n, page, hkv, 128), dtype=torch.uint8, device="cuda") for _ in range(2))
    pool = pages.prepare(n, page, 3, 8)
    pool["refs"][:69990] = 1  # the front is taken: new pages lie at the end
    rows = torch.tensor([1], dtype=torch.int32, device="cuda")
    data = make_prompt([0], [150], 4, hkv=hkv, window=40, sinks=3)
    dev = oattn.to_device(data, "cuda")
    pages.extend(pool, rows, 150)
    table = pool["page_table"][1:2, :3].contiguous()
    assert table.tolist() == [[69990, 69991, 69992]]
    small = {k: dev[k] for k in ("qkv", "k_scale", "v_scale", "seq_lens", "cu_seqlens_q", "config")}
    far = dict(small, k_cache=kc.view(FP8), v_cache=vc.view(FP8), page_table=table)
    out = attention.prompt_fn(far)
    near = dict(small, k_cache=torch.zeros((4, page, hkv, 128), dtype=torch.uint8, device="cuda").view(FP8),
                v_cache=torch.zeros((4, page, hkv, 128), dtype=torch.uint8, device="cuda").view(FP8),
                page_table=torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"))
    assert torch.equal(out, attention.prompt_fn(near))
    assert torch.equal(kc[69990:69993], near["k_cache"].view(torch.uint8)[:3])
    pool["seq_lens"][1] = 150
    pages.fork(pool, rows, torch.tensor([2], dtype=torch.int32, device="cuda"), [kc, vc])
    assert pool["page_table"][2, :3].tolist() == [69990, 69991, 69993]
    assert torch.equal(kc[69993, :22], kc[69992, :22]) and torch.equal(vc[69993, :22], vc[69992, :22])
    pool["refs"][:69990] = 0
    keep = kc[69990:69994].clone()
    assert pages.compact(pool, [kc, vc]).tolist() == [4, 4]
    assert pool["page_table"][1:, :3].tolist() == [[0, 1, 2], [0, 1, 3]] and torch.equal(kc[:4], keep)
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("far pages")


def test_page_ids_and_positions_that_do_not_exist():
    """Reported, not followed: a page id past the cache among the old positions or the new ones, a new position past the
    table."""
    from muse_spark_open_b200 import abi, attention
    for where, value in (((0, 0), 10 ** 6), ((0, 5), 10 ** 6), ((0, 0), -7)):
        data = make_prompt([300], [70], 6)
        data["page_table"][where] = value
        dev = oattn.to_device(data, "cuda")
        before = dev["k_cache"].view(torch.uint8).clone()
        attention.prompt_fn(dev)
        torch.cuda.synchronize()
        with pytest.raises(abi.MskError, match="out of range in attn_prompt"):
            abi.status_for("cuda").raise_if_set("bad page")
        bad = int((dev["k_cache"].view(torch.uint8) != before).flatten(2).any(2).sum())
        assert bad <= 70
    data = make_prompt([300], [70], 6)
    data["seq_lens"][0] = 350  # 70 tokens behind it end past the table's last page
    attention.prompt_fn(oattn.to_device(data, "cuda"))
    torch.cuda.synchronize()
    with pytest.raises(abi.MskError, match="out of range in attn_prompt"):
        abi.status_for("cuda").raise_if_set("past the table")


@pytest.mark.parametrize("seq", [2 ** 31 - 1, 2 ** 31 - 40, 10 ** 9, 500, -1, -500, -2 ** 31])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 0), (100, 2 ** 31 - 1), (2 ** 31 - 1, 7)])
def test_lengths_that_no_request_can_have(seq, window, sinks):
    """One request's length is nonsense: reported, at once, and the other requests are what they were."""
    from muse_spark_open_b200 import abi, attention
    for new in ([50, 40, 30], [9, 7, 8]):
        data = make_prompt([130, 60, 0], new, 12, hkv=1, window=window, sinks=sinks)
        good = attention.prompt_fn(oattn.to_device(data, "cuda"))
        data["seq_lens"][1] = seq
        out = attention.prompt_fn(oattn.to_device(data, "cuda"))
        torch.cuda.synchronize()
        with pytest.raises(abi.MskError, match="out of range in attn_prompt"):
            abi.status_for("cuda").raise_if_set("length")
        a, b = new[0], new[0] + new[1]
        assert torch.equal(out[:a], good[:a]) and torch.equal(out[b:], good[b:])


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("new", [40, 20])  # pairs of CTAs, and single ones
@pytest.mark.parametrize("at", [0, 1, 5, 6, 7, 38, 70, 127, 150])
def test_nan_in_a_visible_key_or_value_is_seen(at, new, splits):
    """A NaN byte in the cache reaches every row that sees it, wherever it lies in the tile, and no other."""
    from muse_spark_open_b200 import abi, attention
    for what in ("k_cache", "v_cache"):
        for channel in (17, 100):
            data = make_prompt([200], [new], 3, hkv=1, window=100)
            seen = [j for j in range(new) if 200 + j - 100 < at <= 200 + j]
            page = int(data["page_table"][0, at // 64])
            if page < 0:
                continue
            data[what].view(torch.uint8)[page, at % 64, 0, channel] = 0x7F
            out = attention.prompt_fn(oattn.to_device(data, "cuda"), splits=splits).cpu().view(new, -1)
            torch.cuda.synchronize()
            abi.status_for("cuda").raise_if_set("nan")
            bad = torch.isnan(out.float()).any(1).nonzero()[:, 0].tolist()
            assert bad == seen, (what, at)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 0), (20, 130), (300, 4)])
@pytest.mark.parametrize("new,at", [(150, 0), (150, 77), (150, 149), (30, 13), (30, 31 - 2)])
def test_a_spoilt_token_spoils_no_earlier_one(new, at, window, sinks, splits):
    """A new token with a NaN value: its own row and the later ones that see it become NaN, the others stay as they were."""
    from muse_spark_open_b200 import abi, attention
    data = make_prompt([90], [new], 8, hkv=1, window=window, sinks=sinks)
    clean = attention.prompt_fn(oattn.to_device(data, "cuda"), splits=splits).view(new, -1)
    data["qkv"][at, 9 * 128 + 70] = float("nan")
    out = attention.prompt_fn(oattn.to_device(data, "cuda"), splits=splits).view(new, -1)
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("nan")
    bad = torch.tensor([j >= at and (window == 0 or j - at < window or 90 + at < sinks) for j in range(new)], device="cuda")
    assert torch.isnan(out[bad].float()).all()
    assert torch.equal(out[~bad], clean[~bad])


def test_prompt_of_many_units_and_heads():
    """More units than SMs, in pairs and alone, with lengths that differ by far: every unit once."""
    for ctx, new in (([0] * 9, [700, 1, 64, 65, 300, 0, 129, 500, 33]), ([50] * 150, [1 + i % 7 for i in range(150)])):
        data = make_prompt(ctx, new, len(new), hkv=4, window=100, sinks=2)
        from muse_spark_open_b200 import abi, attention
        dev = oattn.to_device(data, "cuda")
        out = attention.prompt_fn(dev)
        torch.cuda.synchronize()
        abi.status_for("cuda").raise_if_set("many units")
        rows = new_rows(data)
        k_new, v_new = (dev[n].view(torch.uint8).cpu().view(-1, 4, 128)[rows].view(FP8) for n in ("k_cache", "v_cache"))
        check(data, out.cpu(), k_new, v_new, f"{len(new)} requests")
