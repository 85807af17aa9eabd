"""Gated attention for single tokens and verify blocks with a sliding window and first tokens that stay visible (sinks),
against the 64-bit statement.  Every page that no token sees is taken out of the page table, and every cache position that
no token sees holds NaN bytes: they must be neither needed nor felt.

Tolerances: outputs are BF16 (half a step: 2^-8 of the value).  Queries enter the tensor cores as two E4M3 terms, off by at
most 2^-9 of their binade, 6e-4 rms; with scores of standard deviation 5.5 (norm 62 x 11.3 / sqrt(128)) that moves a score
by 0.0033 rms and a probability by the same share, so an output by about 0.3 % of its norm, and single elements by a few
times that: rtol 2e-2 / atol 1e-2 on elements as for every BF16 output of this framework, 6e-3 on the relative L2 norm."""
import pytest
import torch

from oracle import attention as oattn

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def streaming(data, sinks):
    """`data` with sinks, without the pages that no token sees, and with NaN bytes at every position no token sees."""
    cfg = data["config"]
    cfg["sinks"] = sinks
    w, size = cfg["window"], cfg["page_size"]
    table = data["page_table"]
    kc, vc = (data[n].view(torch.uint8).clone() for n in ("k_cache", "v_cache"))
    keep = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b, c in enumerate(data["seq_lens"].tolist()):
        lo = max(0, c - w + 1) if w else 0
        pos = torch.arange(c)
        pos = pos[(pos >= lo) | (pos < sinks)]
        keep[table[b].long()[pos // size], pos % size] = True
        for lp in range(table.shape[1]):
            if w and lp * size >= sinks and (lp + 1) * size <= lo:
                table[b, lp] = -1
    kc[~keep], vc[~keep] = 0x7F, 0x7F
    data["k_cache"], data["v_cache"] = kc.view(FP8), vc.view(FP8)
    return data


def run_step(data, **kw):
    from muse_spark_open_b200 import abi, attention
    dev = oattn.to_device(data, "cuda")
    out = attention.kernel_fn(dev, **kw)
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    hkv, d = data["config"]["num_kv_heads"], data["config"]["head_dim"]
    k_new, v_new = (dev[n].view(-1, hkv, d).view(torch.uint8)[dev["cache_loc"]].cpu().view(FP8) for n in ("k_cache", "v_cache"))
    return out.cpu(), k_new, v_new


def close(out, ref, what, atol=1e-2):
    out, ref = out.double().reshape(ref.shape), ref
    assert torch.isfinite(out).all(), what
    torch.testing.assert_close(out, ref, rtol=2e-2, atol=atol, msg=lambda m: f"{what}: {m}")
    err = float((out - ref).norm() / ref.norm())
    assert err < 6e-3, (what, err)


CASES = [
    # batch, seq_lens, q_len, window, sinks, page, chunks
    ("one", [1500], 1, 1024, 4, 64, 0),
    ("sinks_inside_the_window", [300, 1023], 1, 1024, 200, 64, 0),
    ("sinks_meet_the_window", [1151, 1152, 1153], 1, 1024, 128, 64, 2),
    ("many_sinks", [4000, 2500, 257], 1, 256, 257, 64, 0),
    ("sink_tile_edges", [2000, 2001, 2002], 1, 100, 128, 64, 4),
    ("one_sink", [700, 65, 0, 1], 1, 64, 1, 16, 8),
    ("window_of_one", [256, 255, 257, 1], 1, 1, 3, 64, 2),
    ("sinks_beyond_the_context", [50, 900], 1, 64, 5000, 64, 0),
    ("big_pages", [3000, 640], 1, 300, 5, 128, 0),
    ("small_pages", [3000, 640], 1, 300, 130, 8, 1),
    ("verify", [1500, 3000], 8, 1024, 4, 64, 0),
    ("verify_small_window", [400, 1000, 3], 8, 5, 2, 32, 2),
    ("verify_many_sinks", [2047, 129, 0], 8, 64, 300, 64, 4),
    ("verify_sinks_in_the_block", [2, 5], 8, 3, 6, 64, 1),
]


@pytest.mark.parametrize("name,seqs,q_len,window,sinks,page,chunks", CASES, ids=[c[0] for c in CASES])
def test_step_with_sinks(name, seqs, q_len, window, sinks, page, chunks):
    data = streaming(oattn.make_input(len(seqs), seqs, seed=len(name) + sinks, q_len=q_len, hq=16, hkv=2, page=page, window=window), sinks)
    out, k_new, v_new = run_step(data, chunks=chunks)
    ref, rk, rv = oattn.ref_stream(data)
    for got, want in ((k_new, rk), (v_new, rv)):
        assert (got.view(torch.uint8) != want.view(torch.uint8)).float().mean() < 5e-3, name
    close(out, oattn.ref_stream(data, new_kv=(k_new, v_new))[0], name)


@pytest.mark.parametrize("batch,hkv", [(80, 4), (300, 1), (37, 8), (150, 2), (111, 4)])
@pytest.mark.parametrize("window,sinks", [(200, 5), (700, 130)])
def test_steps_beyond_one_wave(batch, hkv, window, sinks):
    """More (request, head) pairs than the GPU holds at once: the last wave's contexts are split in two where they fill at most
    half of it; lengths from none to several windows, in any order.

    The largest error of 3e5 elements: two keys that share a row's weight move an output by p (1 - p) (e1 - e2) (v1 - v2), with
    e the scores' errors (each 0.0033 rms, so 0.0047 for the difference) and v of variance 1 (1.41), over the row's norm
    (0.71 per element at p = 1/2): at most 0.25 x 0.0047 x 1.41 / 0.71 = 0.0023 times a product of two standard normals.  Such
    a product passes 17 with probability 1e-8, so were all rows of that kind, 3e5 elements would pass 0.04 three times in a
    thousand runs (and 0.0127, as one here does, some hundred times in each).  A wrong row of the 5000 would move the relative
    L2 norm by 1.4e-2, against 6e-3."""
    g = torch.Generator().manual_seed(batch)
    seqs = torch.randint(0, 1400, (batch,), generator=g).tolist()
    seqs[3], seqs[7], seqs[11] = 0, 1, window
    data = streaming(oattn.make_input(batch, seqs, seed=batch, q_len=1, hq=8 * hkv, hkv=hkv, page=64, window=window), sinks)
    out, k_new, v_new = run_step(data)
    close(out, oattn.ref_stream(data, new_kv=(k_new, v_new))[0], f"{batch} requests", atol=4e-2)
    again = run_step(data)[0]
    assert torch.equal(out, again)


def test_no_sinks_is_what_it_was():
    """sinks = 0 and no `sinks` at all give the same bits; without a window sinks change nothing."""
    for window in (1024, 0):
        data = oattn.make_input(3, [1500, 70, 2900], seed=4, hq=8, hkv=1, window=window)
        base = run_step(data)[0]
        data["config"]["sinks"] = 0
        assert torch.equal(run_step(data)[0], base)
        if window == 0:
            data["config"]["sinks"] = 77
            assert torch.equal(run_step(data)[0], base)


def test_negative_sinks_and_windows_are_refused():
    from muse_spark_open_b200 import abi, attention
    data = oattn.to_device(oattn.make_input(1, [300], seed=3, hq=8, hkv=1), "cuda")
    for bad in ({"sinks": -1}, {"window": -5}):
        with pytest.raises(abi.MskError):
            attention.kernel_fn(dict(data, config=dict(data["config"], **bad)))


def test_layer_step_with_sinks():
    """The whole layer hands `sinks` to its attention: its result equals the one whose pages between the sinks and the
    window are gone, and differs from the step without sinks."""
    from muse_spark_open_b200 import abi, layer
    from oracle import layer as olayer
    weights = olayer.make_weights(3, hidden=1024, hq=8, hkv=1, d=128, n_experts=16, inner=128)
    data = olayer.make_input(3, [700, 1300, 5], 7, q_len=1, hidden=1024, hq=8, hkv=1, d=128, window=128, rope_theta=1e6)
    state = layer.prepare({k: v.cuda() for k, v in weights.items()})
    results = []
    for sinks, cut in ((0, False), (4, False), (4, True)):
        d = dict(data, config=dict(data["config"], sinks=sinks), page_table=data["page_table"].clone(), k_cache=data["k_cache"].clone(),
                 v_cache=data["v_cache"].clone())
        dev = oattn.to_device(streaming(d, sinks) if cut else d, "cuda")
        results.append(layer.kernel_fn(dev, state)[1].clone())
        torch.cuda.synchronize()
        abi.status_for("cuda").raise_if_set("layer")
    assert torch.equal(results[1], results[2])
    assert not torch.equal(results[0], results[1])
