"""Gated attention for prompts (any number of new tokens per request) against the 64-bit statement.  Pages no token sees are
missing from the page table; cache positions no token sees, and the rows the new tokens will be written to, hold NaN bytes.

Tolerances: queries and cache values enter the products exactly, probabilities as FP16 (off by 2^-12 of their value, so an
output row by about 2^-12 of its norm per key that matters), sums in FP32; the result is rounded to BF16 (2^-8 of an
element at most, 2^-8 / sqrt(3) x 0.7 = 1.6e-3 rms).  Elements: rtol 2^-7, atol 4e-3 (rows have norm-one elements times a
gate below 1); relative L2: 3e-3.

A query's rounding to BF16 can fall the other way than in 64 bits: the FP32 chain before it (norm, scale, turn) is off by
about 3 x 2^-24 of an element, a BF16 step is 2^-8 to 2^-7 of it, so 2 x 1.8e-7 / 5.5e-3 = 6.5e-5 of the elements, one row
in 120, has such an element.  Its step is 0.125 for an element in [16, 32) (queries have norm 62, elements of 5.5 rms),
which moves a score by 0.125 x |k| / 11.3, 0.044 at |k| = 4, probabilities by 4.4 % and a row, whose values may cancel to
a third of their norm before RMSNorm, by up to 0.13.  Most such elements are small and their rows stay inside the first
bound; 0.5 % of the rows may leave it, by no more than 0.13."""
import pytest
import torch

from oracle import attention as oattn

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def make_prompt(ctx, new, seed, hkv=2, page=64, window=0, sinks=0, theta=1e6, pad=0, wide=0):
    """Requests with ctx[b] cached and new[b] new tokens; `pad` rows behind the last one, `wide` columns beside qkv."""
    base = oattn.make_input(len(ctx), ctx, seed=seed, q_len=1, hq=8 * hkv, hkv=hkv, page=page, window=window, rope_theta=theta,
                            max_len=max(c + n for c, n in zip(ctx, new)))
    g = torch.Generator().manual_seed(seed + 1)
    t, d = sum(new), 128
    columns = max(1, (max(c + n for c, n in zip(ctx, new)) + page - 1) // page)
    lo = [max(0, c - window + 1) if window else 0 for c in ctx]
    need = [[lp for lp in range(columns) if lp * page < c + n and (lp * page < sinks or (lp + 1) * page > l)] for c, n, l in zip(ctx, new, lo)]
    total = sum(len(v) for v in need) + 2
    perm = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(ctx), columns), -1, dtype=torch.int32)
    at = 0
    for b, v in enumerate(need):
        for lp in v:
            table[b, lp] = perm[at]
            at += 1
    kv = torch.randn((2, total, page, hkv, d), generator=g)
    scale = [float(x.abs().amax()) / 448.0 for x in kv]
    caches = []
    for x, s in zip(kv, scale):
        c8 = oattn.quant_e4m3(x, s).view(torch.uint8)
        seen = torch.zeros(c8.shape[:2], dtype=torch.bool)
        for b, c in enumerate(ctx):
            pos = torch.arange(c)
            pos = pos[(pos >= lo[b]) | (pos < sinks)]
            seen[table[b].long()[pos // page], pos % page] = True
        c8[~seen] = 0x7F
        caches.append(c8.view(FP8))
    row = (2 * 8 * hkv + 2 * hkv) * d
    qkv = torch.randn((t + pad, row + wide), generator=g)
    qkv[:, :9 * hkv * d] *= 2
    qkv[t:] = float("nan")
    data = {"qkv": qkv.to(torch.bfloat16), "k_cache": caches[0], "v_cache": caches[1], "k_scale": torch.tensor(scale[0]), "v_scale": torch.tensor(scale[1]),
            "page_table": table, "seq_lens": torch.tensor(ctx, dtype=torch.int32),
            "cu_seqlens_q": torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32),
            "config": dict(base["config"], batch=len(ctx), sinks=sinks)}
    return data


def new_rows(data):
    """Flat cache rows of the new tokens."""
    page, cu, out = data["config"]["page_size"], data["cu_seqlens_q"].tolist(), []
    for b, c in enumerate(data["seq_lens"].tolist()):
        pos = torch.arange(c, c + cu[b + 1] - cu[b])
        out.append(data["page_table"][b].long()[pos // page] * page + pos % page)
    return torch.cat(out)


def run(data, **kw):
    from muse_spark_open_b200 import abi, attention
    dev = oattn.to_device(data, "cuda")
    out = attention.prompt_fn(dev, **kw)
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    hkv = data["config"]["num_kv_heads"]
    rows = new_rows(data)
    k_new, v_new = (dev[n].view(torch.uint8).cpu().view(-1, hkv, 128)[rows].view(FP8) for n in ("k_cache", "v_cache"))
    return out.cpu(), k_new, v_new, dev


def check(data, out, k_new, v_new, what):
    ref_data = dict(data, qkv=data["qkv"][:, :(18 * data["config"]["num_kv_heads"]) * 128].contiguous())
    _, rk, rv = oattn.ref_stream(ref_data)
    for got, want in ((k_new, rk), (v_new, rv)):
        assert (got.view(torch.uint8) != want.view(torch.uint8)).float().mean() < 2e-3, what
    ref = oattn.ref_stream(ref_data, new_kv=(k_new, v_new))[0]
    out = out.double()[:ref.shape[0]]
    assert torch.isfinite(out).all(), what
    off = (out - ref).abs()
    assert off.max() < 0.13, (what, float(off.max()))
    rows = (off > 4e-3 + 2 ** -7 * ref.abs()).view(-1, 128).any(1)
    assert int(rows.sum()) <= max(1, 0.005 * rows.numel()), (what, int(rows.sum()), rows.numel())
    err = float((out - ref).norm() / ref.norm())
    assert err < 3e-3, (what, err)


CASES = [
    # name, cached, new, window, sinks, page
    ("one_token", [0], [1], 0, 0, 64),
    ("one_tile", [0], [16], 0, 0, 64),
    ("unit_edges", [0, 0, 0], [31, 32, 33], 0, 0, 64),
    ("key_tile_edges", [0, 1, 95, 96, 97], [127, 128, 33, 32, 31], 0, 0, 64),
    ("behind_a_context", [700, 129, 3], [40, 17, 200], 0, 0, 64),
    ("empty_requests", [5, 0, 300, 7], [0, 20, 0, 3], 0, 0, 64),
    ("window", [1500, 0], [70, 300], 200, 0, 64),
    ("window_and_sinks", [1500, 0, 100], [70, 400, 60], 200, 4, 64),
    ("window_of_one", [130, 0], [40, 129], 1, 0, 32),
    ("window_of_one_and_sinks", [130, 0], [40, 129], 1, 3, 32),
    ("many_sinks", [900, 0], [33, 600], 100, 300, 128),
    ("sinks_at_a_tile_edge", [1000, 0], [33, 500], 64, 128, 16),
    ("small_pages", [333], [222], 150, 9, 8),
    ("long", [0], [1100], 0, 0, 64),
    ("many_requests", list(range(0, 360, 9)), [1 + (7 * i) % 23 for i in range(40)], 64, 2, 16),
]


@pytest.mark.parametrize("name,ctx,new,window,sinks,page", CASES, ids=[c[0] for c in CASES])
def test_prompt(name, ctx, new, window, sinks, page):
    data = make_prompt(ctx, new, len(name), window=window, sinks=sinks, page=page)
    out, k_new, v_new, _ = run(data)
    check(data, out, k_new, v_new, name)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
def test_prompt_splits(splits):
    """Keys split over CTAs, more ways than there are tiles among them: some splits are empty."""
    data = make_prompt([900, 10, 300], [20, 40, 1], 3, window=300, sinks=5)
    out, k_new, v_new, _ = run(data, splits=splits)
    check(data, out, k_new, v_new, f"splits {splits}")


@pytest.mark.parametrize("hkv,theta", [(1, 0.0), (4, 1e4), (8, 1e6)])
def test_prompt_heads_and_rope(hkv, theta):
    data = make_prompt([64, 300], [130, 5], hkv, hkv=hkv, theta=theta, window=128, sinks=1)
    out, k_new, v_new, _ = run(data)
    check(data, out, k_new, v_new, f"{hkv} heads")


def test_prompt_rows_behind_the_last_request_stay():
    """A padded batch: rows behind the last request (NaN inputs) are neither read nor written, qkv and out have wider rows."""
    data = make_prompt([10, 200], [30, 55], 5, window=100, sinks=4, pad=40, wide=256)
    dev = oattn.to_device(data, "cuda")
    whole = torch.full((125, 16 * 128 + 64), 7.0, dtype=torch.bfloat16, device="cuda")
    from muse_spark_open_b200 import abi, attention
    attention.prompt_fn(dev, out=whole[:, :2048])
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    assert (whole[85:] == 7.0).all() and (whole[:, 2048:] == 7.0).all()
    rows = new_rows(data)
    k_new, v_new = (dev[n].view(torch.uint8).cpu().view(-1, 2, 128)[rows].view(FP8) for n in ("k_cache", "v_cache"))
    check(data, whole[:85, :2048].cpu(), k_new, v_new, "padded")


@pytest.mark.parametrize("ctx", [0, 20000])
def test_prompt_keys_are_rounded_once(ctx):
    """The cached keys and values are the 64-bit formula's, byte for byte, at far positions too."""
    data = make_prompt([ctx], [700], 21, window=100, sinks=3)
    _, k_new, v_new, _ = run(data)
    cfg = data["config"]
    q, k, v, _ = data["qkv"].double().split([16 * 128, 2 * 128, 2 * 128, 16 * 128], 1)
    k, v = k.reshape(700, 2, 128), v.reshape(700, 2, 128)
    k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + 1e-5)
    freq = (1.0 / (cfg["rope_theta"] ** (torch.arange(0, 128, 2).float() / 128))).double()
    ang = (ctx + torch.arange(700).double())[:, None, None] * freq
    a, b = k[..., 0::2], k[..., 1::2]
    k = torch.stack((a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()), -1).flatten(-2)
    for got, want in ((k_new, k / data["k_scale"].double()), (v_new, v / data["v_scale"].double())):
        want = want.clamp(-448, 448).float().to(FP8).view(torch.uint8)
        assert torch.equal(got.view(torch.uint8).view(want.shape), want)


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("new", [20, 90])
def test_prompt_rows_that_start_on_16_bytes_only(new, splits):
    """Rows of qkv and out that lie at odd multiples of 16 bytes: the same bits as at 32."""
    from muse_spark_open_b200 import abi, attention
    data = make_prompt([150], [new], 15, window=70, sinks=2, wide=8)
    dev = oattn.to_device(data, "cuda")
    want = attention.prompt_fn(dict(dev, qkv=dev["qkv"][:, :-8].contiguous()), splits=splits)
    for width, at in ((2048 + 8, 0), (2048 + 24, 8), (2048 + 16, 8)):
        whole = torch.full((new, width), 7.0, dtype=torch.bfloat16, device="cuda")
        attention.prompt_fn(dev, out=whole[:, at:at + 2048], splits=splits)
        torch.cuda.synchronize()
        abi.status_for("cuda").raise_if_set("attention")
        assert torch.equal(whole[:, at:at + 2048], want)
        assert (whole[:, :at] == 7.0).all() and (whole[:, at + 2048:] == 7.0).all()


def test_prompt_leaves_other_pages_alone_and_replays_bitwise():
    data = make_prompt([100, 0, 77], [65, 33, 1], 6)
    before = data["k_cache"].view(torch.uint8).clone()
    out, _, _, dev = run(data)
    again = run(data)[0]
    assert torch.equal(out, again)
    after = dev["k_cache"].view(torch.uint8).cpu()
    rows = new_rows(data)
    keep = torch.ones(before.shape[0] * before.shape[1], dtype=torch.bool)
    keep[rows] = False
    assert torch.equal(before.view(-1, 256)[keep], after.view(-1, 256)[keep])


def test_prompt_then_tokens_is_one_prompt():
    """A prompt in two pieces, then single tokens, against the whole prompt at once: what the cache holds and the last rows."""
    from muse_spark_open_b200 import abi, attention
    data = make_prompt([0], [150], 8, window=64, sinks=4)
    whole, _, _, dev = run(data)
    parts = oattn.to_device(data, "cuda")
    outs, at = [], 0
    for n in (70, 77):
        piece = dict(parts, qkv=parts["qkv"][at:at + n], seq_lens=torch.tensor([at], dtype=torch.int32, device="cuda"),
                     cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
        outs.append(attention.prompt_fn(piece))
        at += n
    for t in range(at, 150):
        table = data["page_table"][0].long()
        step = dict(parts, qkv=parts["qkv"][t:t + 1].view(1, 1, -1), seq_lens=torch.tensor([t], dtype=torch.int32, device="cuda"),
                    cache_loc=(table[t // 64] * 64 + t % 64).view(1).cuda(), config=dict(data["config"], q_len=1))
        outs.append(attention.kernel_fn(step)[0])
    got = torch.cat(outs).cpu()
    torch.cuda.synchronize()
    abi.status_for("cuda").raise_if_set("attention")
    same = (parts["k_cache"].view(torch.uint8) == dev["k_cache"].view(torch.uint8)).float().mean()
    assert same > 0.999
    torch.testing.assert_close(got.float(), whole.float(), rtol=2e-2, atol=2e-2)


def test_prompt_reports_a_missing_page():
    """A new token without a page is reported and not written; the rest of the call runs."""
    from muse_spark_open_b200 import abi, attention
    data = make_prompt([0, 0], [70, 40], 9)
    data["page_table"][0, 1] = -1
    dev = oattn.to_device(data, "cuda")
    out = attention.prompt_fn(dev)
    torch.cuda.synchronize()
    with pytest.raises(abi.MskError, match="out of range in attn_prompt"):
        abi.status_for("cuda").raise_if_set("attention")
    assert torch.isfinite(out[70:].float()).all()
