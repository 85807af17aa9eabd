"""Cases for the operators of a streaming cache: gated attention with a sliding window and first tokens that stay visible
(single tokens and verify blocks; whole prompts), and the pages of the FP8 cache it reads (fork, extend, free, trim, compact).

Attention, for a request with c tokens in the cache and n new ones, new token j at position t = c + j:
  q = bf16(rope(rms(q_in) * qk_scale_factor, t)),  k = e4m3(rope(rms(k_in), t) / k_scale),  v = e4m3(v_in / v_scale)
  token j sees position s when s <= t and (window == 0 or s > t - window or s < sinks)
  o = softmax(q . (k * k_scale) * sm_scale) (v * v_scale) per head (8 query heads share a key head)
  out = bf16(rms(o) * sigmoid(gate)); the new k and v are written into the cache pages that the page table names.
Pages: `refs[p]` counts the page-table entries that name page p; a page is free when it is 0; new pages are the lowest free
ones, given out in the order of the rows.
"""
import math
import random

import torch

own = False

D, GROUP = 128, 8
FP8 = torch.float8_e4m3fn
EPS = 1e-5
QK = 5.4730064863875


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one user's next token: latency
        _step("token_1", 1, 1, 1500, 1500, 1024, 4, 1, 64),
        # the decode batch of the attention benchmark, with four first tokens kept visible
        _step("tokens_16", 16, 1, 1024, 8192, 1024, 4, 2, 64),
        # eight draft tokens for each of 16 requests
        _step("verify_16", 16, 8, 1024, 8192, 1024, 4, 3, 64),
        # the serving batch of the layer benchmark under a long window: bound by the cache's bytes
        _step("tokens_256", 256, 1, 2048, 16384, 4096, 64, 4, 64),
        # a short question after a long cached conversation
        _prompt("prompt_followup", 1, 19, 19, 7001, 7001, 1024, 4, 5, 64),
        # a mixed batch: prompts of 1 to 1024 tokens behind 0 to 4096 cached ones
        _prompt("prompt_mixed", 16, 1, 1024, 0, 4096, 1024, 4, 6, 64),
        # three long documents under window and sinks
        _prompt("prompt_window", 3, 2500, 4099, 0, 1000, 1024, 64, 7, 64),
        # one document with every earlier token visible: bound by the tensor cores
        _prompt("prompt_full", 1, 8192, 8192, 0, 0, 0, 0, 8, 64),
        # four conversations, two candidate continuations each, one token
        _branch("branch_4x2", 4, 2, 1024, 8192, 1, 1, 9, 64),
        # 64 conversations with three branches of eight draft tokens, a cache of four layers
        _branch("branch_64x3", 64, 3, 1024, 4096, 8, 4, 10, 64),
        # a small server between two bursts: half the requests gone
        _compact("compact_8", 8, 4, 1024, 8192, 1024, 4, 1, 11, 64),
        # a full server: 128 requests, 64 leave, the others keep their window and sinks or everything
        _compact("compact_128", 128, 64, 2048, 16384, 4096, 64, 2, 12, 64),
    ]


def _step(name, batch, q_len, ctx_lo, ctx_hi, window, sinks, lens, page, hkv=4, theta=1e6):
    return _named(name, {"kind": "step", "batch": batch, "q_len": q_len, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "window": window, "sinks": sinks,
                         "lens": lens, "page": page, "hkv": hkv, "theta": theta})


def _prompt(name, batch, new_lo, new_hi, ctx_lo, ctx_hi, window, sinks, lens, page, hkv=4, theta=1e6):
    return _named(name, {"kind": "prompt", "batch": batch, "new_lo": new_lo, "new_hi": new_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "window": window,
                         "sinks": sinks, "lens": lens, "page": page, "hkv": hkv, "theta": theta})


def _branch(name, parents, fan, ctx_lo, ctx_hi, q_len, layers, lens, page, hkv=4):
    return _named(name, {"kind": "branch", "parents": parents, "fan": fan, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "q_len": q_len, "layers": layers,
                         "lens": lens, "page": page, "hkv": hkv})


def _compact(name, requests, gone, ctx_lo, ctx_hi, window, sinks, layers, lens, page, hkv=4):
    return _named(name, {"kind": "compact", "requests": requests, "gone": gone, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "window": window, "sinks": sinks,
                         "layers": layers, "lens": lens, "page": page, "hkv": hkv})


def _named(name, case):
    return {"name": name, **case} if name else case


def _log(rng, lo, hi):
    """A whole number between lo and hi (lo >= 1), spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["step", "step", "prompt", "prompt", "branch", "compact"])
    page, lens = rng.choice([16, 32, 64, 128]), rng.randrange(100, 1 << 30)
    hkv = rng.choice([1, 2, 4, 8])
    window = rng.choice([0, _log(rng, 48, 4096), _log(rng, 48, 4096)])
    sinks = rng.choice([0, rng.randrange(1, 9), rng.randrange(9, 257)])
    if kind == "step":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, 16384 if window else max(64, min(16384, 1000000 // batch)))
        hkv = min(hkv, 4) if batch > 64 else hkv
        return _step(None, batch, rng.choice([1, 1, 8]), rng.randrange(0, hi + 1), hi, window, sinks, lens, page, hkv, rng.choice([0.0, 1e4, 1e6]))
    if kind == "prompt":
        batch, new, ctx = _log(rng, 1, 16), _log(rng, 1, 4096), rng.choice([0, _log(rng, 1, 8192)])
        hkv = min(hkv, 4)
        while batch * hkv * GROUP * new * (new + ctx) > 2.1e9:
            if batch > 1:
                batch = batch // 2
            elif ctx > new:
                ctx = ctx // 2
            else:
                new = new - new // 4
        return _prompt(None, batch, rng.randrange(1, new + 1), new, rng.randrange(0, ctx + 1), ctx, window, sinks, lens, page, hkv, rng.choice([0.0, 1e4, 1e6]))
    if kind == "branch":
        parents = _log(rng, 1, 64)
        hi = _log(rng, 16, 4096)
        return _branch(None, parents, rng.randrange(1, 5), rng.randrange(1, hi + 1), hi, _log(rng, 1, 300), rng.randrange(1, 5), lens, page, min(hkv, 4))
    n = _log(rng, 2, 128)
    hi = _log(rng, 64, 8192)
    return _compact(None, n, rng.randrange(1, n + 1), rng.randrange(1, hi + 1), hi, window, sinks, rng.randrange(1, 3), lens, page, min(hkv, 4))


def _lens(case):
    """The lengths of a case: cached tokens of each request, and new ones."""
    r = random.Random(case["lens"])
    n = case.get("batch") or case.get("parents") or case.get("requests")
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(n)]
    if case["kind"] == "prompt":
        new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
    else:
        new = [case.get("q_len", 0)] * n
    return ctx, new


# ------------------------------------------------------------------------------------------------------------ inputs
def _randn(seed, shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * scale


def _cache(seed, pages, page, hkv):
    """(values e4m3 [pages, page, hkv, 128], scale): N(0, 1) under one scale, its largest value at 448."""
    x = _randn(seed, (pages, page, hkv, D))
    scale = x.abs().amax() / 448.0
    return x.div_(scale).clamp_(-448.0, 448.0).to(FP8), scale.float()


def _table(seed, spans, columns, page, spare):
    """int32 [rows, columns] page table with pages in scattered order, -1 where a row has none; and how many pages there are.
    `spans`: for each row the positions it holds, as two ranges [0, a) and [b, c)."""
    a, b, c = (torch.tensor(v, device="cuda")[:, None] for v in zip(*spans))
    at = torch.arange(columns, device="cuda")[None, :] * page
    held = (at < a) | ((at + page > b) & (at < c))
    count = int(held.sum())
    g = torch.Generator(device="cuda").manual_seed(seed)
    perm = torch.randperm(count + spare, generator=g, device="cuda").to(torch.int32)
    order = torch.cumsum(held.reshape(-1).to(torch.int64), 0).reshape(held.shape) - 1
    return torch.where(held, perm[order.clamp(min=0)], torch.full_like(perm[:1], -1)).contiguous(), count + spare


def prepare(case, seed):
    ctx, new = _lens(case)
    page, hkv = case["page"], case["hkv"]
    if case["kind"] in ("step", "prompt"):
        b, w, sinks = len(ctx), case["window"], case["sinks"]
        # what a server with this window keeps: the sinks' pages, the window's, and room for the new tokens
        spans = [(min(sinks, c), max(0, c - w + 1) if w else 0, c + n) for c, n in zip(ctx, new)]
        columns = -(-max(c + n for c, n in zip(ctx, new)) // page)
        table, pages = _table(seed * 11 + 1, spans, columns, page, 3)
        kc, ks = _cache(seed * 11 + 2, pages, page, hkv)
        vc, vs = _cache(seed * 11 + 3, pages, page, hkv)
        t = sum(new)
        wide = 2 * hkv * GROUP + 2 * hkv
        qkv = _randn(seed * 11 + 4, (t, wide * D))
        qkv[:, :(hkv * GROUP + hkv) * D] *= 2.0  # queries and keys ~ 2N, values and gates ~ N
        qkv = qkv.to(torch.bfloat16)
        cu = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
        seq = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        cfg = {"batch": b, "num_q_heads": hkv * GROUP, "num_kv_heads": hkv, "head_dim": D, "page_size": page, "window": w, "sinks": sinks,
               "rope_theta": case["theta"], "qk_scale_factor": QK, "sm_scale": D ** -0.5}
        data = {"qkv": qkv, "seq_lens": seq, "page_table": table, "k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs, "config": cfg}
        if case["kind"] == "step":
            cfg["q_len"] = case["q_len"]
            pos = (seq.long()[:, None] + torch.arange(case["q_len"], device="cuda")[None, :])
            data["cache_loc"] = (torch.gather(table.long(), 1, pos // page) * page + pos % page).reshape(-1)
            data["qkv"] = qkv.view(b, case["q_len"], -1)
        else:
            data["cu_seqlens_q"] = cu
        return {"case": case, "data": data, "ctx": ctx, "new": new}
    n = len(ctx)
    if case["kind"] == "branch":
        rows, q = n * (1 + case["fan"]), case["q_len"]
        columns = (case["ctx_hi"] + q) // page + 1
        spans = [(0, 0, c) for c in ctx] + [(0, 0, 0)] * (n * case["fan"])
        spare = n * case["fan"] * (2 + q // page) + 5
    else:
        rows, columns = n, (case["ctx_hi"] - 1) // page + 1
        spans, spare = [(0, 0, c) for c in ctx], 5
    table, pages = _table(seed * 11 + 1, spans, columns, page, spare)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[table[table >= 0].long()] = 1
    seq = torch.tensor(ctx + [0] * (rows - n), dtype=torch.int32, device="cuda")
    every = torch.empty((2 * case["layers"], pages, page, hkv, D), dtype=FP8, device="cuda")
    for i in range(2 * case["layers"]):
        every[i] = _cache(seed * 11 + 2 + i, pages, page, hkv)[0]
    pool = {"page_table": table, "seq_lens": seq, "refs": refs, "page_size": page}
    state = {"case": case, "pool": pool, "every": every, "caches": list(every.unbind(0)), "ctx": ctx}
    if case["kind"] == "branch":
        parents = torch.arange(n, dtype=torch.int32, device="cuda").repeat_interleave(case["fan"])
        order = torch.randperm(n * case["fan"], generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
        state["parents"] = parents[order].contiguous()  # branches come in any order
        state["children"] = torch.arange(n, rows, dtype=torch.int32, device="cuda")
    else:
        order = torch.randperm(n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(torch.int32)
        state["gone"], state["kept"] = order[:case["gone"]].contiguous(), order[case["gone"]:].contiguous()
        state["was"] = {k: pool[k].clone() for k in ("page_table", "seq_lens", "refs")}
    return state


# -------------------------------------------------------------------------------------------------------------- runs
def run(state):
    kind = state["case"]["kind"]
    if kind == "step":
        return _run_step(state)
    if kind == "prompt":
        return _run_prompt(state)
    if kind == "branch":
        return _run_branch(state)
    return _run_compact(state)


def _run_step(state):
    data = state["data"]
    if own:
        from muse_spark_open_b200 import attention
        out = attention.kernel_fn(data)
    else:
        b, q = data["config"]["batch"], data["config"]["q_len"]
        out = _plain_attention(data, data["qkv"].reshape(b * q, -1), [q] * b, state["ctx"]).view(b, q, -1)
    return {"out": out, "k_cache": data["k_cache"], "v_cache": data["v_cache"]}


def _run_prompt(state):
    data = state["data"]
    if own:
        from muse_spark_open_b200 import attention
        out = attention.prompt_fn(data)
    else:
        out = _plain_attention(data, data["qkv"], state["new"], state["ctx"])
    return {"out": out, "k_cache": data["k_cache"], "v_cache": data["v_cache"]}


def _run_branch(state):
    """Drop the last branches, branch again, make room for the next tokens: a user's loop over candidate continuations."""
    pool, parents, children, q = state["pool"], state["parents"], state["children"], state["case"]["q_len"]
    if own:
        from muse_spark_open_b200 import pages
        pages.free(pool, children)
        pages.fork(pool, parents, children, state["caches"])
        loc = pages.extend(pool, children, q)
    else:
        _plain_free(pool, children)
        _plain_fork(pool, parents, children, state["every"])
        loc = _plain_extend(pool, children, q)
    return {"cache_loc": loc, **_of(pool), "caches": state["caches"]}


def _run_compact(state):
    """Requests leave, the others give back what their window has passed, and the pages in use move to the front."""
    pool, case = state["pool"], state["case"]
    was = state["was"]  # the requests that were there before
    pool["page_table"].copy_(was["page_table"])
    pool["seq_lens"].copy_(was["seq_lens"])
    pool["refs"].copy_(was["refs"])
    if own:
        from muse_spark_open_b200 import pages
        pages.free(pool, state["gone"])
        pages.trim(pool, state["kept"], case["window"], case["sinks"])
        pages.compact(pool, state["caches"])
    else:
        _plain_free(pool, state["gone"])
        _plain_trim(pool, state["kept"], case["window"], case["sinks"])
        _plain_compact(pool, state["every"])
    return {**_of(pool), "caches": state["caches"]}


def _of(pool):
    return {k: pool[k] for k in ("page_table", "seq_lens", "refs")}


# ------------------------------------------------------------------------------------------------------- plain forms
def _rms(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _rope(x, pos, theta):
    """Pairs (2i, 2i + 1) of the last axis turn by pos * theta^(-2i/128); x [tokens, heads, 128], the angles in 64 bits."""
    if not theta:
        return x
    freq = (1.0 / (theta ** (torch.arange(0, D, 2).float() / D))).to(x.device)
    ang = pos.double()[:, None, None] * freq.double()
    c, s = ang.cos().to(x.dtype), ang.sin().to(x.dtype)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _e4m3(x, scale):
    return (x / scale).clamp(-448.0, 448.0).to(FP8)


def _plain_attention(data, qkv, new, ctx):
    """All requests at once, padded to the most new tokens and, per request, to the positions that any of them sees."""
    cfg = data["config"]
    hkv, hq, page, w, sinks = cfg["num_kv_heads"], cfg["num_q_heads"], cfg["page_size"], cfg["window"], cfg["sinks"]
    dev, table = qkv.device, data["page_table"].long()
    b, most = len(new), max(new)
    n, c = torch.tensor(new, device=dev), data["seq_lens"].long()
    first = torch.cumsum(n, 0) - n
    req = torch.repeat_interleave(torch.arange(b, device=dev), n, output_size=sum(new))
    pos = c[req] + torch.arange(sum(new), device=dev) - first[req]
    q, k, v, gate = qkv.split([hq * D, hkv * D, hkv * D, hq * D], -1)
    q = _rope(_rms(q.double().view(-1, hq, D)) * cfg["qk_scale_factor"], pos, cfg["rope_theta"]).float().to(torch.bfloat16).float()
    k = _rope(_rms(k.double().view(-1, hkv, D)), pos, cfg["rope_theta"])
    row = torch.gather(table[req], 1, (pos // page)[:, None])[:, 0] * page + pos % page
    data["k_cache"].view(-1, hkv, D)[row] = _e4m3(k, data["k_scale"].double())
    data["v_cache"].view(-1, hkv, D)[row] = _e4m3(v.float().view(-1, hkv, D), data["v_scale"])
    # the positions that count for a request: the sinks before its window, then everything from the window's start
    low = [max(0, x - w + 1) if w else 0 for x in ctx]
    front = min(sinks, max(low)) if w else 0
    span = max(x + m - l for x, m, l in zip(ctx, new, low))
    low = torch.tensor(low, device=dev)[:, None]
    at = torch.cat([torch.arange(front, device=dev)[None, :].expand(b, -1), low + torch.arange(span, device=dev)[None, :]], 1)
    real = torch.cat([torch.arange(front, device=dev)[None, :] < low, torch.ones((b, span), dtype=torch.bool, device=dev)], 1)
    held = torch.gather(table, 1, (at // page).clamp(max=table.shape[1] - 1)).clamp(min=0) * page + at % page
    keys = data["k_cache"].view(-1, hkv, D)[held].float() * data["k_scale"]
    vals = data["v_cache"].view(-1, hkv, D)[held].float() * data["v_scale"]
    slot = (first[:, None] + torch.arange(most, device=dev)[None, :].clamp(max=most - 1)).clamp(max=sum(new) - 1)  # [b, most]
    t = c[:, None, None] + torch.arange(most, device=dev)[None, :, None]
    s = at[:, None, :]
    sees = real[:, None, :] & (s <= t)
    if w:
        sees = sees & ((s > t - w) | (s < sinks))
    qb = q[slot].view(b, most, hkv, GROUP, D).permute(0, 2, 3, 1, 4).reshape(b, hkv, GROUP * most, D)
    sc = torch.matmul(qb, keys.permute(0, 2, 3, 1)).view(b, hkv, GROUP, most, -1).mul_(cfg["sm_scale"])
    vals = vals.masked_fill(~sees.any(1)[:, :, None, None], 0.0)
    sc.masked_fill_(~sees[:, None, None], -math.inf)
    sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    total = sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.view(b, hkv, GROUP * most, -1), vals.permute(0, 2, 1, 3)).view(b, hkv, GROUP, most, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(b * most, hq, D)
    j = torch.arange(sum(new), device=dev) - first[req]
    o = o[req * most + j]
    return (_rms(o) * torch.sigmoid(gate.float().view(-1, hq, D))).view(-1, hq * D).to(torch.bfloat16)


def _plain_free(pool, rows):
    r = rows.long()
    ids = pool["page_table"][r]
    pool["refs"].index_add_(0, ids.clamp(min=0).reshape(-1).long(), -(ids >= 0).reshape(-1).to(torch.int32))
    pool["page_table"][r] = -1
    pool["seq_lens"][r] = 0


def _free_pages(refs):
    """The free pages in rising order, in a list as long as there are pages."""
    is_free = refs == 0
    rank = torch.where(is_free, torch.cumsum(is_free.long(), 0) - 1, torch.full_like(refs, refs.numel(), dtype=torch.int64))
    found = torch.full((refs.numel() + 1,), -1, dtype=torch.int64, device=refs.device)
    found.scatter_(0, rank, torch.arange(refs.numel(), device=refs.device))
    return found


def _plain_fork(pool, parents, children, every):
    table, page = pool["page_table"], pool["page_size"]
    p, c = parents.long(), children.long()
    seq = pool["seq_lens"][p].long()
    part, last = seq % page, seq // page
    need = part > 0
    fresh = torch.where(need, _free_pages(pool["refs"])[torch.cumsum(need.long(), 0) - 1], torch.full_like(seq, -1))
    cols = torch.arange(table.shape[1], device=table.device)[None, :]
    held = table[p]
    src = torch.gather(held, 1, last.clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    shared = torch.where(cols < last[:, None], held, torch.full_like(held, -1))
    table[c] = torch.where((cols == last[:, None]) & need[:, None], fresh[:, None].to(torch.int32), shared)
    pool["refs"].index_add_(0, shared.clamp(min=0).reshape(-1).long(), (shared >= 0).reshape(-1).to(torch.int32))
    pool["seq_lens"][c] = seq.to(torch.int32)
    src, fresh, part = src[need], fresh[need], part[need]
    pool["refs"][fresh] = 1
    used = (torch.arange(page, device=table.device)[None, :] < part[:, None])[None, :, :, None, None]
    as_bytes = every.view(torch.uint8)
    as_bytes[:, fresh] = torch.where(used, as_bytes[:, src], as_bytes[:, fresh])


def _plain_extend(pool, rows, q_len):
    table, page = pool["page_table"], pool["page_size"]
    r = rows.long()
    seq = pool["seq_lens"][r].long()
    cols = torch.arange(table.shape[1], device=table.device)[None, :]
    held = table[r]
    want = (cols >= (seq // page)[:, None]) & (cols <= ((seq + q_len - 1) // page)[:, None]) & (held < 0)
    rank = torch.cumsum(want.reshape(-1).long(), 0).view(want.shape) - 1
    held = torch.where(want, _free_pages(pool["refs"])[rank.clamp(min=0)].to(torch.int32), held)
    table[r] = held
    pool["refs"].index_add_(0, held.clamp(min=0).reshape(-1).long(), want.reshape(-1).to(torch.int32))
    pos = seq[:, None] + torch.arange(q_len, device=table.device)[None, :]
    return (torch.gather(held.long(), 1, pos // page) * page + pos % page).reshape(-1)


def _plain_trim(pool, rows, window, sinks):
    table, page = pool["page_table"], pool["page_size"]
    r = rows.long()
    at = torch.arange(table.shape[1], device=table.device)[None, :] * page
    low = (pool["seq_lens"][r].long() - window + 1 if window else torch.zeros_like(r))[:, None]
    held = table[r]
    drop = (at + page <= low) & (at >= sinks) & (held >= 0)
    pool["refs"].index_add_(0, held.clamp(min=0).reshape(-1).long(), -drop.reshape(-1).to(torch.int32))
    table[r] = held.masked_fill(drop, -1)


def _plain_compact(pool, every):
    refs, table = pool["refs"], pool["page_table"]
    live = refs > 0
    count = live.sum()
    at = torch.arange(refs.numel(), device=refs.device)
    src, dst = (live & (at >= count)).nonzero()[:, 0], (~live & (at < count)).nonzero()[:, 0]
    to = at.clone()
    to[src] = dst
    as_bytes = every.view(torch.uint8)
    as_bytes[:, dst] = as_bytes[:, src]
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table))
    refs[dst] = refs[src]
    refs[src] = 0


# -------------------------------------------------------------------------------------------------------------- work
def _seen(ctx, new, w, sinks):
    """(positions of the cache that any new token of a request sees, pairs of new token and position seen)."""
    if not w:
        return ctx, new * ctx + new * (new + 1) // 2
    low = max(0, ctx - w + 1)
    pairs = 0
    for t in range(ctx, ctx + new):
        lo = max(0, t - w + 1)
        pairs += t + 1 - lo + min(sinks, lo)
    return ctx - low + min(sinks, low), pairs


def work(case):
    ctx, new = _lens(case)
    page, hkv = case["page"], case["hkv"]
    token = hkv * D  # bytes of one position in one of the two caches
    if case["kind"] in ("step", "prompt"):
        seen = [_seen(c, n, case["window"], case["sinks"]) for c, n in zip(ctx, new)]
        t = sum(new)
        return {"bytes": 2 * token * sum(s for s, _ in seen) + t * (2 * GROUP * token * 2 + 2 * token * 2 + GROUP * token * 2 + 2 * token),
                "flops": 4 * D * GROUP * hkv * sum(p for _, p in seen)}
    n, layers = len(ctx), case["layers"]
    if case["kind"] == "branch":
        rows, held = n * (1 + case["fan"]), sum(-(-c // page) for c in ctx)
        spare = n * case["fan"] * (2 + case["q_len"] // page) + 5
        moved = case["fan"] * sum(c % page for c in ctx) * token * 2 * layers
        columns = (case["ctx_hi"] + case["q_len"]) // page + 1
        # the pages' counts, the parents' rows read, the children's written; data read and written
        return {"bytes": 2 * moved + 4 * (held + spare) + 4 * n * columns + 4 * (rows - n) * columns + 8 * (rows - n) * case["q_len"], "flops": 0}
    w, sinks = case["window"], case["sinks"]
    total = sum(-(-c // page) for c in ctx)
    keep = 0
    for c in ctx:
        low = max(0, c - w + 1) if w else 0
        keep += sum(1 for p in range(-(-c // page)) if p * page + page > low or p * page < sinks)
    live = keep * (n - case["gone"]) / n  # which requests leave goes by the seed: the expected number
    moves = live * (1 - live / (total + 5))
    columns = (case["ctx_hi"] - 1) // page + 1
    return {"bytes": 2 * moves * page * token * 2 * layers + 8 * (total + 5) + 8 * n * columns, "flops": 0}


# ------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("step", "prompt"):
        return _exact_attention(case, state)
    pool = state["pool"]
    table = [list(r) for r in pool["page_table"].tolist()]
    seq, refs, page = pool["seq_lens"].tolist(), pool["refs"].tolist(), pool["page_size"]
    data = [c.clone().view(torch.uint8) for c in state["caches"]]

    def drop(r, lp):
        if table[r][lp] >= 0:
            refs[table[r][lp]] -= 1
            table[r][lp] = -1

    def lowest(at=[0]):
        while refs[at[0]]:
            at[0] += 1
        return at[0]

    loc = None
    if case["kind"] == "branch":
        moves, loc = [], []
        for p, c in zip(state["parents"].tolist(), state["children"].tolist()):
            for lp in range(len(table[c])):
                drop(c, lp)
            full, part = divmod(seq[p], page)
            for lp in range(full):
                table[c][lp] = table[p][lp]
                if table[p][lp] >= 0:
                    refs[table[p][lp]] += 1
            if part:
                x = lowest()
                refs[x], table[c][full] = 1, x
                moves.append((table[p][full], x, part))
            seq[c] = seq[p]
        for a, b, part in moves:
            for d in data:
                d[b, :part] = d[a, :part]
        for c in state["children"].tolist():
            for t in range(seq[c], seq[c] + case["q_len"]):
                if table[c][t // page] < 0:
                    x = lowest()
                    refs[x], table[c][t // page] = 1, x
                loc.append(table[c][t // page] * page + t % page)
    else:
        for r in state["gone"].tolist():
            for lp in range(len(table[r])):
                drop(r, lp)
            seq[r] = 0
        for r in state["kept"].tolist():
            for lp in range(len(table[r])):
                if case["window"] and lp * page + page - 1 <= seq[r] - case["window"] and lp * page >= case["sinks"]:
                    drop(r, lp)
        live = sum(1 for x in refs if x)
        src, dst = [i for i in range(live, len(refs)) if refs[i]], [i for i in range(live) if not refs[i]]
        to = dict(zip(src, dst))
        table = [[to.get(x, x) for x in r] for r in table]
        for a, b in to.items():
            refs[b], refs[a] = refs[a], 0
        if to:
            a, b = torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda")
            for d in data:
                d[b] = d[a]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = {"page_table": i32(table), "seq_lens": i32(seq), "refs": i32(refs), "caches": [d.view(FP8) for d in data]}
    if loc is not None:
        got["cache_loc"] = torch.tensor(loc, dtype=torch.int64, device="cuda")
    return got


def _exact_attention(case, state):
    data, ctx, new = state["data"], state["ctx"], state["new"]
    cfg = data["config"]
    hkv, w, sinks, page = case["hkv"], case["window"], case["sinks"], case["page"]
    hq = hkv * GROUP
    kc, vc = data["k_cache"].clone(), data["v_cache"].clone()
    flat_k, flat_v = kc.view(-1, hkv, D), vc.view(-1, hkv, D)
    ks, vs = data["k_scale"].double(), data["v_scale"].double()
    x = data["qkv"].reshape(sum(new), -1).double()
    half = torch.arange(D // 2)
    freq = (1.0 / (case["theta"] ** ((2 * half).float() / D))).double().cuda() if case["theta"] else None

    def unit(u):
        return u / torch.sqrt(u.pow(2).sum(-1, keepdim=True) / D + EPS)

    def turn(u, pos):
        if freq is None:
            return u
        z = torch.view_as_complex(u.reshape(*u.shape[:-1], D // 2, 2).contiguous())
        turns = torch.polar(torch.ones_like(pos[:, None] * freq), pos[:, None] * freq)[:, None, :]
        return torch.view_as_real(z * turns).reshape(u.shape)

    outs, at = [], 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        rows = x[at:at + n]
        at += n
        pos = torch.arange(c, c + n, device="cuda")
        q = turn(unit(rows[:, :hq * D].view(n, hq, D)) * cfg["qk_scale_factor"], pos.double()).to(torch.bfloat16).double()
        k = turn(unit(rows[:, hq * D:(hq + hkv) * D].view(n, hkv, D)), pos.double())
        v = rows[:, (hq + hkv) * D:(hq + 2 * hkv) * D].view(n, hkv, D)
        where = data["page_table"][b].long()[pos // page] * page + pos % page
        flat_k[where] = (k / ks).clamp(-448, 448).to(FP8)
        flat_v[where] = (v / vs).clamp(-448, 448).to(FP8)
        s = torch.arange(c + n, device="cuda")
        if w:
            s = s[(s > c - w) | (s < sinks)]
        held = data["page_table"][b].long()[s // page] * page + s % page
        keys, vals = flat_k[held].double() * ks, flat_v[held].double() * vs
        o = torch.empty((n, hq, D), dtype=torch.float64, device="cuda")
        step = max(1, int(4e8 // max(1, len(s) * GROUP)))
        for h in range(hkv):
            for j in range(0, n, step):
                t = pos[j:j + step, None]
                sees = s[None, :] <= t
                if w:
                    sees &= (s[None, :] > t - w) | (s[None, :] < sinks)
                sc = torch.einsum("tgd,sd->tgs", q[j:j + step, h * GROUP:(h + 1) * GROUP], keys[:, h]) * cfg["sm_scale"]
                p = torch.softmax(sc.masked_fill(~sees[:, None, :], -math.inf), -1)
                o[j:j + step, h * GROUP:(h + 1) * GROUP] = torch.einsum("tgs,sd->tgd", p, vals[:, h])
        g = rows[:, (hq + 2 * hkv) * D:].view(n, hq, D)
        outs.append((unit(o) / (1.0 + torch.exp(-g))).reshape(n, hq * D))
    out = torch.cat(outs)
    if case["kind"] == "step":
        out = out.view(len(ctx), case["q_len"], -1)
    return {"out": out, "k_cache": kc, "v_cache": vc}
