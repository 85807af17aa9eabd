"""Gated attention decode / verify: the reference's per-op entry point over the C ABI.

`kernel_fn(data) -> bf16 [B, L, Hq*d]` with the `Inputs` / `Config` fields of
muse_attention_decode/submission.py:37-65; the new tokens' K/V are written into
`data["k_cache"]` / `data["v_cache"]` in place at `data["cache_loc"]`, like the reference.
With a window, `config["sinks"]` (default 0) first positions stay visible to every token.
Nothing derived from `data` is cached between calls; only the RoPE frequency table (a function of
theta and head_dim) is kept per device.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi

_inv_freq: dict = {}


def inv_freq(theta: float, d: int, device) -> torch.Tensor | None:
    """theta^(-2i/d), computed in FP32 exactly as the reference does (reference.py:274)."""
    if not theta:
        return None
    key = (float(theta), d, torch.device(device).index or 0)
    if key not in _inv_freq:
        _inv_freq[key] = (1.0 / (theta ** (torch.arange(0, d, 2).float() / d))).to(device)
    return _inv_freq[key]


def launch(qkv2d: torch.Tensor, out2d: torch.Tensor, data: dict, cfg: dict, chunks: int = 0, stages: int = 0, issuers: int = 0,
           pdl: bool = False, row_groups: int = 0) -> None:
    """qkv2d bf16 [B*L, >= (2Hq+2Hkv)*d] (row stride free), out2d bf16 [B*L, Hq*d]."""
    p = abi.AttnParams()
    p.qkv, p.ld_qkv, p.out, p.ld_out = abi.ptr(qkv2d), qkv2d.stride(0), abi.ptr(out2d), out2d.stride(0)
    kc, vc = data["k_cache"], data["v_cache"]
    p.k_cache, p.v_cache = abi.ptr(kc), abi.ptr(vc)
    p.k_scale, p.v_scale = abi.ptr(data["k_scale"]), abi.ptr(data["v_scale"])
    p.seq_lens, p.page_table = abi.ptr(data["seq_lens"]), abi.ptr(data["page_table"])
    p.max_pages = data["page_table"].shape[1]
    p.cache_loc = abi.ptr(data["cache_loc"])
    f = inv_freq(cfg["rope_theta"], cfg["head_dim"], qkv2d.device)
    p.inv_freq = abi.ptr(f) if f is not None else None
    p.B, p.L, p.Hq, p.Hkv, p.d = cfg["batch"], cfg["q_len"], cfg["num_q_heads"], cfg["num_kv_heads"], cfg["head_dim"]
    p.page_size, p.num_pages, p.window = cfg["page_size"], kc.shape[0], cfg["window"]
    p.sinks = cfg.get("sinks", 0)
    p.qk_scale_factor, p.sm_scale = cfg["qk_scale_factor"], cfg["sm_scale"]
    p.chunks, p.stages, p.issuers, p.pdl, p.row_groups = chunks, stages, issuers, int(pdl), row_groups
    st = abi.status_for(qkv2d.device)
    abi.check(abi.lib().msk_attn_decode(C.byref(p), st.p, abi.stream_ptr()), "msk_attn_decode")


def kernel_fn(data: dict, chunks: int = 0, stages: int = 0) -> torch.Tensor:
    cfg = data["config"]
    b, l, hq, d = cfg["batch"], cfg["q_len"], cfg["num_q_heads"], cfg["head_dim"]
    qkv = data["qkv"]
    if qkv.dtype != torch.bfloat16 or data["k_cache"].dtype != torch.float8_e4m3fn:
        raise abi.MskError("qkv must be bfloat16 and the cache float8_e4m3fn")
    if data["seq_lens"].dtype != torch.int32 or data["page_table"].dtype != torch.int32 or \
            data["cache_loc"].dtype != torch.int64:
        raise abi.MskError("seq_lens / page_table must be int32 and cache_loc int64")
    out = torch.empty((b, l, hq * d), dtype=torch.bfloat16, device=qkv.device)
    launch(qkv.view(b * l, -1), out.view(b * l, hq * d), data, cfg, chunks, stages)
    return out


def prompt_fn(data: dict, out: torch.Tensor | None = None, splits: int = 0) -> torch.Tensor:
    """bf16 [T, Hq*d]: the same attention for prompts, with any number of new tokens per request.

    `data` as for `kernel_fn`, except: qkv is [T, (2Hq+2Hkv)*d] (row stride free), cu_seqlens_q int32 [B + 1] says which
    rows belong to which request, and there is no cache_loc (the rows of the new K/V follow from the page table, whose
    entries must exist for the new positions: `pages.extend`).  `config` needs no q_len.  Rows behind cu_seqlens_q[B]
    (a padded batch) are not touched: they keep what `out` held.  The workspace comes from torch's allocator on the current
    stream, so calls on several streams or in several captured graphs do not share it.
    """
    cfg, qkv, kc, vc = data["config"], data["qkv"], data["k_cache"], data["v_cache"]
    table, seq, cu = data["page_table"], data["seq_lens"], data["cu_seqlens_q"]
    b, hq, hkv, d = cfg["batch"], cfg["num_q_heads"], cfg["num_kv_heads"], cfg["head_dim"]
    if qkv.dtype != torch.bfloat16 or kc.dtype != torch.float8_e4m3fn or vc.dtype != torch.float8_e4m3fn:
        raise abi.MskError("qkv must be bfloat16 and the cache float8_e4m3fn")
    if qkv.dim() != 2 or qkv.shape[1] < (2 * hq + 2 * hkv) * d or qkv.stride(1) != 1:
        raise abi.MskError("qkv must be [tokens, (2Hq+2Hkv)*d] with unit column stride")
    if seq.dtype != torch.int32 or table.dtype != torch.int32 or cu.dtype != torch.int32:
        raise abi.MskError("seq_lens / page_table / cu_seqlens_q must be int32")
    if seq.numel() != b or table.dim() != 2 or table.shape[0] != b or cu.numel() != b + 1 or \
            not (seq.is_contiguous() and table.is_contiguous() and cu.is_contiguous()):
        raise abi.MskError("seq_lens [B], page_table [B, max_pages] and cu_seqlens_q [B + 1] must be contiguous")
    shape = (kc.shape[0], cfg["page_size"], hkv, d)
    if kc.shape != shape or vc.shape != shape or not (kc.is_contiguous() and vc.is_contiguous()):
        raise abi.MskError("k_cache / v_cache must be contiguous [num_pages, page_size, Hkv, d]")
    t, dev = qkv.shape[0], abi.here(qkv, kc, vc, data["k_scale"], data["v_scale"], seq, cu, table)
    if out is None:
        out = torch.empty((t, hq * d), dtype=torch.bfloat16, device=dev)
    elif out.dtype != torch.bfloat16 or out.shape != (t, hq * d) or out.stride(1) != 1:
        raise abi.MskError("out must be bfloat16 [tokens, Hq*d] with unit column stride")
    else:
        abi.here(qkv, out)
    if t == 0:
        return out
    f = inv_freq(cfg["rope_theta"], d, dev)
    p = abi.PromptParams(
        abi.ptr(qkv), qkv.stride(0), abi.ptr(out), out.stride(0), abi.ptr(kc), abi.ptr(vc), abi.ptr(data["k_scale"]), abi.ptr(data["v_scale"]),
        abi.ptr(seq), abi.ptr(cu), abi.ptr(table), table.shape[1], abi.ptr(f), b, t, hq, hkv, d, cfg["page_size"], kc.shape[0],
        cfg["window"], cfg.get("sinks", 0), cfg["qk_scale_factor"], cfg["sm_scale"], splits, 0, None, 0)
    lib, n = abi.lib(), C.c_size_t()
    abi.check(lib.msk_attn_prompt_scratch_bytes(C.byref(p), C.byref(n)), "msk_attn_prompt_scratch_bytes")
    scratch = torch.empty(n.value, dtype=torch.uint8, device=dev)
    p.scratch, p.scratch_bytes = scratch.data_ptr(), n.value
    abi.check(lib.msk_attn_prompt(C.byref(p), abi.status_for(dev).p, abi.stream_ptr()), "msk_attn_prompt")
    return out
