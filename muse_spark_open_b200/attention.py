"""Gated attention decode / verify: the reference's per-op entry point over the C ABI.

`kernel_fn(data) -> bf16 [B, L, Hq*d]` with the `Inputs` / `Config` fields of
muse_attention_decode/submission.py:37-65; the new tokens' K/V are written into
`data["k_cache"]` / `data["v_cache"]` in place at `data["cache_loc"]`, like the reference.
With a window, `config["sinks"]` (default 0) first positions stay visible to every token.
q_len is 1 (decode) or 8 (verify) as in the reference, or any other length: blocks other than 1 and 8, and blocks of 8 with
a window and sinks, write the new rows where the page table says (cache_loc says the same in the reference, submission.py:37-65).
RoPE's angle is the reference's product in 32 bits for tokens and blocks of 8 without sinks, off by up to 2^-11 rad at positions
8192 to 16384 and twice that at twice the position; prompts, other blocks and steps with sinks turn by the exact one.  They may
share a cache: each key has its own token's angle either way, and at position 16384 the two differ by about as much of a score
as the queries' other roundings do.
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


_attn_args, _prompt_args = abi.packer(abi.AttnParams), abi.packer(abi.PromptParams)


def _run_step(qkv: int, ld_qkv: int, out: int, ld_out: int, data: dict, cfg: dict, index: int, chunks: int, stages: int, issuers: int, pdl: bool,
              row_groups: int) -> None:
    kc, d = data["k_cache"], cfg["head_dim"]
    theta = cfg["rope_theta"]
    freq = (_inv_freq.get((float(theta), d, index)) if theta else None)
    if theta and freq is None:
        freq = inv_freq(theta, d, kc.device)
    table = data["page_table"]
    args = _attn_args.pack(
        qkv, ld_qkv, out, ld_out, abi.ptr(kc), abi.ptr(data["v_cache"]), abi.ptr(data["k_scale"]), abi.ptr(data["v_scale"]), abi.ptr(data["seq_lens"]),
        abi.ptr(table), table.shape[1], abi.ptr(data["cache_loc"]), freq.data_ptr() if freq is not None else 0, cfg["batch"], cfg["q_len"],
        cfg["num_q_heads"], cfg["num_kv_heads"], d, cfg["page_size"], kc.shape[0], cfg["window"], cfg["qk_scale_factor"], cfg["sm_scale"], chunks,
        stages, issuers, int(pdl), row_groups, cfg.get("sinks", 0))
    rc = abi.lib().msk_attn_decode(args, abi.status_ptr(index), abi.raw_stream(index))
    if rc:
        abi.check(rc, "msk_attn_decode")


def launch(qkv2d: torch.Tensor, out2d: torch.Tensor, data: dict, cfg: dict, chunks: int = 0, stages: int = 0, issuers: int = 0,
           pdl: bool = False, row_groups: int = 0) -> None:
    """qkv2d bf16 [B*L, >= (2Hq+2Hkv)*d] (row stride free), out2d bf16 [B*L, Hq*d]."""
    _run_step(abi.ptr(qkv2d), qkv2d.stride(0), abi.ptr(out2d), out2d.stride(0), data, cfg, qkv2d.get_device(), chunks, stages, issuers, pdl, row_groups)


def kernel_fn(data: dict, chunks: int = 0, stages: int = 0) -> torch.Tensor:
    cfg = data["config"]
    b, l, wide = cfg["batch"], cfg["q_len"], cfg["num_q_heads"] * cfg["head_dim"]
    qkv = data["qkv"]
    if qkv.dtype != torch.bfloat16 or data["k_cache"].dtype != torch.float8_e4m3fn:
        raise abi.MskError("qkv must be bfloat16 and the cache float8_e4m3fn")
    if data["seq_lens"].dtype != torch.int32 or data["page_table"].dtype != torch.int32 or \
            data["cache_loc"].dtype != torch.int64:
        raise abi.MskError("seq_lens / page_table must be int32 and cache_loc int64")
    if qkv.is_contiguous() and b * l > 0 and qkv.numel() % (b * l) == 0:
        cols = ld = qkv.numel() // (b * l)
    else:
        flat = qkv.view(b * l, -1)
        cols, ld = flat.shape[1] if flat.stride(1) == 1 else 0, flat.stride(0)
    out = torch.empty((b, l, wide), dtype=torch.bfloat16, device=qkv.device)
    if l != 1 and (l != 8 or (cfg["window"] and cfg.get("sinks", 0))) and not chunks and not stages:
        # blocks of other lengths, and verify blocks with sinks: the prompt kernels (16 requests x 8 tokens, window 1024 + 4
        # sinks, in a graph: 22 us against 52 us for the verify kernel, whose results without sinks stay what they were)
        _run_prompt(data, cfg, qkv, b * l, cols, ld, out, wide, None, l, 0)
        return out
    _run_step(abi.ptr(qkv), ld, out.data_ptr(), wide, data, cfg, qkv.get_device(), chunks, stages, 0, False, 0)
    return out


_prompt_bytes: dict = {}


def _run_prompt(data: dict, cfg: dict, qkv: torch.Tensor, t: int, cols: int, ld_qkv: int, out: torch.Tensor | None, ld_out: int,
                cu: torch.Tensor | None, q_len: int, splits: int) -> torch.Tensor:
    """msk_attn_prompt on checked arguments: t rows of `cols` values in qkv (0: not such rows), ld_qkv apart; cu None: q_len
    tokens per request; out None: made here."""
    kc, vc, table, seq, ks, vs = data["k_cache"], data["v_cache"], data["page_table"], data["seq_lens"], data["k_scale"], data["v_scale"]
    b, hq, hkv, d, page = cfg["batch"], cfg["num_q_heads"], cfg["num_kv_heads"], cfg["head_dim"], cfg["page_size"]
    if qkv.dtype != torch.bfloat16 or kc.dtype != torch.float8_e4m3fn or vc.dtype != torch.float8_e4m3fn:
        raise abi.MskError("qkv must be bfloat16 and the cache float8_e4m3fn")
    if cols < (2 * hq + 2 * hkv) * d:
        raise abi.MskError("qkv must be [tokens, (2Hq+2Hkv)*d] with unit column stride")
    if seq.dtype != torch.int32 or table.dtype != torch.int32 or (cu is not None and cu.dtype != torch.int32):
        raise abi.MskError("seq_lens / page_table / cu_seqlens_q must be int32")
    if seq.numel() != b or table.dim() != 2 or table.shape[0] != b or not (seq.is_contiguous() and table.is_contiguous()) or \
            (cu is not None and (cu.numel() != b + 1 or not cu.is_contiguous())):
        raise abi.MskError("seq_lens [B], page_table [B, max_pages] and cu_seqlens_q [B + 1] must be contiguous")
    pages = kc.shape[0]
    shape = (pages, page, hkv, d)
    if kc.shape != shape or vc.shape != shape or not (kc.is_contiguous() and vc.is_contiguous()):
        raise abi.MskError("k_cache / v_cache must be contiguous [num_pages, page_size, Hkv, d]")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise abi.MskError("k_scale / v_scale must be float32")
    index = abi.here((qkv, kc, vc, ks, vs, seq, table) if cu is None else (qkv, kc, vc, ks, vs, seq, table, cu))
    dev = qkv.device
    if out is None:
        out, ld_out = torch.empty((t, hq * d), dtype=torch.bfloat16, device=dev), hq * d
    elif out.get_device() != index:
        raise abi.MskError("the tensors of one call must be on one device")
    if t == 0:
        return out
    theta, window, sinks, max_pages = cfg["rope_theta"], cfg["window"], cfg.get("sinks", 0), table.shape[1]
    freq = 0
    if theta:
        f = _inv_freq.get((float(theta), d, index))
        freq = (inv_freq(theta, d, dev) if f is None else f).data_ptr()
    lib = abi.lib()
    # the workspace's size is a function of sizes alone
    key = (b, t, hq, hkv, d, page, pages, window, sinks, max_pages, splits, q_len)
    nbytes = _prompt_bytes.get(key)
    if nbytes is None:
        n = C.c_size_t()
        p = abi.PromptParams(B=b, T=t, Hq=hq, Hkv=hkv, d=d, page_size=page, num_pages=pages, window=window, sinks=sinks, max_pages=max_pages,
                             splits=splits, q_len=q_len, cu_seqlens_q=None if cu is None else cu.data_ptr())
        abi.check(lib.msk_attn_prompt_scratch_bytes(C.byref(p), C.byref(n)), "msk_attn_prompt_scratch_bytes")
        if len(_prompt_bytes) > 4096:
            _prompt_bytes.clear()
        nbytes = _prompt_bytes[key] = n.value
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    args = _prompt_args.pack(
        qkv.data_ptr(), ld_qkv, out.data_ptr(), ld_out, kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), seq.data_ptr(),
        0 if cu is None else cu.data_ptr(), table.data_ptr(), max_pages, freq, b, t, hq, hkv, d, page, pages, window, sinks,
        cfg["qk_scale_factor"], cfg["sm_scale"], splits, 0, scratch.data_ptr(), nbytes, q_len)
    rc = lib.msk_attn_prompt(args, abi.status_ptr(index), abi.raw_stream(index))
    if rc:
        abi.check(rc, "msk_attn_prompt")
    return out


def prompt_fn(data: dict, out: torch.Tensor | None = None, splits: int = 0) -> torch.Tensor:
    """bf16 [T, Hq*d]: the same attention for prompts, with any number of new tokens per request.

    `data` as for `kernel_fn`, except: qkv is [T, (2Hq+2Hkv)*d] (row stride free), cu_seqlens_q int32 [B + 1] says which
    rows belong to which request, and there is no cache_loc (the rows of the new K/V follow from the page table, whose
    entries must exist for the new positions: `pages.extend`).  `config` needs no q_len.  Rows behind cu_seqlens_q[B]
    (a padded batch) are not touched: they keep what `out` held.  The workspace comes from torch's allocator on the current
    stream, so calls on several streams or in several captured graphs do not share it.
    """
    cfg, qkv = data["config"], data["qkv"]
    t, cols = qkv.shape if qkv.dim() == 2 and qkv.stride(1) == 1 else (0, 0)
    if out is not None and (out.dtype != torch.bfloat16 or out.shape != (t, cfg["num_q_heads"] * cfg["head_dim"]) or out.stride(1) != 1):
        raise abi.MskError("out must be bfloat16 [tokens, Hq*d] with unit column stride")
    return _run_prompt(data, cfg, qkv, t, cols, qkv.stride(0) if cols else 0, out, 0 if out is None else out.stride(0), data["cu_seqlens_q"], 0, splits)
