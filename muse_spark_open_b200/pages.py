"""Pages of a paged cache: what a serving loop does with the page table that `attention` and `layer` read.

`prepare(num_pages, page_size, rows, max_pages, device) -> pool`, a dict of device tensors: page_table int32 [rows,
max_pages] (-1 = no page), seq_lens int32 [rows] (tokens in the cache), refs int32 [num_pages] (table entries that name a
page; 0 = free), and page_size.  A row is one request; `pool["page_table"]` and `pool["seq_lens"]` (or some of their rows)
go into the `data` of attention.kernel_fn / prompt_fn and layer.kernel_fn as they are.  Lists of rows are int32 device
tensors.  `caches` are the tensors whose first axis is the physical page and whose second the slot, K and V of every layer
that uses the pool: at most 128 per call (64 layers), all with the same bytes per token, a multiple of 16, because fork and
compact change the table in the call that moves the data.  A step of a serving loop:

    loc = pages.extend(pool, rows, q_len)                 # room for the next tokens; their cache rows
    ... attention / layer step with pool["page_table"], pool["seq_lens"], cache_loc=loc ...
    pool["seq_lens"][rows] += q_len                       # the tokens that stay (fewer after a rejected draft)
    pages.trim(pool, rows, window, sinks)                 # what the window has passed goes back

Everything happens on the device, in place and in stream order (order the streams yourself when you use several on one pool);
nothing is read back, so all calls can be captured in a CUDA graph.  New pages are the lowest free ones, given out in the order of the rows: results do not depend on scheduling.
Problems with the contents (a row out of range or listed twice, no free page, seq_lens set back into pages that a fork shares
and then extended, cu_seqlens that falls or names more tokens than `tokens`, negative seq_lens) are reported in the status
word (`abi.status_for(device).raise_if_set()`), and the entries concerned are skipped; include/msk.h says how.
The reference has no counterpart: its inputs come with a finished table (muse_attention_decode/reference.py:168-253).
"""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch

from . import abi


def prepare(num_pages: int, page_size: int, rows: int, max_pages: int, device="cuda") -> dict:
    """A pool with every page free and every row empty."""
    if page_size < 1 or page_size & (page_size - 1) or min(num_pages, rows, max_pages) < 1:
        raise abi.MskError("page_size must be a power of two, and num_pages, rows and max_pages at least 1")
    mk = lambda shape, v: torch.full(shape, v, dtype=torch.int32, device=device)  # noqa: E731
    return {"page_table": mk((rows, max_pages), -1), "seq_lens": mk((rows,), 0), "refs": mk((num_pages,), 0), "page_size": page_size}


_pages_args = abi.packer(abi.Pages)
_INT = torch.int32


def _args(pool: dict, *lists: torch.Tensor):
    """(the packed MskPages, its shape, the device) of a pool whose tensors and lists are what the C functions expect."""
    table, seq, refs = pool["page_table"], pool["seq_lens"], pool["refs"]
    if table.dtype != _INT or seq.dtype != _INT or refs.dtype != _INT or table.dim() != 2 or seq.dim() != 1 or refs.dim() != 1 or \
            seq.shape[0] != table.shape[0] or not (table.is_contiguous() and seq.is_contiguous() and refs.is_contiguous()):
        raise abi.MskError("page_table [rows, max_pages], seq_lens [rows] and refs [num_pages] must be contiguous int32")
    for x in lists:
        if x.dtype != _INT or x.dim() != 1 or not x.is_contiguous():
            raise abi.MskError("lists of rows must be contiguous int32 vectors")
    index = abi.here((table, seq, refs, *lists))
    rows, most = table.shape
    pages = refs.shape[0]
    return _pages_args.pack(table.data_ptr(), seq.data_ptr(), refs.data_ptr(), rows, most, pages, pool["page_size"]), (rows, pages), index


def _scratch(pool: dict, q: bytes, shape, n: int):
    """(address, bytes) of the pool's workspace, kept in the pool from its first call on: calls on one pool change the same
    counts and are ordered anyway.  Lists longer than the pool has rows (and a first call inside a graph capture, whose memory
    is the graph's) get memory of their own, for the call."""
    kept = pool.get("scratch")
    if kept is not None and (kept[0] != shape or kept[4] is not pool["refs"] or kept[1] != kept[3].data_ptr()):
        kept = None  # a copy of another pool, with counts of its own (a deep one: the address is still the other pool's)
    if kept is not None and n <= shape[0]:
        return kept[1], kept[2], None
    b = C.c_size_t()
    abi.check(abi.lib().msk_pages_scratch_bytes(q, max(n, shape[0]), C.byref(b)), "msk_pages_scratch_bytes")
    t = torch.empty(b.value, dtype=torch.uint8, device=pool["refs"].device)
    if kept is None and n <= shape[0] and not torch.cuda.is_current_stream_capturing():
        pool["scratch"] = (shape, t.data_ptr(), b.value, t, pool["refs"])
    return t.data_ptr(), b.value, t


def _caches(caches, pool: dict, index: int):
    """(host array of the caches' addresses, how many, bytes per token)"""
    pages, size, token, ptrs = pool["refs"].shape[0], pool["page_size"], 0, []
    for c in caches:
        shape = c.shape
        if len(shape) < 3 or shape[0] != pages or shape[1] != size or not c.is_contiguous():
            raise abi.MskError("caches must be contiguous [num_pages, page_size, ...]")
        if c.get_device() != index:
            raise abi.MskError("the tensors of one call must be on one device")
        bytes_ = math.prod(shape[2:]) * c.element_size()  # not the stride: of an axis of length one it may be anything
        if token and bytes_ != token:
            raise abi.MskError("the caches of one call must have the same bytes per token")
        token = bytes_
        ptrs.append(c.data_ptr())
    return struct.pack(f"{len(ptrs)}P", *ptrs), len(ptrs), token or 16


def extend(pool: dict, rows: torch.Tensor, q_len: int = 1, cu_seqlens: torch.Tensor | None = None,
           tokens: int | None = None) -> torch.Tensor:
    """Pages for the next `q_len` tokens of each row, or for cu_seqlens[j + 1] - cu_seqlens[j] of row j (then `tokens`, which
    has to be given, rows in all, padding included).  Returns cache_loc int64 [len(rows) * q_len] (or [tokens]): the flat cache row of each new
    token, -1 where there is none.  seq_lens stays: the caller advances it when the tokens are in."""
    n = rows.shape[0]
    if cu_seqlens is None:
        tokens = 0
        q, shape, index = _args(pool, rows)
        loc, cu = torch.empty(n * q_len, dtype=torch.int64, device=rows.device), 0
    else:
        if tokens is None or tokens < 0:
            raise abi.MskError("with cu_seqlens, tokens (its last entry or more) has to be given")
        q, shape, index = _args(pool, rows, cu_seqlens)
        if cu_seqlens.shape[0] != n + 1:
            raise abi.MskError("cu_seqlens must have one entry more than rows")
        loc, cu = torch.full((tokens,), -1, dtype=torch.int64, device=rows.device), cu_seqlens.data_ptr()
    ws, size, _own = _scratch(pool, q, shape, n)
    rc = abi.lib().msk_pages_extend(q, rows.data_ptr(), n, q_len, cu, tokens, loc.data_ptr(), ws, size, abi.status_ptr(index),
                                    abi.raw_stream(index))
    if rc:
        abi.check(rc, "msk_pages_extend")
    return loc


def fork(pool: dict, parents: torch.Tensor, children: torch.Tensor, caches) -> None:
    """children[j] becomes a copy of parents[j]: full pages are shared, a last page that is not full is copied (its filled
    part, in every cache).  What the children's rows held goes back.  A parent may have several children; a child must not
    be listed twice nor be a parent."""
    q, shape, index = _args(pool, parents, children)
    n = children.shape[0]
    if parents.shape[0] != n:
        raise abi.MskError("parents and children must have the same length")
    ptrs, count, token = _caches(caches, pool, index)
    ws, size, _own = _scratch(pool, q, shape, n)
    rc = abi.lib().msk_pages_fork(q, parents.data_ptr(), children.data_ptr(), n, ptrs, count, token, ws, size, abi.status_ptr(index),
                                  abi.raw_stream(index))
    if rc:
        abi.check(rc, "msk_pages_fork")


def free(pool: dict, rows: torch.Tensor) -> None:
    """The rows' pages go back, the rows become empty."""
    q, _, index = _args(pool, rows)
    rc = abi.lib().msk_pages_free(q, rows.data_ptr(), rows.shape[0], abi.status_ptr(index), abi.raw_stream(index))
    if rc:
        abi.check(rc, "msk_pages_free")


def trim(pool: dict, rows: torch.Tensor, window: int, sinks: int = 0) -> None:
    """The pages that no later token of the rows sees under this window and these sinks go back (table entries become -1)."""
    q, _, index = _args(pool, rows)
    rc = abi.lib().msk_pages_trim(q, rows.data_ptr(), rows.shape[0], window, sinks, abi.status_ptr(index), abi.raw_stream(index))
    if rc:
        abi.check(rc, "msk_pages_trim")


def compact(pool: dict, caches) -> torch.Tensor:
    """Moves pages in use into free ones at the front, in every cache, until the n pages in use are [0, n); the table
    follows.  Returns int32 [2] on the device: n, and how many pages moved."""
    q, shape, index = _args(pool)
    ptrs, count, token = _caches(caches, pool, index)
    ws, size, _own = _scratch(pool, q, shape, 0)
    result = torch.empty(2, dtype=_INT, device=pool["refs"].device)
    rc = abi.lib().msk_pages_compact(q, ptrs, count, token, result.data_ptr(), ws, size, abi.status_ptr(index), abi.raw_stream(index))
    if rc:
        abi.check(rc, "msk_pages_compact")
    return result
