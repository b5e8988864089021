"""The 4-bit paged KV cache and the page operations of a serving loop, on torch
tensors (device memory and streams come from torch); re-exported by ``ops``.

Layout, rounding and rules are those of include/mb200.h. All lengths, tables
and counts are int32 CUDA tensors that the calls read and change on the device:
nothing is copied to the host, so a decode loop built from these calls can be
captured in a CUDA graph. Workspaces come from torch's allocator on the current
stream (in a capture: from the graph's own pool). Arguments are checked and
passed on by the extension module ``_kv4`` (host/kv4_ext.cpp): a wrong type is a
TypeError, a wrong shape, stride or device a ValueError.
"""
from __future__ import annotations

import torch

from . import _lib

PAGE = 64
HEAD_DIM = 128
PAGE_HEAD_BYTES = 8704  # one page of one kv head: codes and scales of 64 keys and values

_ext = None


def _kv4():
    """The extension module (built beside libmb200.so; there is no fallback)."""
    global _ext
    if _ext is None:
        try:
            from . import _kv4 as ext
        except ImportError as e:
            raise ImportError("metalbench_b200/_kv4.so is missing or does not load: build it with "
                              "`python -m metalbench_b200.build` (there is no fallback)") from e
        _ext = ext
    return _ext


def kv4_cache(num_pages: int, n_kv_heads: int, device=None) -> torch.Tensor:
    """An empty 4-bit cache: uint8 [num_pages, n_kv_heads, 8704] (head dim 128)."""
    if num_pages < 1 or n_kv_heads < 1:
        raise ValueError("kv4_cache: needs at least one page and one head")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    return torch.zeros((num_pages, n_kv_heads, PAGE_HEAD_BYTES), dtype=torch.uint8, device=device)


def kv4_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
               start_pos: torch.Tensor, new_len: torch.Tensor | None = None,
               kv_len: torch.Tensor | None = None) -> None:
    """Store the (already rotated) keys and values of S new tokens a sequence.

    k, v: bf16 [B, S, n_kv_heads, 128], the last axis contiguous (views into a
    fused projection's rows are fine); token s < new_len[b] (default: all S)
    goes to position start_pos[b] + s of sequence b, unless that is kv_len[b] or
    past it: with the lengths that kv_pages_extend keeps there, nothing is stored
    for tokens that it found no pages for. Other slots of the cache stay as they
    are. A token (and head) with a NaN or an infinity, or whose largest and smallest
    number are 2^128 or more apart, reads back as NaN."""
    rc = (_ext or _kv4()).append(k, v, cache, block_table, start_pos, new_len, kv_len)
    if rc:
        _lib.check("mb_kv4_append_bf16", rc)


def kv4_gather(cache: torch.Tensor, block_table: torch.Tensor, start_pos: torch.Tensor, length: int,
               kv_len: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of positions start_pos[b] .. start_pos[b] + length - 1 as
    the numbers they stand for: fp32 [B, length, n_kv_heads, 128], zeros at
    positions kv_len[b] and later."""
    r = (_ext or _kv4()).gather(cache, block_table, start_pos, length, kv_len)
    if type(r) is int:
        _lib.check("mb_kv4_gather_f32", r)
    return r


def attention_kv4(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                  kv_len: torch.Tensor, start_pos: torch.Tensor | None = None,
                  scale: float | None = None, out: torch.Tensor | None = None,
                  max_kv_len: int | None = None) -> torch.Tensor:
    """softmax(scale * q k^T) v over the 4-bit cache (GQA, head dim 128).

    q: bf16 [B, S, n_heads, 128], or [B, n_heads, 128] for one token a sequence;
    heads contiguous, positions any multiple of 8 elements apart. Keys
    0..kv_len[b]-1 are seen; with start_pos, row s sees those at positions <=
    start_pos[b] + s (causal). A row that sees no key becomes zeros. scale:
    1/sqrt(128) by default. max_kv_len: no kv_len is larger (longer ones are
    cut; by default the block table's width); give a bound near the longest
    length when the table is much wider. Good for |q| below 2^111 and for a
    sequence's value scales within a factor of 2^90 of each other (within 2^-50 ..
    2^60 where values of zero stand beside them); values stored with a scale
    below 2^-90 may count as up to 2^-86 more. Sums are fp32; q and the softmax
    weights have 11 bits, and where many rows (64 or more a sequence) take the
    tcgen05 form the keys and values too."""
    r = (_ext or _kv4()).attention(q, cache, block_table, kv_len, start_pos, scale, out, max_kv_len)
    if type(r) is int:
        _lib.check("mb_attention_kv4_bf16", r)
    return r


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def kv_pages_extend(block_table: torch.Tensor, seq_len: torch.Tensor, page_refs: torch.Tensor,
                    new_len: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Room for new_len[b] more tokens of every sequence, in place: new pages
    (the lowest-numbered free ones, in row order) enter block_table, seq_len
    grows. Returns (start_pos, status): the lengths before, and an int32 that is
    0, or the number of pages that were lacking, or -1 for a length out of range
    (then nothing was changed)."""
    r = (_ext or _kv4()).extend(block_table, seq_len, page_refs, new_len)
    if type(r) is int:
        _lib.check("mb_kv_pages_extend", r)
    return r


def kv_pages_fork(pools, block_table: torch.Tensor, seq_len: torch.Tensor, page_refs: torch.Tensor,
                  parent: torch.Tensor) -> torch.Tensor:
    """Row b becomes a fork of row parent[b] as it was before the call, in
    place: its full pages are shared, a partly filled last page is copied (in
    every pool) into a page that was free. parent[b] == b: stays; -1: freed.
    pools: the page tensors [num_pages, ...] of all layers (bf16 or 4-bit).
    Returns an int32 status: 0, or the number of pages that were lacking, or -1
    for an index or length out of range (then nothing was changed)."""
    r = (_ext or _kv4()).fork(pools, block_table, seq_len, page_refs, parent)
    if type(r) is int:
        _lib.check("mb_kv_pages_fork", r)
    return r


def kv_pages_compact(pools, block_table: torch.Tensor, seq_len: torch.Tensor,
                     page_refs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Move the pages in use into 0..live-1, in place, with the fewest moves:
    those from `live` on go, in order, into the free ones below. Returns
    (remap, live): every page's new number (-1: was free) for references held
    outside the table, and the number of pages in use (-1: a table entry was
    out of range or not in use, and nothing was changed)."""
    r = (_ext or _kv4()).compact(pools, block_table, seq_len, page_refs)
    if type(r) is int:
        _lib.check("mb_kv_pages_compact", r)
    return r

