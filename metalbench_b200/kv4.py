"""The 4-bit paged KV cache and the page operations of a serving loop, on torch
tensors (device memory and streams come from torch); re-exported by ``ops``.

Layout, rounding and rules are those of include/mb200.h. All lengths, tables
and counts are int32 CUDA tensors that the calls read and change on the device:
nothing is copied to the host, so a decode loop built from these calls can be
captured in a CUDA graph. Workspaces come from torch's allocator on the current
stream (in a capture: from the graph's own pool).
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

PAGE = 64
HEAD_DIM = 128
PAGE_HEAD_BYTES = 8704  # one page of one kv head: codes and scales of 64 keys and values


_I32, _BF16 = torch.int32, torch.bfloat16


def _refuse(t, name: str, dtype, dev: int, shape) -> None:
    """Say what is wrong with a tensor that did not pass a call's check."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: dtype {t.dtype} is not {dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (no CPU fallback)")
    if t.get_device() != dev:
        raise ValueError(f"{name}: expected a tensor on cuda:{dev}, got one on {t.device}")
    raise ValueError(f"{name}: expected a contiguous tensor of shape {tuple(shape)}, got "
                     f"{tuple(t.shape)} with strides {t.stride()}")


def _rows(t: torch.Tensor, name: str, dev: int, n: int) -> int:
    """Address of a contiguous int32 [n] on device `dev`."""
    if not isinstance(t, torch.Tensor) or t.dtype is not _I32 or t.get_device() != dev or t.shape != (n,) \
            or not t.is_contiguous():
        _refuse(t, name, _I32, dev, (n,))
    return t.data_ptr()


def _table(t: torch.Tensor, name: str, dev: int):
    """B, max_pages and address of a block table on device `dev`."""
    if not isinstance(t, torch.Tensor) or t.dtype is not _I32 or t.get_device() != dev or t.dim() != 2 \
            or not t.is_contiguous() or t.shape[1] == 0:
        _refuse(t, name, _I32, dev, ("B", "max_pages >= 1"))
    B, M = t.shape
    return B, M, t.data_ptr()


def _cache(t: torch.Tensor, name: str):
    """num_pages, heads, device and address of a 4-bit cache."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.uint8 or not t.is_cuda or t.dim() != 3 \
            or t.shape[2] != PAGE_HEAD_BYTES or not t.is_contiguous() or t.numel() == 0 or t.data_ptr() % 16:
        _refuse(t, f"{name}(cache)", torch.uint8, t.get_device() if isinstance(t, torch.Tensor) else 0,
                ("num_pages", "n_kv_heads", PAGE_HEAD_BYTES))
    P, H, _ = t.shape
    return P, H, t.get_device(), t.data_ptr()


def _stream(dev: int) -> int:
    """torch's current stream on the current device `dev`; libmb200 set up there."""
    if dev not in _ready:
        from . import ops
        ops.init(dev)
        _ready.add(dev)
    return _raw_stream(dev)


_ready: set[int] = set()
# the public accessor builds a Stream object first, which takes longer than a small launch
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _fn(name: str):
    return getattr(_lib.lib(), name)


def kv4_cache(num_pages: int, n_kv_heads: int, device=None) -> torch.Tensor:
    """An empty 4-bit cache: uint8 [num_pages, n_kv_heads, 8704] (head dim 128)."""
    if num_pages < 1 or n_kv_heads < 1:
        raise ValueError("kv4_cache: needs at least one page and one head")
    device = device or torch.device("cuda", torch.cuda.current_device())
    return torch.zeros((num_pages, n_kv_heads, PAGE_HEAD_BYTES), dtype=torch.uint8, device=device)


def _token_strides(t: torch.Tensor, name: str, dev: int, B: int, H: int):
    """Batch, token and head strides (elements) of bf16 [B, S, H, 128]."""
    if not isinstance(t, torch.Tensor) or t.dtype is not _BF16 or t.get_device() != dev or t.dim() != 4:
        _refuse(t, name, _BF16, dev, (B, "S", H, HEAD_DIM))
    b, S, h, D = t.shape
    if b != B or h != H or D != HEAD_DIM:
        _refuse(t, name, _BF16, dev, (B, "S", H, HEAD_DIM))
    sb, ss, sh, sd = t.stride()
    if B == 1:
        sb = 0  # a stride that is never taken may be anything
    if S == 1:
        ss = 0
    if H == 1:
        sh = 0
    if sd != 1 or (sb | ss | sh) % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name}: the head dim must be contiguous and 16-byte aligned, the other strides "
                         f"multiples of 8 elements; got strides {t.stride()}")
    return sb, ss, sh


def kv4_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
               start_pos: torch.Tensor, new_len: torch.Tensor | None = None) -> None:
    """Store the (already rotated) keys and values of S new tokens a sequence.

    k, v: bf16 [B, S, n_kv_heads, 128], the last axis contiguous (views into a
    fused projection's rows are fine); token s < new_len[b] (default: all S)
    goes to position start_pos[b] + s of sequence b. Other slots of the cache
    stay as they are."""
    P, H, dev, cp = _cache(cache, "kv4_append")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return kv4_append(k, v, cache, block_table, start_pos, new_len)
    B, M, tp = _table(block_table, "kv4_append(block_table)", dev)
    ks = _token_strides(k, "kv4_append(k)", dev, B, H)
    vs = _token_strides(v, "kv4_append(v)", dev, B, H)
    if k.shape != v.shape:
        raise ValueError("kv4_append: k and v shapes differ")
    sp = _rows(start_pos, "kv4_append(start_pos)", dev, B)
    nl = None if new_len is None else _rows(new_len, "kv4_append(new_len)", dev, B)
    rc = _fn("mb_kv4_append_bf16")(k.data_ptr(), v.data_ptr(), *ks, *vs, cp, P, H, tp, M, sp, nl, B,
                                   k.shape[1], _stream(dev))
    if rc:
        _lib.check("mb_kv4_append_bf16", rc)


def kv4_gather(cache: torch.Tensor, block_table: torch.Tensor, start_pos: torch.Tensor, length: int,
               kv_len: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of positions start_pos[b] .. start_pos[b] + length - 1 as
    the numbers they stand for: fp32 [B, length, n_kv_heads, 128], zeros at
    positions kv_len[b] and later."""
    P, H, dev, cp = _cache(cache, "kv4_gather")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return kv4_gather(cache, block_table, start_pos, length, kv_len)
    B, M, tp = _table(block_table, "kv4_gather(block_table)", dev)
    sp = _rows(start_pos, "kv4_gather(start_pos)", dev, B)
    kl = _rows(kv_len, "kv4_gather(kv_len)", dev, B)
    if length < 0:
        raise ValueError("kv4_gather: negative length")
    k = torch.empty((B, length, H, HEAD_DIM), dtype=torch.float32, device=cache.device)
    v = torch.empty_like(k)
    rc = _fn("mb_kv4_gather_f32")(cp, P, H, tp, M, sp, kl, B, length, k.data_ptr(), v.data_ptr(), _stream(dev))
    if rc:
        _lib.check("mb_kv4_gather_f32", rc)
    return k, v


def _row_stride(t: torch.Tensor, name: str, dev: int, B: int, H: int):
    """S, heads and elements between two positions' rows of bf16 [B, S, heads,
    128] or [B, heads, 128] (S = 1), heads contiguous and a multiple of H."""
    if not isinstance(t, torch.Tensor) or t.dtype is not _BF16 or t.get_device() != dev or t.dim() not in (3, 4):
        _refuse(t, name, _BF16, dev, (B, "S", f"heads (a multiple of {H})", HEAD_DIM))
    shape, st = t.shape, t.stride()
    if len(shape) == 4:
        b, S, Hq, D = shape
        sb, ss, sh, sd = st
    else:
        b, Hq, D = shape
        sb, sh, sd = st
        S, ss = 1, 0
    if b != B or D != HEAD_DIM or Hq == 0 or Hq % H:
        _refuse(t, name, _BF16, dev, (B, "S", f"heads (a multiple of {H})", HEAD_DIM))
    ld = ss if S > 1 else sb if B > 1 else Hq * HEAD_DIM
    if t.numel() and (sd != 1 or (Hq > 1 and sh != HEAD_DIM) or (S > 1 and B > 1 and sb != S * ss)
                      or ld < Hq * HEAD_DIM or ld % 8 or t.data_ptr() % 16):
        raise ValueError(f"{name}: heads must be contiguous, positions evenly spaced (a multiple of 8 "
                         f"elements) and 16-byte aligned; got strides {st}")
    return S, Hq, ld


def attention_kv4(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                  kv_len: torch.Tensor, start_pos: torch.Tensor | None = None,
                  scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale * q k^T) v over the 4-bit cache (GQA, head dim 128).

    q: bf16 [B, S, n_heads, 128], or [B, n_heads, 128] for one token a sequence;
    heads contiguous, positions any multiple of 8 elements apart. Keys
    0..kv_len[b]-1 are seen; with start_pos, row s sees those at positions <=
    start_pos[b] + s (causal). A row that sees no key becomes zeros. scale:
    1/sqrt(128) by default."""
    P, H, dev, cp = _cache(cache, "attention_kv4")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return attention_kv4(q, cache, block_table, kv_len, start_pos, scale, out)
    B, M, tp = _table(block_table, "attention_kv4(block_table)", dev)
    S, Hq, ldq = _row_stride(q, "attention_kv4(q)", dev, B, H)
    kl = _rows(kv_len, "attention_kv4(kv_len)", dev, B)
    sp = None if start_pos is None else _rows(start_pos, "attention_kv4(start_pos)", dev, B)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        ldo = Hq * HEAD_DIM
    else:
        if out.shape != q.shape:
            raise ValueError(f"attention_kv4(out): shape {tuple(out.shape)} is not q's {tuple(q.shape)}")
        ldo = _row_stride(out, "attention_kv4(out)", dev, B, H)[2]
    nb = _fn("mb_attention_kv4_workspace_bytes")(B, S, Hq, H, M)
    ws = torch.empty(nb, dtype=torch.uint8, device=cache.device)
    rc = _fn("mb_attention_kv4_bf16")(q.data_ptr(), ldq, cp, P, tp, M, kl, sp, B, S, Hq, H, HEAD_DIM,
                                      _SCALE if scale is None else scale, out.data_ptr(), ldo,
                                      ws.data_ptr(), nb, _stream(dev))
    if rc:
        _lib.check("mb_attention_kv4_bf16", rc)
    return out


_SCALE = 1.0 / math.sqrt(HEAD_DIM)


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def _pages(block_table, seq_len, page_refs, name: str):
    """Device, sizes and addresses of the three tensors of a page call."""
    if not isinstance(block_table, torch.Tensor) or not block_table.is_cuda:
        raise ValueError(f"{name}: expected CUDA tensors (no CPU fallback)")
    dev = block_table.get_device()
    B, M, tp = _table(block_table, f"{name}(block_table)", dev)
    if not isinstance(page_refs, torch.Tensor) or page_refs.dim() != 1:
        raise ValueError(f"{name}: page_refs must be [num_pages]")
    P = page_refs.shape[0]
    return dev, B, M, P, tp, _rows(seq_len, name, dev, B), _rows(page_refs, name, dev, P)


def _pools(pools, name: str, dev: int, P: int):
    n = len(pools)
    ptrs, sizes = [], []
    for t in pools:
        if t.get_device() != dev or t.dim() < 1 or t.shape[0] != P or not t.is_contiguous():
            raise ValueError(f"{name}: a pool must be a contiguous tensor on cuda:{dev} with {P} pages")
        size = t.nbytes // P if P else 16
        if size == 0 or size % 16 or t.data_ptr() % 16:
            raise ValueError(f"{name}: a pool's pages must be a multiple of 16 bytes and 16-byte aligned")
        ptrs.append(t.data_ptr())
        sizes.append(size)
    if len(set(ptrs)) < n:
        raise ValueError(f"{name}: the same pool twice")
    return (C.c_void_p * n)(*ptrs), (C.c_int64 * n)(*sizes), n


def kv_pages_extend(block_table: torch.Tensor, seq_len: torch.Tensor, page_refs: torch.Tensor,
                    new_len: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Room for new_len[b] more tokens of every sequence, in place: new pages
    (the lowest-numbered free ones, in row order) enter block_table, seq_len
    grows. Returns (start_pos, status): the lengths before, and an int32 that is
    0, or the number of pages that were lacking, or -1 for a length out of range
    (then nothing was changed)."""
    dev, B, M, P, tp, sl, pr = _pages(block_table, seq_len, page_refs, "kv_pages_extend")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return kv_pages_extend(block_table, seq_len, page_refs, new_len)
    nl = _rows(new_len, "kv_pages_extend(new_len)", dev, B)
    start = torch.empty_like(seq_len)
    status = torch.empty(1, dtype=_I32, device=seq_len.device)
    nb = _fn("mb_kv_pages_workspace_bytes")(B, M, P)
    ws = torch.empty(nb, dtype=torch.uint8, device=seq_len.device)
    rc = _fn("mb_kv_pages_extend")(tp, sl, pr, B, M, P, nl, start.data_ptr(), status.data_ptr(),
                                   ws.data_ptr(), nb, _stream(dev))
    if rc:
        _lib.check("mb_kv_pages_extend", rc)
    return start, status


def kv_pages_fork(pools, block_table: torch.Tensor, seq_len: torch.Tensor, page_refs: torch.Tensor,
                  parent: torch.Tensor) -> torch.Tensor:
    """Row b becomes a fork of row parent[b] as it was before the call, in
    place: its full pages are shared, a partly filled last page is copied (in
    every pool) into a page that was free. parent[b] == b: stays; -1: freed.
    pools: the page tensors [num_pages, ...] of all layers (bf16 or 4-bit).
    Returns an int32 status: 0, or the number of pages that were lacking, or -1
    for an index or length out of range (then nothing was changed)."""
    dev, B, M, P, tp, sl, pr = _pages(block_table, seq_len, page_refs, "kv_pages_fork")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return kv_pages_fork(pools, block_table, seq_len, page_refs, parent)
    pa = _rows(parent, "kv_pages_fork(parent)", dev, B)
    ptrs, sizes, n = _pools(pools, "kv_pages_fork", dev, P)
    status = torch.empty(1, dtype=_I32, device=seq_len.device)
    nb = _fn("mb_kv_pages_workspace_bytes")(B, M, P)
    ws = torch.empty(nb, dtype=torch.uint8, device=seq_len.device)
    rc = _fn("mb_kv_pages_fork")(ptrs, sizes, n, tp, sl, pr, B, M, P, pa, status.data_ptr(),
                                 ws.data_ptr(), nb, _stream(dev))
    if rc:
        _lib.check("mb_kv_pages_fork", rc)
    return status


def kv_pages_compact(pools, block_table: torch.Tensor, seq_len: torch.Tensor,
                     page_refs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Move the pages in use into 0..live-1, in place, with the fewest moves:
    those from `live` on go, in order, into the free ones below. Returns
    (remap, live): every page's new number (-1: was free) for references held
    outside the table, and the number of pages in use (-1: a table entry was
    out of range or not in use, and nothing was changed)."""
    dev, B, M, P, tp, sl, pr = _pages(block_table, seq_len, page_refs, "kv_pages_compact")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return kv_pages_compact(pools, block_table, seq_len, page_refs)
    ptrs, sizes, n = _pools(pools, "kv_pages_compact", dev, P)
    remap = torch.empty_like(page_refs)
    live = torch.empty(1, dtype=_I32, device=seq_len.device)
    nb = _fn("mb_kv_pages_workspace_bytes")(B, M, P)
    ws = torch.empty(nb, dtype=torch.uint8, device=seq_len.device)
    rc = _fn("mb_kv_pages_compact")(ptrs, sizes, n, tp, sl, pr, B, M, P, remap.data_ptr(),
                                    live.data_ptr(), ws.data_ptr(), nb, _stream(dev))
    if rc:
        _lib.check("mb_kv_pages_compact", rc)
    return remap, live
