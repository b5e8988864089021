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


def _i32(t: torch.Tensor, name: str, device, shape) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name}: expected an int32 tensor")
    if t.device != device:
        raise ValueError(f"{name}: expected a tensor on {device}")
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor of shape {shape}, got {tuple(t.shape)}")
    return t.data_ptr()


def _table(block_table: torch.Tensor, name: str, device) -> tuple[int, int]:
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError(f"{name}: block_table must be [B, max_pages]")
    B, M = block_table.shape
    _i32(block_table, f"{name}(block_table)", device, (B, M))
    if M == 0:
        raise ValueError(f"{name}: block_table has no columns")
    return B, M


def _cache(cache: torch.Tensor, name: str) -> tuple[int, int]:
    if not isinstance(cache, torch.Tensor) or not cache.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (no CPU fallback)")
    if cache.dtype != torch.uint8 or cache.dim() != 3 or cache.shape[2] != PAGE_HEAD_BYTES \
            or not cache.is_contiguous() or cache.data_ptr() % 16:
        raise ValueError(f"{name}: the cache must be a contiguous, 16-byte aligned uint8 tensor "
                         f"[num_pages, n_kv_heads, {PAGE_HEAD_BYTES}]")
    if cache.shape[0] == 0 or cache.shape[1] == 0:
        raise ValueError(f"{name}: the cache has no pages or no heads")
    return cache.shape[0], cache.shape[1]


def _on_device(fn):
    """Run on the device of the first argument (a tensor, or a list of tensors
    and then the block table) when that is not the current one."""
    def call(*args, **kw):
        t = args[0] if args else None
        if isinstance(t, (list, tuple)):
            t = args[1] if len(args) > 1 else None
        if isinstance(t, torch.Tensor) and t.is_cuda and t.device.index != torch.cuda.current_device():
            with torch.cuda.device(t.device):
                return fn(*args, **kw)
        return fn(*args, **kw)
    call.__name__, call.__doc__, call.__wrapped__ = fn.__name__, fn.__doc__, fn
    return call


def _start(device) -> int:
    from . import ops
    ops.init(device.index)
    return torch.cuda.current_stream().cuda_stream


def kv4_cache(num_pages: int, n_kv_heads: int, device=None) -> torch.Tensor:
    """An empty 4-bit cache: uint8 [num_pages, n_kv_heads, 8704] (head dim 128)."""
    if num_pages < 1 or n_kv_heads < 1:
        raise ValueError("kv4_cache: needs at least one page and one head")
    device = device or torch.device("cuda", torch.cuda.current_device())
    return torch.zeros((num_pages, n_kv_heads, PAGE_HEAD_BYTES), dtype=torch.uint8, device=device)


def _strides(t: torch.Tensor, name: str):
    B, S, H, D = t.shape
    if t.stride(3) != 1 or t.data_ptr() % 16:
        raise ValueError(f"{name}: the head dim must be contiguous and 16-byte aligned")
    st = [s if n > 1 else 0 for s, n in zip(t.stride()[:3], (B, S, H))]
    if any(s % 8 for s in st):
        raise ValueError(f"{name}: strides must be multiples of 8 elements, got {t.stride()}")
    return (C.c_int64 * 3)(*st)


@_on_device
def kv4_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
               start_pos: torch.Tensor, new_len: torch.Tensor | None = None) -> None:
    """Store the (already rotated) keys and values of S new tokens a sequence.

    k, v: bf16 [B, S, n_kv_heads, 128], the last axis contiguous (views into a
    fused projection's rows are fine); token s < new_len[b] (default: all S)
    goes to position start_pos[b] + s of sequence b. Other slots of the cache
    stay as they are."""
    P, H = _cache(cache, "kv4_append")
    B, M = _table(block_table, "kv4_append", cache.device)
    for n, t in (("k", k), ("v", v)):
        if not t.is_cuda or t.device != cache.device:
            raise ValueError(f"kv4_append({n}): expected a tensor on {cache.device}")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"kv4_append({n}): dtype {t.dtype} is not bfloat16")
        if t.dim() != 4 or t.shape[0] != B or t.shape[2] != H or t.shape[3] != HEAD_DIM:
            raise ValueError(f"kv4_append({n}): expected [{B}, S, {H}, {HEAD_DIM}], got {tuple(t.shape)}")
    if k.shape != v.shape:
        raise ValueError("kv4_append: k and v shapes differ")
    sp = _i32(start_pos, "kv4_append(start_pos)", cache.device, (B,))
    nl = _i32(new_len, "kv4_append(new_len)", cache.device, (B,)) if new_len is not None else None
    if k.numel() == 0:
        return
    ks, vs = _strides(k, "kv4_append(k)"), _strides(v, "kv4_append(v)")
    _lib.call("mb_kv4_append_bf16", k.data_ptr(), v.data_ptr(), ks, vs, cache.data_ptr(), P, H,
              block_table.data_ptr(), M, sp, nl, B, k.shape[1], _start(cache.device))


@_on_device
def kv4_gather(cache: torch.Tensor, block_table: torch.Tensor, start_pos: torch.Tensor, length: int,
               kv_len: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of positions start_pos[b] .. start_pos[b] + length - 1 as
    the numbers they stand for: fp32 [B, length, n_kv_heads, 128], zeros at
    positions kv_len[b] and later."""
    P, H = _cache(cache, "kv4_gather")
    B, M = _table(block_table, "kv4_gather", cache.device)
    sp = _i32(start_pos, "kv4_gather(start_pos)", cache.device, (B,))
    kl = _i32(kv_len, "kv4_gather(kv_len)", cache.device, (B,))
    if length < 0:
        raise ValueError("kv4_gather: negative length")
    k, v = (torch.empty((B, length, H, HEAD_DIM), dtype=torch.float32, device=cache.device)
            for _ in range(2))
    if k.numel():
        _lib.call("mb_kv4_gather_f32", cache.data_ptr(), P, H, block_table.data_ptr(), M, sp, kl, B,
                  length, k.data_ptr(), v.data_ptr(), _start(cache.device))
    return k, v


@_on_device
def attention_kv4(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                  kv_len: torch.Tensor, start_pos: torch.Tensor | None = None,
                  scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale * q k^T) v over the 4-bit cache (GQA, head dim 128).

    q: bf16 [B, S, n_heads, 128], or [B, n_heads, 128] for one token a sequence;
    heads contiguous, positions any multiple of 8 elements apart. Keys
    0..kv_len[b]-1 are seen; with start_pos, row s sees those at positions <=
    start_pos[b] + s (causal). A row that sees no key becomes zeros. scale:
    1/sqrt(128) by default."""
    P, H = _cache(cache, "attention_kv4")
    B, M = _table(block_table, "attention_kv4", cache.device)
    if q.dtype != torch.bfloat16:
        raise TypeError(f"attention_kv4(q): dtype {q.dtype} is not bfloat16")
    if q.device != cache.device:
        raise ValueError(f"attention_kv4(q): expected a tensor on {cache.device}")
    single = q.dim() == 3
    x = q.unsqueeze(1) if single else q
    if x.dim() != 4 or x.shape[0] != B or x.shape[3] != HEAD_DIM or x.shape[2] == 0 or x.shape[2] % H:
        raise ValueError(f"attention_kv4(q): expected [{B}, S, n_heads (a multiple of {H}), "
                         f"{HEAD_DIM}], got {tuple(q.shape)}")
    S, Hq = x.shape[1], x.shape[2]
    ldq = _row_stride(x, "attention_kv4(q)")
    kl = _i32(kv_len, "attention_kv4(kv_len)", cache.device, (B,))
    sp = _i32(start_pos, "attention_kv4(start_pos)", cache.device, (B,)) if start_pos is not None else None
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    elif out.dtype != torch.bfloat16 or out.device != q.device or out.shape != q.shape:
        raise ValueError("attention_kv4(out): expected a bf16 tensor of q's shape and device")
    if x.numel() == 0:
        return out
    ldo = _row_stride(out.unsqueeze(1) if single else out, "attention_kv4(out)")
    nb = _lib.lib().mb_attention_kv4_workspace_bytes(B, S, Hq, H, M)
    ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=q.device)
    _lib.call("mb_attention_kv4_bf16", x.data_ptr(), ldq, cache.data_ptr(), P, block_table.data_ptr(),
              M, kl, sp, B, S, Hq, H, HEAD_DIM, 1.0 / math.sqrt(HEAD_DIM) if scale is None else float(scale),
              out.data_ptr(), ldo, ws.data_ptr(), nb, _start(cache.device))
    return out


def _row_stride(x: torch.Tensor, name: str) -> int:
    """Elements between two positions' rows of [B, S, heads, 128], heads contiguous."""
    B, S, H, D = x.shape
    if x.numel() == 0:
        return H * D
    ld = x.stride(1) if S > 1 else (x.stride(0) if B > 1 else H * D)
    if x.stride(3) != 1 or (H > 1 and x.stride(2) != D) or (B > 1 and S > 1 and x.stride(0) != S * ld) \
            or ld < H * D or ld % 8 or x.data_ptr() % 16:
        raise ValueError(f"{name}: heads must be contiguous, positions evenly spaced (a multiple of 8 "
                         f"elements) and 16-byte aligned; got strides {x.stride()}")
    return ld


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def _meta(block_table, seq_len, page_refs, name):
    if not isinstance(block_table, torch.Tensor) or not block_table.is_cuda:
        raise ValueError(f"{name}: expected CUDA tensors (no CPU fallback)")
    dev = block_table.device
    B, M = _table(block_table, name, dev)
    if not isinstance(page_refs, torch.Tensor) or page_refs.dim() != 1:
        raise ValueError(f"{name}: page_refs must be [num_pages]")
    P = page_refs.shape[0]
    return dev, B, M, P, _i32(seq_len, f"{name}(seq_len)", dev, (B,)), _i32(
        page_refs, f"{name}(page_refs)", dev, (P,))


def _pools(pools, name, dev, P):
    n = len(pools)
    ptrs, sizes = (C.c_void_p * max(n, 1))(), (C.c_int64 * max(n, 1))()
    for i, t in enumerate(pools):
        if t.device != dev or not t.is_contiguous() or t.dim() < 1 or t.shape[0] != P:
            raise ValueError(f"{name}: pool {i} must be a contiguous tensor on {dev} with {P} pages")
        size = t.numel() * t.element_size() // P if P else 16
        if size == 0 or size % 16 or t.data_ptr() % 16:
            raise ValueError(f"{name}: pool {i}'s pages must be a multiple of 16 bytes and 16-byte aligned")
        ptrs[i], sizes[i] = t.data_ptr(), size
    if len(set(ptrs[:n])) < n:
        raise ValueError(f"{name}: the same pool twice")
    return ptrs, sizes, n


def _workspace(B, M, P, dev):
    nb = _lib.lib().mb_kv_pages_workspace_bytes(B, M, P)
    return torch.empty(nb, dtype=torch.uint8, device=dev), nb


@_on_device
def kv_pages_extend(block_table: torch.Tensor, seq_len: torch.Tensor, page_refs: torch.Tensor,
                    new_len: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Room for new_len[b] more tokens of every sequence, in place: new pages
    (the lowest-numbered free ones, in row order) enter block_table, seq_len
    grows. Returns (start_pos, status): the lengths before, and an int32 that is
    0, or the number of pages that were lacking, or -1 for a length out of range
    (then nothing was changed)."""
    name = "kv_pages_extend"
    dev, B, M, P, sl, pr = _meta(block_table, seq_len, page_refs, name)
    nl = _i32(new_len, f"{name}(new_len)", dev, (B,))
    start = torch.empty((B,), dtype=torch.int32, device=dev)
    status = torch.empty((1,), dtype=torch.int32, device=dev)
    ws, nb = _workspace(B, M, P, dev)
    _lib.call("mb_kv_pages_extend", block_table.data_ptr(), sl, pr, B, M, P, nl, start.data_ptr(),
              status.data_ptr(), ws.data_ptr(), nb, _start(dev))
    return start, status


@_on_device
def kv_pages_fork(pools, block_table: torch.Tensor, seq_len: torch.Tensor, page_refs: torch.Tensor,
                  parent: torch.Tensor) -> torch.Tensor:
    """Row b becomes a fork of row parent[b] as it was before the call, in
    place: its full pages are shared, a partly filled last page is copied (in
    every pool) into a page that was free. parent[b] == b: stays; -1: freed.
    pools: the page tensors [num_pages, ...] of all layers (bf16 or 4-bit).
    Returns an int32 status: 0, or the number of pages that were lacking, or -1
    for an index or length out of range (then nothing was changed)."""
    name = "kv_pages_fork"
    dev, B, M, P, sl, pr = _meta(block_table, seq_len, page_refs, name)
    pa = _i32(parent, f"{name}(parent)", dev, (B,))
    ptrs, sizes, n = _pools(pools, name, dev, P)
    status = torch.empty((1,), dtype=torch.int32, device=dev)
    ws, nb = _workspace(B, M, P, dev)
    _lib.call("mb_kv_pages_fork", ptrs, sizes, n, block_table.data_ptr(), sl, pr, B, M, P, pa,
              status.data_ptr(), ws.data_ptr(), nb, _start(dev))
    return status


@_on_device
def kv_pages_compact(pools, block_table: torch.Tensor, seq_len: torch.Tensor,
                     page_refs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Move the pages in use into 0..live-1, in place, with the fewest moves:
    those from `live` on go, in order, into the free ones below. Returns
    (remap, live): every page's new number (-1: was free) for references held
    outside the table, and the number of pages in use (-1: a table entry was
    out of range or not in use, and nothing was changed)."""
    name = "kv_pages_compact"
    dev, B, M, P, sl, pr = _meta(block_table, seq_len, page_refs, name)
    ptrs, sizes, n = _pools(pools, name, dev, P)
    remap = torch.empty((P,), dtype=torch.int32, device=dev)
    live = torch.empty((1,), dtype=torch.int32, device=dev)
    ws, nb = _workspace(B, M, P, dev)
    _lib.call("mb_kv_pages_compact", ptrs, sizes, n, block_table.data_ptr(), sl, pr, B, M, P,
              remap.data_ptr(), live.data_ptr(), ws.data_ptr(), nb, _start(dev))
    return remap, live
