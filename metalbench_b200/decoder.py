"""LLaMA decoder layer on libmb200 (torch tensors for device memory only).

Mirrors the reference hook ``mlx/kernels/full/llama_decoder_layer.py``:
``Model(S, D, H, H_kv, FF, base, eps).forward(x, W_qkv, W_o, W_gu, W_down)``,
weights in the reference (in, out) layout. ``DecoderLayer`` packs them once
(K-major, this rank's tensor-parallel shard) and runs the fused kernels;
``PagedKVCache`` holds the rotated keys and values of every sequence in
64-token pages; ``PagedKV4Cache`` holds them in 4 bits, for the layers of a
model together, with the pages' bookkeeping on the device.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib, ops

PAGE = 64


@dataclass
class DecoderConfig:
    d_model: int
    n_heads: int
    n_kv_heads: int
    ffn: int
    head_dim: int = 128
    rope_base: float = 10000.0
    eps: float = 1e-5

    def as_c(self) -> _lib.MbDecoderConfig:
        return _lib.MbDecoderConfig(self.d_model, self.n_heads, self.n_kv_heads, self.head_dim,
                                    self.ffn, float(self.rope_base), float(self.eps))


class PagedKVCache:
    """k, v: [num_pages, Hkv_local, 64, Dh] bf16; block_table [B, max_pages] int32.

    Sequence b owns pages b*max_pages .. b*max_pages+max_pages-1 (a simple
    contiguous assignment; any page permutation works with the kernels)."""

    def __init__(self, batch: int, max_len: int, n_kv_heads: int, head_dim: int = 128,
                 device=None, block_table: torch.Tensor | None = None):
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        self.batch = batch
        self.max_pages = (max_len + PAGE - 1) // PAGE
        n_pages = batch * self.max_pages
        shape = (n_pages, n_kv_heads, PAGE, head_dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        if block_table is None:
            block_table = torch.arange(n_pages, dtype=torch.int32, device=device).view(
                batch, self.max_pages)
        self.block_table = block_table.to(device=device, dtype=torch.int32).contiguous()
        self.max_len = self.max_pages * PAGE

    def write_positions(self, b: int, k: torch.Tensor, v: torch.Tensor, start: int = 0) -> None:
        """Store already-rotated k, v [Hkv, L, Dh] of sequence b at start.. (test/bench set-up)."""
        L = k.shape[1]
        for p in range(start, start + L):
            pg = int(self.block_table[b, p // PAGE])
            self.k[pg, :, p % PAGE] = k[:, p - start]
            self.v[pg, :, p % PAGE] = v[:, p - start]


class PagedKV4Cache:
    """The keys and values of ``n_layers`` layers in 4 bits (layout and rounding
    in include/mb200.h): one page pool a layer, uint8 [num_pages, Hkv, 8704],
    under one block table [batch, max_pages], sequence lengths and page use
    counts, all int32 on the device. Pages are given out as sequences grow,
    shared by forks and returned when the last sequence that holds them ends.

    A step is ``start = cache.extend(new_len)``, then for every layer either
    ``layer(x, cache.layer(i), start, ...)`` or ``append`` and ``attend``. Nothing is
    read back by the host, so steps can be captured in a CUDA graph;
    ``cache.status`` tells, when the program next looks, whether every page
    operation since ``clear_status`` was served (0), replayed ones too. One that
    was not changed nothing, and the tokens that had no room are not stored: the
    status is then the number of pages that were lacking (after several such
    operations the bits of their numbers together), or -1 for a length, parent or
    table entry out of range."""

    def __init__(self, batch: int, max_len: int, n_kv_heads: int, n_layers: int = 1,
                 num_pages: int | None = None, device=None):
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        if batch < 1 or max_len < 1 or n_layers < 1:
            raise ValueError("PagedKV4Cache: batch, max_len and n_layers must be at least 1")
        self.batch, self.n_layers = batch, n_layers
        self.max_pages = (max_len + PAGE - 1) // PAGE
        num_pages = batch * self.max_pages if num_pages is None else num_pages
        self.pools = [ops.kv4_cache(num_pages, n_kv_heads, device) for _ in range(n_layers)]
        self.block_table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=device)
        self.seq_len = torch.zeros(batch, dtype=torch.int32, device=device)
        self.page_refs = torch.zeros(num_pages, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def extend(self, new_len: torch.Tensor) -> torch.Tensor:
        """Room for new_len[b] more tokens a sequence; the positions of the first of them."""
        start, status = ops.kv_pages_extend(self.block_table, self.seq_len, self.page_refs, new_len)
        self.status.bitwise_or_(status)
        return start

    def fork(self, parent: torch.Tensor) -> None:
        """Row b becomes a fork of row parent[b] (its own number: stays; -1: is freed)."""
        self.status.bitwise_or_(ops.kv_pages_fork(self.pools, self.block_table, self.seq_len, self.page_refs,
                                                  parent))

    def compact(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Move the pages in use to the front of every pool: (new numbers, pages in use)."""
        remap, live = ops.kv_pages_compact(self.pools, self.block_table, self.seq_len, self.page_refs)
        self.status.bitwise_or_(live.clamp(max=0))
        return remap, live

    def clear_status(self) -> None:
        self.status.zero_()

    def append(self, i: int, k: torch.Tensor, v: torch.Tensor, start_pos: torch.Tensor,
               new_len: torch.Tensor | None = None) -> None:
        """Store layer i's keys and values [B, S, Hkv, 128] of the new tokens."""
        ops.kv4_append(k, v, self.pools[i], self.block_table, start_pos, new_len, self.seq_len)

    def attend(self, i: int, q: torch.Tensor, start_pos: torch.Tensor | None = None,
               scale: float | None = None, max_kv_len: int | None = None) -> torch.Tensor:
        """Layer i's attention of q [B, S, H, 128] over each sequence's tokens."""
        return ops.attention_kv4(q, self.pools[i], self.block_table, self.seq_len, start_pos, scale,
                                 max_kv_len=max_kv_len)

    def layer(self, i: int) -> "KV4Layer":
        return KV4Layer(self, i)


@dataclass
class KV4Layer:
    """One layer's part of a PagedKV4Cache, as a DecoderLayer takes it."""
    owner: PagedKV4Cache
    index: int


class DecoderLayer:
    def __init__(self, cfg: DecoderConfig, W_qkv: torch.Tensor, W_o: torch.Tensor,
                 W_gu: torch.Tensor, W_down: torch.Tensor, tp_rank: int = 0, tp_world: int = 1):
        for name, t in (("W_qkv", W_qkv), ("W_o", W_o), ("W_gu", W_gu), ("W_down", W_down)):
            ops._cuda(t, f"DecoderLayer({name})", (torch.bfloat16,))
        D, Dh = cfg.d_model, cfg.head_dim
        want = {"W_qkv": (D, D + 2 * cfg.n_kv_heads * Dh), "W_o": (D, D),
                "W_gu": (D, 2 * cfg.ffn), "W_down": (cfg.ffn, D)}
        for name, t in (("W_qkv", W_qkv), ("W_o", W_o), ("W_gu", W_gu), ("W_down", W_down)):
            if tuple(t.shape) != want[name]:
                raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {want[name]}")
        ops.init(W_qkv.device.index)
        self.cfg = cfg
        self.tp_rank, self.tp_world = tp_rank, tp_world
        self.h_kv_local = cfg.n_kv_heads // tp_world
        self.h_local = cfg.n_heads // tp_world
        h = C.c_void_p()
        _lib.call("mb_decoder_layer_create", C.byref(cfg.as_c()), W_qkv.data_ptr(), W_o.data_ptr(),
                  W_gu.data_ptr(), W_down.data_ptr(), tp_rank, tp_world, C.byref(h))
        self._h = h
        torch.cuda.synchronize()

    def close(self):
        if getattr(self, "_h", None):
            _lib.lib().mb_decoder_layer_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def workspace_bytes(self, B: int, S: int, max_kv_len: int) -> int:
        return _lib.lib().mb_decoder_layer_workspace_bytes(self._h, B, S, max_kv_len)

    def forward(self, x: torch.Tensor, cache: "PagedKVCache | KV4Layer", start_pos: torch.Tensor,
                causal: bool = True, out: torch.Tensor | None = None,
                max_kv_len: int | None = None, kv_len: torch.Tensor | None = None,
                x_res32: torch.Tensor | None = None,
                y_res32: torch.Tensor | None = None,
                rstd_in: torch.Tensor | None = None,
                rstd_out: torch.Tensor | None = None,
                new_len: torch.Tensor | None = None) -> torch.Tensor:
        """x: [B, S, D] bf16 (or [S, D] for B = 1); start_pos: int32 [B] on the device.

        The new tokens' keys/values are appended at start_pos[b].. and attention
        reads positions 0..start_pos[b]+S-1. kv_len (= start_pos + S, int32 on
        the device) may be passed in when several layers share it. x_res32 /
        y_res32 (fp32, x's shape) carry the residual stream in fp32 between
        layers: x_res32 is this layer's input residual (x its bf16 rounding),
        y_res32 receives the fp32 output. rstd_in / rstd_out (fp32, one entry
        per token) chain the input RMSNorm factor between layers: rstd_out
        receives rsqrt(mean(y_res32^2) + eps) for the next layer, which takes
        it as rstd_in instead of computing it (rstd_out needs y_res32).

        cache may be a layer of a PagedKV4Cache (``cache.layer(i)``), whose
        pages were extended for this step: keys and values are then held in 4
        bits, kv_len is the cache's seq_len, and new_len (int32 [B]) may say how
        many of the S tokens each sequence has (the rows of y behind them are
        unspecified)."""
        squeeze = x.dim() == 2
        X = x.unsqueeze(0) if squeeze else x
        ops._cuda(X, "DecoderLayer.forward(x)", (torch.bfloat16,))
        B, S, D = X.shape
        for nm, t in (("start_pos", start_pos), ("kv_len", kv_len), ("new_len", new_len)):
            if t is not None and (t.dtype != torch.int32 or t.device != X.device or t.numel() != B
                                  or not t.is_contiguous()):
                raise ValueError(f"{nm} must be a contiguous int32 CUDA tensor with one entry per sequence, "
                                 "on x's device")
        kv4 = isinstance(cache, KV4Layer)
        if kv4:
            own, pool = cache.owner, cache.owner.pools[cache.index]
            if own.batch != B or pool.shape[1] != self.h_kv_local or pool.device != X.device:
                raise ValueError("the 4-bit cache has another batch, number of kv heads or device")
            if kv_len is None:
                kv_len = own.seq_len
            if max_kv_len is None:
                max_kv_len = own.max_pages * PAGE  # the lengths are on the device
            ws_bytes = _lib.lib().mb_decoder_layer_workspace_bytes_kv4(self._h, B, S, max_kv_len)
            # a workspace of the call: captured graphs and other streams keep theirs
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=X.device)
        else:
            if new_len is not None:
                raise ValueError("new_len needs a 4-bit cache")
            if kv_len is None:
                kv_len = (start_pos + S).contiguous()
            if max_kv_len is None:
                max_kv_len = int(kv_len.max().item())
            ws_bytes = self.workspace_bytes(B, S, max_kv_len)
            ws = ops._workspace(ws_bytes, X.device)
        if out is None:
            out = torch.empty_like(X)
        self._kv_len = kv_len  # keep alive until the stream has consumed it
        for nm, t in (("x_res32", x_res32), ("y_res32", y_res32)):
            if t is not None:
                ops._cuda(t, f"DecoderLayer.forward({nm})", (torch.float32,))
                if t.numel() != X.numel():
                    raise ValueError(f"{nm} must have x's shape")
        for nm, t in (("rstd_in", rstd_in), ("rstd_out", rstd_out)):
            if t is not None:
                ops._cuda(t, f"DecoderLayer.forward({nm})", (torch.float32,))
                if t.numel() != B * S:
                    raise ValueError(f"{nm} must hold one float per token")
        if rstd_out is not None and y_res32 is None:
            raise ValueError("rstd_out needs y_res32")
        if kv4:
            ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
            _lib.call("mb_decoder_layer_forward_kv4", self._h, X.data_ptr(), ptr(x_res32), ptr(rstd_in),
                      out.data_ptr(), ptr(y_res32), ptr(rstd_out), B, S, start_pos.data_ptr(),
                      kv_len.data_ptr(), max_kv_len, ptr(new_len), pool.data_ptr(), pool.shape[0],
                      own.block_table.data_ptr(), own.max_pages, 1 if causal else 0, ws.data_ptr(),
                      ws_bytes, ops._stream())
            return out[0] if squeeze else out
        _lib.call("mb_decoder_layer_forward_chain", self._h, X.data_ptr(),
                  0 if x_res32 is None else x_res32.data_ptr(),
                  0 if rstd_in is None else rstd_in.data_ptr(), out.data_ptr(),
                  0 if y_res32 is None else y_res32.data_ptr(),
                  0 if rstd_out is None else rstd_out.data_ptr(), B, S,
                  start_pos.data_ptr(), kv_len.data_ptr(), max_kv_len, cache.k.data_ptr(),
                  cache.v.data_ptr(), cache.block_table.data_ptr(), cache.max_pages,
                  1 if causal else 0, ws.data_ptr(), ws_bytes, ops._stream())
        return out[0] if squeeze else out

    __call__ = forward
