"""Measured cases of the 4-bit paged KV cache: storing tokens in it, attention
over it, and the page operations of a serving loop (fork and free, compaction).

A page holds 64 tokens. The 4-bit cache is uint8 [num_pages, Hkv, 8704]; the
8704 bytes of one page and one kv head (head dim 128) are

    [0, 4096)     key codes: token t at byte 64 t, byte j = dim 2j (low four
                  bits) and dim 2j + 1 (high four bits)
    [4096, 8192)  value codes, the same, but the 16-byte piece c of token t
                  stands at piece c ^ ((t >> 1) & 3)
    [8192, 8448)  per token: bf16 scale, bf16 minimum of the key
    [8448, 8704)  per token: bf16 scale, bf16 minimum of the value

and the value that a code u stands for is minimum + scale * u, with
minimum = min(x), scale = bf16((max(x) - min(x)) / 15) over the token's 128
dims and u = (x - minimum) / scale rounded to the nearest whole number (ties to
even) and clamped to 0..15; u = 0 where scale = 0.

`own` False: the operators in elementary torch operations. `own` True: the
calls a user makes of metalbench_b200.ops.
"""
import math

import numpy as np
import torch

own = False

PAGE, DIM, BLOB = 64, 128, 8704


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one user's decode step: a single short sequence, where latency counts
        dict(name="attend 1 x 517", kind="attend", batch=1, rows=1, hq=32, hkv=8, lo=517, hi=517, empty=0),
        # the decode step of the 8-layer stack that bench.py runs (one layer)
        dict(name="attend 64 x 8193", kind="attend", batch=64, rows=1, hq=64, hkv=8, lo=8193, hi=8193, empty=0),
        # continuous batching: lengths from a few tokens to long ones, some slots of the batch empty
        dict(name="attend ragged 48", kind="attend", batch=48, rows=1, hq=32, hkv=8, lo=3, hi=16000, empty=5),
        # one long document
        dict(name="attend 1 x 131075", kind="attend", batch=1, rows=1, hq=64, hkv=8, lo=131075, hi=131075, empty=0),
        # checking four drafted tokens a sequence at once
        dict(name="attend 16 x 4 rows", kind="attend", batch=16, rows=4, hq=32, hkv=8, lo=2000, hi=4100, empty=0),
        # a piece of a long prompt, after what is in the cache already
        dict(name="attend prompt piece", kind="attend", batch=2, rows=512, hq=32, hkv=8, lo=8000, hi=8192, empty=0),
        # storing the new token of every sequence of a decode batch
        dict(name="store 64 x 1", kind="store", batch=64, rows=1, hkv=8, before=8192, ragged=False),
        # storing whole prompts (the prefill size of the decoder layer), padded to the longest
        dict(name="store 4 x 2048", kind="store", batch=4, rows=2048, hkv=8, before=0, ragged=True),
        # four beams of one short request
        dict(name="fork 4 beams", kind="fork", batch=4, length=300, moved=3, dropped=0, pools=2, page_kib=68, spare=16),
        # a batch whose sequences branch and end, eight layers' caches
        dict(name="fork 64 of 96", kind="fork", batch=96, length=2048, moved=64, dropped=12, pools=8, page_kib=68, spare=200),
        # a small pool after a few requests ended
        dict(name="compact 256 pages", kind="compact", batch=8, pages=256, used=0.6, pools=2, page_kib=68),
        # a large pool after many did
        dict(name="compact 8192 pages", kind="compact", batch=128, pages=8192, used=0.55, pools=4, page_kib=68),
    ]


def _spread(rng, lo, hi):
    """A whole number in lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "store", "fork", "compact"))
    if kind == "attend":
        hkv = rng.choice((1, 2, 4, 8))
        hq = hkv * rng.choice((1, 2, 3, 4, 5, 8, 16))
        rows = rng.choice((1, 1, 1, 2, 3, 5, _spread(rng, 2, 512)))
        batch = _spread(rng, 1, 64)
        # keys in all: at most the largest listed case's; query rows times keys: at most the prompt piece's
        most = min(131075, 64 * 8193 * 8 // (batch * hkv), 2 * 512 * 32 * 8192 // (batch * rows * hq))
        hi = _spread(rng, 1, max(1, most))
        lo = rng.choice((hi, _spread(rng, 1, hi)))
        return dict(kind=kind, batch=batch, rows=rows, hq=hq, hkv=hkv, lo=lo, hi=hi, empty=rng.randint(0, batch // 4))
    if kind == "store":
        batch, hkv = _spread(rng, 1, 64), rng.choice((1, 2, 4, 8))
        rows = _spread(rng, 1, max(1, 4 * 2048 * 8 // (batch * hkv)))
        return dict(kind=kind, batch=batch, rows=rows, hkv=hkv, before=rng.choice((0, _spread(rng, 1, 8192))), ragged=rng.random() < 0.5)
    pools, page_kib = rng.choice((1, 2, 4, 8)), rng.choice((17, 34, 68, 128))
    if kind == "fork":
        batch = _spread(rng, 2, 96)
        moved = rng.randint(1, max(1, 64 * 68 * 8 // max(64 * 68 * 8 // batch, pools * page_kib)))
        moved = min(moved, batch)
        return dict(kind=kind, batch=batch, length=_spread(rng, 1, 2048), moved=moved, dropped=rng.randint(0, (batch - moved) // 2), pools=pools,
                    page_kib=page_kib, spare=moved + rng.randint(0, 99))
    pages = _spread(rng, 16, 8192 * 68 * 4 // (pools * page_kib))
    return dict(kind=kind, batch=_spread(rng, 1, 128), pages=min(pages, 8192), used=round(rng.uniform(0.05, 0.95), 2), pools=pools, page_kib=page_kib)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case, seed):
    rs = np.random.RandomState(seed % (1 << 31))
    lens = np.exp(rs.uniform(math.log(case["lo"]), math.log(case["hi"] + 1e-3), case["batch"])).round().astype(np.int64)
    lens = np.clip(lens, case["lo"], case["hi"])
    lens[rs.permutation(case["batch"])[: case["empty"]]] = 0
    return lens, rs


def _pack_pages(k, v):
    """bf16 k, v [n, hkv, 64, 128] as cache pages uint8 [n, hkv, 8704]."""
    out = torch.empty(k.shape[:2] + (BLOB,), dtype=torch.uint8, device=k.device)
    for at, par, x in ((0, 8192, k), (4096, 8448, v)):
        codes, scale, low = _quantised(x)
        codes = codes.to(torch.uint8)
        packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
        if at:
            t = torch.arange(PAGE, device=k.device)
            piece = torch.arange(4, device=k.device)[None, :] ^ ((t[:, None] >> 1) & 3)
            packed = packed.view(packed.shape[:-1] + (4, 16)).gather(-2, piece[None, None, :, :, None].expand(packed.shape[:-1] + (4, 16))).flatten(-2)
        out[..., at: at + 4096] = packed.flatten(-2)
        out[..., par: par + 256] = torch.stack((scale, low), -1).to(torch.bfloat16).contiguous().view(torch.uint8).flatten(-2)
    return out


def _random_cache(g, pages, hkv, device):
    """A filled cache: keys with some strong channels, values without."""
    cache = torch.empty((pages, hkv, BLOB), dtype=torch.uint8, device=device)
    strength = 0.5 + 2.0 * torch.rand((hkv, 1, DIM), generator=g, device=device) ** 4
    centre = 0.5 * torch.randn((hkv, 1, DIM), generator=g, device=device)
    for a in range(0, pages, 2048):
        n = min(2048, pages - a)
        k = torch.randn((n, hkv, PAGE, DIM), generator=g, device=device) * strength + centre
        v = torch.randn((n, hkv, PAGE, DIM), generator=g, device=device)
        cache[a: a + n] = _pack_pages(k.to(torch.bfloat16), v.to(torch.bfloat16))
    return cache


def _tables(rs, counts, num_pages, most, shared=0):
    """Block table [B, most] with counts[b] pages a row, the first `shared` of
    a row those of row 0, pages in any order; how often each page is used."""
    table = np.full((len(counts), most), -1, dtype=np.int32)
    order = rs.permutation(num_pages).astype(np.int32)
    at = 0
    for b, n in enumerate(counts):
        s = min(shared, n, counts[0]) if b else 0
        table[b, :s] = table[0, :s]
        table[b, s:n] = order[at: at + n - s]
        at += n - s
    used = table[np.arange(most)[None, :] < np.asarray(counts)[:, None]]
    return table, np.bincount(used, minlength=num_pages).astype(np.int32)


def _meta(table, lens, refs):
    """Block table, lengths and page uses as three views of one buffer (and a
    copy that holds the start of a pass)."""
    flat = torch.from_numpy(np.concatenate([table.ravel(), np.asarray(lens, dtype=np.int32), refs])).cuda()
    work = flat.clone()
    n, b = table.size, len(lens)
    return dict(start=flat, work=work, table=work[:n].view(table.shape), lens=work[n: n + b], refs=work[n + b:])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(kind=case["kind"], case=case)
    if case["kind"] == "attend":
        lens, rs = _lengths(case, seed)
        counts = -(-lens // PAGE)
        num = int(counts.sum()) + 3
        table, _ = _tables(rs, counts, num, max(1, int(counts.max())))
        st["cache"] = _random_cache(g, num, case["hkv"], "cuda")
        st["table"] = torch.from_numpy(table).cuda()
        st["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        st["first"] = (st["lens"] - case["rows"]).clamp(min=0)
        q = torch.randn((case["batch"], case["rows"], case["hq"], DIM), generator=g, device="cuda") * 1.5
        st["q"] = q.to(torch.bfloat16)
    elif case["kind"] == "store":
        rs = np.random.RandomState(seed % (1 << 31))
        B, S = case["batch"], case["rows"]
        before = np.maximum(0, case["before"] - rs.randint(0, PAGE, B)) if case["before"] else np.zeros(B, dtype=np.int64)
        new = rs.randint(S // 4, S + 1, B) if case["ragged"] else np.full(B, S)
        counts = -(-before // PAGE)
        most = -(-(case["before"] + S) // PAGE)
        num = B * most + 5
        table, refs = _tables(rs, counts, num, most)
        st["meta"] = _meta(table, before, refs)
        st["new"] = torch.from_numpy(new.astype(np.int32)).cuda()
        st["cache"] = torch.zeros((num, case["hkv"], BLOB), dtype=torch.uint8, device="cuda")
        for n in ("k", "v"):
            # the keys and values of a token lie in one row of a fused projection's output
            row = torch.randn((B, S, 3 * case["hkv"], DIM), generator=g, device="cuda").to(torch.bfloat16)
            st[n] = row[:, :, case["hkv"]: 2 * case["hkv"]]
    elif case["kind"] == "fork":
        rs = np.random.RandomState(seed % (1 << 31))
        B = case["batch"]
        lens = rs.randint(max(1, case["length"] // 2), case["length"] + 1, B)
        counts = -(-lens // PAGE)
        shared = int(min(lens) // PAGE) // 2
        most = -(-case["length"] // PAGE)
        table, refs = _tables(rs, counts, B * most + case["spare"], most, shared)
        st["meta"] = _meta(table, lens, refs)
        parent = np.arange(B)
        rows = rs.permutation(B)
        parent[rows[: case["moved"]]] = rs.randint(0, B, case["moved"])
        parent[rows[case["moved"]: case["moved"] + case["dropped"]]] = -1
        st["parent"] = torch.from_numpy(parent.astype(np.int32)).cuda()
        st["pools"] = _pools(g, case, len(refs))
    else:
        rs = np.random.RandomState(seed % (1 << 31))
        B, P = case["batch"], case["pages"]
        share = np.arange(1, B + 1) / (B * (B + 1) / 2)  # some sequences are much longer than others
        counts = rs.permutation((share * P * case["used"]).astype(np.int64))
        lens = np.maximum(0, counts * PAGE - rs.randint(0, PAGE, B))
        table, refs = _tables(rs, counts, P, int(counts.max()) + 1)
        st["meta"] = _meta(table, lens, refs)
        st["pools"] = _pools(g, case, P)
    return st


def _pools(g, case, pages):
    return [torch.randint(0, 256, (pages, case["page_kib"] * 1024), generator=g, device="cuda", dtype=torch.uint8) for _ in range(case["pools"])]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    if own:
        from metalbench_b200 import ops
        if st["kind"] == "attend":
            return ops.attention_kv4(st["q"], st["cache"], st["table"], st["lens"], start_pos=st["first"])
        m = st["meta"]
        m["work"].copy_(m["start"])
        if st["kind"] == "store":
            start, status = ops.kv_pages_extend(m["table"], m["lens"], m["refs"], st["new"])
            ops.kv4_append(st["k"], st["v"], st["cache"], m["table"], start, new_len=st["new"])
            k, v = ops.kv4_gather(st["cache"], m["table"], start, st["k"].shape[1], kv_len=m["lens"])
            return dict(k=k, v=v, table=m["table"], lens=m["lens"], refs=m["refs"], status=status)
        if st["kind"] == "fork":
            status = ops.kv_pages_fork(st["pools"], m["table"], m["lens"], m["refs"], st["parent"])
            return dict(pools=st["pools"], table=m["table"], lens=m["lens"], refs=m["refs"], status=status)
        remap, live = ops.kv_pages_compact(st["pools"], m["table"], m["lens"], m["refs"])
        return dict(pools=st["pools"], table=m["table"], refs=m["refs"], remap=remap, live=live)
    if st["kind"] == "attend":
        return _attend(st["q"], st["cache"], st["table"], st["lens"], st["first"])
    m = st["meta"]
    m["work"].copy_(m["start"])
    if st["kind"] == "store":
        start = m["lens"].clone()
        status = _extend(m["table"], m["lens"], m["refs"], st["new"])
        _store(st["k"], st["v"], st["cache"], m["table"], start, st["new"])
        k, v = _gather(st["cache"], m["table"], start, st["k"].shape[1], m["lens"])
        return dict(k=k, v=v, table=m["table"], lens=m["lens"], refs=m["refs"], status=status)
    if st["kind"] == "fork":
        status = _fork(st["pools"], m["table"], m["lens"], m["refs"], st["parent"])
        return dict(pools=st["pools"], table=m["table"], lens=m["lens"], refs=m["refs"], status=status)
    remap, live = _compact(st["pools"], m["table"], m["lens"], m["refs"])
    return dict(pools=st["pools"], table=m["table"], refs=m["refs"], remap=remap, live=live)


def _quantised(x):
    """Codes, scale and minimum over the last axis (64 bits: a code's border
    must not move with the rounding of the division)."""
    x = x.double()
    low, high = x.amin(-1), x.amax(-1)
    scale = ((high - low) / 15).to(torch.bfloat16).double()
    u = torch.where(scale[..., None] > 0, (x - low[..., None]) / scale[..., None], 0.0)
    return u.round().clamp(0, 15), scale, low


def _codes(packed):
    """uint8 [..., 64] as float32 codes [..., 128]."""
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2).float()


def _unpack(pages):
    """Cache pages [..., 8704] as float32 keys and values [..., 64, 128]."""
    t = torch.arange(PAGE, device=pages.device)
    piece = torch.arange(4, device=pages.device)[None, :] ^ ((t[:, None] >> 1) & 3)
    kc = pages[..., :4096].unflatten(-1, (PAGE, 64))
    vc = pages[..., 4096:8192].unflatten(-1, (PAGE, 4, 16))
    vc = vc[..., t[:, None], piece, :].flatten(-2)
    par = pages[..., 8192:].contiguous().view(torch.bfloat16).unflatten(-1, (2, PAGE, 2)).float()
    k = par[..., 0, :, 1:] + par[..., 0, :, :1] * _codes(kc)
    v = par[..., 1, :, 1:] + par[..., 1, :, :1] * _codes(vc)
    return k, v


def _attend(q, cache, table, lens, first):
    B, S, H, D = q.shape
    hkv = cache.shape[1]
    G = H // hkv
    k, v = _unpack(cache[table.clamp(min=0)])  # [B, pages, hkv, 64, 128]
    k, v = (x.transpose(1, 2).reshape(B, hkv, -1, D) for x in (k, v))
    qs = q.float().view(B, S, hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, hkv, S * G, D)
    s = (qs @ k.transpose(-1, -2)) / math.sqrt(D)
    del k
    pos = torch.arange(s.shape[-1], device=q.device)
    row = torch.arange(S, device=q.device).repeat_interleave(G)
    last = torch.minimum(lens[:, None] - 1, first[:, None] + row[None, :])  # [B, S*G]
    ok = pos[None, None, :] <= last[:, :, None]
    s = s.masked_fill(~ok[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    del s
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill((pos[None, :] >= lens[:, None])[:, None, :, None], 0.0)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    return o.view(B, hkv, S, G, D).permute(0, 2, 1, 3, 4).reshape(B, S, H, D).to(torch.bfloat16)


def _places(table, start, new, S):
    """Page and slot of each of S new tokens, and which of them are there."""
    s = torch.arange(S, device=table.device)
    pos = start.long()[:, None] + s[None, :]
    ok = s[None, :] < new[:, None]
    page = table.long().gather(1, (pos // PAGE).clamp(max=table.shape[1] - 1))
    return page, pos % PAGE, ok


def _store(k, v, cache, table, start, new):
    page, slot, ok = _places(table, start, new, k.shape[1])
    page, slot = page[ok], slot[ok]
    for at, par, x in ((0, 8192, k), (4096, 8448, v)):
        codes, scale, low = _quantised(x[ok])  # [n, hkv, 128]
        codes = codes.to(torch.uint8)
        packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
        if at:
            piece = torch.arange(4, device=k.device)[None, :] ^ ((slot[:, None] >> 1) & 3)
            packed = packed.unflatten(-1, (4, 16)).gather(-2, piece[:, None, :, None].expand(-1, packed.shape[1], -1, 16)).flatten(-2)
        cache[:, :, at: at + 4096].unflatten(-1, (PAGE, 64))[page, :, slot] = packed
        pars = torch.stack((scale, low), -1).to(torch.bfloat16).view(torch.uint8)
        cache[:, :, par: par + 256].unflatten(-1, (PAGE, 4))[page, :, slot] = pars


def _gather(cache, table, start, S, lens):
    page, slot, ok = _places(table, start, lens - start, S)
    kv = []
    for at, par in ((0, 8192), (4096, 8448)):
        p = page.clamp(min=0)
        packed = cache[:, :, at: at + 4096].unflatten(-1, (PAGE, 64))[p, :, slot]  # [B, S, hkv, 64]
        if at:
            piece = torch.arange(4, device=cache.device) ^ ((slot[..., None] >> 1) & 3)
            packed = packed.unflatten(-1, (4, 16)).gather(-2, piece[:, :, None, :, None].expand(-1, -1, packed.shape[2], -1, 16)).flatten(-2)
        pars = cache[:, :, par: par + 256].unflatten(-1, (PAGE, 4))[p, :, slot].contiguous().view(torch.bfloat16).float()
        x = pars[..., 1:] + pars[..., :1] * _codes(packed)
        kv.append(torch.where(ok[:, :, None, None], x, 0.0))
    return kv


def _pages_of(lens):
    return (lens + PAGE - 1) // PAGE


def _extend(table, lens, refs, new):
    old, then = _pages_of(lens), _pages_of(lens + new)
    need = then - old
    short = (need.sum() - (refs == 0).sum()).clamp(min=0)
    order = torch.argsort((refs != 0).to(torch.uint8), stable=True).to(torch.int32)  # free pages first, lowest first
    col = torch.arange(table.shape[1], device=table.device)
    fresh = (col[None, :] >= old[:, None]) & (col[None, :] < then[:, None]) & (short == 0)
    nth = (need.cumsum(0) - need)[:, None] + col[None, :] - old[:, None]
    page = order[nth.clamp(0, len(order) - 1)]
    table.copy_(torch.where(fresh, page, table))
    refs.index_add_(0, torch.where(fresh, page, 0).flatten().long(), fresh.flatten().to(torch.int32))
    lens.add_(torch.where(short == 0, new, 0))
    return short.to(torch.int32).view(1)


def _fork(pools, table, lens, refs, parent):
    B, M = table.shape
    moved, gone = parent != torch.arange(B, device=table.device), parent < 0
    src = parent.clamp(min=0).long()
    length = torch.where(gone, 0, lens[src])
    tail = moved & ~gone & (length % PAGE != 0)
    short = (tail.sum() - (refs == 0).sum()).clamp(min=0)
    fine = short == 0
    order = torch.argsort((refs != 0).to(torch.uint8), stable=True).to(torch.int32)
    page = order[(tail.cumsum(0) - 1).clamp(0, len(order) - 1)]
    col = torch.arange(M, device=table.device)
    last = (length // PAGE).long()
    old_use = (col[None, :] < _pages_of(lens)[:, None]) & moved[:, None] & fine
    new_use = (col[None, :] < _pages_of(length)[:, None]) & moved[:, None] & fine
    rows = table[src]
    copied = rows.gather(1, last.clamp(max=M - 1)[:, None])[:, 0]  # the page that a tail is copied from
    rows = torch.where((col[None, :] == last[:, None]) & tail[:, None], page[:, None], rows)
    refs.index_add_(0, torch.where(old_use, table, 0).flatten().long(), -old_use.flatten().to(torch.int32))
    refs.index_add_(0, torch.where(new_use, rows, 0).flatten().long(), new_use.flatten().to(torch.int32))
    table.copy_(torch.where(new_use, rows, table))
    lens.copy_(torch.where(fine & moved, length, lens))
    at = (tail & fine).nonzero()[:, 0]
    to, of = page[at].long(), copied[at].long()
    for pool in pools:
        pool[to] = pool[of]
    return short.to(torch.int32).view(1)


def _compact(pools, table, lens, refs):
    P = len(refs)
    used = refs > 0
    live = used.sum()
    at = torch.arange(P, device=refs.device)
    holes = (~used & (at < live)).nonzero()[:, 0]
    movers = (used & (at >= live)).nonzero()[:, 0]
    remap = torch.where(used, at, -1)
    remap[movers] = holes
    for pool in pools:
        pool[holes] = pool[movers]
    col = torch.arange(table.shape[1], device=table.device)
    valid = col[None, :] < _pages_of(lens)[:, None]
    table.copy_(torch.where(valid, remap[torch.where(valid, table, 0).long()].to(torch.int32), table))
    moved = refs[movers]
    refs[movers] = 0
    refs[holes] = moved
    return remap.to(torch.int32), live.to(torch.int32).view(1)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "attend":
        live, rows = case["batch"] - case["empty"], case["rows"]
        lo, hi = case["lo"], case["hi"]
        keys = live * (lo if lo == hi else (hi - lo) / math.log(hi / lo))
        io = 2 * 2 * case["batch"] * rows * case["hq"] * DIM
        return dict(bytes=keys * case["hkv"] * 136 + io, flops=4 * keys * rows * case["hq"] * DIM)
    if case["kind"] == "store":
        tokens = case["batch"] * case["rows"] * (0.625 if case["ragged"] and case["rows"] > 1 else 1.0)
        # read in bf16, stored in 4 bits, and read back as float32 (rows that are not there as zeros)
        moved = tokens * case["hkv"] * (4 * DIM + 2 * 136) + case["batch"] * case["rows"] * case["hkv"] * 8 * DIM
        return dict(bytes=moved, flops=tokens * case["hkv"] * DIM * 10)
    page = case["page_kib"] * 1024 * case["pools"]
    if case["kind"] == "fork":
        pages = case["moved"] * (1 - 1 / case["batch"]) * 63 / 64
        return dict(bytes=2 * page * pages + 8 * case["batch"] * (case["length"] // PAGE + 1), flops=case["batch"])
    pages = case["pages"] * case["used"] * (1 - case["used"])
    return dict(bytes=2 * page * pages + 12 * case["pages"], flops=case["pages"])


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "attend":
        st = prepare(case, seed)
        B, S, H = case["batch"], case["rows"], case["hq"]
        out = torch.zeros((B, S, H, DIM), dtype=torch.float64, device="cuda")
        word = torch.arange(DIM, device="cuda")
        for b, n in enumerate(st["lens"].tolist()):
            if not n:
                continue
            blob = st["cache"][st["table"][b, : -(-n // PAGE)].long()].long()  # [pages, hkv, 8704]
            tok = torch.arange(n, device="cuda")
            pg, t = tok // PAGE, tok % PAGE
            par = st["cache"][st["table"][b, : -(-n // PAGE)].long()][:, :, 8192:].contiguous().view(torch.bfloat16).double()
            for h in range(case["hkv"]):
                byte = t[:, None] * 64 + word[None, :] // 2
                key = (blob[pg[:, None], h, byte] >> (4 * (word % 2))) % 16
                piece = (word[None, :] // 32) ^ ((t[:, None] // 2) % 4)
                byte = 4096 + t[:, None] * 64 + piece * 16 + (word[None, :] % 32) // 2
                val = (blob[pg[:, None], h, byte] >> (4 * (word % 2))) % 16
                key = par[pg, h, 2 * t + 1][:, None] + par[pg, h, 2 * t][:, None] * key
                val = par[pg, h, 128 + 2 * t + 1][:, None] + par[pg, h, 128 + 2 * t][:, None] * val
                G = H // case["hkv"]
                q = st["q"][b, :, h * G: (h + 1) * G].double()
                w = torch.einsum("sgd,nd->sgn", q, key) / DIM ** 0.5
                seen = tok[None, :] <= st["first"][b].item() + torch.arange(S, device="cuda")[:, None]
                w = torch.softmax(w.masked_fill(~seen[:, None, :], -math.inf), -1)
                out[b, :, h * G: (h + 1) * G] = torch.einsum("sgn,nd->sgd", w, val)
        return out
    if case["kind"] == "store":
        st = prepare(case, seed)
        kv = []
        for x in (st["k"], st["v"]):
            x = x.double()
            low = x.min(-1, keepdim=True).values
            step = ((x.max(-1, keepdim=True).values - low) / 15).bfloat16().double()
            u = ((x - low) / step.where(step > 0, torch.ones_like(step))).round().clamp(max=15.0)
            there = torch.arange(x.shape[1], device="cuda")[None, :] < st["new"][:, None]
            kv.append((low + step * u) * there[:, :, None, None])
        return dict(k=kv[0], v=kv[1], table=None, lens=None, refs=None, status=None)
    return None
