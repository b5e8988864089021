"""Plain implementations (64 bits, host) of the 4-bit paged cache and of the
page operations, from their definitions in include/mb200.h."""
import numpy as np

PAGE, DIM, BLOB = 64, 128, 8704


def bf16_round(x):
    """Nearest bf16 (ties to even) of float64 values, as float64."""
    import torch
    return torch.from_numpy(np.asarray(x, dtype=np.float64)).to(torch.bfloat16).double().numpy()


def bf16_bits(x):
    import torch
    return torch.from_numpy(np.asarray(x, dtype=np.float64)).to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)


def quantise(x):
    """x [..., 128] -> codes (uint8), scale, minimum (float64)."""
    x = np.asarray(x, dtype=np.float64)
    low = x.min(-1)
    scale = bf16_round((x.max(-1) - low) / 15)
    div = np.where(scale > 0, scale, 1.0)[..., None]
    u = np.where(scale[..., None] > 0, np.rint((x - low[..., None]) / div), 0.0)
    return np.clip(u, 0, 15).astype(np.uint8), scale, low


def put_token(blob, t, k, v):
    """Store one token's key and value [128] into slot t of a page-and-head blob."""
    for at, par, x in ((0, 8192, k), (4096, 8448, v)):
        u, s, m = quantise(x)
        row = u[0::2] | (u[1::2] << 4)
        if at:
            row = row.reshape(4, 16)
            row = np.stack([row[c ^ ((t >> 1) & 3)] for c in range(4)]).reshape(-1)
        blob[at + 64 * t: at + 64 * t + 64] = row
        blob[par + 4 * t: par + 4 * t + 4] = np.array([bf16_bits(s), bf16_bits(m)], dtype=np.uint16).view(np.uint8)


def get_pages(pages):
    """uint8 [n, 8704] -> dict of keys' and values' codes, scales, minima, each [n, 64, ...] float64."""
    n = pages.shape[0]
    out = {}
    for name, at, par in (("k", 0, 8192), ("v", 4096, 8448)):
        row = pages[:, at: at + 4096].reshape(n, PAGE, 4, 16)
        if at:
            t = np.arange(PAGE)
            row = row[:, t[:, None], np.arange(4)[None] ^ ((t[:, None] >> 1) & 3)]
        row = row.reshape(n, PAGE, 64)
        u = np.stack([row & 15, row >> 4], -1).reshape(n, PAGE, DIM).astype(np.float64)
        p = pages[:, par: par + 256].copy().view(np.uint16).reshape(n, PAGE, 2).astype(np.uint32) << 16
        p = p.view(np.float32).astype(np.float64)
        out[name] = (u, p[..., 0], p[..., 1])
    return out


def attention(q, cache, table, lens, first, scale=DIM ** -0.5):
    """Outputs [B, S, Hq, 128] and, beside each, how far fp32 sums, an fp16
    rounding of every softmax weight and fp32 scores can move it."""
    B, S, Hq, _ = q.shape
    H = cache.shape[1]
    G = Hq // H
    out, slack = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        ids = table[b, : -(-n // PAGE)]
        for h in range(H):
            got = get_pages(cache[ids, h])
            (ku, ks, km), (vu, vs, vm) = ((a.reshape(-1, DIM)[:n], s.reshape(-1)[:n], m.reshape(-1)[:n])
                                          for a, s, m in (got["k"], got["v"]))
            for s in range(S):
                end = n if first is None else min(n, int(first[b]) + s + 1)
                if end <= 0:
                    continue
                for g in range(G):
                    x = q[b, s, h * G + g].astype(np.float64)
                    sc = scale * (ks[:end] * (ku[:end] @ x) + km[:end] * x.sum())
                    mag = scale * (ks[:end] * (ku[:end] @ np.abs(x)) + np.abs(km[:end] * x.sum()))
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    out[b, s, h * G + g] = (p * vs[:end]) @ vu[:end] + p @ vm[:end]
                    size = (p * vs[:end]) @ vu[:end] + p @ np.abs(vm[:end])
                    # an fp32 sum of 128 products, truncated: 128 * 2^-23 of its absolute sum; each
                    # weight rounded to fp16 (2^-11); n/16 accumulations, each within 2^-23; exp2, log2
                    # and the division 2^-16
                    rel = 2 ** -11 + 2 * mag.max() * 2 ** -16 + (end / 16) * 2 ** -23 + 2 ** -16
                    slack[b, s, h * G + g] = rel * size
    return out, slack


# ---- page operations ----------------------------------------------------------
def pages_of(n):
    return -(-n // PAGE)


class Pages:
    """Block table, lengths and uses; every method returns the status and
    changes nothing unless that is 0 (compact: not negative)."""

    def __init__(self, table, lens, refs):
        self.table, self.lens, self.refs = table.copy(), lens.copy(), refs.copy()

    def free(self):
        return [int(p) for p in np.nonzero(self.refs == 0)[0]]

    def extend(self, new):
        B, M = self.table.shape
        for b in range(B):
            if self.lens[b] < 0 or new[b] < 0 or int(self.lens[b]) + int(new[b]) > M * PAGE:
                return -1
        need = [pages_of(int(l) + int(n)) - pages_of(int(l)) for l, n in zip(self.lens, new)]
        free = self.free()
        if sum(need) > len(free):
            return sum(need) - len(free)
        for b in range(B):
            old = pages_of(int(self.lens[b]))
            for i in range(need[b]):
                p = free.pop(0)
                self.table[b, old + i] = p
                self.refs[p] = 1
            self.lens[b] += new[b]
        return 0

    def fork(self, parent, pools):
        B, M = self.table.shape
        P = len(self.refs)
        for b in range(B):
            p = int(parent[b])
            if p < -1 or p >= B or not 0 <= self.lens[b] <= M * PAGE:
                return -1
            for r in {b, p} - {-1}:
                if p != b:
                    row = self.table[r, : pages_of(int(self.lens[r]))]
                    if ((row < 0) | (row >= P)).any():
                        return -1
        tails = [b for b in range(B) if parent[b] >= 0 and parent[b] != b and self.lens[parent[b]] % PAGE]
        free = self.free()
        if len(tails) > len(free):
            return len(tails) - len(free)
        table, lens = self.table.copy(), self.lens.copy()
        for b in range(B):
            if parent[b] == b:
                continue
            for p in table[b, : pages_of(int(lens[b]))]:
                self.refs[p] -= 1
            n = 0 if parent[b] < 0 else int(lens[parent[b]])
            row = table[parent[b], : pages_of(n)].copy()
            if b in tails:
                to = free.pop(0)
                for pool in pools:
                    pool[to] = pool[row[-1]]
                row[-1] = to
            for p in row:
                self.refs[p] += 1
            self.table[b, : len(row)] = row
            self.lens[b] = n
        return 0

    def compact(self, pools):
        P = len(self.refs)
        for b in range(len(self.lens)):
            if not 0 <= self.lens[b] <= self.table.shape[1] * PAGE:
                return -1, np.arange(P)
            row = self.table[b, : pages_of(int(self.lens[b]))]
            if ((row < 0) | (row >= P)).any() or (self.refs[row] <= 0).any():
                return -1, np.arange(P)
        used = self.refs > 0
        live = int(used.sum())
        holes = [p for p in range(live) if not used[p]]
        movers = [p for p in range(live, P) if used[p]]
        remap = np.where(used, np.arange(P), -1)
        for f, t in zip(movers, holes):
            remap[f] = t
            for pool in pools:
                pool[t] = pool[f]
            self.refs[t], self.refs[f] = self.refs[f], 0
        for b in range(len(self.lens)):
            n = pages_of(int(self.lens[b]))
            self.table[b, :n] = remap[self.table[b, :n]]
        return live, remap


def prompt_slack(q, cache, table, lens, first, scale=DIM ** -0.5):
    """Beside each output of attention(), how far the fp16 form for many rows
    may be off: keys, values and weights rounded to fp16 (2^-11 of each, half
    of eps; weights under 2^-30 of the largest may be lost), fp32 sums."""
    B, S, Hq, _ = q.shape
    H = cache.shape[1]
    G = Hq // H
    slack = np.zeros(q.shape)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        ids = table[b, : -(-n // PAGE)]
        for h in range(H):
            got = get_pages(cache[ids, h])
            k, v = ((m[..., None] + s[..., None] * u).reshape(-1, DIM)[:n] for u, s, m in (got["k"], got["v"]))
            x = q[b, :, h * G: (h + 1) * G].astype(np.float64)
            sc = scale * np.einsum("sgd,nd->sgn", x, k)
            # a key's rounding, and 128 products summed in fp32 (2^-16 with truncating adders)
            off = scale * (2 ** -11 + 2 ** -16) * np.einsum("sgd,nd->sgn", np.abs(x), np.abs(k))
            if first is not None:
                hide = np.arange(n)[None, :] > int(first[b]) + np.arange(S)[:, None]
                sc[np.broadcast_to(hide[:, None], sc.shape)] = -np.inf
            top = sc.max(-1, keepdims=True)
            p = np.exp(sc - np.where(np.isfinite(top), top, 0.0))
            tot = p.sum(-1, keepdims=True)
            p = p / np.where(tot > 0, tot, 1.0)
            # a score off by `off` moves its weight and the sum of all by that factor each
            size = np.einsum("sgn,nd->sgd", p * (2 * off + 2 ** -11 + 2 ** -11 + 2 ** -14), np.abs(v)) + n * 2 ** -30 * np.abs(v).max()
            slack[b, :, h * G: (h + 1) * G] = size
    return slack
