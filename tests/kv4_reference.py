"""Plain numpy forms of the 4-bit paged KV cache and of the log-probabilities,
written from the formulas in include/nimf_cuda.h (float32 where the format
fixes the roundings, float64 elsewhere)."""
import math

import numpy as np

F = np.float32


# ------------------------------------------------------------------ the format
def tile_bytes(dim, group):
    return 16 * dim + 256 * (dim // group)


def place(ch, dim, key):
    """(byte of the row, shift) of a channel's code."""
    if key:
        word, nib = (ch % 32 // 8) * (dim // 32) + ch // 32, ch % 8
    else:
        word, nib = (ch % 32 // 4) * (dim // 64) + ch // 64, ch % 4 + 4 * (ch % 64 // 32)
    return word * 4 + nib // 2, 4 * (nib % 2)


def encode(x, group):
    """x [..., dim] float32 -> codes [..., dim], scale, minimum [..., dim / group]."""
    x = np.asarray(x, F)
    g = x.reshape(*x.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        low, high = g.min(-1) + F(0), g.max(-1) + F(0)   # -0 counts as 0
        scale = ((high - low).astype(F) / F(15)).astype(F)
        bad = ~np.isfinite(scale) | ~np.isfinite(g).all(-1)
        step = np.where(bad | (scale == 0), F(1), scale)
        code = np.rint(((g - np.where(bad, F(0), low)[..., None]).astype(F) / step[..., None]).astype(F))
        code = np.where((bad | (scale == 0))[..., None], 0, np.minimum(code, 15))
    scale, low = np.where(bad, F(np.nan), scale), np.where(bad, F(np.nan), low)
    return np.nan_to_num(code).astype(np.uint8).reshape(x.shape), scale.astype(F), low.astype(F)


def decode(code, scale, low):
    """The values that codes stand for, rounded as nimf_kv4_read_dev rounds."""
    g = code.reshape(*scale.shape, -1).astype(F)
    return ((g * scale[..., None]).astype(F) + low[..., None]).astype(F).reshape(code.shape)


class Pool:
    """A cache buffer [blocks][kv heads][block / 16][tile bytes] on the host."""

    def __init__(self, blocks, hkv, dim, bs, group, rng=None):
        self.blocks, self.hkv, self.dim, self.bs, self.group = blocks, hkv, dim, bs, group
        self.tb = tile_bytes(dim, group)
        shape = (blocks, hkv, bs // 16, self.tb)
        self.buf = np.zeros(shape, np.uint8) if rng is None else rng.integers(0, 256, shape).astype(np.uint8)

    def parts(self, key):
        d, ng = self.dim, self.dim // self.group
        codes = 0 if key else 8 * d
        params = 16 * d + (0 if key else 128 * ng)
        return codes, params

    def write(self, slot, key, x):
        """x [hkv, dim] float32 into a slot."""
        blk, r = divmod(int(slot), self.bs)
        code, scale, low = encode(x, self.group)
        codes, params = self.parts(key)
        for h in range(self.hkv):
            tile = self.buf[blk, h, r // 16]
            row = np.zeros(self.dim // 2, np.uint8)
            for ch in range(self.dim):
                b, s = place(ch, self.dim, key)
                row[b] |= np.uint8(code[h, ch] << s)
            at = codes + (r % 16) * (self.dim // 2)
            tile[at:at + self.dim // 2] = row
            for n in range(self.dim // self.group):
                at = params + (n * 16 + r % 16) * 8
                tile[at:at + 8] = np.array([scale[h, n], low[h, n]], F).view(np.uint8)

    def tokens(self, table, n, key):
        """codes [n, hkv, dim], scale and minimum [n, hkv, dim / group] of the
        first n tokens of a block table."""
        t = np.arange(n)
        tiles = self.buf[np.asarray(table)[t // self.bs], :, t % self.bs // 16]   # [n, hkv, tb]
        codes, params = self.parts(key)
        half = self.dim // 2
        rows = np.take_along_axis(tiles, (codes + (t % 16)[:, None] * half + np.arange(half))[:, None, :].repeat(self.hkv, 1), 2)
        byte, shift = zip(*[place(ch, self.dim, key) for ch in range(self.dim)])
        code = (rows[:, :, list(byte)] >> np.array(shift, np.uint8)) & 15
        ng = self.dim // self.group
        at = params + ((np.arange(ng) * 16)[None, :] + (t % 16)[:, None]) * 8          # [n, ng]
        idx = (at[:, :, None] + np.arange(8)).reshape(n, 1, -1).repeat(self.hkv, 1)
        p = np.ascontiguousarray(np.take_along_axis(tiles, idx, 2)).view(F).reshape(n, self.hkv, ng, 2)
        return code, p[..., 0], p[..., 1]


# ------------------------------------------------------------------ operators
def reserve(bs, n_blocks, width, n_new, lens, table, free, n_free, max_rows):
    """Request by request, as the header says it."""
    n = len(lens)
    table, slots, positions = table.copy(), np.full(max_rows, -1, np.int32), np.zeros(max_rows, np.int32)
    cu, out, granted = np.zeros(n + 1, np.int32), np.array(lens, np.int32), np.zeros(n, np.int32)
    asked, row, taken = 0, 0, 0
    n_free = min(max(int(n_free), 0), n_blocks)
    for b in range(n):
        old, new = max(int(lens[b]), 0), max(int(n_new[b]), 0)
        out[b] = old
        cu[b], end = row, row + new
        have, total = -(-old // bs), -(-(old + new) // bs)
        if total <= width and end <= max_rows:
            need = total - have
            if need == 0 or asked + need <= n_free:
                for j in range(need):
                    table[b, have + j] = free[n_free - 1 - asked - j]
                taken += need
                for i in range(new):
                    p = old + i
                    positions[row + i] = p
                    slots[row + i] = table[b, p // bs] * bs + p % bs
                out[b], granted[b] = old + new, 1
            asked += need
        row = end
    cu[n] = row
    return dict(lens=out, table=table, n_free=n_free - taken, cu_rows=cu, slots=slots, positions=positions, granted=granted)


def rope(x, pos, cos_t, sin_t):
    """x [rows, heads, dim] float32, each product and sum rounded."""
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos_t[pos][:, None], sin_t[pos][:, None]
    return np.concatenate(((a * c).astype(F) - (b * s).astype(F), (a * s).astype(F) + (b * c).astype(F)), -1).astype(F)


def attention(pool, table, length, q, scale):
    """Causal attention of q [n, heads, dim], the last n of `length` tokens, in
    64 bits; and a bound on what a float32 computation of the same sums may be
    off, by element.

    With u = 2^-24 (half a float32 step): a score is sum over channels of
    (q scale) ((c - 8) s + (m + 8 s)).  q enters on a grid of 2^-10 of its row's
    largest magnitude Q at most, the rest of a grid step in fp16: off by 2^-23 Q
    a channel.  The tensor core cuts each of its D / 8 partial sums by at most
    2u of it; scale, row factor, log2(e), the sums of q and the FMAs add at most
    16u more.  So with A = sum |q scale| (|c - 8| s + |m + 8 s|) log2(e) a base-2
    score is off by E = A (2u D / 8 + 16u) + 2^-23 Q scale log2(e) sum |c - 8| s.
    A probability is off by E ln 2 for its own score and the same for the
    maximum's, by the exponent's rounding |s - max| 2u and by ex2's own 2^-22,
    so relatively by e = 2 E ln 2 + 2^-22 + 2u |s - max|; w = p s is rounded
    twice (2u) and enters as q does, on a grid of the largest w of 32 tokens:
    2^-23 of that a token.  The weighted sums run over 32 tokens in the tensor
    core (4 steps, 2u each) and over at most n / 32 + 3 units, warps' and CTAs'
    pieces in float32, each with a rescaling (4u); the denominator the same.
    With V = sum p (|c - 8| s + |m + 8 s|):
    |error| <= V (2 max e + 2^-22 + 2u + 8u + 2 * 4u (n / 32 + 8))
               + 2^-23 sum over units (max w) (sum |c - 8|)."""
    n, heads, dim = q.shape
    hkv, u = pool.hkv, 2.0 ** -24
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    if length <= 0:
        return out, tol
    r = heads // hkv
    full = []
    for key in (True, False):
        code, sc, low = pool.tokens(table, length, key)
        sc, low = (v.astype(np.float64).repeat(pool.group, -1) for v in (sc, low))
        full.append((code * sc + low, np.abs(code - 8.0) * sc + np.abs(low + 8 * sc), np.abs(code - 8.0), sc))
    (k, ka, kc, ks), (v, va, vc, vs) = full
    units = -(-length // 32)
    seen = np.arange(length)[None, :] <= (length - n + np.arange(n))[:, None]
    with np.errstate(all="ignore"):
        for h in range(heads):
            g = h // r
            qs = q[:, h].astype(np.float64) * scale
            s = np.where(seen, qs @ k[:, g].T, -np.inf)
            big = np.where(seen, np.abs(qs) @ ka[:, g].T, 0.0) * math.log2(math.e)
            top = s.max(-1, keepdims=True)
            top = np.where(np.isneginf(top), 0.0, top)
            p = np.exp(s - top)
            total = p.sum(-1, keepdims=True)
            p = np.where(total > 0, p / np.where(total > 0, total, 1.0), p)
            pv = np.where(seen, p, 0.0)
            vz = np.where(seen.any(0)[:, None], v[:, g], 0.0)
            vaz = np.where(seen.any(0)[:, None], va[:, g], 0.0)
            out[:, h] = pv @ vz
            far = np.where(seen & (p > 0), np.abs(s - top), 0.0) * math.log2(math.e)
            grid = np.where(seen, np.abs(qs).max(-1, keepdims=True) * (kc[:, g] * ks[:, g]).sum(-1), 0.0) * math.log2(math.e) * 2.0 ** -23
            e = 2 * (big * (u * dim / 4 + 16 * u) + grid).max(-1, keepdims=True) * math.log(2) + 2.0 ** -22
            rel = 2 * (e + 2 * u * (pv * far).sum(-1, keepdims=True)) + 2.0 ** -22 + 10 * u + 8 * u * (length / 32 + 8)
            for n0 in range(0, dim, pool.group):       # the grid of w, unit by unit
                w = np.zeros((n, units * 32))
                w[:, :length] = np.where(seen, pv * np.where(seen.any(0), vs[:, g, n0], 0.0), 0.0)
                c8 = np.zeros((units * 32, pool.group))
                c8[:length] = vc[:, g, n0:n0 + pool.group]
                tol[:, h, n0:n0 + pool.group] = 2.0 ** -23 * w.reshape(n, units, 32).max(-1) @ c8.reshape(units, 32, -1).sum(1)
            tol[:, h] += (pv @ vaz) * rel
    return out, tol + 1e-30


def logprobs(x, ids, top):
    """x [rows, vocab] float32 in 64 bits."""
    rows, vocab = x.shape
    xd = x.astype(np.float64)
    res = dict(logprob=np.zeros(rows), entropy=np.zeros(rows), rank=np.zeros(rows, np.int64),
               top_ids=np.zeros((rows, top), np.int64), top_logprobs=np.zeros((rows, top)))
    for i in range(rows):
        r = xd[i]
        order = np.argsort(-np.where(np.isnan(r), -np.inf, r), kind="stable")[:top]
        m = r.max()
        if np.isnan(m) or m == np.inf:
            lp, ent = np.full(vocab, np.nan), np.nan
        elif m == -np.inf:
            lp, ent = np.full(vocab, -np.inf), 0.0
        else:
            t = r - m
            e = np.exp(t)
            k = np.argmax(r)
            s = e[:k].sum() + e[k + 1:].sum()
            lp = t - np.log1p(s)
            ent = np.log1p(s) - np.where(e > 0, e * np.where(e > 0, t, 0.0), 0.0).sum() / (1 + s)
        ok = 0 <= ids[i] < vocab
        res["logprob"][i] = lp[ids[i]] if ok else (np.nan if np.isnan(lp).all() else -np.inf)
        res["entropy"][i] = ent
        res["rank"][i] = 1 + (r > r[ids[i]]).sum() if ok else 0
        res["top_ids"][i] = order
        res["top_logprobs"][i] = lp[order]
    return res
