"""Numpy restatement of the serving operators (TEST INFRASTRUCTURE: oracle only): the paged K/V cache
and the token draw, written row by row from the definitions of include/eii.h.

The rotation and the attention of a 16-bit cache are the forward pass's own (oracle.forward.rope,
oracle.forward.attention); this module adds the pages, the 4-bit rows and the draw.
"""
import math

import numpy as np

from oracle.forward import DMAX, rs, sat

I64 = np.int64
SAMPLE_C = (744163075, 257059888, 57045411, 7277686)
LOG2E_Q24 = round(math.log2(math.e) * 2 ** 24)
MASKED = -(1 << 31)


# ----------------------------------------------------------------------------------------- 4 bits
def quantise(x):
    """int64 [64] -> (nibbles [64], m, z)."""
    z, hi = int(x.min()), int(x.max())
    m = max(1, -(-(hi - z) // 15))
    return (2 * (x - z) + m) // (2 * m), m, z


class Pool:
    """One pool as bytes [n_pages][n_kv][slab], written and read a row of a head at a time."""

    def __init__(self, data, n_kv, hd, page, bits):
        self.hd, self.page, self.bits = hd, page, bits
        self.row = hd * 2 if bits == 16 else hd // 2
        self.slab = page * (self.row + (0 if bits == 16 else hd // 16))
        self.data = data.reshape(-1, n_kv, self.slab)

    def put(self, page, head, slot, x):
        """Stores int64 [hd]; returns the values that the cache then stands for."""
        b, at = self.data[page, head], slot * self.row
        if self.bits == 16:
            b[at:at + self.row] = x.astype("<i2").view(np.uint8)
            return x.copy()
        out = np.empty_like(x)
        for a in range(self.hd // 64):
            n, m, z = quantise(x[64 * a:64 * a + 64])
            b[at + 32 * a:at + 32 * a + 32] = n[:32] | n[32:] << 4
            w = self.page * self.row + (slot * (self.hd // 64) + a) * 4
            b[w:w + 4] = np.array([m | (z & 0xFFFF) << 16], dtype="<u4").view(np.uint8)
            out[64 * a:64 * a + 64] = z + m * n
        return out

    def get(self, page, head, slot):
        b, at = self.data[page, head], slot * self.row
        if self.bits == 16:
            return b[at:at + self.row].copy().view("<i2").astype(I64)
        out = np.empty(self.hd, I64)
        for a in range(self.hd // 64):
            n = b[at + 32 * a:at + 32 * a + 32].astype(I64)
            w = self.page * self.row + (slot * (self.hd // 64) + a) * 4
            m, z = b[w:w + 2].copy().view("<u2")[0], b[w + 2:w + 4].copy().view("<i2")[0]
            out[64 * a:64 * a + 64] = int(z) + int(m) * np.concatenate([n & 15, n >> 4])
        return out


# ----------------------------------------------------------------------------------------- append
def rotate(x, c, s, shift):
    """int64 [..., hd] with one position's Q30 rows [hd / 2]."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return sat(rs(np.concatenate([a * c - b * s, b * c + a * s], -1), shift), 16)


def append(q, k, v, seq, pos, table, k_pool, v_pool, rope, shift_q, shift_k, q_out, kv_out):
    """q [n][heads][hd] or None, k, v [n][kv][hd]; updates the pools, q_out [n][heads][hd], kv_out [n][2][kv][hd]."""
    for r in range(k.shape[0]):
        if seq[r] < 0 or pos[r] < 0:
            continue
        c, s = rope[0][pos[r]].astype(I64), rope[1][pos[r]].astype(I64)
        if q is not None:
            q_out[r] = rotate(q[r].astype(I64), c, s, shift_q)
        page, slot = int(table[seq[r], pos[r] // k_pool.page]), int(pos[r] % k_pool.page)
        kr = rotate(k[r].astype(I64), c, s, shift_k)
        for h in range(k.shape[1]):
            kv_out[r, 0, h] = k_pool.put(page, h, slot, kr[h])
            kv_out[r, 1, h] = v_pool.put(page, h, slot, v[r, h].astype(I64))


# -------------------------------------------------------------------------------------- attention
def attention(q, seq, length, table, k_pool, v_pool, E, shift_s, prob_bits, shift_c, bits_c, out):
    """q [n][heads][hd] -> out [n][heads][hd] (rows of a negative sequence are left)."""
    n, heads, hd = q.shape
    kv = k_pool.data.shape[1]
    for r in range(n):
        if seq[r] < 0:
            continue
        L = max(int(length[r]), 0)
        for h in range(kv):
            at = [(int(table[seq[r], t // k_pool.page]), h, t % k_pool.page) for t in range(L)]
            K = np.array([k_pool.get(*a) for a in at], I64).reshape(L, hd)
            V = np.array([v_pool.get(*a) for a in at], I64).reshape(L, hd)
            for j in range(h * heads // kv, (h + 1) * heads // kv):
                if L == 0:
                    out[r, j] = 0
                    continue
                s = sat(rs(K @ q[r, j].astype(I64), shift_s), 16)
                d = s.max() - s
                e = np.where(d <= DMAX, E[np.minimum(d, DMAX)], 0).astype(I64)
                Z = int(e.sum())
                P = ((e << prob_bits) + Z // 2) // Z
                out[r, j] = sat(rs(P @ V, shift_c), bits_c)


# --------------------------------------------------------------------------------------- sampling
def weights(row, inv_temp):
    """Integer weights of one row of int64 logits."""
    row = np.asarray(row, I64)
    b2 = (int(inv_temp) * LOG2E_Q24 + (1 << 15)) >> 16
    x = (row.max() - row) * b2  # (below 2^32 2^31)
    n, f = x >> 40, ((x >> 16) & 0xFFFFFF) << 7
    y = np.full(row.size, SAMPLE_C[3], I64)
    for c in (SAMPLE_C[2], SAMPLE_C[1], SAMPLE_C[0], 1 << 30):
        y = c - ((y * f) >> 31)
    s = np.minimum(n, 31)
    return np.where((n <= 30) & (row != MASKED), (y + ((I64(1) << s) >> 1)) >> s, 0)


def draw(row, u, inv_temp=65536, top_k=0, top_p=65536, min_p=0):
    """(token, kept, prob) of one row."""
    w = weights(row, inv_temp)
    order = np.lexsort((np.arange(w.size), -w))
    order = order[w[order] > 0]
    if top_k > 0:
        order = order[:top_k]
    order = order[w[order] >= (min_p << 14)]
    if order.size == 0:
        return -1, 0, 0
    goal = max(1, -(-top_p * int(w[order].sum()) // 65536))
    order = order[:int(np.searchsorted(np.cumsum(w[order]), goal)) + 1]
    mass = int(w[order].sum())
    target = int(u) * mass >> 32
    ids = np.sort(order)
    i = int(ids[np.searchsorted(np.cumsum(w[ids]), target, side="right")])
    return i, order.size, (int(w[i]) * (1 << 30) + mass // 2) // mass


# ----------------------------------------------------------------------------- the model, 4-bit cache
def forward_compressed(mdl, ids):
    """Logits [T, V] of the forward pass (oracle.forward.forward) of one sequence whose k and v rows are kept
    at 4 bits: the rows of every position, its own included, are what their nibbles stand for."""
    from oracle import forward as ofw
    ids = np.asarray(ids, I64)
    T = ids.shape[0]

    def stored(x):
        out = np.empty_like(x)
        for t in range(T):
            for h in range(x.shape[1]):
                n, m, z = quantise(x[t, h])
                out[t, h] = z + m * n
        return out
    x = ofw.embed(mdl, ids)
    plain = ofw.attention

    def attention(qr, kr, v, *args, **kw):
        return plain(qr, stored(kr), stored(v), *args, **kw)
    try:
        ofw.attention = attention
        for l in range(len(mdl["layers"])):
            x = ofw.block_batch(mdl, l, x, T)
    finally:
        ofw.attention = plain
    return ofw.logits_from_y(mdl, ofw.final_norm(mdl, x))
