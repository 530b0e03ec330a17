"""Plain 64-bit forms of the 4-bit-cache operators, on the CPU, from their definitions: loops over requests and
tokens, nothing shared with the package. Byte layout as include/velox_sm100.h documents it."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values():
    """Value of every byte's low seven bits (0x7f: 480, as the cache reads it)."""
    out = np.zeros(128)
    for b in range(128):
        e, m = b >> 3, b & 7
        out[b] = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
    return out


E4M3 = e4m3_values()


def nearest(x, grid, even):
    """Index of the grid value nearest to each x >= 0 (saturating); ties go to the index `even` prefers."""
    hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    lo = hi - 1
    mid = (grid[lo] + grid[hi]) / 2
    up = (x > mid) | ((x == mid) & even(hi))
    return np.where(up, hi, lo)


def quantise(x, divisor):
    """x: f32 [..., D] -> (codes [..., D], scale bytes [..., D/16]); single-precision steps."""
    x = np.asarray(x, dtype=np.float32)
    g = x.reshape(x.shape[:-1] + (-1, 16))
    amax = np.abs(g).max(-1)
    s = (np.float32(divisor) * amax).astype(np.float32) / np.float32(6)
    sb = nearest(s.astype(np.float64), E4M3[:127], lambda i: i % 2 == 0)
    ds = E4M3[sb].astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        v = np.where(ds > 0, (g * np.float32(divisor)).astype(np.float32) / np.where(ds > 0, ds, 1), 0).astype(np.float32)
    c = nearest(np.abs(v).astype(np.float64), LEVELS, lambda i: i % 2 == 0)
    c = c + 8 * (np.signbit(v) & (ds > 0))
    return c.reshape(x.shape).astype(np.uint8), sb.astype(np.uint8)


def values(codes, scales, divisor):
    sign = np.where(codes & 8, -1.0, 1.0)
    v = sign * LEVELS[codes & 7] * np.repeat(E4M3[scales & 127], 16, axis=-1)
    return v / divisor


def k_code_at(D, tau, byte):
    return tau * (D // 2) + byte


def v_code_at(D, tau, byte):
    w = D // 16
    p, t, j = tau // 8, tau // 2 % 4, tau % 2
    return 8 * D + (((p * 8 + byte // w) * 4 + t) * 2 + j) * w + byte % w


def k_scale_at(D, tau, group):
    w = D // 64
    return 16 * D + (((tau % 8) * 4 + group // w) * 2 + tau // 8) * w + group % w


def v_scale_at(D, tau, group):
    return 17 * D + ((group * 4 + tau // 2 % 4) * 2 + tau // 8) * 2 + tau % 2


class Cache:
    """numpy view of a cache's bytes [pages, kv_heads, page/16, 18 D]."""

    def __init__(self, storage, page, D, kdiv, vdiv):
        self.s, self.page, self.D, self.kdiv, self.vdiv = storage, page, D, kdiv, vdiv
        self.hkv = storage.shape[1]
        b = np.arange(D // 2)
        g = np.arange(D // 16)
        self.at = [(k_code_at(D, t, b), v_code_at(D, t, b), k_scale_at(D, t, g), v_scale_at(D, t, g)) for t in range(16)]

    def block(self, slot):
        off = slot % self.page
        return self.s[slot // self.page, :, off // 16, :], self.at[off % 16]

    def write(self, slot, k, v):
        """k, v: f32 [kv_heads, D]"""
        blk, (kc, vc, ks, vs) = self.block(slot)
        for x, div, ci, si in ((k, self.kdiv, kc, ks), (v, self.vdiv, vc, vs)):
            c, s = quantise(x, div)
            blk[:, ci] = c[:, 0::2] | (c[:, 1::2] << 4)
            blk[:, si] = s

    def read(self, slot):
        blk, (kc, vc, ks, vs) = self.block(slot)
        out = []
        for div, ci, si in ((self.kdiv, kc, ks), (self.vdiv, vc, vs)):
            by = blk[:, ci]
            c = np.stack([by & 15, by >> 4], -1).reshape(self.hkv, self.D)
            out.append(values(c, blk[:, si], div))
        return out


def norm_rope(x, weight, eps, offset, rope, positions, interleaved):
    """f64 [T, H, D]"""
    y = np.array(x, dtype=np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * ((1.0 if offset else 0.0) + weight.astype(np.float64))
    if rope is not None:
        rot = rope.shape[1]
        for t in range(y.shape[0]):
            if not 0 <= positions[t] < rope.shape[0]:
                continue
            c, s = rope[positions[t], : rot // 2].astype(np.float64), rope[positions[t], rot // 2:].astype(np.float64)
            a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
            u, v = y[t][:, a].copy(), y[t][:, b].copy()
            y[t][:, a], y[t][:, b] = u * c - v * s, v * c + u * s
    return y


def plan(cached, new, table, free, taken, page, tokens):
    table = table.copy()
    cols = table.shape[1]
    cu, kv = [0], []
    pos, slot = -np.ones(tokens, np.int64), -np.ones(tokens, np.int64)
    used, status, t = taken, 0, 0
    for b in range(len(cached)):
        c, n = max(0, int(cached[b])), max(0, int(new[b]))
        have, full = -(-c // page), -(-(c + n) // page)
        if full > cols:
            status |= 2
        mapped = have
        for i in range(have, min(full, cols)):
            if used < len(free):
                table[b, i] = free[used]
                mapped = i + 1
            else:
                table[b, i] = -1
                status |= 1
            used += 1
        kv.append(min(c + n, mapped * page))
        for i in range(n):
            if t < tokens:
                p = c + i
                pos[t] = p
                if p // page < cols and table[b, p // page] >= 0:
                    slot[t] = table[b, p // page] * page + p % page
            else:
                status |= 4
            t += 1
        cu.append(t)
    return table, np.array(cu), np.array(kv, dtype=np.int64), pos, slot, min(used, len(free)), status


def attention(q, cache, table, cu, kv_lens, scale, causal, window):
    """(out, bound's ingredients): f64 [T, H, D] with NaN in the rows of no request, sum_j p_j |v_j|, and the
    largest sum_d |q_d k_jd| * scale of each row and head."""
    T, H, D = q.shape
    out = np.full((T, H, D), np.nan)
    spread = np.zeros((T, H, D))
    reach = np.zeros((T, H))
    G = H // cache.hkv
    for b in range(len(kv_lens)):
        n = cu[b + 1] - cu[b]
        L = min(int(kv_lens[b]), table.shape[1] * cache.page)
        k, v, there = np.zeros((L, cache.hkv, D)), np.zeros((L, cache.hkv, D)), np.zeros(L, bool)
        for j in range(L):
            page = table[b, j // cache.page]
            if 0 <= page < cache.s.shape[0]:
                k[j], v[j] = cache.read(int(page) * cache.page + j % cache.page)
                there[j] = True
        for i in range(n):
            row, p = cu[b] + i, L - n + i
            see = there.copy()
            j = np.arange(L)
            if causal:
                see &= j <= p
            if window > 0:
                see &= j > p - window
            for h in range(H):
                if not see.any():
                    out[row, h] = 0.0
                    continue
                kk, vv, qq = k[see, h // G], v[see, h // G], q[row, h]
                s = kk @ qq * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[row, h], spread[row, h] = w @ vv, w @ np.abs(vv)
                reach[row, h] = (np.abs(kk) @ np.abs(qq)).max() * scale
    return out, spread, reach


def attention_bound(out, spread, reach, tokens, vmax, D):
    """Largest difference an exact-arithmetic reader may see, per element. Probabilities are rounded to f16 (2^-11 of
    each, so 2^-11 sum p|v|; those under 2^-22 of the largest are subnormal: 2^-33 of the largest each). A score is a sum of
    D products in f32 (each partial sum at most `reach`, one rounding of 2^-24 each, doubled for truncating adders, and
    two more multiplications), in the exponent of p: p is off by that relative amount, and so is the sum of the p; exp2 itself is
    good to 2^-22. Sums over `tokens` probabilities: positive terms, chains no longer than tokens / 16 + 64. The result is rounded to
    bf16: 2^-8 of the value."""
    rel = 2.0 ** -11 + 2 * (reach[..., None] * (2 * D + 4) * 2.0 ** -24 + 2.0 ** -22) + 2 * (tokens / 16 + 64) * 2.0 ** -24
    return 2.0 ** -8 * np.abs(out) + rel * spread * (1 + 2.0 ** -8) + tokens * 2.0 ** -33 * vmax + 1e-30
