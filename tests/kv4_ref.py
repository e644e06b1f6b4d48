"""The 4-bit K/V cache in numpy and 64 bits: the format's definition, its bytes, attention over
it, and how far a result in f32 may be from it."""
import numpy as np

HD, BLK, HALF, BLOCK = 64, 64, 64 * 36, 64 * 72


def quantise(x):
    """x f32 / f16 [..., 64] -> (n' int [..., 64], c, d f64 [...]), as include/madi_q8.h defines them."""
    x = np.asarray(x).astype(np.float32)
    bad = ~(np.abs(x) <= 57344).all(-1)
    x = np.where(bad[..., None], np.float32(0), x)
    lo, hi = x.min(-1), x.max(-1)
    c = (lo + (hi - lo) * np.float32(8 / 15)).astype(np.float16).astype(np.float64)
    lo, hi, x = lo.astype(np.float64), hi.astype(np.float64), x.astype(np.float64)
    r = np.maximum((c - lo) / 8, (hi - c) / 7)
    _, e = np.frexp(r)
    step = np.ldexp(1.0, np.maximum(e - 8, -24))
    d = np.ceil(r / step) * step
    z = np.floor((x - c[..., None]) / np.where(d > 0, d, 1)[..., None] + 0.5)
    z = np.where((d > 0)[..., None], z, 0)
    assert z.min(initial=0) >= -8 and z.max(initial=0) <= 7
    z[bad] = 0
    return z.astype(np.int64), np.where(bad, np.nan, c), np.where(bad, 0.0, d)


def values(z, c, d):
    return c[..., None] + d[..., None] * z


def pack(data, kv, s, h, row, z, c, d):
    """Write one group into the u8 bytes data [slots][heads][blocks][4608]; kv 0: K, 1: V."""
    blk = data[s, h, row // BLK, kv * HALF:(kv + 1) * HALF]
    u = (z + 8).astype(np.uint8)
    r = row % BLK
    blk[r * 32:(r + 1) * 32] = u[0::2] | (u[1::2] << 4)
    blk[2048 + 4 * r:2052 + 4 * r] = np.array([c, d], np.float16).view(np.uint8)


def unpack(data, kv, max_tok):
    """(n', c, d) of all rows: [slots][heads][max_tok][64], [slots][heads][max_tok] x 2."""
    S, H, B, _ = data.shape
    half = data[..., kv * HALF:(kv + 1) * HALF]
    u = half[..., :2048].reshape(S, H, B * BLK, 32)[:, :, :max_tok]
    z = np.stack((u & 15, u >> 4), -1).reshape(S, H, max_tok, HD).astype(np.int64) - 8
    cd = np.ascontiguousarray(half[..., 2048:]).view(np.float16).reshape(S, H, B * BLK, 2)[:, :, :max_tok]
    return z, cd[..., 0].astype(np.float64), cd[..., 1].astype(np.float64)


def random_cache(g, slots, heads, max_tok, written, spread=1.0):
    """Bytes of a cache whose rows < written[s] hold bell-shaped codes; all other bytes are 0xFF
    (their c and d are NaN)."""
    data = np.full((slots, heads, (max_tok + BLK - 1) // BLK, BLOCK), 0xFF, np.uint8)
    rows = data.shape[2] * BLK
    for kv, sp in ((0, 1.0), (1, 0.5 * spread)):
        z = np.clip(np.rint(g.standard_normal((slots, heads, rows, HD)) * 3.2 + 0.5), -8, 7).astype(np.int64) + 8
        c = (g.standard_normal((slots, heads, rows)) * 0.2 * sp).astype(np.float16)
        d = np.maximum(0.3 + 0.04 * g.standard_normal((slots, heads, rows)), 0.05) * sp
        m, e = np.frexp(d)
        d = np.ldexp(np.ceil(m * 256), e - 8)                          # 8 significant bits
        half = data[..., kv * HALF:(kv + 1) * HALF]
        codes = (z[..., 0::2] | (z[..., 1::2] << 4)).astype(np.uint8).reshape(slots, heads, -1, BLK, 32)
        cd = np.stack((c, d.astype(np.float16)), -1).view(np.uint8).reshape(slots, heads, -1, BLK, 4)
        there = (np.arange(rows) < np.asarray(written).reshape(-1, 1, 1)).reshape(slots, 1, -1, BLK, 1)
        hc = half[..., :2048].reshape(slots, heads, -1, BLK, 32)
        hp = half[..., 2048:].reshape(slots, heads, -1, BLK, 4)
        half[..., :2048] = np.where(there, codes, hc).reshape(half[..., :2048].shape)
        half[..., 2048:] = np.where(there, cd, hp).reshape(half[..., 2048:].shape)
    return data


def key_counts(slots, rows, max_tok, pos=None, lens=None):
    """L [slots][rows]."""
    if pos is not None:
        return np.minimum(np.asarray(pos, np.int64).reshape(-1, 1) + np.arange(rows) + 1, max_tok)
    top = np.full(slots, max_tok) if lens is None else np.minimum(np.asarray(lens, np.int64), max_tok)
    return np.repeat(top.reshape(-1, 1), rows, 1)


def attend(q, data, max_tok, heads, L, n=None, f16=False, p16=False):
    """(out, bound) f64 [slots][rows][heads * 64]: the exact result, and how far a kernel with f32
    sums may be from it.

    With u = 2^-23 (a tensor-core sum may cut its last place instead of rounding it):
      score: the 64 products are summed in 4 steps of 16, twice (two f16 parts of q), then scaled
        and shifted by c sum(q): 16 u of the sum of magnitudes covers the roundings, the parts'
        missing bits (2^-22 of each q) and sum(q)'s own sum, the magnitudes being
        |q| (|c| + 24 d) / 8 since z = n' + 8 <= 15 and 8 sum(q) are combined;
      weight: relative error e_p = that + u |s| log2 e (the subtraction in base 2) + 4 u (exp2);
      output: numerator and denominator both carry e_p: 2 e_p sum p|v|; the products' two f16
        parts of p d (2 u, plus at most 2^-24 2^-14 of the largest weight each where the low part
        is subnormal) and the sums over L / 16 steps, at most 2 L / 16 + 16 u of sum p (|c| + 16 d).
    f16: the output's rounding, 2^-11 of the value (2^-25 at the least).
    p16: the weights are rounded to f16 (2^-11 each, in numerator and denominator; 2^-25 where
    they are subnormal)."""
    S, T, _ = q.shape
    H = data.shape[1]
    G = heads // H
    kz, kc, kd = unpack(data, 0, max_tok)
    vz, vc, vd = unpack(data, 1, max_tok)
    out = np.zeros((S, T, heads * HD))
    tol = np.zeros_like(out)
    u = 2.0 ** -23
    for s in range(S):
        for i in range(T if n is None else min(T, int(n[s]))):
            m = int(L[s, i])
            if m == 0:
                continue
            for h in range(heads):
                x = np.asarray(q[s, i, h * HD:(h + 1) * HD], np.float64)
                k = values(kz[s, h // G, :m], kc[s, h // G, :m], kd[s, h // G, :m])
                v = values(vz[s, h // G, :m], vc[s, h // G, :m], vd[s, h // G, :m])
                z = k @ x / 8
                p = np.exp(z - z.max())
                p /= p.sum()
                o = p @ v
                mag = np.abs(x).sum() / 8 * (np.abs(kc[s, h // G, :m]) + 24 * kd[s, h // G, :m])
                ep = (16 * u * mag + u * 1.4427 * np.abs(z - z.max()) + 4 * u).max()
                a = p @ np.abs(v)
                b = p @ (np.abs(vc[s, h // G, :m]) + 16 * vd[s, h // G, :m])
                t = 2 * ep * a + (2 * m / 16 + 16) * u * b + m * 2.0 ** -38 * vd[s, h // G, :m].max()
                if p16:
                    t = t + 2 * 2.0 ** -11 * a + m * 2.0 ** -25 * np.abs(v).max() * p.max() * 2
                if f16:
                    t = t + np.maximum(2.0 ** -11 * (np.abs(o) + t), 2.0 ** -25)
                out[s, i, h * HD:(h + 1) * HD] = o
                tol[s, i, h * HD:(h + 1) * HD] = t
    return out, tol
