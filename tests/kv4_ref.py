"""The 4-bit cache's format and operators in numpy float64, from their
definitions (include/ferrum_hip.h), one element at a time where that is plainest."""
import numpy as np


def quantise(x):
    """x [..., hd] f32 -> scales f16 [..., hd / 32], levels uint8 [..., hd]."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    with np.errstate(invalid="ignore", over="ignore"):
        a = np.abs(b)
        m = np.take_along_axis(b, np.argmax(np.where(np.isnan(a), -1, a), axis=-1)[..., None], -1)
        d = np.clip(m.astype(np.float64) / -8, -65504, 65504).astype(np.float16)
        w = d.astype(np.float64)
        q = np.clip(np.rint(np.where(w != 0, b.astype(np.float64) / np.where(w != 0, w, 1), 0)), -8, 7) + 8
    odd = ~np.isfinite(b).all(axis=-1, keepdims=True)
    d = np.where(odd, np.float16(np.nan), d)
    q = np.where(odd, 8, q)
    return d[..., 0], q.astype(np.uint8).reshape(x.shape)


def values(d, q):
    return (q.astype(np.float64) - 8) * np.repeat(d.astype(np.float64), 32, axis=-1)


def k_place(key, ch, hd):
    """Byte and shift of a key's channel in a head's plane."""
    g, b, i = ch % 32 // 8, ch // 32, ch % 8
    return key * (hd // 2) + (g * (hd // 32) + b) * 4 + i // 2, 4 * (i % 2)


def v_place(key, ch, hd):
    if hd == 32:
        h, n, e, unit, units = ch // 16, ch % 16 // 2, ch % 2, ch % 16 // 2, 8
    else:
        p, h, n, e = ch // 64, ch % 64 // 32, ch % 32 // 2, ch % 2
        unit, units = n * (hd // 64) + p, hd // 4
    return ((key // 8 * units + unit) * 8 + key % 8) * 2 + h, 4 * e


def unpack(plane, d, hd, keys, v):
    """Values of positions `keys` of one head: plane uint8 [cap * hd / 2], d f16 [cap / 8, hd / 32, 8]."""
    place = v_place if v else k_place
    at = [[place(k, c, hd) for c in range(hd)] for k in keys]
    q = np.array([[plane[o] >> s & 15 for o, s in row] for row in at], np.uint8).reshape(len(keys), hd)
    sc = np.array([[d[k // 8, b, k % 8] for b in range(hd // 32)] for k in keys], np.float16).reshape(len(keys), -1)
    return values(sc, q), q, sc


def pack(d, q, cap, v):
    """One head's planes from scales [keys, hd / 32] and levels [keys, hd] (unused positions zero)."""
    keys, hd = q.shape
    plane, sc = np.zeros(cap * hd // 2, np.uint8), np.zeros((cap // 8, hd // 32, 8), np.float16)
    place = v_place if v else k_place
    key, ch = np.meshgrid(np.arange(keys), np.arange(hd), indexing="ij")
    o = np.empty((keys, hd, 2), np.int64)
    for c in range(hd):
        a, s = place(np.arange(keys), c, hd)
        o[:, c, 0], o[:, c, 1] = a, s
    np.bitwise_or.at(plane, o[..., 0].ravel(), (q.astype(np.uint8) << o[..., 1].astype(np.uint8)).ravel())
    k = np.arange(keys)
    for b in range(hd // 32):
        sc[k // 8, b, k % 8] = d[:, b]
    return plane, sc


def rotate(x, pos, rope_dim, base, neox, ff=None, linear=1.0):
    """apply_rope of x [..., heads, hd] at pos [...], angles in f32 as there, the rest in float64."""
    y = x.astype(np.float64)
    half = rope_dim // 2
    for i in range(half):
        freq = np.float32(np.power(np.float64(np.float32(base)), -2.0 * i / rope_dim))
        f = np.float32(1.0) if ff is None else np.float32(ff[i])
        th = (np.asarray(pos).astype(np.float32) * freq / f * (np.float32(1.0) / np.float32(linear))).astype(np.float64)
        a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
        u, v = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
        c, s = np.cos(th)[..., None], np.sin(th)[..., None]
        y[..., a], y[..., b] = u * c - v * s, u * s + v * c
    return y


def attention(q, k, v, first, end, softcap=0.0, slopes=None, qpos=None, kpos=None):
    """q [rows, heads, hd]; k, v [n_kv, keys, hd] float64; first, end [rows].
    Returns out [rows, heads, hd], lse [rows, heads], weight [n_kv, keys]."""
    rows, heads, hd = q.shape
    group = heads // k.shape[0]
    keys = np.arange(k.shape[1])
    out, lse, weight = np.zeros(q.shape), np.full((rows, heads), -np.inf), np.zeros(k.shape[:2])
    for r in range(rows):
        see = keys[first[r]:max(first[r], end[r])]
        if not len(see):
            continue
        for h in range(heads):
            z = k[h // group, see] @ q[r, h].astype(np.float64) / np.sqrt(hd)
            if softcap:
                z = softcap * np.tanh(z / softcap)
            if slopes is not None:
                kp = see if kpos is None else kpos[h // group, see]
                z = z - np.float64(slopes[h]) * np.abs(int(qpos[r]) - kp.astype(np.int64))
            m = z.max()
            e = np.exp(z - m)
            out[r, h] = (e / e.sum()) @ v[h // group, see]
            lse[r, h] = m + np.log(e.sum())
            weight[h // group, see] += e / e.sum()
    return out, lse, weight


def evict(weight, n, keep, recent):
    """Rows of one head that stay."""
    if n <= keep:
        return list(range(n))
    free = n - recent
    key = [np.inf if np.isnan(w) else w for w in weight[:free]]
    nan = [np.isnan(w) for w in weight[:free]]
    heavy = sorted(range(free), key=lambda j: (not nan[j], -key[j], j))[:keep - recent]
    return sorted(heavy) + list(range(free, n))
