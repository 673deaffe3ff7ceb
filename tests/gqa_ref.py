"""Prompts and drafted trees over f32 key/value caches, what is accepted of a tree, and
edited logits, from their definitions in float64 (numpy only)."""
import numpy as np


def angles(pos, rope_dim, base, freq_factors, linear):
    """[rows, rope_dim / 2] float32: the angle as the framework forms it (the frequency rounded
    from 64 bits, position * frequency / factor * (1 / linear) in 32)."""
    i = np.arange(rope_dim // 2, dtype=np.float64)
    freq = np.power(np.float64(np.float32(base)), -2.0 * i / max(rope_dim, 1)).astype(np.float32)
    ff = np.ones(rope_dim // 2, np.float32) if freq_factors is None else np.asarray(freq_factors, np.float32)
    return np.asarray(pos, np.float32)[:, None] * freq / ff * (np.float32(1) / np.float32(linear))


def rotate(x, pos, rope_dim, base, neox, freq_factors=None, linear=1.0):
    """x [rows, heads, hd] rotated, float64."""
    x = np.asarray(x, np.float64).copy()
    if rope_dim == 0:
        return x
    t = angles(pos, rope_dim, base, freq_factors, linear).astype(np.float64)[:, None]
    half = rope_dim // 2
    ia, ib = (np.arange(half), np.arange(half) + half) if neox else (2 * np.arange(half), 2 * np.arange(half) + 1)
    a, b = x[..., ia], x[..., ib]
    x[..., ia], x[..., ib] = a * np.cos(t) - b * np.sin(t), a * np.sin(t) + b * np.cos(t)
    return x


def path(parent, t):
    """Rows from the root of row t to t itself; a parent that is not before its row is none."""
    out = [t]
    while 0 <= parent[t] < t:
        t = int(parent[t])
        out.append(t)
    return out[::-1]


def attend(q, k, v, seen):
    """q [rows, H, hd] over k, v [keys, G, hd] with seen [rows, keys]: the outputs [rows, H,
    hd], and what their bound is made of: each output row's sum of weight * the value row's
    largest magnitude, and its largest sum of |q k| / sqrt(hd)."""
    rows, heads, hd = q.shape
    group = heads // k.shape[1]
    out, mass, size = np.zeros((rows, heads, hd)), np.zeros((rows, heads)), np.zeros((rows, heads))
    used = seen.any(axis=0)
    k, v, seen = k[used], v[used], seen[:, used]
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = np.where(seen, q[:, h] @ kh.T / np.sqrt(hd), -np.inf)
        a = np.where(seen, np.abs(q[:, h]) @ np.abs(kh).T / np.sqrt(hd), 0.0)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        out[:, h], mass[:, h], size[:, h] = p @ vh, p @ np.abs(vh).max(axis=1), a.max(axis=1)
    return out, mass, size


def bound(mass, size, hd, keys):
    """How far an output may be off, per (row, head).  A score: both operands cut to 22 bits and
    the product of their lower terms left out, 3 * 2^-22 of its terms, and 3 hd / 16 + 4 sums
    and roundings in f32 of 2^-24 (rotated rows, 2^-22, before them); an error of d in every
    score moves a normalised sum by 2 d of its mass.  The second product: 3 * 2^-22 and f32 sums
    over 6 products a tile of 32 keys, each of which is off by 2^-24 of the mass; the rest (exp2, sums
    of weights, the quotient) 16 * 2^-24.  A weight below 2^-13 of the largest loses lower-term bits:
    2^-11 of it, 2^-24 of the largest, of at most `keys` such."""
    d = size * (4 * 2.0**-22 + (3 * hd / 16 + 4) * 2.0**-24)
    return mass * (2 * d + 3 * 2.0**-22 + (6 * -(-keys // 32) + 16) * 2.0**-24) + mass * min(keys, 64) * 2.0**-24


def accept(parent, tokens, chosen):
    """The accepted rows of one tree, in order."""
    if len(parent) == 0:
        return []
    out = [0]
    while True:
        fits = [t for t in range(out[-1] + 1, len(parent)) if parent[t] == out[-1] and tokens[t] == chosen[out[-1]]]
        if not fits:
            return out
        out.append(fits[0])


def edit(logits, lists, repetition=None, frequency=None, presence=None, biases=None, allowed=None):
    """One row: lists is every counted id; biases a list of (id, value), the last of an id counts."""
    x = np.asarray(logits, np.float64).copy()
    v = len(x)
    ids = [i for i in lists if i < v]
    count = np.bincount(np.asarray(ids, np.int64), minlength=v) if ids else np.zeros(v, np.int64)
    hit = count > 0
    if repetition is not None and repetition > 0:
        x = np.where(hit, np.where(x > 0, x / repetition, x * repetition), x)
    if frequency is not None:
        x = np.where(hit, x - frequency * count, x)
    if presence is not None:
        x = np.where(hit, x - presence, x)
    for i, b in dict((i, b) for i, b in biases or [] if i < v).items():
        x[i] += b
    return x if allowed is None else np.where(allowed, x, -np.inf)
