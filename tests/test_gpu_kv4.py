"""The 4-bit key/value cache (fh_kv4_*) against its definitions in float64
(kv4_ref): the bytes that append writes, attention for single tokens and prompts
under every score option, the weights, the eviction, and their refusals."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

HEADS = [(4, 4, 32), (14, 2, 64), (12, 12, 64), (32, 8, 128), (40, 2, 64), (5, 1, 128)]


def gpu(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def ints(values):
    return gpu(np.asarray(values, np.uint32).view(np.int32))


class Box:
    """A cache whose unused rows hold the worst that memory can: NaN and huge
    scales.  Rows below `lens` hold quantised normals, kept here as float64."""

    def __init__(self, seqs, n_kv, hd, cap, lens, seed, tracked=False, k_std=1.0, v_std=1.0, repeat=1):
        """repeat: so many times the sequences given, one set after the other."""
        import ferrum_hip
        import torch

        rng = np.random.default_rng(seed)
        self.seqs, self.n_kv, self.hd, self.cap, self.lens = seqs, n_kv, hd, cap, list(lens)
        nb = hd // 32
        kp, vp = (rng.integers(0, 256, (seqs, n_kv, cap * hd // 2), dtype=np.uint8) for _ in range(2))
        junk = np.array([0x7E00, 0x7BFF, 0xFC00, 0xFBFF, 0x7C00, 0xFE01], np.uint16)
        kd, vd = (rng.choice(junk, (seqs, n_kv, cap // 8, nb, 8)).view(np.float16) for _ in range(2))
        self.k, self.v = (np.zeros((seqs, n_kv, cap, hd)) for _ in range(2))
        self.vstep = np.zeros((seqs, n_kv, cap, hd))
        self.kstep = np.zeros((seqs, n_kv, cap, hd))
        for s in range(seqs):
            n = min(self.lens[s], cap)
            for h in range(n_kv):
                for plane, sc, val, std, step, isv in ((kp, kd, self.k, k_std, self.kstep, False),
                                                       (vp, vd, self.v, v_std, self.vstep, True)):
                    x = (rng.standard_normal((n, hd)) * std * np.exp(0.3 * rng.standard_normal(hd))).astype(np.float32)
                    d, q = ref.quantise(x)
                    new, nd = ref.pack(d, q, cap, isv)
                    key, ch = np.arange(n), np.arange(nb)
                    val[s, h, :n] = ref.values(d, q)
                    step[s, h, :n] = np.abs(np.repeat(d.astype(np.float64), 32, axis=1))
                    sc[s, h][key[:, None] // 8, ch[None], key[:, None] % 8] = d
                    if isv:  # (positions share no byte, but an octet's bytes interleave)
                        used = np.zeros(cap * hd // 2, bool)
                        one = np.full((n, hd), 15, np.uint8)
                        used = ref.pack(d, one, cap, True)[0] != 0
                        plane[s, h][used] = new[used]
                    else:
                        plane[s, h, :n * hd // 2] = new[:n * hd // 2]
        if repeat > 1:
            again = lambda x: np.tile(x, (repeat,) + (1,) * (x.ndim - 1))  # noqa: E731
            kp, kd, vp, vd, self.k, self.v, self.kstep, self.vstep = map(
                again, (kp, kd, vp, vd, self.k, self.v, self.kstep, self.vstep))
            self.seqs = seqs = seqs * repeat
            self.lens = self.lens * repeat
        self.pos = np.tile(np.arange(cap, dtype=np.int32), (seqs, n_kv, 1)) if tracked else None
        self.weight = rng.random((seqs, n_kv, cap)).astype(np.float32) if tracked else None
        planes = [gpu(kp), gpu(kd), gpu(vp), gpu(vd)]
        self.c = ferrum_hip.KV4Cache(seqs, n_kv, hd, cap, *planes, gpu(self.pos) if tracked else None,
                                     gpu(self.weight) if tracked else None)
        torch.cuda.synchronize()

    def plane(self, name):
        p = self.c.planes[name]
        return None if p is None else p.cpu().numpy()


def rows_of(lens, news):
    off = np.concatenate([[0], np.cumsum(news)])
    return off, [(s, off[s] + t, lens[s] + t, t) for s in range(len(news)) for t in range(news[s])]


def check_attention(box, q, lens, news, out, lse, first=None, end=None, softcap=0.0, slopes=None, qpos=None,
                    weight=None):
    """Each output within its own bound.  With a_j = sum_c |q_c| 8 step_jc / sqrt(hd) (what
    a score's partial sums can reach; plus the distance term, plus the cap) a score has at
    most 8 roundings of 2^-24 of a_j, so a weight is off by 2^-21 a_j and, with the
    normaliser, an output by 2^-21 sum_j p_j (a_j + mean a) 8 step_j; the weights' own
    roundings (exp2 2^-23, scale 2^-24, two f16 terms 2^-22) and the sums' (4 a tile of at
    most twice the mass; 64 tiles add up as sqrt) give 2^-18 of the mass sum_j p_j 8 step_j."""
    n_heads, hd = q.shape[1], q.shape[2]
    group = n_heads // box.n_kv
    total_w = np.zeros((box.seqs, box.n_kv, box.cap))
    tol_w = np.zeros_like(total_w)
    off, _ = rows_of(lens, news)
    for s in range(box.seqs):
        rows = np.arange(off[s], off[s + 1])
        at = lens[s] + np.arange(news[s])
        keys = min(lens[s] + news[s], box.cap)
        lo = np.zeros(news[s], np.int64) if first is None else np.minimum(np.asarray(first, np.int64)[rows], keys)
        hi = np.minimum(at + 1 if end is None else np.asarray(end, np.int64)[rows], keys)
        bad = at >= keys
        none = ~bad & (lo >= hi)
        assert np.isnan(out[rows[bad]]).all() and (out[rows[none]] == 0).all()
        if lse is not None:
            assert np.isnan(lse[rows[bad]]).all() and (lse[rows[none]] == -np.inf).all()
        ok = ~bad & ~none
        if not ok.any():
            continue
        rows, lo, hi, at = rows[ok], lo[ok], hi[ok], at[ok]
        here = np.arange(hi.max())
        seen = (here >= lo[:, None]) & (here < hi[:, None])
        for h in range(n_heads):
            g, x = h // group, q[rows, h].astype(np.float64)
            k, v = box.k[s, g, :len(here)], box.v[s, g, :len(here)]
            ks, vs = 8 * box.kstep[s, g, :len(here)], 8 * box.vstep[s, g, :len(here)]
            score, a = x @ k.T / np.sqrt(hd), np.abs(x) @ ks.T / np.sqrt(hd)
            if softcap:
                score = softcap * np.tanh(score / softcap)
                a = a + softcap * (np.abs(score) > 0.4 * softcap) + np.abs(score)
            if slopes is not None:
                kp = here if box.pos is None else box.pos[s, g, :len(here)].astype(np.int64)
                me = at if qpos is None else np.asarray(qpos, np.int64)[rows]
                far = np.float64(slopes[h]) * np.abs(me[:, None] - kp)
                score, a = score - far, a + far
            score = np.where(seen, score, -np.inf)
            top = score.max(axis=1, keepdims=True)
            mass = np.exp(score - top).sum(axis=1, keepdims=True)
            z, p = (top + np.log(mass))[:, 0], np.exp(score - top) / mass
            abar = (p * a).sum(axis=1, keepdims=True)
            tol = 2.0 ** -21 * ((p * (a + abar)) @ vs) + 2.0 ** -18 * (p @ vs)
            err = np.abs(out[rows, h] - p @ v)
            assert (err <= tol).all(), (s, h, float((err / tol).max()))
            if lse is not None:
                assert (np.abs(lse[rows, h] - z) <= 2.0 ** -21 * abar[:, 0] + 2.0 ** -20 * (1 + np.abs(z))).all()
            total_w[s, g, :len(here)] += p.sum(axis=0)
            tol_w[s, g, :len(here)] += (p * (2.0 ** -21 * (a + abar) + 2.0 ** -20 * (1 + np.abs(z[:, None])))).sum(axis=0)
    if weight is not None:
        want = box.weight.astype(np.float64) + total_w
        # (one rounding of the stored sum, sqrt(columns) of the columns' own)
        tol = tol_w + 2.0 ** -21 * total_w + 2.0 ** -23 * want
        assert (np.abs(weight - want) <= tol).all(), float((np.abs(weight - want) / np.maximum(tol, 1e-300)).max())


def attend(fh, box, n_heads, lens, news, seed, use_off, masks=None, softcap=0.0, slopes=None, qpos=None, weigh=False,
           max_keys=None, ld_pad=0, tail=0):
    import ferrum_hip
    import torch

    rng = np.random.default_rng(seed)
    total, hd = sum(news) + tail, box.hd
    q = rng.standard_normal((total, n_heads, hd)).astype(np.float32)
    ld = n_heads * hd + ld_pad
    qb = np.full((total, ld), np.nan, np.float32)
    qb[:, :n_heads * hd] = q.reshape(total, -1)
    off, _ = rows_of(lens, news)
    first, end = (None, None) if masks is None else masks
    pad = lambda x: None if x is None else ints(list(x) + [0] * tail)  # noqa: E731
    out = torch.full((total, n_heads * hd), 7.0, device="cuda")
    lse = torch.full((total, n_heads), 7.0, device="cuda")
    sc = ferrum_hip.AttnScore(softcap, None if slopes is None else gpu(slopes, np.float32), pad(qpos), pad(first), pad(end))
    mk = max(a + b for a, b in zip(lens, news)) if max_keys is None else max_keys
    args = (fh, box.c, gpu(qb), ld, total, n_heads, ints(off) if use_off else None, max(news), ints(lens), mk, sc)
    torch.cuda.synchronize()
    ferrum_hip.kv4_attention_async(*args, out, lse)
    if weigh:
        ferrum_hip.kv4_weigh_async(*args, lse)
    fh.sync()
    o, z = out.cpu().numpy(), lse.cpu().numpy()
    if tail:
        assert (o[-tail:] == 7).all() and (z[-tail:] == 7).all()
        o, z, q = o[:-tail], z[:-tail], q[:-tail]
    check_attention(box, q, lens, news, o.reshape(-1, n_heads, hd), z, first, end, softcap,
                    None if slopes is None else np.asarray(slopes, np.float32), qpos,
                    box.plane("weight") if weigh else None)
    return o


# ---- append and read ------------------------------------------------------------


@pytest.mark.parametrize("n_heads,n_kv,hd", HEADS)
@pytest.mark.parametrize("lens,news", [([0], [1]), ([7, 0, 8, 3], [1, 1, 1, 1]), ([5, 0], [30, 30]), ([3, 8, 20], [0, 17, 4])])
@pytest.mark.parametrize("rope", [None, "norm", "neox", "part"])
@pytest.mark.parametrize("pad", [0, 3])  # (rows that are 16-byte aligned, and rows that are not)
def test_append_writes_the_formats_bytes(fh, n_heads, n_kv, hd, lens, news, rope, pad):
    import ferrum_hip
    import torch

    rng = np.random.default_rng(sum(lens) + hd)
    cap, seqs, total = 40, len(lens), sum(news)
    box = Box(seqs, n_kv, hd, cap, lens, 1, tracked=True)
    before = {n: box.plane(n).copy() for n in ("k", "k_d", "v", "v_d", "pos", "weight")}
    wide = (n_heads + 2 * n_kv) * hd
    x = rng.standard_normal((total, n_heads + 2 * n_kv, hd)).astype(np.float32)
    if rope is None and total:  # blocks at the edges of the format
        e = x[0, n_heads:, :32]
        e[0] = 0
        e[-1] = np.where(np.arange(32) % 2, 2.0, -2.0)
        if n_kv > 1:
            e[1] = np.arange(32) * 0.5 - 8
            e[-2] = 3e6
        if total > 2:
            x[1, n_heads, 5] = np.inf
            x[1, n_heads + n_kv, hd - 1] = np.nan
            x[2, n_heads:] *= np.float32(1e-7)
    off, places = rows_of(lens, news)
    pos = rng.integers(0, 5000, total)
    rd = 0 if rope is None else hd // 2 if rope == "part" else hd
    ff = rng.uniform(0.5, 2, rd // 2).astype(np.float32) if rope == "part" else None
    lin = 2.0 if rope == "part" else 1.0
    buf = np.full((total, wide + pad), np.nan, np.float32)
    buf[:, :wide] = x.reshape(total, wide)
    q = torch.full((total, n_heads * hd), float("nan"), device="cuda")
    uniform = len(set(news)) == 1
    args = (gpu(buf), wide + pad, total, n_heads, None if uniform else ints(off), max(news), ints(lens), ints(pos), rd, 1e4,
            ferrum_hip.ROPE_NORM if rope == "norm" else ferrum_hip.ROPE_NEOX, None if ff is None else gpu(ff), lin, q)
    torch.cuda.synchronize()
    ferrum_hip.kv4_append_async(fh, box.c, *args)
    fh.sync()
    turned = ref.rotate(x[:, :n_heads + n_kv], pos, rd, 1e4, rope != "norm", ff, lin)
    k, v = turned[:, n_heads:].astype(np.float32), x[:, n_heads + n_kv:]
    got_q = q.cpu().numpy().reshape(total, n_heads, hd)
    assert np.allclose(got_q, turned[:, :n_heads], rtol=2.0 ** -23, atol=2.0 ** -45)  # one f32 rounding of a float64 result
    after = {n: box.plane(n) for n in before}
    touched = {n: np.zeros(before[n].shape, bool) for n in before}
    (dk, qk), (dv, qv) = ref.quantise(k), ref.quantise(v)
    for s, row, at, _ in places:
        if at >= cap:
            continue
        for h in range(n_kv):
            for name, lev, sc, isv in (("k", qk, dk, False), ("v", qv, dv, True)):
                _, gq, gd = ref.unpack(after[name][s, h], after[name + "_d"][s, h], hd, [at], isv)
                assert np.array_equal(gq[0], lev[row, h]), (name, s, row, h)
                assert np.array_equal(gd[0].view(np.uint16) & 0x7FFF, sc[row, h].view(np.uint16) & 0x7FFF)
                assert np.array_equal(np.isnan(gd[0]) | (gd[0] == sc[row, h]), np.ones(hd // 32, bool))
                place = ref.v_place if isv else ref.k_place
                for c in range(hd):
                    touched[name][s, h, place(at, c, hd)[0]] = True
                touched[name + "_d"][s, h, at // 8, :, at % 8] = True
            assert after["pos"][s, h, at] == pos[row] and after["weight"][s, h, at] == 0
            touched["pos"][s, h, at] = touched["weight"][s, h, at] = True
    for n in before:  # every other byte as it was
        keep = ~touched[n]
        a, b = (z.view(np.uint16) if z.dtype == np.float16 else z for z in (after[n], before[n]))
        assert np.array_equal(a[keep], b[keep]), n


def test_append_past_the_capacity_stores_what_fits(fh):
    import ferrum_hip
    import torch

    box = Box(2, 1, 64, 16, [12, 16], 3, tracked=True)
    x = np.random.default_rng(0).standard_normal((16, 3 * 64)).astype(np.float32)
    old = box.plane("k").copy()
    q = torch.zeros((16, 64), device="cuda")
    torch.cuda.synchronize()
    ferrum_hip.kv4_append_async(fh, box.c, gpu(x), 192, 16, 1, None, 8, ints([12, 16]), q=q)
    fh.sync()
    new = box.plane("k")
    assert np.array_equal(old[0, 0, :12 * 32], new[0, 0, :12 * 32]) and np.array_equal(old[1], new[1])
    _, lev, _ = ref.unpack(new[0, 0], box.plane("k_d")[0, 0], 64, range(12, 16), False)
    assert np.array_equal(lev, ref.quantise(x[:4, 64:128])[1])
    assert np.array_equal(q.cpu().numpy(), x[:, :64])  # no rotation: q as it is, for every row


@pytest.mark.parametrize("n_heads,n_kv,hd", HEADS)
def test_read_gives_the_values_the_blocks_stand_for(fh, n_heads, n_kv, hd):
    import ferrum_hip
    import torch

    box = Box(3, n_kv, hd, 24, [24, 24, 24], 9)
    first, rows = [0, 5, 20], 7
    k, v = (torch.zeros((3, rows, n_kv * hd), device="cuda") for _ in range(2))
    f = ints(first)
    torch.cuda.synchronize()
    ferrum_hip.kv4_read_async(fh, box.c, f, rows, k, v)
    fh.sync()
    for got, want in ((k, box.k), (v, box.v)):
        got = got.cpu().numpy().reshape(3, rows, n_kv, hd)
        for s in range(3):
            n = min(rows, 24 - first[s])
            assert np.array_equal(got[s, :n], want[s, :, first[s]:first[s] + n].transpose(1, 0, 2).astype(np.float32))
            assert np.isnan(got[s, n:]).all()


# ---- attention ------------------------------------------------------------------


@pytest.mark.parametrize("n_heads,n_kv,hd", HEADS)
@pytest.mark.parametrize("lens", [[0], [1], [31, 32, 33], [7, 0, 300, 64, 255]])
def test_decode(fh, n_heads, n_kv, hd, lens):
    cap = -(-(max(lens) + 1) // 8) * 8
    box = Box(len(lens), n_kv, hd, cap, [n + 1 for n in lens], 4)
    attend(fh, box, n_heads, lens, [1] * len(lens), 5, False)


@pytest.mark.parametrize("n_heads,n_kv,hd", [(14, 2, 64), (4, 4, 32), (8, 2, 128)])
def test_decode_of_long_rows_splits_the_keys(fh, n_heads, n_kv, hd):
    lens = [2500, 9, 1777]
    box = Box(3, n_kv, hd, 2504, [n + 1 for n in lens], 6, tracked=True)
    attend(fh, box, n_heads, lens, [1] * 3, 7, False, weigh=True)


@pytest.mark.parametrize("n_heads,n_kv,hd", HEADS)
@pytest.mark.parametrize("lens,news", [([0], [2]), ([0], [45]), ([13, 0, 40], [3, 70, 1]), ([0, 5], [0, 33])])
def test_prompts(fh, n_heads, n_kv, hd, lens, news):
    cap = -(-max(a + b for a, b in zip(lens, news)) // 8) * 8
    box = Box(len(lens), n_kv, hd, cap, [a + b for a, b in zip(lens, news)], 8, tracked=True)
    attend(fh, box, n_heads, lens, news, 9, True, weigh=True, ld_pad=5, tail=3)


# Enough columns (at least 512 workgroups of 128, three quarters of them in use) for the form
# in which columns share each key's expansion.
MANY = [(8, 2, 64, 32), (8, 2, 128, 32), (12, 12, 64, 6)]


@pytest.mark.parametrize("n_heads,n_kv,hd,repeat", MANY)
@pytest.mark.parametrize("kind", ["causal", "documents", "prefix", "holes", "beyond"])
@pytest.mark.parametrize("options", [False, True])
def test_many_rows(fh, n_heads, n_kv, hd, repeat, kind, options):
    lens, news = [0, 41, 7, 130] * repeat, [120, 101, 117, 128] * repeat
    if n_kv == 12:
        lens, news = [0, 41, 7, 130] * repeat, [480, 501, 417, 510] * repeat
    top = max(a + b for a, b in zip(lens, news))
    box = Box(4, n_kv, hd, -(-top // 8) * 8, [a + b for a, b in zip(lens, news)][:4], 18, repeat=repeat)
    masks = None if kind == "causal" else masks_of(kind, lens, news, np.random.default_rng(2))
    slopes = 2.0 ** (-8.0 * np.arange(1, n_heads + 1) / n_heads) if options else None
    attend(fh, box, n_heads, lens, news, 19, True, masks, softcap=3.0 if options else 0.0, slopes=slopes, ld_pad=4, tail=2)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("repeat", [1, 64])  # (few columns, and many)
def test_values_far_apart(fh, repeat, hd):
    """A document of huge keys and values beside one of tiny ones, a NaN in a third, and blocks of
    very different size: each row has the accuracy of what it sees."""
    import torch

    n_kv = 2
    lens, news = [0, 0] * repeat, [96, 96] * repeat
    box = Box(2, n_kv, hd, 96, [96, 96], 80, repeat=repeat)
    nb = hd // 32
    scale = np.ones((96, nb))
    scale[32:40] = 2.0 ** 12
    scale[40:64] = 2.0 ** -9
    scale[:, nb // 2:] *= 2.0 ** -3
    by = scale.reshape(12, 8, nb).transpose(0, 2, 1)
    for name, val, step, f in (("k_d", box.k, box.kstep, np.where(by > 1, 4.0, 0.5)), ("v_d", box.v, box.vstep, by)):
        old = box.plane(name)
        new = (old.astype(np.float32) * f).astype(np.float16)  # (the smallest are subnormal: rounded again)
        ratio = np.repeat((new.astype(np.float64) / old.astype(np.float64)).transpose(0, 1, 2, 4, 3).reshape(
            box.seqs, n_kv, 96, nb), 32, axis=3)
        val *= ratio
        step *= np.abs(ratio)
        if name == "v_d":
            new[:, :, 9, 0, 3] = np.nan  # key 75
        box.c.planes[name].copy_(gpu(new))
    torch.cuda.synchronize()
    # documents: keys 0 .. 31, 32 .. 39, 40 .. 63, 64 .. 74, and rows of the last see 64 .. 74 too
    first, end = [], []
    for s in range(2 * repeat):
        for t in range(96):
            f = 0 if t < 32 else 32 if t < 40 else 40 if t < 64 else 64
            first.append(f)
            end.append(min(t + 1, 75))
    attend(fh, box, 8, lens, news, 81, True, (first, end))


@pytest.mark.parametrize("n_heads,n_kv,hd,rows", [(2, 2, 64, 1), (8, 1, 64, 1), (9, 1, 64, 1), (4, 2, 64, 4), (6, 2, 32, 2),
                                                  (2, 2, 32, 8), (4, 1, 128, 2), (3, 1, 128, 3)])
@pytest.mark.parametrize("kind", ["causal", "window", "holes"])
def test_few_columns_around_tiles(fh, n_heads, n_kv, hd, rows, kind):
    """Lengths around one tile of keys, two, the tiles that a workgroup's waves have, and its parts."""
    lens = [0, 30, 31, 32, 33, 62, 63, 64, 65, 127, 255, 256, 257, 511, 513, 1000, 1023, 2040]
    news = [rows] * len(lens)
    box = Box(len(lens), n_kv, hd, 2048, [a + rows for a in lens], 84, tracked=True)
    masks = None
    if kind == "window":
        masks = [max(0, a + t - 40) for a in lens for t in range(rows)], [a + t + 1 for a in lens for t in range(rows)]
    elif kind == "holes":
        masks = masks_of(kind, lens, news, np.random.default_rng(3))
    attend(fh, box, n_heads, lens, news, 85, rows > 1, masks, weigh=True)


def masks_of(kind, lens, news, rng):
    first, end = [], []
    for at, new in zip(lens, news):
        for t in range(new):
            row = at + t
            if kind == "window":
                f, e = max(0, row - 9), row + 1
            elif kind == "documents":
                f, e = at + t // 11 * 11, row + 1
            elif kind == "prefix":
                f, e = 0, max(row + 1, at + new // 2)
            elif kind == "holes":  # some rows see nothing, some one key
                f, e = [(0, row + 1), (row, row + 1), (5, 5), (row + 1, row), (0, 1)][t % 5]
            else:  # beyond what is there
                f, e = int(rng.integers(0, 5)), 0xFFFFFFFF if t % 2 else at + new + 50
            first.append(f)
            end.append(e)
    return first, end


@pytest.mark.parametrize("n_heads,n_kv,hd", [(14, 2, 64), (4, 4, 32), (8, 2, 128)])
@pytest.mark.parametrize("kind", ["window", "documents", "prefix", "holes", "beyond"])
@pytest.mark.parametrize("rows", ["one", "many"])
def test_masks(fh, n_heads, n_kv, hd, kind, rows):
    lens, news = ([70, 3, 33], [1, 1, 1]) if rows == "one" else ([20, 0, 7], [40, 77, 9])
    box = Box(3, n_kv, hd, 80, [a + b for a, b in zip(lens, news)], 10, tracked=True)
    attend(fh, box, n_heads, lens, news, 11, rows == "many", masks_of(kind, lens, news, np.random.default_rng(1)), weigh=True)


@pytest.mark.parametrize("n_heads,n_kv,hd", [(14, 2, 64), (4, 4, 32), (8, 2, 128)])
@pytest.mark.parametrize("softcap", [0.0, 2.0, 30.0])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("rows", ["one", "many"])
def test_caps_and_biases(fh, n_heads, n_kv, hd, softcap, biased, rows):
    lens, news = ([170, 3], [1, 1]) if rows == "one" else ([20, 0], [40, 67])
    box = Box(2, n_kv, hd, 176, [a + b for a, b in zip(lens, news)], 12, tracked=True)
    slopes = 2.0 ** (-8.0 * np.arange(1, n_heads + 1) / n_heads) if biased else None
    attend(fh, box, n_heads, lens, news, 13, rows == "many", softcap=softcap, slopes=slopes, weigh=True)


@pytest.mark.parametrize("repeat", [1, 64])  # (few columns, and many)
@pytest.mark.parametrize("softcap", [0.0, 1e-44, 3e38])
def test_scores_of_no_size_and_caps_of_any(fh, repeat, softcap):
    """Rows of zero, of subnormal and of ordinary queries under a mask: with scores or a cap next to
    nothing the weights are all alike, with a cap beyond every score it changes nothing."""
    import ferrum_hip
    import torch

    seqs, rows, n_kv, hd = 2 * repeat, 48, 2, 64
    box = Box(2, n_kv, hd, 48, [48, 48], 82, repeat=repeat)
    q = np.random.default_rng(83).standard_normal((seqs, rows, 8, hd)).astype(np.float32)
    size = np.where(np.arange(rows) % 3 == 0, 0.0, np.where(np.arange(rows) % 3 == 1, 1e-41, 1.0))
    q = (q * size[None, :, None, None]).astype(np.float32)
    first = np.tile(np.arange(rows) // 11 * 11, seqs)
    out, lse = torch.zeros((seqs * rows, 8 * hd), device="cuda"), torch.zeros((seqs * rows, 8), device="cuda")
    sc = ferrum_hip.AttnScore(softcap, None, None, ints(first), None)
    args = (fh, box.c, gpu(q.reshape(seqs * rows, -1)), 8 * hd, seqs * rows, 8, None, rows, ints([0] * seqs), rows, sc)
    torch.cuda.synchronize()
    ferrum_hip.kv4_attention_async(*args, out, lse)
    fh.sync()
    # (a cap of 1e-44 leaves scores that no rounding of exp tells from 0)
    check_attention(box, q.reshape(-1, 8, hd) * np.float32(softcap != 1e-44), [0] * seqs, [rows] * seqs,
                    out.cpu().numpy().reshape(-1, 8, hd), lse.cpu().numpy(), first.tolist())


@pytest.mark.parametrize("n_heads,n_kv,hd,lens,news", [(8, 2, 128, [0], [700]), (4, 4, 64, [600, 0, 37], [530, 1, 300]),
                                                       (6, 1, 32, [1100, 513], [70, 129]), (2, 2, 64, [0] * 40, [33] * 40)])
@pytest.mark.parametrize("kind", ["causal", "window", "documents", "prefix", "beyond"])
@pytest.mark.parametrize("options", [False, True])
def test_weights_of_long_prompts(fh, n_heads, n_kv, hd, lens, news, kind, options):
    """Several groups of keys, parts of the rows and batches of columns; rows that see none of a group."""
    top = max(a + b for a, b in zip(lens, news))
    box = Box(len(lens), n_kv, hd, -(-top // 8) * 8, [a + b for a, b in zip(lens, news)], 87, tracked=True)
    masks = None if kind == "causal" else masks_of(kind, lens, news, np.random.default_rng(4))
    slopes = 2.0 ** (-8.0 * np.arange(1, n_heads + 1) / n_heads) if options else None
    attend(fh, box, n_heads, lens, news, 88, True, masks, softcap=4.0 if options else 0.0, slopes=slopes, weigh=True, tail=3)


def test_bias_goes_by_positions_not_rows(fh):
    """A cache whose rows are no longer their positions (as after an eviction)."""
    box = Box(2, 2, 64, 104, [100, 61], 14, tracked=True)
    box.pos = np.sort(np.random.default_rng(3).integers(0, 900, box.pos.shape), axis=2).astype(np.int32)
    box.c.planes["pos"].copy_(gpu(box.pos))
    slopes = 2.0 ** (-8.0 * np.arange(1, 15) / 14)
    attend(fh, box, 14, [99, 60], [1, 1], 15, False, slopes=slopes, qpos=[950, 901], weigh=True)


@pytest.mark.parametrize("k_std,v_std", [(1e-3, 1e-4), (8.0, 1e3), (1.0, 3e4)])
def test_scales_far_from_one(fh, k_std, v_std):
    lens = [600, 33]
    box = Box(2, 2, 128, 608, [n + 1 for n in lens], 16, k_std=k_std, v_std=v_std)
    attend(fh, box, 8, lens, [1, 1], 17, False)


def test_one_large_value_among_small_ones(fh):
    """The weights' f16 range follows the largest value scale; the others keep their bits."""
    import torch

    lens = [300]
    box = Box(1, 1, 64, 304, [301], 20)
    d = box.plane("v_d").copy()
    d[0, 0, 10, 1, 3] = np.float16(900.0)  # key 83, block 1
    box.vstep[0, 0, 83, 32:] = 900.0
    old = box.v[0, 0, 83, 32:].copy()
    lev, _, _ = ref.unpack(box.plane("v")[0, 0], d[0, 0], 64, [83], True)
    box.v[0, 0, 83, 32:] = lev[0, 32:]
    assert not np.array_equal(old, lev[0, 32:])
    box.c.planes["v_d"].copy_(gpu(d))
    torch.cuda.synchronize()
    attend(fh, box, 7, lens, [1], 21, False)


def test_rows_beyond_the_bounds_are_nan_and_nothing_else_is(fh):
    import ferrum_hip
    import torch

    box = Box(3, 2, 64, 32, [32, 32, 10], 22)
    q = torch.randn((3, 14 * 64), device="cuda")
    out = torch.zeros_like(q)
    lens = ints([32, 0xFFFFFFFF, 9])  # at the capacity, far past it, inside
    torch.cuda.synchronize()
    ferrum_hip.kv4_attention_async(fh, box.c, q, 14 * 64, 3, 14, None, 1, lens, 64, None, out)
    fh.sync()
    o = out.cpu().numpy()
    assert np.isnan(o[:2]).all() and np.isfinite(o[2]).all()
    ferrum_hip.kv4_attention_async(fh, box.c, q, 14 * 64, 3, 14, None, 1, ints([8, 9, 7]), 9, None, out)
    fh.sync()
    o = out.cpu().numpy()
    assert np.isfinite(o[0]).all() and np.isnan(o[1]).all() and np.isfinite(o[2]).all()


def test_offsets_that_decrease_or_run_out_stay_inside(fh):
    import ferrum_hip
    import torch

    box = Box(3, 2, 64, 32, [8, 8, 8], 23)
    q = torch.randn((6, 14 * 64), device="cuda")
    out = torch.full_like(q, 7.0)
    off = ints([2, 1, 900, 0xFFFFFFFF])  # nothing; rows 1 .. 5; nothing (behind the end)
    torch.cuda.synchronize()
    ferrum_hip.kv4_attention_async(fh, box.c, q, 14 * 64, 6, 14, off, 4, None, 32, None, out)
    fh.sync()
    o = out.cpu().numpy()
    assert (o[0] == 7).all() and (o[5] == 7).all()  # (max_rows 4: rows 1 .. 4)
    assert np.isfinite(o[1:5]).all() and (o[1:5] != 7).any()


def test_a_nan_key_reaches_only_the_rows_that_see_it(fh):
    import ferrum_hip
    import torch

    for name in ("k_d", "v_d"):
        box = Box(1, 2, 64, 64, [60], 24)
        box.c.planes[name][0, 0, 5, 1, 0] = float("nan")  # key 40 of head 0
        q = torch.randn((20, 14 * 64), device="cuda")
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        ferrum_hip.kv4_attention_async(fh, box.c, q, 14 * 64, 20, 14, None, 20, ints([30]), 64, None, out)
        fh.sync()
        o = out.cpu().numpy().reshape(20, 14, 64)
        assert np.isfinite(o[:10]).all() and np.isfinite(o[10:, 7:]).all()
        assert np.isnan(o[10:, :7]).any(axis=(1, 2)).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("name", ["k_d", "v_d"])
def test_a_nan_key_among_many_rows(fh, hd, name):
    """In every fourth sequence: its neighbours and the rows before it stay as they were, and a NaN
    among the values is none of the scores'."""
    import ferrum_hip
    import torch

    seqs, rows = 128, 64
    box = Box(4, 2, hd, 64, [64] * 4, 25, repeat=seqs // 4)
    q = torch.randn((seqs * rows, 8 * hd), device="cuda")
    outs = []
    for bad in (False, True):
        if bad:
            box.c.planes[name][::4, 0, 5, 1, 0] = float("nan")  # key 40 of head 0
        out, lse = torch.zeros_like(q), torch.zeros((seqs * rows, 8), device="cuda")
        torch.cuda.synchronize()
        ferrum_hip.kv4_attention_async(fh, box.c, q, 8 * hd, seqs * rows, 8, ints(np.arange(seqs + 1) * rows), rows,
                                       ints([0] * seqs), 64, None, out, lse)
        fh.sync()
        outs.append((out.cpu().numpy().reshape(seqs, rows, 8, hd), lse.cpu().numpy().reshape(seqs, rows, 8)))
    (o, z), (ob, zb) = outs
    hit = np.zeros((seqs, rows, 8), bool)
    hit[::4, 40:, :4] = True
    assert np.isfinite(o).all() and np.array_equal(ob[~hit], o[~hit]) and np.array_equal(zb[~hit], z[~hit])
    assert np.isnan(ob[hit]).any(axis=-1).all()
    if name == "k_d":
        assert np.isnan(zb[hit]).all()
    else:
        # The scores are the same bits, but the running maximum goes by the values' exponents too, and a
        # NaN has none: other powers of two stand before the sums, so exp2's arguments round elsewhere.
        # Either sum is within 2^-20 of itself (exp2 2^-23 and its argument 2^-22, 64 terms' additions
        # at most 2^-21 together in sequences of 8, 2 and 4), its log and the product 2^-23 (1 + |z|).
        assert (np.abs(zb[hit] - z[hit]) <= 2.0 ** -19 + 2.0 ** -22 * (1 + np.abs(z[hit]))).all()


# ---- eviction -------------------------------------------------------------------


@pytest.mark.parametrize("n_heads,n_kv,hd", HEADS)
@pytest.mark.parametrize("lens,keep,recent", [([30, 5, 17], 16, 4), ([200, 64, 65], 64, 0), ([200, 150, 90], 70, 70),
                                              ([33], 1, 0), ([1500, 1500], 1100, 100)])
def test_evict(fh, n_heads, n_kv, hd, lens, keep, recent):
    import ferrum_hip
    import torch

    cap, kcap = -(-max(lens) // 8) * 8, -(-keep // 8) * 8
    box = Box(len(lens), n_kv, hd, cap, lens, 30, tracked=True)
    w = box.weight
    w[:, :, ::3] = 0.25  # ties: the first ones stay
    w[:, 0, 4] = np.nan
    w[:, 0, 6], w[:, 0, 7] = 0.0, -0.0
    box.pos = (box.pos * 3 + 1).astype(np.int32)
    box.c.planes["weight"].copy_(gpu(w))
    box.c.planes["pos"].copy_(gpu(box.pos))
    to = Box(len(lens), n_kv, hd, kcap, [0] * len(lens), 31, tracked=True)
    names = ("k", "k_d", "v", "v_d", "pos", "weight")
    before = {n: to.plane(n).copy() for n in names}
    src = {n: box.plane(n).copy() for n in names}
    ln = ints(lens)
    torch.cuda.synchronize()
    ferrum_hip.kv4_evict_async(fh, box.c, to.c, ln, max(lens), keep, recent, ln)
    fh.sync()
    assert list(ln.cpu().numpy()) == [min(n, keep) for n in lens]
    after = {n: to.plane(n) for n in names}
    for n in names:
        assert np.array_equal(src[n].view(np.uint8), box.plane(n).view(np.uint8)), n  # the source is read only
    for s, n in enumerate(lens):
        for h in range(n_kv):
            kept = ref.evict(w[s, h], n, keep, recent)
            m = len(kept)
            assert m == min(n, keep)
            assert np.array_equal(after["pos"][s, h, :m], box.pos[s, h, kept])
            assert np.array_equal(after["weight"][s, h, :m].view(np.uint32), w[s, h, kept].view(np.uint32))
            for name, isv in (("k", False), ("v", True)):
                _, lev, sc = ref.unpack(after[name][s, h], after[name + "_d"][s, h], hd, range(m), isv)
                _, lw, sw = ref.unpack(src[name][s, h], src[name + "_d"][s, h], hd, kept, isv)
                assert np.array_equal(lev, lw) and np.array_equal(sc.view(np.uint16), sw.view(np.uint16))
                if m < kcap:
                    _, lev, sc = ref.unpack(after[name][s, h], after[name + "_d"][s, h], hd, range(m, kcap), isv)
                    _, lw, sw = ref.unpack(before[name][s, h], before[name + "_d"][s, h], hd, range(m, kcap), isv)
                    assert np.array_equal(lev, lw) and np.array_equal(sc.view(np.uint16), sw.view(np.uint16))


# ---- together -------------------------------------------------------------------


@pytest.mark.parametrize("src_pos,dst_pos,dst_weight", [(True, False, False), (False, True, True), (True, True, False)])
def test_evict_with_fewer_planes_and_lengths_cut(fh, src_pos, dst_pos, dst_weight):
    """Planes that one side lacks, lengths above max_len and the capacity, the lengths' own place kept."""
    import ferrum_hip
    import torch

    lens, cap, max_len, keep, recent = [90, 64, 300, 20, 0], 96, 80, 33, 5
    box = Box(5, 2, 64, cap, [min(n, cap) for n in lens], 89, tracked=True)
    p = box.c.planes
    src = ferrum_hip.KV4Cache(5, 2, 64, cap, p["k"], p["k_d"], p["v"], p["v_d"], p["pos"] if src_pos else None, p["weight"])
    to = Box(5, 2, 64, 40, [0] * 5, 90, tracked=True)
    t = to.c.planes
    dst = ferrum_hip.KV4Cache(5, 2, 64, 40, t["k"], t["k_d"], t["v"], t["v_d"], t["pos"] if dst_pos else None,
                              t["weight"] if dst_weight else None)
    untouched = {n: to.plane(n).copy() for n, own in (("pos", dst_pos), ("weight", dst_weight)) if not own}
    ln, new = ints(lens), ints([7] * 5)
    torch.cuda.synchronize()
    ferrum_hip.kv4_evict_async(fh, src, dst, ln, max_len, keep, recent, new)
    fh.sync()
    assert list(ln.cpu().numpy()) == lens and list(new.cpu().numpy()) == [33, 33, 33, 20, 0]
    for n, old in untouched.items():
        assert np.array_equal(to.plane(n).view(np.uint8), old.view(np.uint8))
    k, v = (torch.zeros((5, keep, 2 * 64), device="cuda") for _ in range(2))
    ferrum_hip.kv4_read_async(fh, dst, None, keep, k, v)
    fh.sync()
    k, v = (x.cpu().numpy().reshape(5, keep, 2, 64) for x in (k, v))
    for s, n in enumerate(min(n, max_len) for n in lens):
        for h in range(2):
            kept = ref.evict(box.weight[s, h], n, keep, recent)
            assert np.array_equal(k[s, :len(kept), h], box.k[s, h, kept].astype(np.float32))
            assert np.array_equal(v[s, :len(kept), h], box.v[s, h, kept].astype(np.float32))
            if dst_pos:
                assert np.array_equal(to.plane("pos")[s, h, :len(kept)], box.pos[s, h, kept] if src_pos else kept)
            if dst_weight:
                assert np.array_equal(to.plane("weight")[s, h, :len(kept)], box.weight[s, h, kept])


@pytest.mark.parametrize("n_heads,n_kv,hd,rows", [(14, 2, 64, 1), (64, 1, 64, 1), (8, 2, 128, 1), (6, 3, 32, 50)])
def test_the_same_call_gives_the_same_bits(fh, n_heads, n_kv, hd, rows):
    """Keys dealt over workgroups are joined in order; no length array: caches that begin with the call."""
    import ferrum_hip
    import torch

    lens = [3000, 17] if rows == 1 else None
    news = [rows, rows]
    box = Box(2, n_kv, hd, 3008, [a + rows for a in lens] if lens else news, 91, tracked=True)
    q = gpu(np.random.default_rng(92).standard_normal((2 * rows, n_heads * hd)).astype(np.float32))
    results = []
    for _ in range(3):
        out, lse = torch.zeros_like(q), torch.zeros((2 * rows, n_heads), device="cuda")
        box.c.planes["weight"].copy_(gpu(box.weight))
        torch.cuda.synchronize()
        args = (fh, box.c, q, n_heads * hd, 2 * rows, n_heads, None, rows, ints(lens) if lens else None, 3008, None)
        ferrum_hip.kv4_attention_async(*args, out, lse)
        ferrum_hip.kv4_weigh_async(*args, lse)
        fh.sync()
        results.append((out.cpu().numpy(), lse.cpu().numpy(), box.plane("weight").copy()))
    for r in results[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(r, results[0]))
    o, z, w = results[0]
    check_attention(box, q.cpu().numpy().reshape(-1, n_heads, hd), lens or [0, 0], news, o.reshape(-1, n_heads, hd), z, weight=w)


@pytest.mark.parametrize("keep,recent", [(16000, 100), (20000, 20000), (39999, 1), (1, 0)])
@pytest.mark.parametrize("values", ["distinct", "few", "one"])
def test_evict_from_long_caches(fh, keep, recent, values):
    """More rows than are held in registers; cuts between weights and within ties."""
    import ferrum_hip
    import torch

    lens, cap, rng = [40000, 16385, 16384, 30011], 40000, np.random.default_rng(86)
    src, dst = (ferrum_hip.KV4Cache.alloc(4, 1, 32, c, True) for c in (cap, -(-keep // 8) * 8))
    w = rng.random((4, 1, cap)).astype(np.float32) ** 4
    w = w if values == "distinct" else np.floor(w * 7).astype(np.float32) if values == "few" else np.ones_like(w)
    src.planes["weight"].copy_(gpu(w))
    src.planes["pos"].copy_(torch.arange(cap, dtype=torch.int32, device="cuda"))
    new = ints([0] * 4)
    torch.cuda.synchronize()
    ferrum_hip.kv4_evict_async(fh, src, dst, ints(lens), cap, keep, recent, new)
    fh.sync()
    assert list(new.cpu().numpy()) == [min(n, keep) for n in lens]
    pos, got = dst.planes["pos"].cpu().numpy(), dst.planes["weight"].cpu().numpy()
    for s, n in enumerate(lens):
        kept = ref.evict(w[s, 0], n, keep, recent)
        assert np.array_equal(pos[s, 0, :len(kept)], kept) and np.array_equal(got[s, 0, :len(kept)], w[s, 0, kept])


def test_a_run_of_them_together(fh):
    """A prompt, its weights, an eviction and decode steps over what is left: the
    attention of every step is that of the rows that a float64 account keeps."""
    import ferrum_hip
    import torch

    n_heads, n_kv, hd, keep, recent, prompt = 14, 2, 64, 40, 8, 60
    rng = np.random.default_rng(40)
    caches = [ferrum_hip.KV4Cache.alloc(1, n_kv, hd, 72, tracked=True) for _ in range(2)]
    wide = (n_heads + 2 * n_kv) * hd
    k, v = [np.zeros((0, hd)) for _ in range(n_kv)], [np.zeros((0, hd)) for _ in range(n_kv)]
    ln, at = torch.zeros(1, dtype=torch.int32, device="cuda"), 0
    for rows in [prompt] + [1] * 6:
        x = rng.standard_normal((rows, n_heads + 2 * n_kv, hd)).astype(np.float32)
        pos = np.arange(at, at + rows)
        qkv, q = gpu(x.reshape(rows, wide)), torch.empty((rows, n_heads * hd), device="cuda")
        out, lse, p = torch.empty_like(q), torch.empty((rows, n_heads), device="cuda"), ints(pos)
        torch.cuda.synchronize()
        used = int(ln.item())
        ferrum_hip.kv4_append_async(fh, caches[0], qkv, wide, rows, n_heads, None, rows, ln, p, hd, 1e6, 1, None, 1.0, q)
        args = (fh, caches[0], q, n_heads * hd, rows, n_heads, None, rows, ln, used + rows, None)
        ferrum_hip.kv4_attention_async(*args, out, lse)
        ferrum_hip.kv4_weigh_async(*args, lse)
        fh.sync()
        turned = ref.rotate(x[:, :n_heads + n_kv], pos, hd, 1e6, True)
        for h in range(n_kv):
            k[h] = np.concatenate([k[h], ref.values(*ref.quantise(turned[:, n_heads + h].astype(np.float32)))])
            v[h] = np.concatenate([v[h], ref.values(*ref.quantise(x[:, n_heads + n_kv + h]))])
        o, _, _ = ref.attention(turned[:, :n_heads].astype(np.float32), np.stack(k), np.stack(v), [0] * rows,
                                used + np.arange(rows) + 1)
        got = out.cpu().numpy().reshape(o.shape)
        # (1e-5 of the values' size: every score here is below 2^4, see check_attention)
        assert np.abs(got - o).max() <= 1e-5 * np.abs(np.stack(v)).max()
        ln += rows
        at += rows
        torch.cuda.synchronize()
        if int(ln.item()) > keep:
            w = caches[0].planes["weight"].cpu().numpy()
            n = int(ln.item())
            ferrum_hip.kv4_evict_async(fh, caches[0], caches[1], ln, n, keep, recent, ln)
            fh.sync()
            caches.reverse()
            for h in range(n_kv):
                stay = ref.evict(w[0, h], n, keep, recent)
                k[h], v[h] = k[h][stay], v[h][stay]
        torch.cuda.synchronize()


def test_captured_calls_replay_as_they_ran(fh):
    import ferrum_hip
    import torch

    rng = np.random.default_rng(50)
    lens = [900, 17, 333]
    n_heads, n_kv, hd = 14, 2, 64
    box = Box(3, n_kv, hd, 904, [n + 1 for n in lens], 51, tracked=True)
    wide = (n_heads + 2 * n_kv) * hd
    x = gpu(rng.standard_normal((3, wide)).astype(np.float32))
    q, out = torch.empty((3, n_heads * hd), device="cuda"), torch.empty((3, n_heads * hd), device="cuda")
    lse, ln = torch.empty((3, n_heads), device="cuda"), ints(lens)
    weight = box.c.planes["weight"].clone()

    def calls():
        ferrum_hip.kv4_append_async(fh, box.c, x, wide, 3, n_heads, None, 1, ln, None, hd, 1e6, 1, None, 1.0, q)
        args = (fh, box.c, q, n_heads * hd, 3, n_heads, None, 1, ln, 901, None)
        ferrum_hip.kv4_attention_async(*args, out, lse)
        ferrum_hip.kv4_weigh_async(*args, lse)

    torch.cuda.synchronize()
    calls()  # (the workspace exists from here on)
    fh.sync()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    try:
        with torch.cuda.graph(g, stream=s):
            fh.set_stream(torch.cuda.current_stream().cuda_stream)
            calls()
    finally:
        fh.set_stream(None)
    seen = []
    for i in range(4):
        for how in (g.replay, calls):
            box.c.planes["weight"].copy_(weight)
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            how()
            torch.cuda.synchronize()
            fh.sync()
            seen.append((out.cpu().numpy().view(np.uint32).copy(), box.plane("weight").view(np.uint32).copy()))
    assert np.isfinite(seen[0][0].view(np.float32)).all()
    assert all(np.array_equal(a, seen[0][0]) and np.array_equal(b, seen[0][1]) for a, b in seen)


def test_capture_needs_a_first_run_and_outlives_larger_ones():
    """On a fresh context the calls that need workspace refuse to be captured; after one
    run they can be, and a larger call later leaves the captured graph as it was."""
    import ferrum_hip
    import torch

    def args(c, box, rows, lens):
        q = torch.randn((len(lens) * rows, 8 * 128), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
        out, lse = torch.empty_like(q), torch.empty((len(lens) * rows, 8), device="cuda")
        return (c, box.c, q, 1024, len(lens) * rows, 8, None, rows, ints(lens), max(lens) + rows, None), out, lse

    with ferrum_hip.Context(0) as c:
        box = Box(1, 2, 128, 1024, [1000], 61, tracked=True)
        start = box.c.planes["weight"].clone()
        spare = Box(1, 2, 128, 512, [0], 62, tracked=True)
        a, out, lse = args(c, box, 100, [900])
        ln, new = ints([1000]), ints([0])

        def calls():
            ferrum_hip.kv4_attention_async(*a, out, lse)
            ferrum_hip.kv4_weigh_async(*a, lse)
            ferrum_hip.kv4_evict_async(c, box.c, spare.c, ln, 1000, 500, 20, new)

        def capture():
            g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            refused = []
            try:
                with torch.cuda.graph(g, stream=s):
                    c.set_stream(torch.cuda.current_stream().cuda_stream)
                    try:
                        calls()
                    except ferrum_hip.FerrumHipError as e:
                        refused.append(e)
            finally:
                c.set_stream(None)
            return g, refused

        torch.cuda.synchronize()
        _, refused = capture()
        assert refused and "outside capture first" in refused[0].msg
        calls()
        c.sync()
        box.c.planes["weight"].copy_(start)
        torch.cuda.synchronize()
        calls()
        c.sync()
        want = [t.clone() for t in (out, box.c.planes["weight"], spare.c.planes["pos"], new)]
        g, refused = capture()
        assert not refused
        big = Box(4, 2, 128, 2048, [2000] * 4, 63, tracked=True)
        b, out2, lse2 = args(c, big, 300, [1700] * 4)
        to = Box(4, 2, 128, 1600, [0] * 4, 64, tracked=True)
        ferrum_hip.kv4_attention_async(*b, out2, lse2)
        ferrum_hip.kv4_weigh_async(*b, lse2)
        ferrum_hip.kv4_evict_async(c, big.c, to.c, ints([2000] * 4), 2000, 1600, 20, ints([0] * 4))
        c.sync()
        for _ in range(3):
            box.c.planes["weight"].copy_(start)
            out.fill_(float("nan"))
            new.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want, (out, box.c.planes["weight"], spare.c.planes["pos"], new)))


def test_planes_beyond_four_gibibytes(fh):
    """The last of 20 sequences, whose levels lie past 2^32 bytes of their planes."""
    import ferrum_hip
    import torch

    seqs, n_kv, hd, cap, n = 20, 8, 128, 1 << 19, 70
    small = Box(1, n_kv, hd, 80, [n + 1], 70, tracked=True)
    nb = hd // 32
    zeros = lambda dt, *s: torch.zeros((seqs, n_kv, *s), dtype=dt, device="cuda")  # noqa: E731
    k, v = zeros(torch.uint8, cap * hd // 2), zeros(torch.uint8, cap * hd // 2)
    assert k.numel() > 2 ** 32
    kd, vd = zeros(torch.float16, cap // 8, nb, 8), zeros(torch.float16, cap // 8, nb, 8)
    weight = zeros(torch.float32, cap)
    p = small.c.planes
    for big, name in ((k, "k"), (kd, "k_d"), (v, "v"), (vd, "v_d")):
        big[-1, :, :p[name].shape[2]] = p[name][0]
    c = ferrum_hip.KV4Cache(seqs, n_kv, hd, cap, k, kd, v, vd, None, weight)
    one = dict(total=seqs, q=torch.randn((seqs, 32 * hd), device="cuda"))
    lens = ints([0] * (seqs - 1) + [n])
    out, lse = torch.empty_like(one["q"]), torch.empty((seqs, 32), device="cuda")
    ref_out, ref_lse = torch.empty((1, 32 * hd), device="cuda"), torch.empty((1, 32), device="cuda")
    small.c.planes["weight"].zero_()
    torch.cuda.synchronize()
    args = (fh, c, one["q"], 32 * hd, seqs, 32, None, 1, lens, n + 1, None)
    ferrum_hip.kv4_attention_async(*args, out, lse)
    ferrum_hip.kv4_weigh_async(*args, lse)
    args = (fh, small.c, one["q"][-1:], 32 * hd, 1, 32, None, 1, ints([n]), n + 1, None)
    ferrum_hip.kv4_attention_async(*args, ref_out, ref_lse)
    ferrum_hip.kv4_weigh_async(*args, ref_lse)
    rk, rv = (torch.empty((seqs, n, n_kv * hd), device="cuda") for _ in range(2))
    sk, sv = (torch.empty((1, n, n_kv * hd), device="cuda") for _ in range(2))
    ferrum_hip.kv4_read_async(fh, c, None, n, rk, rv)
    ferrum_hip.kv4_read_async(fh, small.c, None, n, sk, sv)
    fh.sync()
    # (the two differ in how many workgroups share the keys, by roundings only)
    assert torch.allclose(out[-1], ref_out[0], rtol=1e-5, atol=1e-5) and torch.allclose(lse[-1], ref_lse[0], rtol=1e-5)
    assert torch.allclose(weight[-1, :, :n + 1], small.c.planes["weight"][0, :, :n + 1], rtol=1e-5, atol=1e-6)
    assert torch.equal(rk[-1], sk[0]) and torch.equal(rv[-1], sv[0])
    x = torch.randn((seqs, (32 + 16) * hd), device="cuda")
    to = ferrum_hip.KV4Cache.alloc(seqs, n_kv, hd, 64)
    new = ints([0] * seqs)
    torch.cuda.synchronize()
    ferrum_hip.kv4_append_async(fh, c, x, 48 * hd, seqs, 32, None, 1, lens)
    ferrum_hip.kv4_append_async(fh, small.c, x[-1:], 48 * hd, 1, 32, None, 1, ints([n]))
    weight[-1, :, :n] = torch.rand((n_kv, n), device="cuda")
    small.c.planes["weight"][0, :, :n] = weight[-1, :, :n]
    torch.cuda.synchronize()
    to1 = ferrum_hip.KV4Cache.alloc(1, n_kv, hd, 64)
    ferrum_hip.kv4_evict_async(fh, c, to, ints([0] * (seqs - 1) + [n + 1]), n + 1, 60, 5, new)
    ferrum_hip.kv4_evict_async(fh, small.c, to1, ints([n + 1]), n + 1, 60, 5, ints([0]))
    fh.sync()
    for name in ("k", "k_d", "v", "v_d"):
        assert torch.equal(to.planes[name][-1], to1.planes[name][0]), name


def test_two_contexts_on_two_streams_at_once(fh):
    import ferrum_hip
    import torch

    box = Box(2, 2, 128, 2048, [2048, 2048], 60)
    q = [torch.randn((2, 8 * 128), device="cuda") for _ in range(2)]
    lens = ints([2047, 1500])
    want, got = [torch.empty_like(a) for a in q], [torch.zeros_like(a) for a in q]
    torch.cuda.synchronize()
    for a, o in zip(q, want):
        ferrum_hip.kv4_attention_async(fh, box.c, a, 1024, 2, 8, None, 1, lens, 2048, None, o)
    fh.sync()
    with ferrum_hip.Context(0) as c1, ferrum_hip.Context(0) as c2:
        for _ in range(20):
            for c, a, o in zip((c1, c2), q, got):
                ferrum_hip.kv4_attention_async(c, box.c, a, 1024, 2, 8, None, 1, lens, 2048, None, o)
        c1.sync()
        c2.sync()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


# ---- refusals -------------------------------------------------------------------


def test_refusals(fh):
    import ferrum_hip as F
    import torch

    ok = F.KV4Cache.alloc(2, 2, 64, 32, tracked=True)
    bare = F.KV4Cache.alloc(2, 2, 64, 32)
    q, out = torch.zeros((2, 8 * 64), device="cuda"), torch.zeros((2, 4 * 64), device="cuda")
    ln = ints([0, 0])
    p = ok.planes

    def att(cache=ok, q=q, ld=512, total=2, heads=4, off=None, rows=1, score=None, out=out):
        return lambda: F.kv4_attention_async(fh, cache, q, ld, total, heads, off, rows, ln, 32, score, out)

    def cache(**kw):
        a = dict(seqs=2, n_kv=2, head_dim=64, capacity=32, k=p["k"], k_d=p["k_d"], v=p["v"], v_d=p["v_d"])
        a.update(kw)
        return F.KV4Cache(**a)

    cases = [
        (F.FH_ERR_INVALID, "cache is NULL", att(cache=None)),
        (F.FH_ERR_INVALID, "plane of the cache is NULL", att(cache=cache(v_d=None))),
        (F.FH_ERR_INVALID, "16-byte aligned", att(cache=cache(k=p["k"].data_ptr() + 8))),
        (F.FH_ERR_INVALID, "no sequences", att(cache=cache(seqs=0))),
        (F.FH_ERR_LIMIT, "head width 96", att(cache=cache(head_dim=96))),
        (F.FH_ERR_INVALID, "multiple of 8", att(cache=cache(capacity=12))),
        (F.FH_ERR_INVALID, "multiple of 8", att(cache=cache(capacity=0))),
        (F.FH_ERR_LIMIT, "too large", att(cache=cache(capacity=1 << 40))),
        (F.FH_ERR_DIM, "multiple of n_kv_heads", att(heads=3)),
        (F.FH_ERR_DIM, "multiple of n_kv_heads", att(heads=0)),
        (F.FH_ERR_DIM, "ld is below", att(ld=255)),
        (F.FH_ERR_DIM, "do not divide", att(total=3)),
        (F.FH_ERR_LIMIT, "too large", att(total=1 << 40)),
        (F.FH_ERR_INVALID, "q or out is NULL", att(q=None)),
        (F.FH_ERR_INVALID, "q or out is NULL", att(out=None)),
        (F.FH_ERR_INVALID, "must not be q", att(out=q)),
        (F.FH_ERR_INVALID, "softcap", att(score=F.AttnScore(-1.0))),
        (F.FH_ERR_INVALID, "softcap", att(score=F.AttnScore(float("nan")))),
        (F.FH_ERR_INVALID, "no weight plane", lambda: F.kv4_weigh_async(fh, bare, q, 512, 2, 4, None, 1, ln, 32, None, out)),
        (F.FH_ERR_INVALID, "lse is NULL", lambda: F.kv4_weigh_async(fh, ok, q, 512, 2, 4, None, 1, ln, 32, None, None)),
        (F.FH_ERR_DIM, "ld is below", lambda: F.kv4_append_async(fh, ok, q, 511, 2, 4, None, 1, ln)),
        (F.FH_ERR_DIM, "rope_dim", lambda: F.kv4_append_async(fh, ok, q, 512, 2, 4, None, 1, ln, rope_dim=66)),
        (F.FH_ERR_DIM, "rope_dim", lambda: F.kv4_append_async(fh, ok, q, 512, 2, 4, None, 1, ln, rope_dim=7)),
        (F.FH_ERR_INVALID, "rope_type", lambda: F.kv4_append_async(fh, ok, q, 512, 2, 4, None, 1, ln, rope_dim=8, rope_type=5)),
        (F.FH_ERR_DIM, "RoPE scaling", lambda: F.kv4_append_async(fh, ok, q, 512, 2, 4, None, 1, ln, rope_dim=8, linear_factor=0.0)),
        (F.FH_ERR_INVALID, "must not be qkv", lambda: F.kv4_append_async(fh, ok, q, 512, 2, 4, None, 1, ln, q=q)),
        (F.FH_ERR_INVALID, "qkv is NULL", lambda: F.kv4_append_async(fh, ok, None, 512, 2, 4, None, 1, ln)),
        (F.FH_ERR_LIMIT, "workgroups", lambda: F.kv4_append_async(fh, cache(seqs=65535, n_kv=1), q, 512, 1 << 29, 2, ln, 1 << 29, ln)),
        (F.FH_ERR_INVALID, "no weight plane", lambda: F.kv4_evict_async(fh, bare, ok, ln, 32, 8, 0, ln)),
        (F.FH_ERR_INVALID, "share a plane", lambda: F.kv4_evict_async(fh, ok, ok, ln, 32, 8, 0, ln)),
        (F.FH_ERR_DIM, "above the capacity", lambda: F.kv4_evict_async(fh, ok, bare, ln, 32, 33, 0, ln)),
        (F.FH_ERR_DIM, "caches differ", lambda: F.kv4_evict_async(fh, ok, F.KV4Cache.alloc(2, 1, 64, 32), ln, 32, 8, 0, ln)),
        (F.FH_ERR_INVALID, "keep must be", lambda: F.kv4_evict_async(fh, ok, bare, ln, 32, 0, 0, ln)),
        (F.FH_ERR_INVALID, "keep must be", lambda: F.kv4_evict_async(fh, ok, bare, ln, 32, 8, 9, ln)),
        (F.FH_ERR_INVALID, "len or new_len", lambda: F.kv4_evict_async(fh, ok, bare, None, 32, 8, 0, ln)),
        (F.FH_ERR_INVALID, "k or v is NULL", lambda: F.kv4_read_async(fh, ok, None, 4, None, out)),
        (F.FH_ERR_LIMIT, "2^32", lambda: F.kv4_read_async(fh, ok, None, 1 << 40, out, out)),
    ]
    for code, text, call in cases:
        with pytest.raises(F.FerrumHipError, match=text.replace("^", r"\^")) as e:
            call()
        assert e.value.code == code, text
    # empty calls are valid
    F.kv4_append_async(fh, ok, None, 512, 0, 4, None, 0, ln)
    F.kv4_attention_async(fh, ok, None, 512, 0, 4, None, 0, ln, 32, None, None)
    F.kv4_weigh_async(fh, ok, None, 512, 0, 4, None, 0, ln, 32, None, None)
    F.kv4_read_async(fh, ok, None, 0, None, None)
    fh.sync()
