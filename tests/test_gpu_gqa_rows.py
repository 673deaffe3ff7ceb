"""Prompts and drafted trees over f32 caches (fh_gqa_attention_rope_prefill_async,
fh_gqa_attention_rope_tree_async) against their definitions in float64 (gqa_ref)."""
import numpy as np
import pytest

import gqa_ref as ref

pytestmark = pytest.mark.gpu

HEADS = [(2, 2, 8), (4, 1, 16), (4, 4, 32), (14, 2, 64), (12, 12, 64), (32, 8, 128), (5, 1, 128)]
JUNK = np.array([np.nan, np.inf, -np.inf, 3e38, -3e38], np.float32)


def gpu(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def ints(values):
    return gpu(np.asarray(values, np.int64).astype(np.uint32).view(np.int32))


class Call:
    """One call's inputs and what it should give.  Cache rows that nothing has been written
    to hold NaN, infinities and the largest numbers."""

    def __init__(self, heads, lens, news, seed, cap=None, parents=None, rope=("neox", None), base=10000.0, factors=False,
                 linear=1.0, pos=None, before=0, behind=0, max_keys=None, max_rows=None, q_std=1.0, v_std=1.0, pad=0):
        self.h, self.g, self.hd = heads
        self.lens, self.news, self.seqs = list(lens), list(news), len(lens)
        self.cap = cap or max(a + n for a, n in zip(lens, news)) + 3
        self.max_rows = max(list(news) + [0]) if max_rows is None else max_rows
        self.max_keys = self.cap if max_keys is None else max_keys
        self.total = before + sum(news) + behind
        self.off = np.concatenate([[0], np.cumsum(news)]) + before
        self.parents, self.kind, self.base, self.linear = parents, rope[0], base, linear
        self.rope_dim = 0 if self.kind is None else rope[1] or self.hd
        rng = np.random.default_rng(seed)
        self.ff = np.exp(0.5 * rng.standard_normal(self.rope_dim // 2)).astype(np.float32) if factors else None
        wide = (self.h + 2 * self.g) * self.hd
        self.ld = wide + pad
        self.qkv = rng.standard_normal((self.total, self.ld)).astype(np.float32)
        self.qkv[:, :self.h * self.hd] *= q_std
        self.qkv[:, wide - self.g * self.hd:wide] *= v_std
        self.k, self.v = (rng.choice(JUNK, (self.seqs, self.cap, self.g * self.hd)) for _ in range(2))
        spread = np.exp(0.3 * rng.standard_normal(self.g * self.hd)).astype(np.float32)
        for s, n in enumerate(self.lens):
            m = min(n, self.cap)
            self.k[s, :m] = rng.standard_normal((m, self.g * self.hd)).astype(np.float32) * spread
            self.v[s, :m] = rng.standard_normal((m, self.g * self.hd)).astype(np.float32) * np.float32(v_std)
        self.pos = rng.integers(0, pos, self.total) if pos else None

    def run(self, fh, out=None):
        import ferrum_hip
        import torch

        self.dk, self.dv = gpu(self.k), gpu(self.v)
        self.dqkv = gpu(self.qkv)
        self.out = torch.full((self.total, self.h * self.hd), 77.0, device="cuda") if out is None else out
        self.doff, self.dlen = ints(self.off), ints(self.lens)
        self.dpos = None if self.pos is None else ints(self.pos)
        self.dff = None if self.ff is None else gpu(self.ff)
        self.dpar = None
        if self.parents is not None:
            flat = np.full(self.total, -7)
            for s, p in enumerate(self.parents):
                flat[self.off[s]:self.off[s + 1]] = p
            self.dpar = ints(flat)
        torch.cuda.synchronize()
        self.again(fh)
        fh.sync()
        return self.out.cpu().numpy().reshape(self.total, self.h, self.hd)

    def again(self, fh):
        import ferrum_hip

        head = (fh, self.dqkv, self.ld, self.total, self.h, self.g, self.hd, self.dk, self.dv, self.seqs, self.cap,
                self.doff, self.max_rows, self.dlen, self.max_keys)
        turn = (self.rope_dim, self.base, ferrum_hip.ROPE_NEOX if self.kind == "neox" else ferrum_hip.ROPE_NORM, self.dff,
                self.linear, self.out)
        if self.parents is None:
            ferrum_hip.gqa_attention_rope_prefill_async(*head, self.dpos, *turn)
        else:
            ferrum_hip.gqa_attention_rope_tree_async(*head, self.dpar, self.dpos, *turn)

    def check(self, fh):
        got = self.run(fh)
        k, v = self.dk.cpu().numpy(), self.dv.cpu().numpy()
        want_k, want_v = self.k.astype(np.float64), self.v.astype(np.float64)
        touched = np.zeros(self.total, bool)
        limit = min(self.cap, self.max_keys)
        worst = 0.0
        for s in range(self.seqs):
            n, at = min(self.news[s], self.max_rows), self.lens[s]
            rows = slice(self.off[s], self.off[s] + n)
            touched[rows] = True
            if n == 0:
                continue
            x = self.qkv[rows, :(self.h + 2 * self.g) * self.hd].reshape(n, -1, self.hd)
            par = None if self.parents is None else self.parents[s]
            ways = [list(range(t + 1)) if par is None else ref.path(par, t) for t in range(n)]
            where = np.array([at + len(w) - 1 for w in ways]) if self.pos is None else self.pos[rows]
            turned = ref.rotate(x[:, :self.h + self.g], where, self.rope_dim, self.base, self.kind == "neox", self.ff, self.linear)
            fit = min(n, max(0, limit - at))
            want_k[s, at:at + fit] = turned[:fit, self.h:].reshape(fit, self.g * self.hd)
            want_v[s, at:at + fit] = x[:fit, self.h + self.g:].reshape(fit, self.g * self.hd)
            assert np.isnan(got[rows][fit:]).all()
            if fit == 0:
                continue
            seen = np.zeros((fit, self.cap), bool)
            for t in range(fit):
                seen[t, :at] = True
                seen[t, [at + a for a in ways[t]]] = True
            out, mass, size = ref.attend(turned[:fit, :self.h], want_k[s].reshape(self.cap, self.g, self.hd),
                                         want_v[s].reshape(self.cap, self.g, self.hd), seen)
            tol = ref.bound(mass, size, self.hd, at + fit)
            err = np.abs(got[rows][:fit] - out).max(axis=2)
            assert np.isfinite(err).all()
            assert (err <= tol).all(), (s, float((err / tol).max()))
            worst = max(worst, float((err / np.maximum(mass, 1e-300)).max()))
        assert (got[~touched] == 77.0).all()
        # what is not rotated is stored as it is; a rotated channel is off by 4 roundings of its pair's size
        np.testing.assert_array_equal(v, want_v.astype(np.float32))
        new = np.isfinite(want_k)
        np.testing.assert_array_equal(k[~new], self.k[~new])
        size = np.abs(want_k[new]) + (3.0 * max(1.0, np.abs(self.qkv).max()) if self.rope_dim else 0.0)
        assert (np.abs(k[new] - want_k[new]) <= 4 * 2.0**-24 * size).all()
        return worst


def trees(news, seed, wide=8):
    """Each row continues one of the `wide` before it; some none, some a row that is not before it."""
    rng = np.random.default_rng(seed)
    out = []
    for n in news:
        p = np.array([-1] + [int(rng.integers(max(0, t - wide), t)) for t in range(1, n)])[:n]
        if n > 20:
            p[n // 2], p[n // 3], p[n - 1] = -1, n + 5, n - 1
        out.append(p)
    return out


@pytest.mark.parametrize("heads", HEADS)
def test_prompts_of_different_lengths(fh, heads):
    Call(heads, [0, 5, 100, 0, 31, 64], [1, 33, 7, 0, 129, 64], 1).check(fh)


@pytest.mark.parametrize("heads", HEADS)
def test_trees_of_different_sizes(fh, heads):
    news = [1, 33, 7, 0, 65, 24]
    Call(heads, [0, 5, 100, 3, 31, 64], news, 2, parents=trees(news, 3)).check(fh)


@pytest.mark.parametrize("rope", [("neox", None), ("norm", None), ("neox", 8), ("norm", 24), (None, None)])
@pytest.mark.parametrize("tree", [False, True])
def test_rotations(fh, rope, tree):
    news = [9, 40]
    Call((4, 2, 32), [20, 3], news, 4, rope=rope, parents=trees(news, 5) if tree else None, base=1e6, factors=rope[0] is not None,
         linear=4.0, pos=60000, pad=5).check(fh)


@pytest.mark.parametrize("heads,lens,news", [((14, 2, 64), [3000], [5]), ((32, 8, 128), [5000], [17]), ((4, 4, 32), [4097], [70]),
                                             ((12, 12, 64), [1, 2500], [40, 1]), ((40, 2, 64), [2000], [9])])
@pytest.mark.parametrize("tree", [False, True])
def test_long_caches_dealt_over_workgroups(fh, heads, lens, news, tree):
    Call(heads, lens, news, 6, parents=trees(news, 7) if tree else None).check(fh)


@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128), (4, 4, 32)])
def test_longer_prompts(fh, heads):
    Call(heads, [0, 70], [700, 513], 8).check(fh)


def test_a_large_tree(fh):
    for n in (64, 200, 1024):
        Call((4, 2, 64), [77], [n], 9, parents=trees([n], 10, 30)).check(fh)


@pytest.mark.parametrize("shape", ["chain", "star", "roots"])
def test_special_trees(fh, shape):
    n = 50
    p = {"chain": np.arange(n) - 1, "star": np.where(np.arange(n) > 0, 0, -1), "roots": np.full(n, -1)}[shape]
    Call((14, 2, 64), [40], [n], 11, parents=[p]).check(fh)


def test_a_chain_is_a_prompt(fh):
    a = Call((14, 2, 64), [100, 7], [40, 33], 12, parents=[np.arange(40) - 1, np.arange(33) - 1])
    b = Call((14, 2, 64), [100, 7], [40, 33], 12)
    np.testing.assert_array_equal(a.run(fh), b.run(fh))
    np.testing.assert_array_equal(a.dk.cpu().numpy(), b.dk.cpu().numpy())


@pytest.mark.parametrize("tree", [False, True])
def test_rows_outside_and_beyond(fh, tree):
    """Rows before the first and behind the last sequence, rows past max_rows, rows past the
    capacity or max_keys."""
    par = lambda news: trees(news, 13) if tree else None  # noqa: E731
    Call((4, 2, 64), [10, 0], [20, 30], 14, before=3, behind=40, parents=par([20, 30])).check(fh)
    Call((4, 2, 64), [10, 0], [20, 30], 15, max_rows=12, parents=par([20, 30])).check(fh)
    Call((4, 2, 64), [60, 64, 200, 3], [20, 30, 4, 8], 16, cap=64, parents=par([20, 30, 4, 8])).check(fh)
    Call((4, 2, 64), [30, 2], [20, 30], 17, cap=100, max_keys=40, parents=par([20, 30])).check(fh)


def test_equal_parts_without_offsets(fh):
    import ferrum_hip
    import torch

    a = Call((14, 2, 64), [0, 0, 0], [11, 11, 11], 18)
    want = a.run(fh)
    out = torch.zeros_like(a.out)
    ferrum_hip.gqa_attention_rope_prefill_async(fh, a.dqkv, a.ld, 33, 14, 2, 64, a.dk, a.dv, 3, a.cap, None, 0, None, a.cap, None,
                                                64, 10000.0, ferrum_hip.ROPE_NEOX, None, 1.0, out)
    fh.sync()
    np.testing.assert_array_equal(out.cpu().numpy().reshape(want.shape), want)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("heads", [(4, 2, 64), (4, 2, 128), (4, 4, 32), (2, 1, 8)])
@pytest.mark.parametrize("where", ["k", "v"])
def test_what_is_not_finite_reaches_the_rows_that_see_it(fh, bad, heads, where):
    news = [40]
    for parents in (None, trees(news, 19)):
        a = Call(heads, [50], news, 20, parents=parents, rope=(None, None))
        plain = a.run(fh)
        col = (a.h + (0 if where == "k" else a.g)) * a.hd + 3  # kv head 0
        a.qkv[30, col] = bad
        got = a.run(fh)
        ways = [list(range(t + 1)) if parents is None else ref.path(parents[0], t) for t in range(40)]
        sees = np.array([30 in w for w in ways])
        hit = np.zeros((40, a.h), bool)
        hit[sees, :a.h // a.g] = True
        # (a value's other channels may or may not come out as numbers)
        assert np.isfinite(got[~hit]).all()
        tol = np.abs(plain[~hit]).max() * 1e-5
        np.testing.assert_allclose(got[~hit], plain[~hit], rtol=0, atol=tol)
        if where == "v" or np.isnan(bad):
            assert not np.isfinite(got[hit][:, 3]).any()


@pytest.mark.parametrize("tree", [False, True])
def test_values_and_keys_far_apart(fh, tree):
    """A row's accuracy does not hang on keys beside it that it does not see, nor on large
    values of little weight."""
    news = [64]
    a = Call((4, 2, 64), [32], news, 21, parents=trees(news, 22) if tree else None, rope=(None, None))
    a.qkv[63, a.h * a.hd:] *= 2.0**40  # the last row's key and value
    a.v[0, 5] *= 2.0**-30
    a.v[0, 6] *= 2.0**12
    a.k[0, 7] *= 2.0**-20
    a.qkv[10, :a.h * a.hd] *= 2.0**-30
    # the last row itself: all weight on itself or none, sizes beyond the bound's reach
    got = a.run(fh)
    for t in (0, 10, 40, 62):
        way = list(range(t + 1)) if not tree else ref.path(a.parents[0], t)
        if 63 in way:
            continue
        x = a.qkv[:, :8 * 64].reshape(64, 8, 64)
        k = np.concatenate([a.k[0, :32].reshape(32, 2, 64), x[way, 4:6]]).astype(np.float64)
        v = np.concatenate([a.v[0, :32].reshape(32, 2, 64), x[way, 6:]]).astype(np.float64)
        out, mass, size = ref.attend(x[t:t + 1, :4].astype(np.float64), k, v, np.ones((1, len(k)), bool))
        tol = ref.bound(mass, size, 64, len(k))[0]
        assert (np.abs(got[t] - out[0]).max(axis=1) <= tol).all()


def test_large_scores(fh):
    """Weights that fall on one key, and scores of some hundreds (their bound grows with them)."""
    Call((14, 2, 64), [200], [40], 23, q_std=30.0).check(fh)
    Call((4, 2, 128), [200], [40], 24, q_std=1e-3, v_std=1e-6).check(fh)
    Call((4, 2, 32), [200], [40], 25, v_std=1e6).check(fh)


def test_the_same_bits_again(fh):
    a = Call((14, 2, 64), [3000, 100], [16, 9], 26)
    one = a.run(fh).copy()
    for _ in range(3):
        a.out.zero_()
        a.again(fh)
        fh.sync()
        np.testing.assert_array_equal(a.out.cpu().numpy().reshape(one.shape), one)


@pytest.mark.parametrize("tree", [False, True])
def test_captured_and_replayed(fh, tree):
    import torch

    news = [16, 30]
    a = Call((14, 2, 64), [2900, 100], news, 27, cap=4000, parents=trees(news, 28) if tree else None)
    a.run(fh)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    fh.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            a.again(fh)
        fh.set_stream(None)
        big = Call((32, 8, 128), [600], [300], 29)  # the workspace grows in between
        rng = np.random.default_rng(30)
        for i in range(3):
            a.qkv = rng.standard_normal(a.qkv.shape).astype(np.float32)
            a.lens = [2900 - 700 * i, 100 + i]
            a.dqkv.copy_(gpu(a.qkv))
            a.dlen.copy_(ints(a.lens))
            a.dk.copy_(gpu(np.nan_to_num(a.k, nan=0.5, posinf=0.5, neginf=0.5).clip(-5, 5)))
            a.dv.copy_(gpu(np.nan_to_num(a.v, nan=0.5, posinf=0.5, neginf=0.5).clip(-5, 5)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = a.out.clone()
            big.check(fh)
            a.out.zero_()
            torch.cuda.synchronize()
            a.again(fh)
            fh.sync()
            assert torch.equal(got, a.out)
    finally:
        fh.set_stream(None)


def test_refusals(fh):
    import ferrum_hip as m
    import torch

    t = torch.zeros(1 << 14, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")

    def call(tree=False, qkv=t, ld=512, total=8, h=4, g=2, hd=64, k=t, v=t, seqs=2, cap=16, off=None, rows=0, ln=i, keys=16,
             par=i, rope=64, kind=1, linear=1.0, out=None):
        out = t[4096:] if out is None else out
        args = (fh, qkv, ld, total, h, g, hd, k, v, seqs, cap, off, rows, ln, keys)
        if tree:
            m.gqa_attention_rope_tree_async(*args, par, None, rope, 1e4, kind, None, linear, out)
        else:
            m.gqa_attention_rope_prefill_async(*args, None, rope, 1e4, kind, None, linear, out)

    for tree in (False, True):
        for kw, code in ((dict(h=5), m.FH_ERR_DIM), (dict(g=0), m.FH_ERR_DIM), (dict(h=0), m.FH_ERR_DIM),
                         (dict(rope=65), m.FH_ERR_DIM), (dict(rope=128), m.FH_ERR_DIM), (dict(linear=0.0), m.FH_ERR_DIM),
                         (dict(linear=float("nan")), m.FH_ERR_DIM), (dict(kind=2), m.FH_ERR_INVALID),
                         (dict(hd=48, rope=0), m.FH_ERR_LIMIT), (dict(hd=256, rope=0), m.FH_ERR_LIMIT),
                         (dict(ld=511), m.FH_ERR_DIM), (dict(total=7), m.FH_ERR_DIM), (dict(seqs=0), m.FH_ERR_INVALID),
                         (dict(cap=0), m.FH_ERR_INVALID), (dict(cap=1 << 31), m.FH_ERR_LIMIT), (dict(seqs=65536, total=0), m.FH_ERR_LIMIT),
                         (dict(qkv=None), m.FH_ERR_INVALID), (dict(k=None), m.FH_ERR_INVALID), (dict(out=t), m.FH_ERR_INVALID),
                         (dict(k=t[1:]), m.FH_ERR_INVALID), (dict(v=t[2:]), m.FH_ERR_INVALID), (dict(out=t[4097:]), m.FH_ERR_INVALID)):
            with pytest.raises(m.FerrumHipError) as e:
                call(tree, **kw)
            assert e.value.code == code, kw
    with pytest.raises(m.FerrumHipError) as e:
        call(True, par=None)
    assert e.value.code == m.FH_ERR_INVALID
    with pytest.raises(m.FerrumHipError) as e:
        call(True, total=2050, seqs=2)
    assert e.value.code == m.FH_ERR_LIMIT
    call(total=0)
    fh.sync()
