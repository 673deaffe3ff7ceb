"""Penalties, biases and masks on logits (fh_logits_edit_async) against float64."""
import numpy as np
import pytest

import gqa_ref as ref

pytestmark = pytest.mark.gpu


def gpu(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(values):
    return gpu(np.asarray(values, np.int64).astype(np.uint32).view(np.int32))


def pack(allowed):
    """[masks, vocab] truth values as words of 32 bits (bits past the vocabulary 0)."""
    m, v = allowed.shape
    bits = np.zeros((m, -(-v // 32) * 32), np.uint8)
    bits[:, :v] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view("<u4")


def run(fh, rows, vocab, seed, history=0, tree=None, off=None, biases=0, masks=0, params=("rep", "freq", "pres"), in_place=False,
        mask_of=True, repeat=False):
    import ferrum_hip
    import torch

    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, vocab)) * 4).astype(np.float32)
    x[0, 0], x[-1, -1] = -np.inf, 0.0
    kw, one = {}, [dict() for _ in range(rows)]
    lists = [[] for _ in range(rows)]
    if history:
        n = [int(rng.integers(0, history + 1)) for _ in range(rows)]
        n[0] = history
        recent = (rng.random(sum(n) + 3) ** 3 * vocab * 1.05).astype(np.int64)  # (some past the vocabulary)
        end = np.cumsum(n) + 3
        ranges = np.stack([end - n, end], axis=1)
        if rows > 1:
            ranges[1] = [9, 4]  # decreasing: empty
            n[1] = 0
        for r in range(rows):
            lists[r] += recent[ranges[r, 0]:ranges[r, 1]].tolist() if n[r] else []
        kw.update(recent=ints(recent), ranges=ints(ranges))
    if tree:
        parts = [rows // tree] * tree if off is None else list(np.diff(off))
        first = np.concatenate([[0], np.cumsum(parts)])[:-1] if off is None else off[:-1]
        parent, tokens = np.full(rows, -1), rng.integers(0, min(vocab, 50) + 1, rows)
        covered = np.zeros(rows, bool)
        for b, n in zip(first, parts):
            covered[b:b + n] = True
            for t in range(1, n):
                parent[b + t] = rng.integers(max(0, t - 6), t) if rng.random() < 0.9 else -1
            for t in range(n):
                lists[b + t] += tokens[[b + a for a in ref.path(parent[b:b + n], t)]].tolist()
        for r in np.flatnonzero(~covered):
            lists[r].append(int(tokens[r]))
        kw.update(parent=ints(parent), tokens=ints(tokens), seqs=len(parts), off=None if off is None else ints(off))
    for name, key, lo, hi in (("repetition", "rep", 0.8, 1.5), ("frequency", "freq", -0.5, 0.7), ("presence", "pres", -0.5, 0.7)):
        if key in params:
            p = rng.uniform(lo, hi, rows).astype(np.float32)
            if key == "rep" and rows > 2:
                p[2] = -1.0  # off
            kw[name] = gpu(p)
            for r in range(rows):
                one[r][name] = float(p[r])
    if biases:
        n = rng.integers(0, biases + 1, rows)
        o = np.concatenate([[0], np.cumsum(n)])
        ids = rng.integers(0, vocab + 2, o[-1] + 1) if not repeat else rng.integers(0, 3, o[-1] + 1)
        b = (rng.standard_normal(o[-1] + 1) * 5).astype(np.float32)
        kw.update(bias_off=ints(o), bias_id=ints(ids), bias=gpu(b))
        for r in range(rows):
            one[r]["biases"] = list(zip(ids[o[r]:o[r + 1]].tolist(), b[o[r]:o[r + 1]].astype(np.float64).tolist()))
    if masks:
        allowed = rng.random((masks, vocab)) < rng.choice([0.0, 0.05, 0.9, 1.0], (masks, 1))
        of = rng.integers(0, masks + 1, rows) if mask_of else np.arange(rows)
        if mask_of and rows > 3:
            of[3] = 0xFFFFFFFF
        kw.update(mask=gpu(pack(allowed).view(np.int32)), masks=masks, mask_of=ints(of) if mask_of else None)
        for r in range(rows):
            if of[r] < masks:
                one[r]["allowed"] = allowed[of[r]]
    d = gpu(x)
    out = d if in_place else torch.full_like(d, 9.0)
    ferrum_hip.logits_edit_async(fh, d, rows, vocab, ferrum_hip.LogitsEdit(**kw), out)
    fh.sync()
    got = out.cpu().numpy()
    if not in_place:
        np.testing.assert_array_equal(d.cpu().numpy(), x)
    for r in range(rows):
        want = ref.edit(x[r], lists[r], **one[r])
        np.testing.assert_array_equal(np.isneginf(got[r]), np.isneginf(want))
        ok = np.isfinite(want)
        # each of at most five operations rounds a number no larger than the sum of all that went in
        count = np.bincount(np.array([i for i in lists[r] if i < vocab] or [0], np.int64), minlength=vocab)
        size = np.abs(x[r].astype(np.float64)) * 1.5 + 0.7 * count + 1 + np.abs(want, where=ok, out=np.zeros(vocab)) * 2
        for i, b in one[r].get("biases", []):
            if i < vocab:
                size[i] += abs(b)
        assert (np.abs(got[r][ok] - want[ok]) <= 5 * 2.0**-24 * size[ok]).all()
    return got


VOCABS = [1, 31, 32, 33, 1000, 2048, 2049, 50257]


@pytest.mark.parametrize("vocab", VOCABS)
def test_everything_at_once(fh, vocab):
    run(fh, 5, vocab, 1, history=200, biases=20, masks=3)
    run(fh, 12, vocab, 2, history=50, tree=3, biases=5, masks=12, mask_of=False)


@pytest.mark.parametrize("part", ["none", "history", "tree", "biases", "masks"])
def test_each_part_alone(fh, part):
    kw = {"none": dict(params=()), "history": dict(history=90), "tree": dict(tree=2), "biases": dict(biases=30, params=()),
          "masks": dict(masks=4, params=())}[part]
    run(fh, 6, 5000, 3, **kw)


@pytest.mark.parametrize("params", [("rep",), ("freq",), ("pres",), ("rep", "pres")])
def test_each_penalty(fh, params):
    run(fh, 4, 3000, 4, history=300, params=params)


def test_one_row_and_many(fh):
    run(fh, 1, 151936, 5, history=5000, biases=300, masks=1)
    run(fh, 64, 4096, 6, history=40, masks=64, mask_of=False)
    run(fh, 300, 700, 7, history=3, tree=10)


def test_trees_by_offsets_and_rows_outside(fh):
    run(fh, 30, 800, 8, tree=3, off=np.array([2, 9, 9, 25]))
    run(fh, 1024, 64, 9, tree=1)


def test_in_place_and_repeated_ids(fh):
    run(fh, 7, 3001, 10, history=100, biases=10, masks=2, in_place=True)
    run(fh, 7, 3001, 11, biases=40, repeat=True)


def test_a_mask_that_leaves_nothing(fh):
    import ferrum_hip
    import torch

    x = torch.randn((2, 100), device="cuda")
    x[0, 5], x[1, 6] = float("nan"), float("inf")
    mask = torch.zeros((1, 4), dtype=torch.int32, device="cuda")
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    ferrum_hip.logits_edit_async(fh, x, 2, 100, ferrum_hip.LogitsEdit(mask=mask, masks=1), out)
    fh.sync()
    assert torch.isneginf(out[0]).all()
    assert torch.equal(out[1], x[1])  # row 1 has no mask


def test_refusals(fh):
    import ferrum_hip as m
    import torch

    x = torch.zeros((4, 16), device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    for kw, code in ((dict(ranges=i), m.FH_ERR_INVALID), (dict(tokens=i), m.FH_ERR_INVALID), (dict(tokens=i, seqs=3), m.FH_ERR_DIM),
                     (dict(bias_off=i), m.FH_ERR_INVALID), (dict(bias_off=i, bias_id=i), m.FH_ERR_INVALID)):
        with pytest.raises(m.FerrumHipError) as e:
            m.logits_edit_async(fh, x, 4, 16, m.LogitsEdit(**kw), x)
        assert e.value.code == code, kw
    for args, code in (((x, 4, 0, m.LogitsEdit(), x), m.FH_ERR_INVALID), ((None, 4, 16, m.LogitsEdit(), x), m.FH_ERR_INVALID),
                       ((x, 4, 16, m.LogitsEdit(), None), m.FH_ERR_INVALID), ((x, 4, 16, None, x), m.FH_ERR_INVALID),
                       ((x, 4, 1 << 31, m.LogitsEdit(), x), m.FH_ERR_LIMIT),
                       ((x, 2050, 16, m.LogitsEdit(tokens=i, seqs=2), x), m.FH_ERR_LIMIT)):
        with pytest.raises(m.FerrumHipError) as e:
            m.logits_edit_async(fh, *args)
        assert e.value.code == code
    m.logits_edit_async(fh, None, 0, 16, m.LogitsEdit(), None)
