"""Prompts whose tiles of keys are packed once (fh_gqa_attention_rope_prefill_async with many
columns and keys): against the definition in float64, what is not finite, rows of very different
sizes, shares of the keys, and growth of the workspace."""
import numpy as np
import pytest

import gqa_ref as ref
from test_gpu_gqa_rows import Call, gpu, ints

pytestmark = pytest.mark.gpu

# query heads, kv heads, width; new rows: more than 1024 columns of a kv head
MANY = [((32, 1, 64), [40, 33, 0, 17]), ((64, 2, 128), [40, 36]), ((48, 1, 32), [30, 25]), ((40, 1, 16), [40, 1, 28]), ((64, 1, 8), [30, 17])]


def packed(heads, lens, news, seed, **kw):
    """A call long enough for it: kv heads * sequences * columns * tiles of the capacity > 3 * 2^19."""
    cols = max(news) * heads[0] // heads[1]
    cap = 32 * (-(-(3 << 19) // (heads[1] * len(news) * cols)) + 2) + 5
    assert cols > 1024
    return Call(heads, lens, news, seed, cap=cap, **kw)


@pytest.mark.parametrize("heads,news", MANY)
def test_prompts_of_different_lengths(fh, heads, news):
    packed(heads, [0] * len(news), news, 40).check(fh)
    packed(heads, [65, 1, 300, 31][:len(news)], news, 41, before=2, behind=5).check(fh)


@pytest.mark.parametrize("rope", [("neox", None), ("norm", None), ("neox", 8), ("norm", 24), (None, None)])
def test_rotations(fh, rope):
    packed((32, 1, 64), [7, 90], [40, 12], 42, rope=rope, factors=True, linear=2.0, pos=50000, pad=3).check(fh)
    packed((32, 1, 64), [7, 90], [40, 12], 42, rope=rope).check(fh)


@pytest.mark.parametrize("heads,news", MANY[:3])
def test_shares_of_a_long_cache(fh, heads, news):
    """Few column blocks over many keys: their shares are joined in two levels."""
    packed(heads, [3000, 1111, 40, 2][:len(news)], news, 43).check(fh)


def test_a_long_prompt(fh):
    Call((14, 2, 64), [0], [2000], 44).check(fh)


def test_rows_past_the_capacity(fh):
    a = packed((32, 1, 64), [0, 0], [40, 40], 45)
    packed((32, 1, 64), [a.cap - 13, a.cap + 7], [40, 40], 45).check(fh)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("heads,news", [MANY[0], MANY[1], MANY[4]])
@pytest.mark.parametrize("where", ["q", "k", "v"])
def test_what_is_not_finite_reaches_the_rows_that_see_it(fh, bad, heads, news, where):
    a = packed(heads, [50] * len(news), news, 46, rope=(None, None))
    plain = a.run(fh)
    at, group = 11, a.h // a.g
    col = {"q": group - 1, "k": a.h, "v": a.h + a.g}[where] * a.hd + 3  # kv head 0
    a.qkv[at, col] = bad
    got = a.run(fh)
    hit = np.zeros(got.shape[:2], bool)
    if where == "q":
        hit[at, group - 1] = True
    else:
        hit[at:news[0], :group] = True
    assert np.isnan(got[hit]).all()
    np.testing.assert_allclose(got[~hit], plain[~hit], rtol=0, atol=1e-5 * np.abs(plain).max())


@pytest.mark.parametrize("heads,news", MANY)
def test_rows_of_different_sizes_are_as_exact(fh, heads, news):
    """Keys and values up to 2^40 apart in one kv head's tiles, which are not packed then; the other
    sequences' are."""
    a = packed(heads, [64] * len(news), news, 47, rope=(None, None))
    a.v[0, 5] *= 2.0**-30
    a.v[0, 6] *= 2.0**10
    a.k[0, 7] *= 2.0**-20
    a.k[0, 40] *= 0.0
    a.v[1, 41] *= 0.0  # (zeros are no size)
    a.check(fh)


def test_the_same_bits_alone_and_beside_others(fh):
    """A sequence whose tiles are not packed does not change what others give."""
    heads, news = MANY[0]
    a = packed(heads, [64] * 4, news, 48)
    one = a.run(fh).copy()
    a.v[1, 5] *= 2.0**-30
    two = a.run(fh)
    rows = slice(a.off[1], a.off[2])
    keep = np.ones(a.total, bool)
    keep[rows] = False
    np.testing.assert_array_equal(two[keep], one[keep])
    # v row 5 has little weight of its own left
    assert np.abs(two[rows] - one[rows]).max() > 0


def test_captured_and_replayed(fh):
    import torch

    a = packed((32, 1, 64), [700, 100], [40, 35], 49)
    a.k, a.v = (np.nan_to_num(x, nan=0.5, posinf=0.5, neginf=0.5).clip(-5, 5) for x in (a.k, a.v))
    a.run(fh)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    fh.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            a.again(fh)
        fh.set_stream(None)
        big = Call((32, 8, 128), [600], [300], 50)
        for i in range(4):
            a.lens = [700 - 200 * i, 100 + i]
            a.v = a.v.copy()
            a.v[1, 5] *= 2.0**-20 if i == 1 else 2.0**20 if i == 2 else 1.0  # (packed or not, from replay to replay)
            a.dlen.copy_(ints(a.lens))
            a.dk.copy_(gpu(a.k))
            a.dv.copy_(gpu(a.v))
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
            a.k, a.v = a.dk.cpu().numpy(), a.dv.cpu().numpy()
        a.lens = [0, 0]
        a.check(fh)
    finally:
        fh.set_stream(None)


def test_single_rows_over_long_caches(fh):
    """One row a sequence over shares of a long cache: every head width, odd lengths."""
    for heads in ((8, 4, 8), (8, 4, 16), (8, 2, 32), (14, 2, 64), (4, 4, 128)):
        for tree in (False, True):
            Call(heads, [4001, 31, 0, 1999], [1, 1, 1, 1], 51, parents=[np.array([-1])] * 4 if tree else None).check(fh)


def test_many_sequences(fh):
    """More column blocks than there are shares planned for, and sequences without rows between."""
    rng = np.random.default_rng(52)
    lens, news = rng.integers(0, 90, 300), rng.integers(0, 4, 300)
    for parents in (None, [np.arange(n) - 1 for n in news]):
        Call((4, 2, 32), lens, news, 53, parents=parents).check(fh)
        Call((4, 2, 32), lens[:120], news[:120], 54, parents=parents and parents[:120]).check(fh)
