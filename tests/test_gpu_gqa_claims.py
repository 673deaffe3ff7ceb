"""What the header says of prompts' and trees' accuracy over f32 caches, where the other tests do not
hold it: ordinary rows to 1e-5, partial rotations of aligned rows, values of both ends of the range."""
import numpy as np
import pytest

import gqa_ref as ref
from test_gpu_gqa_rows import Call, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("heads,lens,news", [((14, 2, 64), [0, 500, 2000], [200, 64, 30]), ((32, 8, 128), [0, 3000], [130, 40]),
                                             ((12, 12, 64), [700], [255]), ((4, 4, 32), [0, 90], [64, 300]),
                                             ((14, 2, 64), [0, 0, 0, 0], [900, 800, 1000, 640]), ((32, 8, 128), [0], [1400])])
def test_ordinary_rows_within_1e_5(fh, heads, lens, news, tree):
    """Unit-normal rows: 1e-5 of the sum of weight * the value row's largest magnitude, far inside the
    bound that counts every rounding at its worst."""
    if tree and max(news) > 700:
        news = [n // 8 for n in news]
    assert Call(heads, lens, news, 80, parents=trees(news, 81) if tree else None).check(fh) <= 1e-5


# (aligned rows: the queries are turned where they are loaded, pairs of channels d and d + half)
@pytest.mark.parametrize("width,rope", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 96), (128, 128), (32, 32)])
@pytest.mark.parametrize("tree", [False, True])
def test_partial_rotations_of_split_halves(fh, width, rope, tree):
    news = [9, 40]
    Call((4, 2, width), [20, 3], news, 82, rope=("neox", rope), parents=trees(news, 83) if tree else None, base=1e4, pos=5000).check(fh)


@pytest.mark.parametrize("width,rope", [(64, 32), (64, 36), (128, 32), (128, 64), (128, 96), (128, 20)])
@pytest.mark.parametrize("kind", ["neox", "norm"])
def test_partial_rotations_over_packed_tiles(fh, width, rope, kind):
    """More than 1024 columns of a kv head and 3 * 2^19 pairs of a column and a tile: each tile is packed once."""
    a = Call((16, 4, width), [0], [2000], 84, rope=(kind, rope), base=1e4)
    assert a.g * (2000 * a.h // a.g) * (a.cap // 32) > 3 << 19
    a.check(fh)


@pytest.mark.parametrize("width", [32, 64, 128])
@pytest.mark.parametrize("rope", [("neox", 16), ("norm", 16), ("norm", 6)])
def test_partial_rotations_of_both_paths(fh, width, rope):
    """Halves that the loads turn in place (norm 16) and such that the first launch turns (neox 16, norm 6)."""
    Call((4, 2, width), [20, 3], [9, 40], 86, rope=rope, base=1e4, pos=5000, factors=True, linear=2.0).check(fh)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("heads", [(4, 2, 64), (4, 2, 128), (2, 1, 8)])
def test_value_rows_of_both_ends_of_the_range(fh, heads, tree):
    """Rows of zeros and of 2^-86 beside rows of 2^27: each keeps its weight in the sums."""
    news = [48]
    a = Call(heads, [64], news, 87, parents=trees(news, 88) if tree else None, rope=(None, None))
    g, hd = a.g, a.hd
    v = a.v[0, :64].reshape(64, g, hd)
    v /= np.abs(v).max(axis=2, keepdims=True)
    v[0:20] = 0.0
    v[20:40] *= np.float32(2.0**-86)
    v[40:64] *= np.float32(2.0**27)
    x = a.qkv[:, (a.h + g) * hd:(a.h + 2 * g) * hd].reshape(48, g, hd)
    x /= np.abs(x).max(axis=2, keepdims=True)
    x[:16] = 0.0
    a.qkv[:, (a.h + g) * hd:(a.h + 2 * g) * hd] = x.reshape(48, -1)
    a.check(fh)
