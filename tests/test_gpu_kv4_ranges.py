"""The 4-bit cache's attention over keys and values whose blocks differ widely in size:
every row is as exact as what it sees, whichever kernel the number of rows selects."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import Box, gpu, ints

pytestmark = pytest.mark.gpu


def rescaled(box, name, factor):
    """The box's keys (name k) or values (v) with block b of key j times factor [keys, blocks], powers of two."""
    hd, keys = box.hd, factor.shape[0]
    by = factor.reshape(keys // 8, 8, -1).transpose(0, 2, 1)
    old = box.plane(name + "_d").astype(np.float64)
    new = (old * by).astype(np.float16)
    assert np.isfinite(new).all()
    # (subnormal scales are rounded again)
    by_key = lambda d: np.repeat(d.astype(np.float64).transpose(0, 1, 2, 4, 3).reshape(  # noqa: E731
        box.seqs, box.n_kv, keys, hd // 32), 32, axis=3)
    val, step = (box.k, box.kstep) if name == "k" else (box.v, box.vstep)
    ratio = by_key(new) / by_key(old)
    val *= ratio
    step *= ratio
    box.c.planes[name + "_d"].copy_(gpu(new))


def attend(fh, box, q, rows, first=None):
    """Caches that begin with the call, `rows` rows a sequence; each channel within its own bound.
    The bound is that of test_gpu_kv4.check_attention (8 roundings of a score's partial sums,
    2^-18 of the mass of its block's largest magnitudes) and what the header leaves out: of
    each of the n keys a weight times its block's scale counts down to 2^-34 of the row's
    largest, which is 8 n 2^-34 of that in a channel."""
    import ferrum_hip
    import torch

    n_heads, hd = q.shape[1], box.hd
    total, group = box.seqs * rows, n_heads // box.n_kv
    out = torch.full((total, n_heads * hd), 7.0, device="cuda")
    lse = torch.full((total, n_heads), 7.0, device="cuda")
    sc = ferrum_hip.AttnScore(0.0, None, None, None if first is None else ints(np.tile(first, box.seqs)))
    qb = gpu(q.reshape(total, -1))
    torch.cuda.synchronize()
    ferrum_hip.kv4_attention_async(fh, box.c, qb, n_heads * hd, total, n_heads, None, rows, None, rows, sc, out, lse)
    fh.sync()
    o, z = out.cpu().numpy().reshape(box.seqs, rows, n_heads, hd), lse.cpu().numpy().reshape(box.seqs, rows, n_heads)
    q = q.reshape(box.seqs, rows, n_heads, hd).astype(np.float64)
    here = np.arange(rows)
    seen = (here <= here[:, None]) & (here >= (0 if first is None else np.asarray(first)[:, None]))
    worst = 0.0
    for s in range(box.seqs):
        for h in range(n_heads):
            g, x = h // group, q[s, :, h]
            k, v = box.k[s, g, :rows], box.v[s, g, :rows]
            ks, vs = 8 * box.kstep[s, g, :rows], 8 * box.vstep[s, g, :rows]
            a = np.abs(x) @ ks.T / np.sqrt(hd)
            score = np.where(seen, x @ k.T / np.sqrt(hd), -np.inf)
            top = score.max(axis=1, keepdims=True)
            mass = np.exp(score - top).sum(axis=1, keepdims=True)
            p = np.exp(score - top) / mass
            abar = (p * a).sum(axis=1, keepdims=True)
            least = (p * vs.max(axis=1)).max(axis=1, keepdims=True) * seen.sum(axis=1, keepdims=True) * 2.0 ** -34
            tol = 2.0 ** -21 * ((p * (a + abar)) @ vs) + 2.0 ** -18 * (p @ vs) + least
            worst = max(worst, float((np.abs(o[s, :, h] - p @ v) / tol).max()))
            lz = (top + np.log(mass))[:, 0]
            assert (np.abs(z[s, :, h] - lz) <= 2.0 ** -21 * abar[:, 0] + 2.0 ** -20 * (1 + np.abs(lz))).all()
    assert worst <= 1, worst


# (few columns; and enough of them for the form in which columns share each key's expansion)
FORMS = [1, 64]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("repeat", FORMS)
@pytest.mark.parametrize("up,std", [(15, 0.5), (20, 0.02), (26, 2.0 ** -12)])
def test_a_late_key_with_one_large_value_block_leaves_the_rows_before_it_exact(fh, repeat, hd, up, std):
    box = Box(2, 2, hd, 96, [96, 96], 101, v_std=std, repeat=repeat)
    factor = np.ones((96, hd // 32))
    factor[90, 1] = 2.0 ** up
    rescaled(box, "v", factor)
    q = np.random.default_rng(102).standard_normal((box.seqs * 96, 8, hd)).astype(np.float32)
    attend(fh, box, q, 96)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("repeat", FORMS)
@pytest.mark.parametrize("down", [10, 16, 20])
def test_value_blocks_of_a_key_far_apart(fh, repeat, hd, down):
    """Every third key's last block, and a document that has no other keys."""
    box = Box(2, 2, hd, 96, [96, 96], 103, v_std=4.0, repeat=repeat)
    factor = np.ones((96, hd // 32))
    factor[::3, -1] = 2.0 ** -down
    factor[64:80, -1] = 2.0 ** -down
    rescaled(box, "v", factor)
    q = np.random.default_rng(104).standard_normal((box.seqs * 96, 8, hd)).astype(np.float32)
    first = np.where(np.arange(96) < 64, 0, np.where(np.arange(96) < 80, 64, 80))
    attend(fh, box, q, 96, first)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("repeat", FORMS)
@pytest.mark.parametrize("down", [14, 18, 22])
@pytest.mark.parametrize("late", [False, True])
def test_key_blocks_far_apart_under_queries_of_the_small_one(fh, repeat, hd, down, late):
    """Keys' first blocks 2^down above their last, where the queries have all their weight: of
    every key, or of one late key alone."""
    box = Box(2, 2, hd, 96, [96, 96], 105, k_std=2.0 ** -10, repeat=repeat)
    factor = np.ones((96, hd // 32))
    factor[90 if late else slice(None), 0] = 2.0 ** down
    rescaled(box, "k", factor)
    q = np.random.default_rng(106).standard_normal((box.seqs * 96, 8, hd)).astype(np.float32) * np.float32(2.0 ** 11)
    q[..., :hd - 32] = 0
    attend(fh, box, q, 96)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("repeat", FORMS)
def test_a_sliding_window_by_its_formula(fh, repeat, hd):
    """first = row + 1 - w, below 0 for the first rows: they see all that is before them."""
    box = Box(2, 2, hd, 96, [96, 96], 107, repeat=repeat)
    q = np.random.default_rng(108).standard_normal((box.seqs * 96, 8, hd)).astype(np.float32)
    attend(fh, box, q, 96, np.arange(96) + 1 - 9)


@pytest.mark.parametrize("n_heads,hd,keys", [(1, 128, 32760), (5, 128, 32760), (16, 64, 65536), (8, 32, 262144)])
def test_a_long_row_over_many_workgroups(fh, n_heads, hd, keys):
    """The keys of one unit of columns are dealt over 128, 64, 32 and 64 workgroups, whose parts the
    last to arrive joins in several passes."""
    from test_gpu_kv4 import attend as attend_box

    box = Box(1, 1, hd, keys, [keys], 109, tracked=True)
    attend_box(fh, box, n_heads, [keys - 1], [1], 110, False, weigh=True)


@pytest.mark.parametrize("n_heads,n_kv,hd", [(8, 2, 32), (8, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("repeat", [1, 90])
def test_bias_by_positions_that_are_not_rows_in_prompts(fh, n_heads, n_kv, hd, repeat):
    """Distances from the cache's own positions (gaps, as after an eviction) under a cap, and the weights."""
    from test_gpu_kv4 import attend as attend_box

    lens, news = [0, 41, 7, 130] * repeat, [70, 61, 57, 68] * repeat
    top = max(a + b for a, b in zip(lens, news))
    box = Box(4, n_kv, hd, -(-top // 8) * 8, [a + b for a, b in zip(lens, news)][:4], 111, tracked=True, repeat=repeat)
    rng = np.random.default_rng(112)
    box.pos = np.sort(rng.integers(0, 3000, box.pos.shape), axis=2).astype(np.int32)
    box.c.planes["pos"].copy_(gpu(box.pos))
    slopes = 2.0 ** (-8.0 * np.arange(1, n_heads + 1) / n_heads)
    qpos = rng.integers(0, 3000, sum(news))  # (in front of some keys, behind others)
    attend_box(fh, box, n_heads, lens, news, 113, True, softcap=6.0, slopes=slopes, qpos=qpos, weigh=True)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("repeat", [1, 90])
def test_rows_of_prompts_beyond_the_bound(fh, repeat, hd):
    """Rows at or past max_keys are NaN, the others as without that bound; the NaN rows weigh nothing."""
    import ferrum_hip
    import torch

    rows, most, n_heads = 96, 70, 8
    box = Box(4, 2, hd, 96, [96] * 4, 114, tracked=True, repeat=repeat)
    total = box.seqs * rows
    q = torch.randn((total, n_heads * hd), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    got = []
    for keys in (rows, most):
        out, lse = torch.zeros_like(q), torch.zeros((total, n_heads), device="cuda")
        weight = box.c.planes["weight"]
        weight.zero_()
        torch.cuda.synchronize()
        args = (fh, box.c, q, n_heads * hd, total, n_heads, None, rows, None, keys, None)
        ferrum_hip.kv4_attention_async(*args, out, lse)
        ferrum_hip.kv4_weigh_async(*args, lse)
        fh.sync()
        got.append((out.cpu().numpy().reshape(box.seqs, rows, -1), lse.cpu().numpy().reshape(box.seqs, rows, -1),
                    weight.cpu().numpy()))
    (o, z, _), (ob, zb, wb) = got
    assert np.isnan(ob[:, most:]).all() and np.isnan(zb[:, most:]).all()
    # (the same products and sums; how the keys are dealt may differ: 1e-5 of the values' size)
    assert np.abs(ob[:, :most] - o[:, :most]).max() <= 1e-5 * np.abs(box.v).max()
    assert np.abs(zb[:, :most] - z[:, :most]).max() <= 1e-5
    assert (wb[:, :, most:] == 0).all() and np.isfinite(wb).all()
    # each row's heads give 1 each; 2^-18 of a weight (its score's and its lse's roundings) and of the sums
    assert np.allclose(wb.sum(axis=2), most * n_heads / 2, rtol=2.0 ** -17)
