"""Acceptance of drafted trees ends where the cache does: a node whose keys and values were
not stored is not accepted, and what is accepted lies in the cache."""
import numpy as np
import pytest

import gqa_ref as ref
from llama_tiny import OracleLlamaRow
from test_gpu_llama_rows import MODELS, build, close
from test_gpu_tree_accept import draft, gpu, ints, run

pytestmark = pytest.mark.gpu


def way_within(parent, tokens, chosen, at, limit):
    """The accepted rows of a tree over `at` cache rows of which `limit` exist."""
    stored = max(0, min(len(parent), limit - at))
    return ref.accept(parent[:stored], tokens[:stored], chosen[:stored])


def call(fh, trees, lens, cap, planes, kv_dim, alias=False, caches=True, max_keys=None):
    """The call's outputs, and the caches before and after."""
    import ferrum_hip
    import torch

    news = [len(t[0]) for t in trees]
    seqs, total = len(trees), sum(news)
    off = np.concatenate([[0], np.cumsum(news)])
    parent, tokens, chosen = (ints(np.concatenate([t[i] for t in trees])) for i in range(3))
    before = np.random.default_rng(40).standard_normal((planes, seqs, cap, kv_dim)).astype(np.float32)
    d = [gpu(p) for p in before]
    table = torch.tensor([x.data_ptr() for x in d], dtype=torch.int64, device="cuda")
    path, count, nxt, ln = (torch.full((n,), 7, dtype=torch.int32, device="cuda") for n in (total, seqs, seqs, seqs))
    length, doff = ints(lens), ints(off)
    new_len = length if alias else ln
    torch.cuda.synchronize()
    ferrum_hip.tree_accept_async(fh, parent, tokens, chosen, total, doff, seqs, max(news), length, table if caches else None,
                                 planes if caches else 0, kv_dim, cap, path, count, nxt, new_len,
                                 *([] if max_keys is None else [max_keys]))
    fh.sync()
    path = path.cpu().numpy()
    paths = [path[off[s]:off[s + 1]].tolist() for s in range(seqs)]
    return paths, count.tolist(), nxt.tolist(), new_len.tolist(), before, [x.cpu().numpy() for x in d]


def check(fh, trees, lens, cap, limit, planes=2, kv_dim=64, **kw):
    paths, count, nxt, new_len, before, after = call(fh, trees, lens, cap, planes, kv_dim, **kw)
    cut = 0
    want = before.copy()
    for s, t in enumerate(trees):
        way = way_within(*t, lens[s], limit)
        cut += len(way) < len(ref.accept(*t))
        assert paths[s] == way + [-1] * (len(t[0]) - len(way)), s
        assert (count[s], new_len[s], nxt[s]) == (len(way), lens[s] + len(way), int(t[2][way[-1]]) if way else 7), s
        for i, p in enumerate(way):
            want[:, s, lens[s] + i] = before[:, s, lens[s] + p]
    for p in range(planes):
        np.testing.assert_array_equal(after[p], want[p])
    return cut


def test_a_child_past_the_capacity_is_not_accepted(fh):
    """Three cache rows are left: rows 0, 1 and 2 are stored, row 3 is not."""
    tree = (np.array([-1, 0, 0, 0]), np.array([5, 11, 12, 13]), np.array([13, 1, 2, 3]))
    assert check(fh, [tree], [29], 32, 32) == 1
    assert check(fh, [tree], [28], 32, 32) == 0


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("kv_dim", [6, 128])
def test_paths_that_leave_the_cache(fh, alias, kv_dim):
    rng = np.random.default_rng(41)
    for _ in range(6):
        trees = [draft(n, rng, 0.9, 3) for n in (20, 40, 1, 300)]
        chain = (np.arange(30) - 1, np.arange(30) + 50, np.arange(30) + 51)
        # the last rows of the cache, the very last one, and none
        assert check(fh, trees + [chain], [44, 47, 49, 30, 45], 50, 50, kv_dim=kv_dim, alias=alias) >= 1
        check(fh, trees + [chain], [50, 60, 50, 49, 3], 50, 50, kv_dim=kv_dim, alias=alias)


def test_rows_outside_beyond_and_in_place(fh):
    """Rows outside all sequences, rows past max_rows, lengths in place, no caches."""
    rng = np.random.default_rng(8)
    trees = [draft(n, rng, 0.9, 3) for n in (20, 40)]
    run(fh, trees, [10, 3], 80, 2, 64, 9, before=5)
    run(fh, trees, [10, 3], 80, 2, 64, 10, max_rows=13, alias=True)
    run(fh, trees, [10, 3], 80, 0, 64, 12)
    assert check(fh, trees, [10, 30], 33, 33) == 1  # (rows past the capacity)


def test_without_caches_there_is_no_bound(fh):
    tree = (np.array([-1, 0, 0, 0]), np.array([5, 11, 12, 13]), np.array([13, 1, 2, 3]))
    paths, count, nxt, new_len, _, _ = call(fh, [tree], [29], 32, 1, 8, caches=False)
    assert (paths, count, nxt, new_len) == ([[0, 3, -1, -1]], [2], [3], [31])


@pytest.mark.parametrize("name", ["qwen", "wide"])
def test_a_step_behind_an_acceptance_at_the_end_of_the_context(fh, orc, name):
    """The draft that the model agrees with lies past the context, one it does not agree with inside:
    the row goes on with the first alone, and the next token's scores are the oracle's."""
    import torch

    cfg, w, m = build(fh, orc, name, 2)
    cap = cfg["context"]
    rng = np.random.default_rng(42)
    text = [rng.integers(0, cfg["vocab"], n).tolist() for n in (cap - 3, cap - 9)]
    root = [3, 4]
    m.prompt_async(ints(np.concatenate(text)), [len(t) for t in text])
    m.pos.copy_(ints([len(t) for t in text]))
    m.tokens.copy_(ints(root))
    tokens, parents = ints([[3, 21, 22, 23], [4, 21, 22, 23]]).flatten(), ints([[-1, 0, 0, 0]] * 2).flatten()
    chosen = ints([[23, 31, 32, 33]] * 2).flatten()
    torch.cuda.synchronize()
    m.verify_async(tokens, parents, 4, cap - 3)
    m.accept_async(chosen)
    fh.sync()
    assert m.count.tolist() == [1, 2] and m.path.tolist() == [[0, -1, -1, -1], [0, 3, -1, -1]]
    assert m.pos.tolist() == [cap - 2, cap - 7] and m.tokens.tolist() == [23, 33]
    m.feed_async(cap - 2)
    fh.sync()
    for r, t in enumerate((text[0] + [3, 23], text[1] + [4, 23, 33])):
        oracle = OracleLlamaRow(orc, w, cfg)
        assert close(m.z[r].cpu().numpy(), [oracle.feed(x) for x in t][-1]), r
    m.free()


@pytest.mark.parametrize("alias", [False, True])
def test_rows_that_the_attention_had_no_place_for(fh, alias):
    """max_keys below the capacity, above it, and without caches."""
    rng = np.random.default_rng(43)
    trees = [draft(n, rng, 0.9, 3) for n in (20, 40, 300)] + [(np.arange(30) - 1, np.arange(30) + 50, np.arange(30) + 51)]
    assert check(fh, trees, [24, 27, 29, 10], 400, 30, alias=alias, max_keys=30) >= 2
    check(fh, trees, [24, 27, 29, 10], 400, 0, alias=alias, max_keys=0)
    check(fh, trees, [24, 27, 29, 10], 400, 400, alias=alias, max_keys=1 << 40)
    paths, count, _, new_len, _, _ = call(fh, trees[3:], [10], 400, 1, 8, caches=False, max_keys=30)
    assert (paths, count, new_len) == ([list(range(20)) + [-1] * 10], [20], [30])


def test_drafts_past_max_pos_are_not_accepted(fh, orc):
    """A step with a bound that the rows have outgrown, as a captured one replayed too often has: the
    drafts it had no place for are left, and the next token's scores are the oracle's."""
    import torch

    cfg, w, m = build(fh, orc, "qwen", 2)
    rng = np.random.default_rng(44)
    text = [rng.integers(0, cfg["vocab"], n).tolist() for n in (20, 17)]
    m.prompt_async(ints(np.concatenate(text)), [20, 17])
    m.pos.copy_(ints([20, 17]))
    tokens, parents = ints([3, 21, 22, 23, 4, 21, 22, 23]), ints([-1, 0, 0, 0] * 2)
    chosen = ints([23, 31, 32, 33] * 2)
    torch.cuda.synchronize()
    m.verify_async(tokens, parents, 4, 18)  # rows up to 21
    fh.sync()
    finite = torch.isfinite(m.zt).all(dim=1).tolist()
    assert finite == [True, True, False, False] + [True] * 4
    m.accept_async(chosen)
    fh.sync()
    assert m.count.tolist() == [1, 2] and m.path.tolist() == [[0, -1, -1, -1], [0, 3, -1, -1]]
    assert m.pos.tolist() == [21, 19] and m.tokens.tolist() == [23, 33]
    m.feed_async(21)
    fh.sync()
    for r, t in enumerate((text[0] + [3, 23], text[1] + [4, 23, 33])):
        oracle = OracleLlamaRow(orc, w, cfg)
        assert close(m.z[r].cpu().numpy(), [oracle.feed(x) for x in t][-1]), r
    m.free()
