"""What is accepted of drafted trees, and the caches made compact (fh_tree_accept_async)."""
import numpy as np
import pytest

import gqa_ref as ref

pytestmark = pytest.mark.gpu


def gpu(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(values):
    return gpu(np.asarray(values, np.int64).astype(np.uint32).view(np.int32))


def draft(n, rng, agree, wide=8):
    """A tree of n rows whose tokens the model agrees with where `agree` says so."""
    parent = np.array([-1] + [int(rng.integers(max(0, t - wide), t)) for t in range(1, n)])[:n]
    tokens, chosen = rng.integers(0, 1000, n), rng.integers(1000, 2000, n)
    for t in range(n - 1, 0, -1):
        if rng.random() < agree:
            chosen[parent[t]] = tokens[t]
    return parent, tokens, chosen


def run(fh, trees, lens, cap, planes, kv_dim, seed, before=0, max_rows=None, alias=False, off=True):
    import ferrum_hip
    import torch

    news = [len(t[0]) for t in trees]
    seqs, total = len(trees), before + sum(news) + 2
    o = np.concatenate([[0], np.cumsum(news)]) + before
    flat = [np.full(total, x) for x in (-1, 5, 5)]
    for s, t in enumerate(trees):
        for dst, src in zip(flat, t):
            dst[o[s]:o[s + 1]] = src
    most = max(news) if max_rows is None else max_rows
    rng = np.random.default_rng(seed)
    cache = rng.standard_normal((planes, seqs, cap, kv_dim)).astype(np.float32)
    d = [gpu(p) for p in cache]
    table = torch.tensor([x.data_ptr() for x in d], dtype=torch.int64, device="cuda")
    parent, tokens, chosen = (ints(x) for x in flat)
    path = torch.full((total,), 7, dtype=torch.int32, device="cuda")
    count, nxt, ln = (torch.full((seqs,), 7, dtype=torch.int32, device="cuda") for _ in range(3))
    length = ints(lens)
    new_len = length if alias else ln
    ferrum_hip.tree_accept_async(fh, parent, tokens, chosen, total, ints(o), seqs, most, length, table, planes, kv_dim, cap, path,
                                 count, nxt, new_len)
    fh.sync()
    path = path.cpu().numpy()
    want = cache.copy()
    used = np.zeros(total, bool)
    for s, (par, tok, cho) in enumerate(trees):
        n = min(news[s], most)
        way = ref.accept(par[:n], tok[:n], cho[:n])
        used[o[s]:o[s] + n] = True
        assert path[o[s]:o[s] + n].tolist() == way + [-1] * (n - len(way))
        assert int(count[s]) == len(way) and int(new_len[s]) == lens[s] + len(way)
        assert int(nxt[s]) == (cho[way[-1]] if way else 7)
        for i, t in enumerate(way):
            if lens[s] + t < cap:
                want[:, s, lens[s] + i] = cache[:, s, lens[s] + t]
    assert (path[~used] == 7).all()
    for p in range(planes):
        np.testing.assert_array_equal(d[p].cpu().numpy(), want[p])


@pytest.mark.parametrize("agree", [0.0, 0.3, 0.8, 1.0])
@pytest.mark.parametrize("kv_dim", [8, 96, 128, 1024, 1030])
def test_paths_and_caches(fh, agree, kv_dim):
    rng = np.random.default_rng(3)
    trees = [draft(n, rng, agree) for n in (1, 16, 64, 0, 33, 2)]
    run(fh, trees, [0, 10, 100, 4, 31, 62], 170, 4, kv_dim, 4)


def test_long_paths(fh):
    rng = np.random.default_rng(5)
    chain = lambda n: (np.arange(n) - 1, np.arange(n) + 50, np.arange(n) + 51)  # noqa: E731
    run(fh, [chain(1024), draft(1024, rng, 1.0, 3), draft(300, rng, 1.0, 4)], [5, 0, 40], 1100, 2, 64, 6)
    # every second row of a chain is a dead end: each accepted row moves
    n = 600
    parent = np.array([-1] + [max(0, t - 2) if t % 2 == 0 else t - 1 for t in range(1, n)])
    tokens, chosen = np.arange(n), np.where(np.arange(n) % 2 == 0, np.arange(n) + 2, 0)
    run(fh, [(parent, tokens, chosen)], [3], 700, 3, 128, 7)


def test_rows_outside_beyond_and_in_place(fh):
    rng = np.random.default_rng(8)
    trees = [draft(n, rng, 0.9, 3) for n in (20, 40)]
    run(fh, trees, [10, 3], 80, 2, 64, 9, before=5)
    run(fh, trees, [10, 3], 80, 2, 64, 10, max_rows=13, alias=True)
    run(fh, trees, [10, 30], 33, 2, 64, 11)  # rows past the capacity
    run(fh, trees, [10, 3], 80, 0, 64, 12)


def test_equal_tokens_take_the_first(fh):
    run(fh, [(np.array([-1, 0, 0, 1, 2]), np.array([1, 5, 5, 6, 6]), np.array([5, 6, 6, 9, 8]))], [0], 8, 1, 32, 13)


def test_bad_parents_end_nowhere(fh):
    run(fh, [(np.array([3, 0, 2, 9, 1]), np.array([5, 5, 5, 5, 5]), np.full(5, 5))], [0], 8, 1, 32, 14)


def test_equal_parts_and_no_lengths(fh):
    import ferrum_hip
    import torch

    rng = np.random.default_rng(15)
    trees = [draft(12, rng, 0.8) for _ in range(3)]
    flat = [ints(np.concatenate([t[i] for t in trees])) for i in range(3)]
    path = torch.zeros(36, dtype=torch.int32, device="cuda")
    count, nxt, ln = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(3))
    ferrum_hip.tree_accept_async(fh, *flat, 36, None, 3, 0, None, None, 0, 0, 0, path, count, nxt, ln)
    fh.sync()
    for s, t in enumerate(trees):
        way = ref.accept(*t)
        assert path[12 * s:12 * s + 12].tolist() == way + [-1] * (12 - len(way))
        assert int(ln[s]) == len(way) == int(count[s]) and int(nxt[s]) == t[2][way[-1]]


def test_refusals(fh):
    import ferrum_hip as m
    import torch

    i = torch.zeros(4096, dtype=torch.int32, device="cuda")
    p = torch.zeros(4, dtype=torch.int64, device="cuda")

    def call(par=i, total=8, off=None, seqs=2, rows=4, planes=p, n=1, dim=64, cap=32, path=i, count=i):
        m.tree_accept_async(fh, par, i, i, total, off, seqs, rows, i, planes, n, dim, cap, path, count, i, i)

    for kw, code in ((dict(seqs=0), m.FH_ERR_INVALID), (dict(seqs=65536, total=0), m.FH_ERR_LIMIT), (dict(total=7), m.FH_ERR_DIM),
                     (dict(total=2050), m.FH_ERR_LIMIT), (dict(off=i, rows=1025, total=2000), m.FH_ERR_LIMIT),
                     (dict(par=None), m.FH_ERR_INVALID), (dict(path=None), m.FH_ERR_INVALID), (dict(count=None), m.FH_ERR_INVALID),
                     (dict(planes=None), m.FH_ERR_INVALID), (dict(dim=0), m.FH_ERR_INVALID), (dict(cap=0), m.FH_ERR_INVALID),
                     (dict(n=65536), m.FH_ERR_LIMIT)):
        with pytest.raises(m.FerrumHipError) as e:
            call(**kw)
        assert e.value.code == code, kw
