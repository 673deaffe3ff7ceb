"""Prompts and trees over f32 caches as they are used: sizes at random, two captured graphs of one
context, another stream, single tokens behind an accepted tree, caches at odd addresses."""
import numpy as np
import pytest

import gqa_ref as ref
from llama_tiny import QWEN, OracleLlamaRow, make_weights
from test_gpu_gqa_rows import Call, gpu, ints, trees
from test_gpu_kv4_llama import close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(12))
def test_sizes_at_random(fh, seed):
    rng = np.random.default_rng(100 + seed)
    for _ in range(4):
        hd = int(rng.choice([8, 16, 32, 64, 128]))
        g = int(rng.choice([1, 2, 3, 8]))
        heads = (g * int(rng.choice([1, 3, 4, 7])), g, hd)
        seqs = int(rng.integers(1, 9))
        tree = bool(rng.integers(0, 2))
        lens = [int(x) for x in np.exp(rng.uniform(0, np.log(3000), seqs))]
        news = [int(x) for x in np.exp(rng.uniform(0, np.log(80 if tree else 250), seqs))]
        if seqs > 2:
            lens[0], news[1] = 0, 0
        rope = [("neox", None), ("norm", None), (None, None)][int(rng.integers(0, 3))]
        print(heads, lens, news, tree, rope, flush=True)
        Call(heads, lens, news, seed, parents=trees(news, seed) if tree else None, rope=rope).check(fh)


def finite(x):
    return np.nan_to_num(x, nan=0.5, posinf=0.5, neginf=0.5).clip(-5, 5)


def test_two_graphs_of_one_context(fh):
    """A tree at width 128 and a prompt, captured one after the other, replayed in turns with eager calls
    between: they share the workspace."""
    import torch

    one = Call((32, 8, 128), [2900, 40, 700], [40, 7, 21], 60, parents=trees([40, 7, 21], 61))
    two = Call((14, 2, 64), [0, 300], [130, 90], 62)
    graphs, stream = [], torch.cuda.Stream()
    for a in (one, two):
        a.k, a.v = finite(a.k), finite(a.v)
        a.run(fh)
    fh.set_stream(stream.cuda_stream)
    try:
        for a in (one, two):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                a.again(fh)
        fh.set_stream(None)
        want = []
        for a in (one, two):
            a.again(fh)
            fh.sync()
            want.append(a.out.clone())
        for turn in range(4):
            for i in ((0, 1), (1, 0))[turn % 2]:
                a = (one, two)[i]
                a.out.zero_()
                torch.cuda.synchronize()
                graphs[i].replay()
                torch.cuda.synchronize()
                assert torch.equal(a.out, want[i]), (turn, i)
            Call((12, 12, 64), [500], [9], 63).check(fh)
    finally:
        fh.set_stream(None)


def test_on_another_stream(fh):
    """Everything enqueued on a caller's stream, inputs made there and not waited for."""
    import torch

    a = Call((14, 2, 64), [900, 3], [30, 12], 64)
    want = a.run(fh)
    stream = torch.cuda.Stream()
    fh.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            source, a.dqkv = a.dqkv, torch.zeros_like(a.dqkv)
            a.out.fill_(77.0)
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(4):
                big = (big @ big) * 1e-3
            a.dqkv.copy_(source)
            a.again(fh)
            got = a.out.clone()
        stream.synchronize()
    finally:
        fh.set_stream(None)
    np.testing.assert_array_equal(got.cpu().numpy().reshape(want.shape), want)


def test_single_tokens_behind_an_accepted_tree(fh, orc):
    import ferrum_hip

    w = make_weights(orc, QWEN, 3, True, True)
    m = ferrum_hip.LlamaDevice.from_weights(fh, w, QWEN, 1)
    oracle = OracleLlamaRow(orc, w, QWEN)
    rng = np.random.default_rng(65)
    ids = [int(x) for x in rng.integers(0, QWEN["vocab"], 8)]
    for t in ids:
        z = m.forward_one(t)
        want = oracle.feed(t)
    first = int(want.argmax())
    path = [first]  # what the model itself would go on with
    walk = OracleLlamaRow(orc, w, QWEN)
    for t in ids:
        walk.feed(t)
    for _ in range(3):
        path.append(int(walk.feed(path[-1]).argmax()))
    assert close(z, want) and m.pos.cpu().tolist() == [8]
    # row 0, a wrong draft, the right ones behind it
    tokens = [path[0], (path[1] + 1) % QWEN["vocab"], path[1], path[2], (path[3] + 1) % QWEN["vocab"]]
    m.verify_async(ints(tokens), ints([-1, 0, 0, 2, 3]), 5, 8)
    fh.sync()
    m.accept_async(m.zt.argmax(dim=1).int())
    fh.sync()
    assert m.path.cpu().tolist() == [[0, 2, 3, -1, -1]] and m.pos.cpu().tolist() == [11]
    assert m.tokens.cpu().tolist() == [path[3]]
    m.next_pos = 11
    for t in path[:3]:
        oracle.feed(t)
    for t in [path[3]] + [int(x) for x in rng.integers(0, QWEN["vocab"], 4)]:
        assert close(m.forward_one(t), oracle.feed(t))
    m.free()


@pytest.mark.parametrize("kv_dim", [1, 6, 128, 260])
def test_acceptance_in_caches_at_odd_addresses(fh, kv_dim):
    """Caches that begin 4 bytes past a 16-byte line, trees of up to 1024 rows, lengths in place."""
    import ferrum_hip
    import torch

    rng = np.random.default_rng(66 + kv_dim)
    news, lens, cap = [1024, 1, 0, 333], [7, 0, 3, 700], 1040
    off = np.concatenate([[0], np.cumsum(news)])
    total = int(off[-1])
    parent = np.concatenate([[-1] + [int(rng.integers(max(0, t - 2), t)) for t in range(1, n)] if n else [] for n in news])
    tokens, chosen = rng.integers(0, 3, total), rng.integers(0, 3, total)
    planes = [torch.randn(len(news) * cap * kv_dim + 4, device="cuda") for _ in range(3)]
    views = [p[1:1 + len(news) * cap * kv_dim].view(len(news), cap, kv_dim) for p in planes]
    before = [v.cpu().numpy().copy() for v in views]
    address = torch.tensor([v.data_ptr() for v in views], dtype=torch.int64, device="cuda")
    path, count, nxt, ln = ints(np.zeros(total)), ints(np.zeros(4)), ints([5] * 4), ints(lens)
    torch.cuda.synchronize()
    ferrum_hip.tree_accept_async(fh, ints(parent), ints(tokens), ints(chosen), total, ints(off), 4, 1024, ln, address, 3, kv_dim,
                                 cap, path, count, nxt, ln)
    fh.sync()
    for s, n in enumerate(news):
        rows = slice(off[s], off[s + 1])
        way = ref.accept(parent[rows], tokens[rows], chosen[rows])
        assert path.cpu().tolist()[rows] == way + [-1] * (n - len(way)) and count.cpu().tolist()[s] == len(way)
        assert ln.cpu().tolist()[s] == lens[s] + len(way)
        assert nxt.cpu().tolist()[s] == (chosen[rows][way[-1]] if way else 5)
        for v, old in zip(views, before):
            want = old[s].copy()
            for i, p in enumerate(way):
                if lens[s] + p < cap:
                    want[lens[s] + i] = old[s][lens[s] + p]
            np.testing.assert_array_equal(v[s].cpu().numpy(), want)
    for p in planes:
        assert p.isfinite().all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("heads", [(4, 2, 64), (32, 2, 64), (4, 2, 128), (80, 2, 128), (4, 4, 32), (2, 1, 8)])
@pytest.mark.parametrize("where", ["q", "k", "v", "cached k", "cached v"])
def test_every_channel_of_a_row_that_sees_what_is_not_finite(fh, bad, heads, where):
    """And no bit of the others, at every number of columns of a workgroup."""
    for parents in (None, trees([40], 67)):
        a = Call(heads, [50], [40], 68, parents=parents, rope=(None, None))
        plain = a.run(fh)
        at, group = 29, a.h // a.g
        if where == "cached k":
            a.k[0, at, 2] = bad
        elif where == "cached v":
            a.v[0, at, 2] = bad
        else:
            a.qkv[at, {"q": group - 1, "k": a.h, "v": a.h + a.g}[where] * a.hd + 3] = bad
        got = a.run(fh)
        ways = [list(range(t + 1)) if parents is None else ref.path(parents[0], t) for t in range(40)]
        hit = np.zeros((40, a.h), bool)
        if where == "q":
            hit[at, group - 1] = True
        else:
            hit[["cached" in where or at in w for w in ways], :group] = True
        assert np.isnan(got[hit]).all()
        np.testing.assert_array_equal(got[~hit], plain[~hit])
