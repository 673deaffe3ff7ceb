"""LlamaDevice over f32 caches: prompts at once, drafted trees, what is accepted of
them, and the run of all of these with edited logits, against the oracle's token by
token decode."""
import numpy as np
import pytest

import gqa_ref as ref
from llama_tiny import LLAMA, QWEN, OracleLlamaRow, make_weights

pytestmark = pytest.mark.gpu

MODELS = {"qwen": (QWEN, True, True), "llama": (LLAMA, False, False),
          "wide": (dict(QWEN, head_dim=64, n_heads=2, n_kv=1), True, True),
          "one": (dict(LLAMA, head_dim=8, n_heads=12, n_kv=12, rope_dim=8), False, True)}


def build(fh, orc, name, rows, context=None):
    import ferrum_hip

    cfg, biases, tied = MODELS[name]
    cfg = dict(cfg, context=context or cfg["context"])
    w = make_weights(orc, cfg, 3, biases, tied)
    return cfg, w, ferrum_hip.LlamaDevice.from_weights(fh, w, cfg, rows)


def ints(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32).ravel())).cuda()


def close(got, want):
    """The rule of the step by step tests: 2e-5 of the largest score."""
    return np.abs(got - want).max() <= 2e-5 * np.abs(want).max()


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("rows", [1, 3])
def test_prompts_then_steps(fh, orc, name, rows):
    import torch

    cfg, w, m = build(fh, orc, name, rows)
    rng = np.random.default_rng(rows)
    oracle = [OracleLlamaRow(orc, w, cfg) for _ in range(rows)]
    pos = np.zeros(rows, np.int64)
    for lens in ([20, 1, 13][:rows], [3, 5, 1][:rows]):
        ids = [rng.integers(0, cfg["vocab"], n) for n in lens]
        m.pos.copy_(ints(pos))
        torch.cuda.synchronize()
        m.prompt_async(ints(np.concatenate(ids)), lens)
        fh.sync()
        for r in range(rows):
            want = [oracle[r].feed(t) for t in ids[r]][-1]
            assert close(m.z[r].cpu().numpy(), want), r
        pos += lens
    for _ in range(2):
        ids = rng.integers(0, cfg["vocab"], rows)
        m.tokens.copy_(ints(ids))
        m.pos.copy_(ints(pos))
        torch.cuda.synchronize()
        m.feed_async(int(pos.max()))
        fh.sync()
        for r in range(rows):
            assert close(m.z[r].cpu().numpy(), oracle[r].feed(ids[r])), r
        pos += 1
    m.free()


def test_forward_one_goes_on_behind_a_prompt(fh, orc):
    cfg, w, m = build(fh, orc, "qwen", 1)
    oracle = OracleLlamaRow(orc, w, cfg)
    ids = np.random.default_rng(5).integers(0, cfg["vocab"], 30)
    for t in ids[:4]:
        assert close(m.forward_one(int(t)), oracle.feed(t))
    m.prompt_async(ints(ids[4:20]), [16])
    fh.sync()
    want = [oracle.feed(t) for t in ids[4:20]][-1]
    assert close(m.z[0].cpu().numpy(), want)
    m.next_pos = 20
    for t in ids[20:]:
        assert close(m.forward_one(int(t)), oracle.feed(t))
    m.free()


def tree(rng, n, vocab):
    parent = np.array([-1] + [int(rng.integers(max(0, t - 5), t)) for t in range(1, n)])
    return parent, rng.integers(0, vocab, n)


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 9), (3, 12), (5, 20)])
def test_trees_score_as_their_paths(fh, orc, name, rows, n):
    import torch

    cfg, w, m = build(fh, orc, name, rows)
    rng = np.random.default_rng(n)
    lens = rng.integers(1, cfg["context"] - n - 8, rows)
    text = [rng.integers(0, cfg["vocab"], k).tolist() for k in lens]
    m.prompt_async(ints(np.concatenate(text)), lens)
    m.pos.copy_(ints(lens))
    torch.cuda.synchronize()
    for _ in range(2):
        trees = [tree(rng, n, cfg["vocab"]) for _ in range(rows)]
        chosen = rng.integers(0, cfg["vocab"], (rows, n))
        for r, (parent, tokens) in enumerate(trees):
            for t in range(1, n):
                if rng.random() < 0.5:
                    chosen[r, parent[t]] = tokens[t]
        m.verify_async(ints([t[1] for t in trees]), ints([t[0] for t in trees]), n, int(max(len(t) for t in text)))
        fh.sync()
        z = m.zt.cpu().numpy().reshape(rows, n, -1)
        for r, (parent, tokens) in enumerate(trees):
            for t in {0, n - 1, n // 2}:
                oracle = OracleLlamaRow(orc, w, cfg)
                want = [oracle.feed(x) for x in text[r] + tokens[ref.path(parent, t)].tolist()][-1]
                assert close(z[r, t], want), (r, t)
        m.accept_async(ints(chosen))
        fh.sync()
        for r, (parent, tokens) in enumerate(trees):
            way = ref.accept(parent, tokens, chosen[r])
            assert m.path[r].tolist() == way + [-1] * (n - len(way)) and int(m.count[r]) == len(way)
            text[r] += tokens[way].tolist()
            assert int(m.pos[r]) == len(text[r]) and int(m.tokens[r]) == chosen[r, way[-1]]
        if max(len(t) for t in text) + n > cfg["context"]:
            break
    # the caches hold the accepted text: a plain step from there
    if max(len(t) for t in text) < cfg["context"]:
        ids = m.tokens.cpu().numpy()
        m.feed_async(max(len(t) for t in text))
        fh.sync()
        for r in range(rows):
            oracle = OracleLlamaRow(orc, w, cfg)
            want = [oracle.feed(x) for x in text[r] + [int(ids[r])]][-1]
            assert close(m.z[r].cpu().numpy(), want), r
    m.free()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("rows", [1, 4])
def test_a_drafted_run_with_edits_has_the_ids_of_a_plain_one(fh, orc, rows, captured):
    """Prompt, then trees: verified, their logits edited (penalties over the text and each node's
    own path, a bias, a grammar mask), sampled, accepted; against single tokens with the same
    edits.  Drafts are the plain run's tokens, some of them spoilt."""
    import ferrum_hip as F
    import torch

    cfg, w, m = build(fh, orc, "qwen", rows, context=96)
    vocab, n, steps = cfg["vocab"], 6, 24
    rng = np.random.default_rng(rows)
    lens = rng.integers(3, 20, rows)
    text = [rng.integers(0, vocab, k).tolist() for k in lens]
    first = rng.integers(0, vocab, rows)
    allowed = rng.random(vocab) < 0.8
    bits = np.packbits(np.pad(allowed, (0, -vocab % 32)).astype(np.uint8), bitorder="little").view("<i4")
    mask = torch.from_numpy(bits.copy()).cuda().view(1, -1)
    bias = dict(bias_id=ints([7, 400]), bias=torch.tensor([2.0, -3.0], device="cuda"))
    full = lambda v, k: torch.full((k,), v, device="cuda")  # noqa: E731
    greedy = F.SamplingParams(0.0, 0, 1.0, 1.0)

    def edit(k, ranges, hist, **tree):
        # the last row alone has biases; every row has the one mask
        return F.LogitsEdit(recent=hist, ranges=ranges, repetition=full(1.3, k), frequency=full(0.2, k), presence=full(0.1, k),
                            bias_off=ints([0] * k + [2]), mask=mask, mask_of=torch.zeros(k, dtype=torch.int32, device="cuda"),
                            masks=1, **bias, **tree)

    def prime():
        m.reset()
        m.prompt_async(ints(np.concatenate(text)), lens)
        fh.sync()
        m.pos.copy_(ints(lens))
        m.tokens.copy_(ints(first))
        torch.cuda.synchronize()

    # token by token
    prime()
    plain = [t + [int(f)] for t, f in zip(text, first)]
    margins = []
    for k in range(steps):
        at = lens + k
        hist = ints([t + [0] * (128 - len(t)) for t in plain])
        ranges = ints([[128 * r, 128 * r + len(plain[r])] for r in range(rows)])
        m.pos.copy_(ints(at))
        e = edit(rows, ranges, hist)
        torch.cuda.synchronize()
        m.feed_async(int(at.max()))
        F.logits_edit_async(fh, m.z, rows, vocab, e, m.z)
        F.sample_rows_async(fh, m.z, rows, vocab, greedy, None, None, None, m.tokens)
        fh.sync()
        z = np.sort(m.z.cpu().numpy(), axis=1)
        margins.append((z[:, -1] - z[:, -2]) / np.abs(z[:, -1]))
        for r in range(rows):
            plain[r].append(int(m.tokens[r]))
    assert allowed[[t for p, k in zip(plain, lens) for t in p[k + 1:]]].all()

    # by trees
    prime()
    hist, ranges = torch.zeros((rows, 128), dtype=torch.int32, device="cuda"), torch.zeros((rows * n, 2), dtype=torch.int32, device="cuda")
    dtok, dpar, ids = (torch.zeros(rows * n, dtype=torch.int32, device="cuda") for _ in range(3))
    e = edit(rows * n, ranges, hist, parent=dpar, tokens=dtok, seqs=rows)
    out = torch.empty((rows * n, vocab), device="cuda")

    def round_():
        m.verify_async(dtok, dpar, n, 96 - n)
        F.logits_edit_async(fh, m.zt, rows * n, vocab, e, out)
        F.sample_rows_async(fh, out, rows * n, vocab, greedy, None, None, None, ids)
        m.accept_async(ids)

    graph = None
    done = [list(t) for t in text]  # accepted into the cache
    rounds = 0
    while min(len(d) - k for d, k in zip(done, lens)) < steps - n:
        nxt = [int(m.tokens[r]) for r in range(rows)]
        par, tok = np.zeros((rows, n), np.int64), np.zeros((rows, n), np.int64)
        for r in range(rows):
            guess = plain[r][len(done[r]) + 1:len(done[r]) + n]
            guess += [0] * (n - 1 - len(guess))
            # node 1 a wrong draft beside the right one; the chain goes on from node 2
            par[r], tok[r] = [-1, 0, 0, 2, 3, 4], [nxt[r], (guess[0] + 1) % vocab] + guess[:n - 2]
            if rng.random() < 0.5:
                tok[r, int(rng.integers(2, n))] = int(rng.integers(0, vocab))
        dtok.copy_(ints(tok))
        dpar.copy_(ints(par))
        hist.copy_(ints([d + [0] * (128 - len(d)) for d in done]).view(rows, 128))
        ranges.copy_(ints([[128 * (r // n), 128 * (r // n) + len(done[r // n])] for r in range(rows * n)]).view(-1, 2))
        torch.cuda.synchronize()
        if captured and graph is None and rounds:
            stream = torch.cuda.Stream()
            graph = torch.cuda.CUDAGraph()
            fh.set_stream(stream.cuda_stream)
            with torch.cuda.graph(graph, stream=stream):
                round_()
            fh.set_stream(None)
        if graph:
            graph.replay()
            torch.cuda.synchronize()
        else:
            round_()
            fh.sync()
        for r in range(rows):
            way = [t for t in m.path[r].tolist() if t >= 0]
            assert way == ref.accept(par[r], tok[r], ids.cpu().numpy().reshape(rows, n)[r])
            done[r] += tok[r, way].tolist()
            assert int(m.pos[r]) == len(done[r])
        rounds += 1
    assert min(np.min(x) for x in margins) > 1e-4  # (no near-tie that rounding could turn)
    for r in range(rows):
        k = min(len(done[r]), len(plain[r]))
        assert done[r][:k] == plain[r][:k]
    assert rounds < steps
    m.free()


def test_refusals(fh, orc):
    import ferrum_hip as F
    import torch

    m = F.LlamaDevice(fh, dict(QWEN, kv="q4"), 2)
    ids = torch.zeros(8, dtype=torch.int32, device="cuda")
    with pytest.raises(F.FerrumHipError, match="needs the f32 cache"):
        m.verify_async(ids, ids, 4, 0)
    m = F.LlamaDevice(fh, QWEN, 2)
    with pytest.raises(F.FerrumHipError, match="follows verify_async"):
        m.accept_async(ids)
    for n in (0, 1025):
        with pytest.raises(F.FerrumHipError, match="1 to 1024"):
            m.verify_async(ids, ids, n, 0)
    for tokens, parents, what in ((ids.long(), ids, "tokens are an int32"), (ids, ids[:6], "6 parents for 2 trees of 4"),
                                  (ids.cpu(), ids, "model's device"), (ids, ids.repeat(2)[::2], "side by side")):
        with pytest.raises(F.FerrumHipError, match=what):
            m.verify_async(tokens, parents, 4, 0)
    for lens, what in (([4], "2 lengths"), ([4, 0], "2 lengths"), ([2, 1], "8 tokens for 3")):
        with pytest.raises(F.FerrumHipError, match=what):
            m.prompt_async(ids, lens)
    m.pos.fill_(QWEN["context"] - 3)
    with pytest.raises(F.DimMismatch, match="KvCache full"):
        m.prompt_async(ids, [4, 4])
