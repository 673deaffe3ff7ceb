"""LlamaDevice over 4-bit caches: prompts fed at once, batched steps and eviction,
against a float64 walk of the model over the keys and values that the device's
caches stand for (read back), and the caches against that walk's own keys."""
import numpy as np
import pytest

from llama_tiny import LLAMA, QWEN, make_weights

pytestmark = pytest.mark.gpu


class Walk:
    """LlamaModel::forward_one in float64 whose attention reads the device's cache."""

    def __init__(self, orc, w, cfg):
        self.c, f64 = cfg, (lambda a: np.asarray(a, np.float64))
        d, qd, kvd, ffn = cfg["d"], cfg["n_heads"] * cfg["head_dim"], cfg["n_kv"] * cfg["head_dim"], cfg["ffn"]
        W = lambda name, n, k: f64(orc.q8_0_dequant(w[name], n * k).reshape(n, k))  # noqa: E731
        self.tok, self.norm = W("token_embd", cfg["vocab"], d), f64(w["output_norm"])
        self.head = W("output", cfg["vocab"], d) if "output" in w else self.tok
        self.layers = []
        for i in range(cfg["layers"]):
            p = f"blk.{i}."
            bias = lambda s, n: f64(w.get(p + f"attn_{s}.bias", np.zeros(n)))  # noqa: E731
            self.layers.append(dict(
                an=f64(w[p + "attn_norm"]), fn=f64(w[p + "ffn_norm"]), q=W(p + "attn_q", qd, d), k=W(p + "attn_k", kvd, d),
                v=W(p + "attn_v", kvd, d), o=W(p + "attn_output", d, qd), g=W(p + "ffn_gate", ffn, d),
                u=W(p + "ffn_up", ffn, d), dn=W(p + "ffn_down", d, ffn), qb=bias("q", qd), kb=bias("k", kvd), vb=bias("v", kvd)))

    def rope(self, x, pos):
        hd, base = self.c["head_dim"], self.c["rope_base"]
        half, y = hd // 2, x.reshape(-1, hd).copy()
        ang = pos * base ** (-2.0 * np.arange(half) / hd)
        a, b = y[:, :half].copy(), y[:, half:].copy()
        y[:, :half], y[:, half:] = a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)
        return y

    def step(self, token, pos, caches):
        """caches[i]: (k, v) [n_kv, rows, hd] that the token sees, its own row the last
        one.  Returns the scores, and each layer's own key and value."""
        c, own = self.c, []
        rms = lambda x, g: x / np.sqrt((x * x).mean() + c["eps"]) * g  # noqa: E731
        x = self.tok[token].copy()
        for L, (k, v) in zip(self.layers, caches):
            h = rms(x, L["an"])
            q = self.rope(L["q"] @ h + L["qb"], pos)
            own.append((self.rope(L["k"] @ h + L["kb"], pos), (L["v"] @ h + L["vb"]).reshape(-1, c["head_dim"])))
            att = []
            for n in range(c["n_heads"]):
                g = n // (c["n_heads"] // c["n_kv"])
                s = k[g] @ q[n] / np.sqrt(c["head_dim"])
                e = np.exp(s - s.max())
                att.append(e / e.sum() @ v[g])
            x = x + L["o"] @ np.concatenate(att)
            h = rms(x, L["fn"])
            a = L["g"] @ h
            x = x + L["dn"] @ (a / (1 + np.exp(-a)) * (L["u"] @ h))
        return self.head @ rms(x, self.norm), own


def read(m, i):
    """Layer i's caches as float64 [rows, n_kv, capacity, hd]."""
    import ferrum_hip
    import torch

    c = m.blocks[i]["k"]
    k, v = (torch.empty((m.rows, c.capacity, m.kv_dim), device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    ferrum_hip.kv4_read_async(m.ctx, c, None, c.capacity, k, v)
    m.ctx.sync()
    return tuple(a.cpu().numpy().astype(np.float64).reshape(m.rows, c.capacity, m.nkv, m.hd).transpose(0, 2, 1, 3)
                 for a in (k, v))


def close(got, want):
    """Scores of a whole model: the framework's 1e-5 rule on sums of d terms, each at
    most the row's own size, through two blocks' residuals and norms (as the f32 cache's
    batched test allows)."""
    return np.abs(got - want).max() <= 1e-4 * np.abs(want).max()


def check_own(own, caches, at):
    """The cached row is the quantised one: within half a step of the walk's (a step at the
    clamped end), the step being the block's largest value / 8."""
    for (k, v), (kc, vc) in zip(own, caches):
        for x, y in ((k, kc[:, at]), (v, vc[:, at])):
            step = np.abs(x.reshape(-1, 32)).max(axis=1) / 8
            off = np.abs(x - y).reshape(-1, 32)
            assert (off <= (1.01 * step + 1e-4)[:, None]).all() and np.median(off / step[:, None]) < 0.35


@pytest.mark.parametrize("rows", [1, 2, 5])
def test_prompt_steps_and_eviction_match_the_walk(fh, orc, rows):
    import ferrum_hip
    import torch

    cfg = dict(QWEN, kv="q4", kv_tracked=True)
    w = make_weights(orc, QWEN, 3, True, True)
    walk = Walk(orc, w, QWEN)
    m = ferrum_hip.LlamaDevice.from_weights(fh, w, cfg, rows)
    rng = np.random.default_rng(rows)
    lens = rng.integers(1, 30, rows)
    lens[0] = 20
    prompts = [rng.integers(0, QWEN["vocab"], n) for n in lens]
    m.prefill_async(torch.from_numpy(np.concatenate(prompts).astype(np.int32)).cuda(), lens)
    fh.sync()
    z = m.z.cpu().numpy()
    caches = [read(m, i) for i in range(m.layers)]
    for r in range(rows):
        for t in (0, lens[r] - 1):
            seen = [(k[r, :, :t + 1], v[r, :, :t + 1]) for k, v in caches]
            want, own = walk.step(prompts[r][t], t, seen)
            check_own(own, [(k[r], v[r]) for k, v in caches], t)
        assert close(z[r], want), r
    # a second block of the prompt, then steps, an eviction and more steps
    pos, used = lens.copy(), lens.copy()

    def place():
        m.pos.copy_(torch.from_numpy(pos.astype(np.int32)))
        m.used.copy_(torch.from_numpy(used.astype(np.int32)))
        torch.cuda.synchronize()

    place()
    more = rng.integers(0, QWEN["vocab"], (rows, 3))
    m.prefill_async(torch.from_numpy(more.ravel().astype(np.int32)).cuda(), [3] * rows)
    pos, used = pos + 3, used + 3
    for phase in ("before", "after"):
        for _ in range(3):
            ids = rng.integers(0, QWEN["vocab"], rows)
            place()
            m.tokens.copy_(torch.from_numpy(ids.astype(np.int32)))
            torch.cuda.synchronize()
            m.feed_async(int(pos.max()))
            fh.sync()
            z = m.z.cpu().numpy()
            caches = [read(m, i) for i in range(m.layers)]
            for r in range(rows):
                seen = [(k[r, :, :used[r] + 1], v[r, :, :used[r] + 1]) for k, v in caches]
                want, own = walk.step(ids[r], pos[r], seen)
                check_own(own, [(k[r], v[r]) for k, v in caches], used[r])
                assert close(z[r], want), (phase, r)
            pos, used = pos + 1, used + 1
        if phase == "before":
            place()
            weights = [b["k"].planes["weight"].cpu().numpy() for b in m.blocks]
            for i, wt in enumerate(weights):  # every query gave each kv head its group's weight, 1 a head
                for r in range(rows):
                    assert np.allclose(wt[r, :, :used[r]].sum(axis=1), used[r] * 2, rtol=1e-4)
            m.evict_async(16, 4)
            fh.sync()
            used = np.minimum(used, 16)
            assert np.array_equal(m.used.cpu().numpy(), used)
            for i, b in enumerate(m.blocks):
                p = b["k"].planes["pos"].cpu().numpy()
                for r in range(rows):
                    for h in range(m.nkv):
                        kept = p[r, h, :used[r]]
                        assert (np.diff(kept) > 0).all() and kept[-1] == pos[r] - 1
                        if pos[r] > 16:
                            heavy = set(np.argsort(-weights[i][r, h, :pos[r] - 4], kind="stable")[:12])
                            assert set(kept[:-4]) == heavy
    m.free()


def test_forward_one_over_a_4_bit_cache_evicts_and_goes_on(fh, orc):
    import ferrum_hip

    cfg = dict(QWEN, context=16, kv="q4", kv_tracked=True)
    w = make_weights(orc, QWEN, 4, True, True)
    walk = Walk(orc, w, QWEN)
    m = ferrum_hip.LlamaDevice.from_weights(fh, w, cfg, 1)
    ids = np.random.default_rng(1).integers(0, QWEN["vocab"], 24)
    used = 0
    for pos, t in enumerate(ids):
        if used == 16:
            with pytest.raises(ferrum_hip.DimMismatch, match="KvCache full"):
                m.forward_one(int(t))
            m.evict_async(10, 3)
            used = 10
        z = m.forward_one(int(t))
        seen = [tuple(a[0, :, :used + 1] for a in read(m, i)) for i in range(m.layers)]
        assert close(z, walk.step(t, pos, seen)[0]), pos
        used += 1
    m.free()


def test_refusals(fh, orc):
    import ferrum_hip as F
    import torch

    with pytest.raises(F.FerrumHipError, match="head width 32, 64 or 128"):
        F.LlamaDevice(fh, dict(LLAMA, kv="q4"), 1)
    with pytest.raises(F.FerrumHipError, match="cache type"):
        F.LlamaDevice(fh, dict(QWEN, kv="q5"), 1)
    m = F.LlamaDevice(fh, QWEN, 2)
    tokens = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(F.FerrumHipError, match="needs the 4-bit cache"):
        m.prefill_async(tokens, [2, 2])
    with pytest.raises(F.FerrumHipError, match="needs a tracked"):
        m.evict_async(4, 1)
    m = F.LlamaDevice(fh, dict(QWEN, kv="q4"), 2)
    with pytest.raises(F.FerrumHipError, match="needs a tracked"):
        m.evict_async(4, 1)
    for lens, what in (([4], "2 lengths"), ([4, 0], "2 lengths"), ([2, 1], "4 tokens for 3")):
        with pytest.raises(F.FerrumHipError, match=what):
            m.prefill_async(tokens, lens)
    m.used.fill_(QWEN["context"] - 1)
    with pytest.raises(F.DimMismatch, match="KvCache full"):
        m.prefill_async(tokens, [2, 2])
