"""LlamaDevice over 4-bit caches at the head widths, rotations and files that the tiny
Qwen2 model does not have: prompts, steps, an eviction and more steps against the
float64 walk over the device's own caches."""
import numpy as np
import pytest

import llama_tiny
from test_gpu_kv4_llama import Walk, check_own, close, read

pytestmark = pytest.mark.gpu

BASE = dict(vocab=384, d=128, layers=2, ffn=192, context=64, rope_base=1e6, eps=1e-6)
MODELS = {  # (cfg, biases, tied)
    "neox64": (dict(BASE, n_heads=6, n_kv=2, head_dim=64, rope_type=1), True, True),
    "norm64": (dict(BASE, n_heads=4, n_kv=4, head_dim=64, rope_type=0, rope_dim=32), False, False),
    "neox128": (dict(BASE, n_heads=5, n_kv=1, head_dim=128, rope_type=1), True, False),
    "norm128": (dict(BASE, n_heads=4, n_kv=2, head_dim=128, rope_type=0), False, True),
    "scaled32": (dict(llama_tiny.QWEN, rope_linear=2.0), True, True),
}


class AnyRope(Walk):
    """Either rotation, of the first rope_dim channels, with linear scaling and frequency factors."""

    def rope(self, x, pos):
        c = self.c
        y = x.reshape(-1, c["head_dim"]).copy()
        rd = c.get("rope_dim", c["head_dim"])
        i = np.arange(rd // 2)
        ang = pos * c["rope_base"] ** (-2.0 * i / rd) / c.get("freqs", np.ones(rd // 2)) / c.get("rope_linear", 1.0)
        a, b = (i, i + rd // 2) if c["rope_type"] else (2 * i, 2 * i + 1)
        u, v = y[:, a].copy(), y[:, b].copy()
        y[:, a], y[:, b] = u * np.cos(ang) - v * np.sin(ang), u * np.sin(ang) + v * np.cos(ang)
        return y


def run(m, walk, cfg, seed):
    import torch

    rows, rng = m.rows, np.random.default_rng(seed)
    pos, used = np.zeros(rows, np.int64), np.zeros(rows, np.int64)

    def check(ids, what):
        """The last token of every row, at pos - 1 and cache row used - 1."""
        m.ctx.sync()
        z = m.z.cpu().numpy()
        caches = [read(m, i) for i in range(m.layers)]
        for r in range(rows):
            seen = [(k[r, :, :used[r]], v[r, :, :used[r]]) for k, v in caches]
            want, own = walk.step(ids[r], pos[r] - 1, seen)
            check_own(own, [(k[r], v[r]) for k, v in caches], used[r] - 1)
            assert close(z[r], want), (what, r)

    def place():
        m.pos.copy_(torch.from_numpy(pos.astype(np.int32)))
        m.used.copy_(torch.from_numpy(used.astype(np.int32)))
        torch.cuda.synchronize()

    for lens in (rng.integers(1, 34, rows), rng.integers(1, 5, rows)):
        prompts = [rng.integers(0, cfg["vocab"], n) for n in lens]
        place()
        m.prefill_async(torch.from_numpy(np.concatenate(prompts).astype(np.int32)).cuda(), lens)
        pos, used = pos + lens, used + lens
        check([p[-1] for p in prompts], "prompt")
    for phase in ("before", "after"):
        for _ in range(2):
            ids = rng.integers(0, cfg["vocab"], rows)
            place()
            m.tokens.copy_(torch.from_numpy(ids.astype(np.int32)))
            torch.cuda.synchronize()
            m.feed_async(int(pos.max()), int(used.max()))
            pos, used = pos + 1, used + 1
            check(ids, phase)
        if phase == "before":
            place()
            m.evict_async(12, 5)
            m.ctx.sync()
            used = np.minimum(used, 12)


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("name", sorted(MODELS))
def test_models_of_other_shapes(fh, orc, name, rows):
    import ferrum_hip

    cfg, biases, tied = MODELS[name]
    w = llama_tiny.make_weights(orc, cfg, 9, biases, tied)
    m = ferrum_hip.LlamaDevice.from_weights(fh, w, dict(cfg, kv="q4", kv_tracked=True), rows)
    run(m, AnyRope(orc, w, cfg), cfg, rows)
    m.free()


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("name,arch", [("norm64", "llama"), ("neox128", "qwen2")])
def test_files_over_4_bit_caches(fh, orc, tmp_path, name, arch, rows):
    import ferrum_hip
    from test_gpu_gguf_import import llama_path

    cfg, biases, tied = MODELS[name]
    w = llama_tiny.make_weights(orc, cfg, 10, biases, tied)
    m = ferrum_hip.LlamaDevice.from_gguf(fh, llama_path(tmp_path, w, cfg, arch), rows=rows, kv="q4", kv_tracked=True)
    assert m.kv == "q4" and m.tracked and m.hd == cfg["head_dim"] and m.cap == cfg["context"]
    run(m, AnyRope(orc, w, cfg), cfg, 20 + rows)
    m.free()


def test_a_file_with_f32_matrices_and_rope_scaling(fh, orc, tmp_path):
    import ferrum_gguf
    import ferrum_hip
    from test_gpu_gguf_import import llama_path

    cfg, biases, tied = MODELS["neox64"]
    w = llama_tiny.make_weights(orc, cfg, 11, biases, tied)
    freqs = np.random.default_rng(2).uniform(0.5, 4.0, cfg["head_dim"] // 2).astype(np.float32)

    def extra(b):
        b.str("qwen2.rope.scaling.type", "linear").f32("qwen2.rope.scaling.factor", 2.0)
        b.tensor("rope_freqs.weight", [cfg["head_dim"] // 2], ferrum_gguf.GGML_F32, freqs.tobytes())

    path = llama_path(tmp_path, w, cfg, "qwen2", f32_names=("token_embd", "blk.0.attn_k", "blk.1.ffn_down"), extra=extra)
    m = ferrum_hip.LlamaDevice.from_gguf(fh, path, rows=2, capacity=50, kv="q4", kv_tracked=True)
    assert m.head.is_f32 and m.blocks[0]["qkv"].is_f32 and m.rope_linear == 2.0 and m.cap == 50
    run(m, AnyRope(orc, w, dict(cfg, rope_linear=2.0, freqs=freqs)), cfg, 30)
    m.free()


@pytest.mark.parametrize("rows", [1, 4])
def test_a_captured_step_replays_as_it_runs(fh, orc, rows):
    """Tokens, positions and cache rows change on the device between replays; after an eviction the
    step is captured again."""
    import ferrum_hip
    import torch

    cfg, biases, tied = MODELS["neox64"]
    w = llama_tiny.make_weights(orc, cfg, 12, biases, tied)
    pair = [ferrum_hip.LlamaDevice.from_weights(fh, w, dict(cfg, kv="q4", kv_tracked=True), rows) for _ in range(2)]
    rng = np.random.default_rng(rows)
    ids = torch.from_numpy(rng.integers(0, cfg["vocab"], 20 * rows).astype(np.int32)).cuda()
    place = torch.full((rows,), 20, dtype=torch.int32, device="cuda")
    for m in pair:
        m.prefill_async(ids, [20] * rows)
        m.ctx.sync()
    for part in range(2):
        eager, other = pair
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        eager.pos.copy_(place)
        eager.used.copy_(place - 20 * part + (10 if part else 0))
        other.pos.copy_(eager.pos)
        other.used.copy_(eager.used)
        kept = [other.blocks[i]["k"].planes["weight"].clone() for i in range(other.layers)]
        torch.cuda.synchronize()
        other.feed_async(40)  # (workspaces; the row is fed again below)
        fh.sync()
        for i in range(other.layers):
            other.blocks[i]["k"].planes["weight"].copy_(kept[i])
        try:
            with torch.cuda.graph(g, stream=s):
                fh.set_stream(torch.cuda.current_stream().cuda_stream)
                other.feed_async(40)
        finally:
            fh.set_stream(None)
        for _ in range(5):
            tok = torch.from_numpy(rng.integers(0, cfg["vocab"], rows).astype(np.int32)).cuda()
            for m in pair:
                m.tokens.copy_(tok)
            torch.cuda.synchronize()
            eager.feed_async(40)
            fh.sync()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(eager.z, other.z) and torch.isfinite(other.z).all()
            for a, b in zip(eager.blocks, other.blocks):
                assert all(torch.equal(a["k"].planes[n], b["k"].planes[n]) for n in ("k", "v", "pos", "weight"))
            for m in pair:
                m.pos += 1
                m.used += 1
            place += 1
            torch.cuda.synchronize()
        del g
        for m in pair:
            m.evict_async(10, 4)
        fh.sync()
    for m in pair:
        m.free()
