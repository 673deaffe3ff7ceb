"""LlamaDevice over 4-bit caches: what forward_one, prefill_async and evict_async
leave to each other, and restarts."""
import numpy as np
import pytest

from llama_tiny import QWEN, make_weights
from test_gpu_kv4_llama import Walk, close, read

pytestmark = pytest.mark.gpu


def positions(m, rows):
    """Positions of the first `rows` cache rows, [layers, n_kv, rows]."""
    return np.stack([b["k"].planes["pos"].cpu().numpy()[0, :, :rows] for b in m.blocks])


def test_eviction_after_forward_one_keeps_the_newest_rows(fh, orc):
    """The row of the last token that forward_one fed is among the recent ones, at every length."""
    import ferrum_hip

    m = ferrum_hip.LlamaDevice.from_weights(fh, make_weights(orc, QWEN, 4, True, True),
                                            dict(QWEN, context=16, kv="q4", kv_tracked=True), 1)
    ids = np.random.default_rng(1).integers(0, QWEN["vocab"], 40)
    used = 0
    for pos, t in enumerate(ids):
        m.forward_one(int(t))
        used += 1
        if used == 16 or pos == 3:
            m.evict_async(10, 3)
            fh.sync()
            used = min(used, 10)
            assert m.used.cpu().tolist() == [used]
            kept = positions(m, used)
            assert (np.diff(kept, axis=2) > 0).all()
            assert (kept[:, :, -3:] == np.arange(pos - 2, pos + 1)).all(), pos
    m.free()


def run(m, ids):
    return [m.forward_one(int(t)) for t in ids]


@pytest.mark.parametrize("how", ["next_pos", "reset"])
@pytest.mark.parametrize("first", [5, 16, 30])  # (a few tokens, a full cache, one that has been cut)
def test_a_second_text_is_as_on_a_fresh_device(fh, orc, how, first):
    import ferrum_hip

    cfg, w = dict(QWEN, context=16, kv="q4", kv_tracked=True), make_weights(orc, QWEN, 4, True, True)
    rng = np.random.default_rng(2)
    one, two = rng.integers(0, QWEN["vocab"], first), rng.integers(0, QWEN["vocab"], 12)
    m = ferrum_hip.LlamaDevice.from_weights(fh, w, cfg, 1)
    for t in one:
        if m.next_used == 16:
            m.evict_async(9, 2)
        m.forward_one(int(t))
    if how == "reset":
        m.reset()
    else:
        m.next_pos = 0
    assert (m.next_pos, m.next_used) == (0, 0) and m.used.cpu().tolist() == m.pos.cpu().tolist() == [0]
    got = run(m, two)
    fresh = ferrum_hip.LlamaDevice.from_weights(fh, w, cfg, 1)
    assert np.array_equal(got, run(fresh, two)) and np.isfinite(got).all()
    m.free()
    fresh.free()


def test_going_back_feeds_the_same_rows_again(fh, orc):
    """next_pos moved back takes next_used with it, until rows have been evicted: then only with next_used."""
    import ferrum_hip

    cfg, w = dict(QWEN, context=16, kv="q4", kv_tracked=True), make_weights(orc, QWEN, 4, True, True)
    ids = np.random.default_rng(3).integers(0, QWEN["vocab"], 16)
    m = ferrum_hip.LlamaDevice.from_weights(fh, w, cfg, 1)
    z = run(m, ids)
    m.next_pos = 9
    assert m.next_used == 9
    assert np.array_equal(run(m, ids[9:]), z[9:])
    m.evict_async(10, 5)
    assert (m.next_pos, m.next_used) == (16, 10)
    with pytest.raises(ferrum_hip.FerrumHipError, match="set next_used"):
        m.next_pos = 14
    want = m.forward_one(7)
    m.next_used = 10
    m.next_pos = 16
    assert (m.next_pos, m.next_used) == (16, 10)
    assert np.array_equal(m.forward_one(7), want)
    m.free()


def test_forward_one_goes_on_behind_a_prompt_and_an_eviction(fh, orc):
    """A prompt at once, its place handed on by next_pos alone, tokens, an eviction, a second prompt:
    each result against a float64 walk over the device's own caches."""
    import ferrum_hip
    import torch

    cfg, w = dict(QWEN, context=24, kv="q4", kv_tracked=True), make_weights(orc, QWEN, 4, True, True)
    walk = Walk(orc, w, QWEN)
    m = ferrum_hip.LlamaDevice.from_weights(fh, w, cfg, 1)
    ids = np.random.default_rng(5).integers(0, QWEN["vocab"], 60).astype(np.int32)
    pos = used = 0

    def check(z):
        seen = [tuple(a[0, :, :used] for a in read(m, i)) for i in range(m.layers)]
        assert close(z, walk.step(ids[pos - 1], pos - 1, seen)[0]), pos

    for prompt, tokens in ((11, 6), (5, 4)):
        m.prefill_async(torch.from_numpy(ids[pos:pos + prompt]).cuda(), [prompt])
        pos, used = pos + prompt, used + prompt
        m.next_pos = pos
        assert m.next_used == used
        fh.sync()
        check(m.z[0].cpu().numpy())
        for _ in range(tokens):
            z = m.forward_one(int(ids[pos]))
            pos, used = pos + 1, used + 1
            check(z)
        m.evict_async(12, 4)
        fh.sync()
        used = min(used, 12)
        assert m.next_used == used and (positions(m, used)[:, :, -4:] == np.arange(pos - 4, pos)).all()
    m.free()


def test_cache_rows_beyond_the_position(fh, orc):
    """Rows whose texts' positions start again behind other rows: feed_async is told how many there are."""
    import ferrum_hip
    import torch

    w = make_weights(orc, QWEN, 4, True, True)
    walk = Walk(orc, w, QWEN)
    m = ferrum_hip.LlamaDevice.from_weights(fh, w, dict(QWEN, kv="q4"), 3)
    lens, pos = np.array([20, 1, 37]), np.array([3, 0, 2])
    ids = np.random.default_rng(6).integers(0, QWEN["vocab"], lens.sum() + 3).astype(np.int32)
    m.prefill_async(torch.from_numpy(ids[:-3]).cuda(), lens)
    fh.sync()
    m.pos.copy_(torch.from_numpy(pos.astype(np.int32)))
    m.used.copy_(torch.from_numpy(lens.astype(np.int32)))
    m.tokens.copy_(torch.from_numpy(ids[-3:]))
    torch.cuda.synchronize()
    m.feed_async(int(pos.max()), int(lens.max()))
    fh.sync()
    z = m.z.cpu().numpy()
    caches = [read(m, i) for i in range(m.layers)]
    for r in range(3):
        seen = [(k[r, :, :lens[r] + 1], v[r, :, :lens[r] + 1]) for k, v in caches]
        assert close(z[r], walk.step(ids[-3 + r], pos[r], seen)[0]), r
    m.free()


def test_prefill_takes_32_bit_ids_only(fh):
    """torch's own ids are 64-bit: read as pairs of 32 they would be others."""
    import ferrum_hip
    import torch

    m = ferrum_hip.LlamaDevice(fh, dict(QWEN, kv="q4"), 2)
    ids = torch.randint(0, QWEN["vocab"], (5,), device="cuda")
    for tokens, what in ((ids, "int32 tensor, not torch.int64"), (ids.int().cpu(), "on the model's device"),
                         (ids.int().repeat(2)[::2], "side by side")):
        with pytest.raises(ferrum_hip.FerrumHipError, match=what):
            m.prefill_async(tokens, [3, 2])


@pytest.mark.parametrize("kv", ["f32", "q4"])
def test_reset_clears_every_row(fh, kv):
    import ferrum_hip

    m = ferrum_hip.LlamaDevice(fh, dict(QWEN, kv=kv), 3)
    for t in [m.pos] + ([m.used] if kv == "q4" else []):
        t.fill_(7)
    m.next_pos = 5
    assert m.pos.cpu().tolist() == [7, 7, 7]  # (several rows' counters are the caller's)
    m.reset()
    assert m.next_pos == 0 and m.pos.cpu().tolist() == [0, 0, 0]
    if kv == "q4":
        assert m.next_used == 0 and m.used.cpu().tolist() == [0, 0, 0]
    for name in ("next_pos", "next_used"):
        with pytest.raises(ferrum_hip.FerrumHipError, match="no position"):
            setattr(m, name, -1)
    assert (m.next_pos, m.next_used) == (0, 0)
