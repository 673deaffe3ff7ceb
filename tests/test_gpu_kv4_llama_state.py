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
