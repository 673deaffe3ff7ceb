"""What LlamaDevice keeps between verify_async and accept_async, on the CPU: the calls into the
library are recorded, not made."""
import gc
import types
import weakref

import pytest

torch = pytest.importorskip("torch")

import ferrum_hip as F  # noqa: E402

CALLS = ("embed_rows_async", "rmsnorm_async", "linear_forward_async", "swiglu_async", "gqa_attention_rope_tree_async",
         "gqa_attention_rope_prefill_async", "tree_accept_async", "gqa_attention_decode_async", "rope_async")


class Ctx:
    def __init__(self, calls):
        self.calls = calls

    def sync(self):
        self.calls.append(("sync", ()))


@pytest.fixture
def model(monkeypatch):
    """rows, device -> a LlamaDevice without weights; its calls gather in m.calls."""
    calls = []
    for name in CALLS:
        monkeypatch.setattr(F, name, lambda *a, _n=name, **k: calls.append((_n, a)))
    waits = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a, **k: waits.append(a))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a, **k: types.SimpleNamespace(synchronize=lambda: None))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(F.LlamaDevice, "_ids", lambda *a: None)
    empty = torch.empty

    def make(rows, device="cpu", vocab=64):
        cfg = dict(vocab=vocab, d=8, n_heads=2, n_kv=1, head_dim=8, layers=1, ffn=16, context=64)
        with monkeypatch.context() as patch:
            patch.setattr(torch, "device", lambda *a: device)
            m = F.LlamaDevice(Ctx(calls), cfg, rows)
        m.blocks = [dict.fromkeys(("qkv", "qkv_b", "o", "gate_up", "down", "attn_norm", "ffn_norm"),) |
                    {"k": empty(8, device=device), "v": empty(8, device=device), "glu": False}]
        m.head = m.tok_w = m.out_norm = None
        m.calls, m.waits = calls, waits
        return m

    return make


def ids(rows, n):
    return torch.zeros((rows, n), dtype=torch.int32)


def test_trees_of_every_size_share_one_set_of_buffers(model):
    m = model(2)
    seen = {}
    for n in list(range(1, 65)) + list(range(64, 0, -1)):
        m.verify_async(ids(2, n), ids(2, n), n, 0)
        assert m.zt.shape == (2 * n, 64) and m.zt.is_contiguous()
        m.accept_async(ids(2, n))
        assert m.path.shape == (2, n) and m.count.shape == (2,)
        seen[m.zt.untyped_storage().data_ptr()] = m.zt.untyped_storage().nbytes()
    # sets that were grown out of stay (a captured graph may hold them): no more than the last one again
    assert sum(seen.values()) <= 2 * max(seen.values())
    assert max(seen.values()) <= 2 * 2 * 64 * 64 * 4
    last = m.zt.untyped_storage().data_ptr()
    m.verify_async(ids(2, 33), ids(2, 33), 33, 0)
    assert m.zt.untyped_storage().data_ptr() == last


def test_a_first_tree_has_what_it_needs_and_no_more(model):
    m = model(2)
    m.verify_async(ids(2, 5), ids(2, 5), 5, 0)
    assert m.zt.untyped_storage().nbytes() == 2 * 5 * 64 * 4
    m.verify_async(ids(2, 1024), ids(2, 1024), 1024, 0)
    assert m.zt.untyped_storage().nbytes() == 2 * 1024 * 64 * 4


def test_inputs_live_until_the_device_has_been_waited_for(model, monkeypatch):
    m = model(2)
    alive = []

    def step():
        given = [ids(2, 4) for _ in range(3)]
        alive.extend(weakref.ref(t) for t in given)
        m.verify_async(given[0], given[1], 4, 0)
        m.accept_async(given[2])

    step()
    m.waits.clear()  # (the buffers')
    for _ in range(20):
        step()
    m.calls.clear()
    gc.collect()
    assert not m.waits and all(r() is not None for r in alive)
    for _ in range(500):
        step()
        m.calls.clear()
    gc.collect()
    # not for ever: what was kept goes when the device has been waited for
    assert m.waits and sum(r() is not None for r in alive) <= 3 * 64
    before = len(m.waits)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for _ in range(100):  # (in a capture nothing waits)
        step()
    assert len(m.waits) == before


def test_a_tree_that_is_verified_again_keeps_the_first_ones_inputs(model):
    m = model(1)
    first = ids(1, 4)
    ref = weakref.ref(first)
    m.verify_async(first, ids(1, 4), 4, 0)
    del first
    m.verify_async(ids(1, 4), ids(1, 4), 4, 0)
    m.calls.clear()
    gc.collect()
    assert ref() is not None


@pytest.mark.parametrize("between", ["reset", "forward_one", "prompt_async"])
def test_what_moves_the_rows_ends_a_verified_tree(model, between, monkeypatch):
    m = model(1)
    m.z = torch.zeros((1, 64))
    m.verify_async(ids(1, 4), ids(1, 4), 4, 0)
    if between == "reset":
        m.reset()
    elif between == "forward_one":
        m.forward_one(3)
    else:
        monkeypatch.setattr(torch.Tensor, "cuda", lambda t: t)
        m.prompt_async(ids(1, 4), [4])
    with pytest.raises(F.FerrumHipError, match="follows verify_async"):
        m.accept_async(ids(1, 4))


def test_buffers_lie_on_the_models_device(model):
    """(meta stands for a device that is not the current one)"""
    m = model(2, device="meta")
    m.verify_async(ids(2, 4), ids(2, 4), 4, 0)
    assert m.zt.device.type == "meta"
    for name, args in m.calls:
        for t in args:
            if isinstance(t, torch.Tensor) and t.dtype == torch.float32:
                assert t.device.type == "meta", name


def test_a_prompts_buffers_lie_on_the_models_device(model):
    m = model(2)
    m.z = torch.zeros((2, 64))
    m.prompt_async(ids(1, 5), [2, 3])
    tensors = [t for _, args in m.calls for t in args if isinstance(t, torch.Tensor)]
    assert len(tensors) > 20 and all(t.device.type == "cpu" for t in tensors)


@pytest.mark.parametrize("where", ["gqa_attention_rope_prefill_async", "swiglu_async"])
def test_a_prompt_that_a_block_refuses_waits_for_what_runs(model, monkeypatch, where):
    """(its buffers go back to torch when it ends)"""
    m = model(2)
    m.z = torch.zeros((2, 64))

    def refuse(*a):
        raise F.FerrumHipError(F.FH_ERR_LIMIT, "no")

    monkeypatch.setattr(F, where, refuse)
    with pytest.raises(F.FerrumHipError, match="no"):
        m.prompt_async(ids(1, 5), [2, 3])
    names = [name for name, _ in m.calls]
    assert "embed_rows_async" in names and names[-1] == "sync"


def test_a_model_made_in_inference_mode_sees_what_is_written(model):
    with torch.inference_mode():
        m = model(1)
        m.z = torch.zeros((1, 64))
        m.forward_one(5)
        m.pos.fill_(7)
        m.verify_async(ids(1, 2), ids(1, 2), 2, 9)
        assert m.pos.tolist() == [7]
        m.next_pos = 3
        m.verify_async(ids(1, 2), ids(1, 2), 2, 9)
        assert m.pos.tolist() == [3]


def test_a_prompt_that_does_not_fit_leaves_the_place(model):
    """forward_one's place is the program's to step by, also behind a prompt that was refused."""
    m = model(1)
    m.z = torch.zeros((1, 64))
    for t in range(60):
        m.forward_one(t)
    with pytest.raises(F.DimMismatch, match="KvCache full"):
        m.prompt_async(ids(1, 5), [5])  # (4 places are left)
    assert m.pos.tolist() == [59] and m.next_pos == 60
    m.prompt_async(ids(1, 4), [4])
    assert m.pos.tolist() == [60]
    prompts = [args for name, args in m.calls if name == "gqa_attention_rope_prefill_async"]
    assert len(prompts) == 1 and prompts[0][14] == 64  # (max_keys)
