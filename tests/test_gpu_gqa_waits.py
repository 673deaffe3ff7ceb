"""Calls on the context's own stream whose outputs torch's stream fills first, with a wait between
the two streams: nothing of the fill is left, and the same bits come again."""
import numpy as np
import pytest

import gqa_ref as ref
from llama_tiny import QWEN, make_weights
from test_gpu_gqa_rows import Call, gpu, ints, trees
from test_gpu_tree_accept import draft

pytestmark = pytest.mark.gpu


def wait():
    import torch

    torch.cuda.synchronize()


@pytest.mark.parametrize("tree", [False, True])
def test_the_same_bits_again(fh, tree):
    news = [16, 9]
    a = Call((14, 2, 64), [3000, 100], news, 70, parents=trees(news, 71) if tree else None)
    one = a.run(fh).copy()
    for _ in range(3):
        a.out.fill_(55.0)
        wait()
        a.again(fh)
        fh.sync()
        np.testing.assert_array_equal(a.out.cpu().numpy().reshape(one.shape), one)


def test_equal_parts_without_offsets(fh):
    import ferrum_hip
    import torch

    a = Call((14, 2, 64), [0, 0, 0], [11, 11, 11], 72)
    want = a.run(fh)
    out = torch.full_like(a.out, 55.0)
    wait()
    ferrum_hip.gqa_attention_rope_prefill_async(fh, a.dqkv, a.ld, 33, 14, 2, 64, a.dk, a.dv, 3, a.cap, None, 0, None, a.cap, None,
                                                64, 10000.0, ferrum_hip.ROPE_NEOX, None, 1.0, out)
    fh.sync()
    np.testing.assert_array_equal(out.cpu().numpy().reshape(want.shape), want)


def test_accepted_in_equal_parts_without_lengths(fh):
    import ferrum_hip
    import torch

    rng = np.random.default_rng(73)
    drafts = [draft(12, rng, 0.8) for _ in range(3)]
    flat = [ints(np.concatenate([t[i] for t in drafts])) for i in range(3)]
    path = torch.full((36,), 9, dtype=torch.int32, device="cuda")
    count, nxt, ln = (torch.full((3,), 9, dtype=torch.int32, device="cuda") for _ in range(3))
    wait()
    ferrum_hip.tree_accept_async(fh, *flat, 36, None, 3, 0, None, None, 0, 0, 0, path, count, nxt, ln)
    fh.sync()
    for s, t in enumerate(drafts):
        way = ref.accept(*t)
        assert path[12 * s:12 * s + 12].tolist() == way + [-1] * (12 - len(way))
        assert int(ln[s]) == len(way) == int(count[s]) and int(nxt[s]) == t[2][way[-1]]


@pytest.mark.parametrize("vocab", [33, 2049, 50257])
def test_edits_leave_nothing_of_the_output(fh, vocab):
    import ferrum_hip
    import torch

    x = torch.randn((5, vocab), device="cuda")
    hist = torch.arange(0, 20, device="cuda", dtype=torch.int32)
    ranges, freq = ints([[0, 20]] * 5), torch.full((5,), 0.5, device="cuda")
    out = torch.full_like(x, 9.0)
    wait()
    ferrum_hip.logits_edit_async(fh, x, 5, vocab, ferrum_hip.LogitsEdit(recent=hist, ranges=ranges, frequency=freq), out)
    fh.sync()
    want = x.clone()
    want[:, :20] -= 0.5
    assert torch.equal(out, want)


def test_chosen_ids_from_torch(fh, orc):
    """The ids that the acceptance takes are torch's, waited for."""
    import ferrum_hip

    m = ferrum_hip.LlamaDevice.from_weights(fh, make_weights(orc, QWEN, 3, True, True), QWEN, 2)
    tokens, parents = ints([5, 6, 7, 8, 9, 10]), ints([-1, 0, 1] * 2)
    wait()
    m.verify_async(tokens, parents, 3, 0)
    fh.sync()
    chosen = m.zt.argmax(dim=1).int()
    want = chosen.cpu().numpy().reshape(2, 3)
    wait()
    m.accept_async(chosen)
    fh.sync()
    for r, tok in enumerate(([5, 6, 7], [8, 9, 10])):
        way = ref.accept([-1, 0, 1], tok, want[r])
        assert m.path[r].tolist() == way + [-1] * (3 - len(way)) and int(m.tokens[r]) == want[r][way[-1]]
    m.free()
