"""Where LlamaDevice goes on over f32 caches: forward_one and next_pos leave self.pos to the
program that steps by it, and prompts and trees of a single row go on where forward_one would."""
import numpy as np
import pytest

from test_gpu_llama_rows import build, close, ints
from llama_tiny import OracleLlamaRow

pytestmark = pytest.mark.gpu


def fed(orc, w, cfg, ids):
    oracle = OracleLlamaRow(orc, w, cfg)
    return [oracle.feed(int(t)) for t in ids]


def test_steps_behind_forward_one(fh, orc):
    """The stepping of a batch (self.pos plus one, feed_async) behind tokens that forward_one fed."""
    import torch

    cfg, w, m = build(fh, orc, "qwen", 1)
    ids = np.random.default_rng(50).integers(0, cfg["vocab"], 12)
    want = fed(orc, w, cfg, ids)
    for t in range(6):
        assert close(m.forward_one(int(ids[t])), want[t])
        assert m.pos.tolist() == [t]
    for t in range(6, 12):
        m.tokens.fill_(int(ids[t]))
        m.pos.add_(1)
        torch.cuda.synchronize()
        m.feed_async(t)
        fh.sync()
        assert close(m.z[0].cpu().numpy(), want[t]), t
    m.free()


def test_next_pos_leaves_the_place_of_steps(fh, orc):
    cfg, w, m = build(fh, orc, "llama", 1)
    ids = np.random.default_rng(51).integers(0, cfg["vocab"], 4)
    want = fed(orc, w, cfg, ids)
    m.pos.fill_(3)
    m.next_pos = 0
    assert m.pos.tolist() == [3] and m.next_pos == 0
    for t in range(3):
        assert close(m.forward_one(int(ids[t])), want[t])
    m.free()


@pytest.mark.parametrize("name", ["qwen", "wide"])
def test_trees_go_on_behind_forward_one(fh, orc, name):
    import torch

    cfg, w, m = build(fh, orc, name, 1)
    ids = np.random.default_rng(52).integers(0, cfg["vocab"], 14)
    want = fed(orc, w, cfg, ids)
    for t in range(8):
        m.forward_one(int(ids[t]))
    # row 0, a wrong draft, the right ones behind it
    tokens, parents = ints([ids[8], 7, ids[9], ids[10]]), ints([-1, 0, 0, 2])
    m.verify_async(tokens, parents, 4, 8)
    fh.sync()
    z = m.zt.cpu().numpy()
    for node, t in ((0, 8), (2, 9), (3, 10)):
        assert close(z[node], want[t]), node
    chosen = ints([ids[9], 1, ids[10], ids[11]])
    torch.cuda.synchronize()
    m.accept_async(chosen)
    fh.sync()
    assert m.pos.tolist() == [11] and m.tokens.tolist() == [ids[11]]
    # a second tree at the place that the first left
    tokens = ints([ids[11], ids[12]])
    parents = ints([-1, 0])
    torch.cuda.synchronize()
    m.verify_async(tokens, parents, 2, 11)
    fh.sync()
    assert close(m.zt[1].cpu().numpy(), want[12])
    m.next_pos = 11
    for t in range(11, 14):
        assert close(m.forward_one(int(ids[t])), want[t])
    m.free()


def test_prompts_go_on_behind_forward_one_and_next_pos(fh, orc):
    import torch

    cfg, w, m = build(fh, orc, "qwen", 1)
    ids = np.random.default_rng(53).integers(0, cfg["vocab"], 30)
    want = fed(orc, w, cfg, ids)
    for t in range(4):
        m.forward_one(int(ids[t]))
    m.prompt_async(ints(ids[4:10]), [6])
    fh.sync()
    assert close(m.z[0].cpu().numpy(), want[9])
    m.next_pos = 10
    m.prompt_async(ints(ids[10:20]), [10])
    fh.sync()
    assert close(m.z[0].cpu().numpy(), want[19])
    # back, over what was fed
    m.next_pos = 7
    m.prompt_async(ints(ids[7:20]), [13])
    fh.sync()
    assert close(m.z[0].cpu().numpy(), want[19])
    # a place that the program itself wrote counts, whatever forward_one fed before
    m.next_pos = 2
    m.forward_one(int(ids[2]))
    m.pos.fill_(20)
    torch.cuda.synchronize()
    m.prompt_async(ints(ids[20:29]), [9])
    fh.sync()
    want_behind = fed(orc, w, cfg, ids[:29])[28]
    assert close(m.z[0].cpu().numpy(), want_behind)
    m.free()


def test_a_place_that_a_graph_moved_counts(fh, orc):
    import torch

    cfg, w, m = build(fh, orc, "qwen", 1)
    ids = np.random.default_rng(54).integers(0, cfg["vocab"], 20)
    want = fed(orc, w, cfg, ids)
    m.forward_one(int(ids[0]))
    m.tokens.fill_(int(ids[1]))
    m.pos.fill_(1)
    torch.cuda.synchronize()
    m.feed_async(16)  # (the workspace is as large as it gets)
    fh.sync()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    fh.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            m.pos.add_(1)
            m.feed_async(16)
    finally:
        fh.set_stream(None)
    m.next_pos = 1
    m.forward_one(int(ids[1]))
    for t in range(2, 6):
        m.tokens.fill_(int(ids[t]))
        graph.replay()
        torch.cuda.synchronize()
        assert close(m.z[0].cpu().numpy(), want[t]), t
    assert m.pos.tolist() == [5]
    m.pos.add_(1)
    torch.cuda.synchronize()
    m.prompt_async(ints(ids[6:12]), [6])
    fh.sync()
    assert close(m.z[0].cpu().numpy(), want[11])
    m.free()


@pytest.mark.parametrize("how", ["forward_one", "next_pos"])
def test_a_place_that_replayed_trees_moved_counts(fh, orc, how):
    """A captured step of trees, replayed behind forward_one or next_pos: a prompt goes on where it left off."""
    import torch

    cfg, w, m = build(fh, orc, "qwen", 1)
    ids = np.random.default_rng(55).integers(0, cfg["vocab"], 24)
    want = fed(orc, w, cfg, ids)
    tokens, parents, chosen = ints([0, 0]), ints([-1, 0]), ints([0, 0])
    m.verify_async(tokens, parents, 2, 30)
    m.accept_async(chosen)
    fh.sync()
    m.reset()
    for t in range(4):
        m.forward_one(int(ids[t]))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    m.pos.fill_(4)
    torch.cuda.synchronize()
    fh.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            m.verify_async(tokens, parents, 2, 30)
            m.accept_async(chosen)
    finally:
        fh.set_stream(None)
    if how == "forward_one":
        m.next_pos = 3
        m.forward_one(int(ids[3]))
        m.pos.fill_(4)
    else:
        m.pos.fill_(4)
        torch.cuda.synchronize()
        m.next_pos = 2
    for t in (4, 6, 8):
        tokens.copy_(ints(ids[t:t + 2]))
        chosen.copy_(ints([ids[t + 1], ids[t + 2]]))
        graph.replay()
        torch.cuda.synchronize()
    assert m.pos.tolist() == [10]
    m.prompt_async(ints(ids[10:16]), [6])
    fh.sync()
    assert close(m.z[0].cpu().numpy(), want[15])
    m.free()


def test_a_capture_refuses_a_place_that_is_not_written(fh, orc):
    import ferrum_hip
    import torch

    cfg, w, m = build(fh, orc, "qwen", 1)
    ids = ints([1, 2])
    m.verify_async(ids, ints([-1, 0]), 2, 10)
    fh.sync()
    m.forward_one(3)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    fh.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            torch.zeros(1, device="cuda")
            with pytest.raises(ferrum_hip.FerrumHipError, match="before the capture"):
                m.verify_async(ids, ids, 2, 10)
    finally:
        fh.set_stream(None)
    m.free()
