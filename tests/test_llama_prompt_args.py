"""What LlamaDevice.prompt_async refuses before it touches a device, over either cache."""
import types

import pytest


def device(F, kv):
    m = object.__new__(F.LlamaDevice)
    m.rows, m.kv, m.d, m.ctx = 2, kv, 128, None  # (a call that goes on ends here)
    setattr(m, "used" if kv == "q4" else "pos", types.SimpleNamespace(device="cuda:0"))
    return m


@pytest.mark.parametrize("kv", ["f32", "q4"])
@pytest.mark.parametrize("dtype,place,step,what", [("int64", "cuda:0", 1, "int32"), ("int32", "cpu", 1, "model's device"),
                                                   ("int32", "cuda:1", 1, "model's device"), ("int32", "cuda:0", 2, "side by side")])
def test_ids_that_the_kernels_cannot_read(kv, dtype, place, step, what):
    torch = pytest.importorskip("torch")
    import ferrum_hip as F

    class Ids(torch.Tensor):  # (says it is elsewhere)
        is_cuda, device = place != "cpu", place

    tokens = torch.zeros(4 * step, dtype=getattr(torch, dtype))[::step].as_subclass(Ids)
    with pytest.raises(F.FerrumHipError, match=what) as e:
        device(F, kv).prompt_async(tokens, [3, 1])
    assert e.value.code == F.FH_ERR_INVALID and "prompt_async" in str(e.value)
