"""What LlamaDevice.prefill_async refuses before it touches a device."""
import pytest


def device(F, rows=2, place="cuda:0"):
    m = object.__new__(F.LlamaDevice)
    m.rows, m.kv, m.d = rows, "q4", 128
    m.ctx = None  # (a call that goes on ends here)
    m.used = device_tensor(place)
    return m


def device_tensor(place):
    import types

    return types.SimpleNamespace(device=place)


@pytest.mark.parametrize("dtype,place,step,what", [
    ("int64", "cuda:0", 1, "int32"), ("int16", "cuda:0", 1, "int32"), ("float32", "cuda:0", 1, "int32"),
    ("int32", "cpu", 1, "model's device"), ("int32", "cuda:1", 1, "model's device"), ("int32", "cuda:0", 2, "side by side")])
def test_ids_that_the_kernels_cannot_read(dtype, place, step, what):
    torch = pytest.importorskip("torch")
    import ferrum_hip as F

    class Ids(torch.Tensor):  # (says it is elsewhere)
        is_cuda, device = place != "cpu", place

    tokens = torch.zeros(4 * step, dtype=getattr(torch, dtype))[::step].as_subclass(Ids)
    with pytest.raises(F.FerrumHipError, match=what) as e:
        device(F).prefill_async(tokens, [3, 1])
    assert e.value.code == F.FH_ERR_INVALID


def test_ids_that_are_no_tensor():
    import ferrum_hip as F

    for tokens in ([1, 2, 3, 4], None, 0):
        with pytest.raises(F.FerrumHipError, match="int32"):
            device(F).prefill_async(tokens, [3, 1])
