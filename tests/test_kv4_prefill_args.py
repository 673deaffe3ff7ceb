"""What LlamaDevice.prefill_async refuses before it touches a device."""
import pytest


def device(F, rows=2):
    m = object.__new__(F.LlamaDevice)
    m.rows, m.kv, m.d = rows, "q4", 128
    m.ctx = None  # (a call that goes on ends here)
    return m


@pytest.mark.parametrize("dtype,cuda,step,what", [("int64", True, 1, "int32"), ("int16", True, 1, "int32"),
                                                   ("float32", True, 1, "int32"), ("int32", False, 1, "on the device"),
                                                   ("int32", True, 2, "side by side")])
def test_ids_that_the_kernels_cannot_read(dtype, cuda, step, what):
    torch = pytest.importorskip("torch")
    import ferrum_hip as F

    class Ids(torch.Tensor):  # (says it is on the GPU)
        is_cuda = cuda

    tokens = torch.zeros(4 * step, dtype=getattr(torch, dtype))[::step].as_subclass(Ids)
    with pytest.raises(F.FerrumHipError, match=what) as e:
        device(F).prefill_async(tokens, [3, 1])
    assert e.value.code == F.FH_ERR_INVALID


def test_ids_that_are_no_tensor():
    import ferrum_hip as F

    for tokens in ([1, 2, 3, 4], None, 0):
        with pytest.raises(F.FerrumHipError, match="int32"):
            device(F).prefill_async(tokens, [3, 1])
