"""A grammar mask given without its count masks (fh_logits_edit_async through LogitsEdit)."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_mask_without_its_count_is_applied(fh):
    import ferrum_hip
    import torch

    x = torch.randn((3, 70), device="cuda")
    mask = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    mask[0, 1] = 1 << 5  # id 37
    mask[1] = -1
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    ferrum_hip.logits_edit_async(fh, x, 3, 70, ferrum_hip.LogitsEdit(mask=mask), out)
    fh.sync()
    want = torch.full((70,), -torch.inf, device="cuda")
    want[37] = x[0, 37]
    assert torch.equal(out[0], want)
    assert torch.equal(out[1:], x[1:])  # mask 1 leaves every id, row 2 has none
