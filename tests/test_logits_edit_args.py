"""How many masks a LogitsEdit has (CPU: nothing here launches a kernel)."""
import pytest


def test_masks_are_counted_from_the_tensor():
    torch = pytest.importorskip("torch")
    import ferrum_hip as F

    mask = torch.zeros((3, 5), dtype=torch.int32)
    assert F.LogitsEdit(mask=mask).masks == 3
    assert F.LogitsEdit(mask=mask, masks=2).masks == 2
    assert F.LogitsEdit(mask=mask, masks=0).masks == 0
    assert F.LogitsEdit().masks == 0 and not F.LogitsEdit().mask
    assert F.LogitsEdit(mask=mask.numpy()).masks == 3


def test_masks_that_cannot_be_counted_are_refused():
    torch = pytest.importorskip("torch")
    import ferrum_hip as F

    for mask in (torch.zeros(15, dtype=torch.int32), 4096):
        with pytest.raises(F.FerrumHipError, match="masks") as e:
            F.LogitsEdit(mask=mask)
        assert e.value.code == F.FH_ERR_INVALID
        assert F.LogitsEdit(mask=mask, masks=1).masks == 1
