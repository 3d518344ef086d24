"""Calls of the Python binding that it refuses, with tensors on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32, device="cuda")


def test_fewer_masks_than_rows(rt):
    """Without mask_row every row has a mask of its own, so a mask without rows is one too few."""
    logits, starts = torch.ones((2, 40), device="cuda"), i32(2)
    for masks in (0, 1):
        with pytest.raises((ValueError, rt.RtHipError)):
            rt.adjust_logits(logits, starts, rt.LogitRules(mask=i32(masks, 2)))
    rt.adjust_logits(logits[:0], starts, rt.LogitRules(mask=i32(0, 2)))
    rt.adjust_logits(logits, starts, rt.LogitRules(mask=i32(0, 2), mask_row=i32(2) - 1))
    assert (logits == 1).all()
