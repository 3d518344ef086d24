"""Calls of the Python binding that it refuses, with tensors on the GPU."""
import pytest
import torch

from paged4 import filled

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


MANY = 2**32 + 1  # the call's 32 bits would take it as 1


def test_more_rows_than_32_bits(rt):
    # (rows of many tensors are one row's memory, where the strides may be anything)
    one = torch.zeros(64, dtype=torch.bfloat16, device="cuda")
    kv = filled(rt, 2, 16, 1, 64)
    slots = torch.empty(MANY, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        rt.paged_read(kv, slots)
    rows = one.as_strided((MANY, 1, 64), (0, 64, 1))
    for call in (lambda: rt.paged_append(kv, rows, rows, slots), lambda: rt.paged_read(kv, slots, out=(rows, rows)),
                 lambda: rt.paged_attention(rows, kv, i32(1, 1), i32(2), i32(1), 0.1, out=rows)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    logits = torch.empty((MANY, 1), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        rt.adjust_logits(logits, i32(2), rt.LogitRules())
    del logits
    with pytest.raises(ValueError, match="32 bits"):
        rt.adjust_logits(torch.ones((1, 40), device="cuda"), slots, rt.LogitRules())
    with pytest.raises(ValueError, match="32 bits"):
        rt.LogitRules(mask=slots[:, None])
    bias = slots.view(torch.float32)
    with pytest.raises(ValueError, match="32 bits"):
        rt.LogitRules(bias=bias, bias_token=slots, bias_start=i32(2))
    adapters = rt.Adapters(one.view(1, 8, 8), one[:8].view(1, 1, 8), torch.ones(1, device="cuda"))
    y, x = torch.zeros(1, device="cuda").expand(MANY, 1), one.as_strided((MANY, 8), (0, 1))
    with pytest.raises(ValueError, match="32 bits"):
        rt.lora_add(y, x, adapters, i32(2), i32(1))
    with pytest.raises(ValueError, match="32 bits"):
        rt.lora_add(y[:1], x[:1], adapters, slots, slots[1:])
