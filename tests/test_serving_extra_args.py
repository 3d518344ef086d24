"""Arguments that adjust_logits and lora_add refuse: a status and a message, before
anything reaches the device (no GPU needed)."""
import ctypes as C

import pytest

from conftest import load_package

ARG, SHAPE, ALIGN, UNSUPPORTED = 1, 2, 3, 6


@pytest.fixture(scope="module")
def rt():
    return load_package().rt_hip


@pytest.fixture(scope="module")
def mem():
    """Addresses of 24 separate, 16-byte aligned pieces of 4096 bytes."""
    buf = C.create_string_buffer(24 * 4096 + 64)
    base = (C.addressof(buf) + 63) & ~63
    yield [base + 4096 * i for i in range(24)]
    del buf


def rules(rt, m, **over):
    a = dict(history=m[3], history_cols=16, history_len=m[4], prompt_len=m[5], repetition=m[6], presence=m[7], frequency=m[8],
             bias_start=m[9], bias_token=m[10], bias=m[11], mask=m[12], mask_stride=2, mask_row=m[13], n_bias=5, n_masks=3)
    a.update(over)
    return C.byref(rt.LogitRulesStruct(**a))


def adjust(rt, m, **over):
    a = dict(logits=m[0], stride=50, dtype=rt.F32, vocab=50, row_start=m[1], n_seq=2, n_rows=6, tokens=m[2],
             rules=rules(rt, m))
    a.update(over)
    return rt.library().status("rt_hip_adjust_logits", *a.values(), None)


def adapters(rt, m, **over):
    a = dict(a=m[5], b=m[6], scale=m[7], dtype=rt.BF16, n_adapters=2, rank=8, k=64, n=48)
    a.update(over)
    return C.byref(rt.LoraStruct(**a))


def lora(rt, m, **over):
    a = dict(y=m[0], y_stride=48, x=m[1], x_dtype=rt.F32, x_stride=64, lora=adapters(rt, m), row_start=m[2], adapter=m[3],
             n_seq=2, n_rows=4)
    a.update(over)
    return rt.library().status("rt_hip_lora_add", *a.values(), None)


@pytest.mark.parametrize("over, code", [
    (dict(dtype=6), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED), (dict(rules=None), ARG), (dict(vocab=0), ARG),
    (dict(vocab=(1 << 20) + 1, stride=1 << 21), SHAPE), (dict(n_seq=-1), ARG), (dict(n_seq=4097), SHAPE), (dict(n_rows=-1), ARG),
    (dict(logits=None), ARG), (dict(row_start=None), ARG), (dict(stride=49), ARG), (dict(stride=1 << 46), SHAPE)])
def test_adjust_refuses(rt, mem, over, code):
    assert adjust(rt, mem, **over) == code
    assert b"rt_hip_adjust_logits" in rt.library().lib.rt_hip_last_error()


@pytest.mark.parametrize("over, code", [
    (dict(history_len=None), ARG), (dict(history_cols=0), ARG), (dict(history_cols=1 << 30), SHAPE), (dict(bias_start=None), ARG),
    (dict(bias_token=None), ARG), (dict(n_bias=-1), ARG), (dict(n_masks=-1), ARG), (dict(mask_stride=1), ARG),
    (dict(mask_row=None), ARG), (dict(mask_stride=1 << 46), SHAPE)])
def test_rules_refused(rt, mem, over, code):
    assert adjust(rt, mem, rules=rules(rt, mem, **over)) == code


def test_adjust_refuses_overlap(rt, mem):
    for name in ("history", "history_len", "prompt_len", "repetition", "presence", "frequency", "bias_start", "bias_token",
                 "bias", "mask", "mask_row"):
        assert adjust(rt, mem, rules=rules(rt, mem, **{name: mem[0] + 4})) == ARG, name
    assert adjust(rt, mem, tokens=mem[0] + 1196) == ARG
    assert adjust(rt, mem, row_start=mem[0]) == ARG
    assert adjust(rt, mem, logits=mem[0] + 2) == ALIGN
    assert adjust(rt, mem, n_seq=0) == 0
    assert adjust(rt, mem, n_rows=0, logits=None) == 0


@pytest.mark.parametrize("over, code", [
    (dict(y=None), ARG), (dict(x=None), ARG), (dict(lora=None), ARG), (dict(row_start=None), ARG), (dict(adapter=None), ARG),
    (dict(x_dtype=2), UNSUPPORTED), (dict(x_dtype=7), UNSUPPORTED), (dict(y_stride=47), ARG), (dict(x_stride=63), ARG),
    (dict(x_stride=66), ALIGN), (dict(n_seq=-1), ARG), (dict(n_seq=4097), SHAPE), (dict(n_rows=-1), ARG),
    (dict(n_rows=(1 << 24) + 1), SHAPE), (dict(y_stride=1 << 46), SHAPE)])
def test_lora_refuses(rt, mem, over, code):
    assert lora(rt, mem, **over) == code
    assert b"rt_hip_lora_add" in rt.library().lib.rt_hip_last_error()


@pytest.mark.parametrize("over, code", [
    (dict(a=None), ARG), (dict(b=None), ARG), (dict(scale=None), ARG), (dict(dtype=0), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED),
    (dict(n_adapters=-1), ARG), (dict(rank=0), SHAPE), (dict(rank=136), SHAPE), (dict(rank=12), ALIGN), (dict(k=60), ALIGN),
    (dict(k=0), SHAPE), (dict(n=0), SHAPE), (dict(n=(1 << 20) + 1), SHAPE)])
def test_adapters_refused(rt, mem, over, code):
    assert lora(rt, mem, lora=adapters(rt, mem, **over)) == code
    if code != ARG:
        assert rt.library().lib.rt_hip_lora_workspace_bytes(adapters(rt, mem, **over), 2, 4) == -1


def test_lora_refuses_overlap(rt, mem):
    assert lora(rt, mem, y=mem[1]) == ARG
    assert lora(rt, mem, lora=adapters(rt, mem, a=mem[0] + 16)) == ARG
    assert lora(rt, mem, lora=adapters(rt, mem, b=mem[0] + 752)) == ARG
    assert lora(rt, mem, adapter=mem[0]) == ARG
    assert lora(rt, mem, x=mem[1] + 8) == ALIGN
    assert lora(rt, mem, lora=adapters(rt, mem, a=mem[5] + 8)) == ALIGN
    assert lora(rt, mem, y=mem[0] + 2) == ALIGN
    assert lora(rt, mem, n_rows=0, x=None, y=None) == 0
    assert lora(rt, mem, n_seq=0) == 0
    assert lora(rt, mem, lora=adapters(rt, mem, n_adapters=0)) == 0


def test_binding_checks_before_it_calls(rt):
    torch = pytest.importorskip("torch")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        rt.LogitRules(repetition=torch.ones(2))
    with pytest.raises(ValueError, match="history_len"):
        rt.LogitRules(history=i32(2, 4))
    with pytest.raises(ValueError, match="bias_start"):
        rt.LogitRules(bias=torch.ones(2))
    with pytest.raises(ValueError, match="mask_row needs mask"):
        rt.LogitRules(mask_row=i32(2))
    with pytest.raises(ValueError, match="GPU"):
        rt.adjust_logits(torch.zeros(2, 8), i32(2), rt.LogitRules())
    a, b = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 48, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        rt.Adapters(a, b, torch.ones(2))
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        rt.Adapters(a.float(), b.float(), torch.ones(2))
