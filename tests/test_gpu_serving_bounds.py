"""Starts, lengths and numbers that are out of range: rows outside every request, and memory beside
the rows, keep their bits."""
import numpy as np
import pytest
import torch

import test_gpu_adjust_logits as adjust
import test_gpu_lora_add as lora
import test_gpu_paged4_attention as attention
from helpers import say

pytestmark = pytest.mark.gpu

INT_MAX, INT_MIN = 2**31 - 1, -(2**31)


def claimed(starts, rows):
    """Rows that the requests have, by the rule for starts that are out of range: each between 0 and rows, an end below
    its start none."""
    mine = np.zeros(rows, bool)
    for a, b in zip(starts, starts[1:]):
        a = min(max(a, 0), rows)
        mine[a:min(max(b, a), rows)] = True
    return mine


STARTS = [[5, 2, 10**9], [-4, -3, INT_MAX], [9, 100, INT_MAX], [INT_MAX, INT_MAX, INT_MAX], [INT_MIN, 1, 1], [3, 3, 4], [2, 0, 1]]


@pytest.mark.parametrize("q", attention.TYPES)
@pytest.mark.parametrize("n", [4, 70])
@pytest.mark.parametrize("starts", STARTS)
def test_attention4(rt, q, n, starts):
    say("bounds attention4", q, n, starts)
    step = attention.Step(rt, q, 4, 2, 128, 16, [(n, 200), (n, 333)], seed=9, byte=0, behind=3, joint=True)
    rows, heads = step.q.shape[:2]
    whole = torch.full((rows + 2, heads + 2, 128), -77.0, dtype=step.q.dtype, device="cuda")
    out = whole[1:-1].flatten(1)[:, :heads * 128].view(rows, heads, 128)  # (rows with something behind each)
    for lens in ([200, 333], [INT_MAX, -5], [0, 1], [INT_MIN, INT_MAX]):
        whole.fill_(-77.0)
        rt.paged_attention(step.q, step.kv, step.table, attention.i32(starts), attention.i32(lens), 0.1, out=out)
        mine = torch.from_numpy(claimed(starts, rows)).cuda()
        assert (out[~mine] == -77.0).all() and not (out[mine] == -77.0).any()
        whole[1:-1, :heads][mine] = -77.0
        assert (whole == -77.0).all()


@pytest.mark.parametrize("dtype", adjust.DTYPES)
@pytest.mark.parametrize("starts", STARTS)
def test_adjust_logits(rt, dtype, starts):
    say("bounds adjust", dtype, starts)
    c = adjust.Case(5000, [6, 2], dtype, seed=7, spread=300, pad=3)
    c.history_len, c.prompt_len = np.array([INT_MAX, 20]), np.array([INT_MIN, 5])
    c.history[:, ::7], c.tokens[2:4] = -1, [5000, INT_MAX]
    c.mask_row[::3] = [INT_MIN, 3, INT_MAX]
    bias_start = [[-4, 10**9, 2], [INT_MAX, INT_MIN, 3], list(c.bias_start)]
    for at in bias_start:
        before = c.store.clone()
        rt.adjust_logits(c.logits, adjust.i32(starts), c.rules(rt, bias_start=adjust.i32(at)), tokens=adjust.i32(c.tokens))
        mine = np.concatenate([claimed(starts, 8), [False, False]])
        bits = torch.int32 if dtype == torch.float32 else torch.int16
        changed = (c.store.view(bits) != before.view(bits)).cpu().numpy()
        assert not changed[~mine].any() and not changed[:, 5000:].any()
        assert changed[mine].any() == mine.any()


@pytest.mark.parametrize("x", list(lora.TYPES))
@pytest.mark.parametrize("starts", STARTS)
def test_lora_add(rt, x, starts):
    say("bounds lora", x, starts)
    for rows in ([4, 4], [70, 10]):
        c = lora.Case(rows, [0, 1], 2, 16, 64, 60, lora.TYPES[x], seed=1, y_pad=5, behind=3)
        total = c.y.shape[0]
        for adapter in ([0, 1], [1, -1], [2, INT_MAX], [INT_MIN, 0]):
            before = c.store.clone()
            rt.lora_add(c.y, c.x, rt.Adapters(c.a, c.b, c.scale), lora.i32(starts), lora.i32(adapter))
            # (a row that two requests claim is undefined, and none of these starts has one)
            mine = np.zeros(total, bool)
            for s, a in enumerate(adapter):
                if 0 <= a < 2:
                    mine |= claimed(starts[s:s + 2], total)
            same = (c.store == before).cpu().numpy()
            assert same[~mine].all() and same[:, 60:].all() and not same[mine, :60].all(1).any()
