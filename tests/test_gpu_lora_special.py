"""rt_hip_lora_add where a factor is an infinity, a NaN or next to float32's end: what the
definition gives in float64, infinity for infinity, and the other values as exact as ever
(tolerances: test_gpu_lora_add)."""
import math

import pytest
import torch

from helpers import say
from test_gpu_lora_add import TYPES, Case, i32

pytestmark = pytest.mark.gpu


def run(rt, c):
    """Checks c.y after the call against float64 on the CPU, and returns it."""
    c.y, c.store = c.y.cpu(), c.store.cpu()
    x, a, b, scale = (t.cpu() for t in (c.x, c.a, c.b, c.scale))
    on_gpu = (c.x, c.a, c.b, c.scale)
    c.x, c.a, c.b, c.scale = x, a, b, scale
    want, tol = c.want()
    c.x, c.a, c.b, c.scale = on_gpu
    y = c.y.cuda()
    rt.lora_add(y, c.x, rt.Adapters(c.a, c.b, c.scale), i32(c.starts), i32(c.adapter))
    got = y.cpu().double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want)) | ((got - want).abs() <= tol.nan_to_num(0.0, 0.0))
    bad = torch.nonzero(~same)
    assert same.all(), (len(bad), bad[:4].tolist(), got[~same][:4].tolist(), want[~same][:4].tolist())
    return want


ROWS = {"few": ([1, 3, 2, 5], [0, 1, -1, 0]), "many": ([40, 33, 50], [1, 0, 1])}


@pytest.mark.parametrize("x", list(TYPES))
@pytest.mark.parametrize("w", ["bf16", "f16"])
@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("rank, k, n", [(8, 64, 40), (16, 520, 300), (40, 264, 129), (128, 1032, 96)])
def test_infinite_weights(rt, x, w, rows, rank, k, n):
    """An infinity in a reaches all of its adapter's rows, one in b a column of them."""
    say("lora infinite weights", x, w, rows, rank, k, n)
    for where in ("a", "b", "both"):
        c = Case(*ROWS[rows], 2, rank, k, n, TYPES[x], TYPES[w], seed=rank)
        if where != "b":
            c.a[0, rank - 3, k - 1] = math.inf
        if where != "a":
            c.b[1, n - 1, 0], c.b[1, 7, rank - 1], c.b[0, 3, 5] = -math.inf, math.inf, math.nan
        want = run(rt, c)
        assert torch.isinf(want).any() and torch.isfinite(want).any()


@pytest.mark.parametrize("x", list(TYPES))
@pytest.mark.parametrize("w", ["bf16", "f16"])
@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("rank, k, n", [(8, 64, 40), (64, 520, 300)])
def test_infinite_rows(rt, x, w, rows, rank, k, n):
    """An infinity in x, met by weights of one sign (infinite sums) and of both (NaN)."""
    say("lora infinite rows", x, w, rows, rank, k, n)
    for one_sign in (True, False):
        c = Case(*ROWS[rows], 2, rank, k, n, TYPES[x], TYPES[w], seed=rank)
        if one_sign:
            c.a, c.b = c.a.abs(), c.b.abs()
        c.x[0, 5], c.x[3, k - 2], c.x[-1, 0] = math.inf, -math.inf, math.nan
        want = run(rt, c)
        assert torch.isinf(want).any() == one_sign and torch.isnan(want).any()


@pytest.mark.parametrize("w", ["bf16", "f16"])
@pytest.mark.parametrize("rows", list(ROWS))
def test_the_largest_numbers(rt, w, rows):
    """Rows that bfloat16 would round to infinities, whose products are finite."""
    say("lora largest", w, rows)
    c = Case(*ROWS[rows], 2, 16, 264, 70, torch.float32, TYPES[w], seed=1)
    c.a[:, :, 9] *= 1e-3
    c.b[:] = (c.b * 1e-2).to(c.b.dtype)
    c.x[0, 9], c.x[4, 9] = torch.finfo(torch.float32).max, -3.4e38
    assert torch.isfinite(run(rt, c)).all()


def test_others_keep_their_bits(rt):
    """What a row of NaN or an infinite column has beside it is as without them."""
    for rows in ROWS.values():
        c = Case(*rows, 2, 32, 512, 260, seed=9)
        adapters = rt.Adapters(c.a, c.b, c.scale)
        plain = rt.lora_add(c.y.clone(), c.x, adapters, i32(c.starts), i32(c.adapter))
        c.x[1] = math.nan
        got = rt.lora_add(c.y.clone(), c.x, adapters, i32(c.starts), i32(c.adapter))
        got[1] = plain[1]
        assert torch.equal(got, plain)
        c.b[:, 100] = math.inf
        got = rt.lora_add(c.y.clone(), c.x, adapters, i32(c.starts), i32(c.adapter))
        got[1], got[:, 100] = plain[1], plain[:, 100]
        assert torch.equal(got, plain)
