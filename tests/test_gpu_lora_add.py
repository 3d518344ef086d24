"""rt_hip_lora_add against its definition in float64.

Tolerances, from the roundings: with T = sum |a_jk x_k| of a rank's sum and U = |scale|
sum_j |b_cj| T_j of an output's, every factor enters with its 24 bits (2^-24 each, a
limb's product left out below that), the sums over k and the rank are of f32 products
in f32: at most k + rank + slices additions of 2^-24 relative to a partial sum, whose
roundings are independent, six standard deviations sqrt((k + rank) / 3) * 2^-24 * 6;
the result rounds once more with what y held.
"""
import math

import numpy as np
import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x, np.int64), device="cuda").to(torch.int32)


class Case:
    def __init__(self, rows, adapter, m, rank, k, n, x=torch.float32, w=torch.bfloat16, seed=0, x_pad=0, y_pad=0, behind=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        total = sum(rows) + behind
        self.x = (r(total, k + x_pad) * torch.exp(r(total, 1))).to(x)[:, :k]
        self.a, self.b = r(m, rank, k).to(w), r(m, n, rank).to(w)
        self.scale = r(m)
        self.store = r(total, n + y_pad)
        self.y = self.store[:, :n]
        self.starts, self.adapter, self.rows = np.concatenate([[0], np.cumsum(rows)]), adapter, rows
        self.m, self.rank, self.k, self.n = m, rank, k, n

    def want(self):
        want, tol = self.y.double(), torch.zeros_like(self.y, dtype=torch.float64)
        for s, i in enumerate(self.adapter):
            if not 0 <= i < self.m:
                continue
            at = slice(int(self.starts[s]), int(self.starts[s + 1]))
            x, a, b = self.x[at].double(), self.a[i].double(), self.b[i].double()
            scale = float(self.scale[i])
            want[at] += scale * ((x @ a.T) @ b.T)
            u = abs(scale) * ((x.abs() @ a.abs().T) @ b.abs().T)
            tol[at] = u * 2.0**-24 * (6 * math.sqrt((self.k + self.rank) / 3) + 8) + 2.0**-24 * want[at].abs()
        return want, tol

    def check(self, rt, stream=None):
        want, tol = self.want()
        before = self.store.clone()
        out = rt.lora_add(self.y, self.x, rt.Adapters(self.a, self.b, self.scale), i32(self.starts), i32(self.adapter), stream=stream)
        assert out is self.y
        torch.cuda.synchronize()
        err = (self.y.double() - want).abs()
        assert (err <= tol).all(), (err.max().item(), torch.nonzero(~(err <= tol))[:4].tolist())
        same = (tol == 0) & (want == before[:, :self.n].double())
        assert torch.equal(self.y[same], before[:, :self.n][same])
        assert torch.equal(self.store[:, self.n:], before[:, self.n:])


TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("x", list(TYPES))
@pytest.mark.parametrize("w", ["bf16", "f16"])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 104, 128])
def test_ranks(rt, x, w, rank):
    say("lora ranks", x, w, rank)
    Case([1, 3, 16, 17, 0, 40, 1], [1, -1, 0, 2, 1, 0, 2], 3, rank, 264, 200, TYPES[x], TYPES[w], seed=rank).check(rt)


@pytest.mark.parametrize("w", ["bf16", "f16"])
@pytest.mark.parametrize("k, n, x_pad, y_pad", [
    (8, 1, 0, 0), (8, 4, 8, 0), (120, 3, 0, 1), (128, 256, 0, 0), (136, 257, 4, 3), (512, 255, 0, 1), (520, 64, 0, 4),
    (4096, 1000, 0, 0), (10240, 260, 0, 0), (2560, 5001, 0, 0)])
def test_shapes(rt, w, k, n, x_pad, y_pad):
    say("lora shapes", w, k, n, x_pad, y_pad)
    Case([1, 5, 33], [0, 1, 0], 2, 16, k, n, w=TYPES[w], seed=k + n, x_pad=x_pad, y_pad=y_pad, behind=2).check(rt)
    Case([1], [0], 1, 32, k, n, w=TYPES[w], seed=k, x_pad=x_pad, y_pad=y_pad).check(rt)


@pytest.mark.parametrize("rows", [[1] * 64, [1] * 65, [2, 1] * 100, [1] * 4096, [700, 1, 900], [5000]])
def test_requests(rt, rows):
    """As many requests as a wave has lanes, and more; long chunks; adapters that are none among them."""
    say("lora requests", len(rows))
    rng = np.random.default_rng(len(rows))
    adapter = rng.integers(-2, 9, len(rows))
    Case(rows, adapter.tolist(), 8, 16, 256, 132, seed=3).check(rt)
    Case(rows, [-1] * len(rows), 8, 16, 256, 132, seed=4).check(rt)


def test_starts_out_of_range(rt):
    """Rows outside the tensors: nothing outside is read or written."""
    c = Case([4, 4], [0, 1], 2, 16, 64, 64, seed=1)
    adapters = rt.Adapters(c.a, c.b, c.scale)
    for starts in ([-5, 2, 10**9], [8, 8, 8], [9, 100, 2**31 - 1], [6, 3, 1]):
        rt.lora_add(c.y, c.x, adapters, i32(starts), i32([0, 1]))
    rt.lora_add(c.y, c.x, adapters, i32([0, 4, 8]), i32([2**31 - 1, -(2**31)]))
    torch.cuda.synchronize()
    assert torch.isfinite(c.y).all()


def test_special_numbers(rt):
    """Infinities and NaN of a row reach that row alone; zeros stay what they are."""
    c = Case([3, 20], [0, 1], 2, 16, 64, 40, seed=2)
    c.x[1, 5], c.x[7, 0] = math.inf, math.nan
    clean = c.y.clone()
    c.x[9] = 0.0
    rt.lora_add(c.y, c.x, rt.Adapters(c.a, c.b, c.scale), i32(c.starts), i32(c.adapter))
    finite = torch.isfinite(c.y).all(1)
    assert not torch.isfinite(c.y[1]).any() and not torch.isfinite(c.y[7]).any()
    finite[[1, 7]] = True
    assert finite.all()
    assert torch.equal(c.y[9], clean[9])


def test_far_adapters(rt):
    """Offsets past 2^32 bytes: the last of many adapters."""
    m, rank, k, n = 2100, 128, 8192, 64
    a = torch.zeros((m, rank, k), dtype=torch.bfloat16, device="cuda")
    b = torch.zeros((m, n, rank), dtype=torch.bfloat16, device="cuda")
    c = Case([2, 1], [0, 0], 1, rank, k, n, seed=6)
    a[m - 1], b[m - 1] = c.a[0], c.b[0]
    want, tol = c.want()
    scale = torch.zeros(m, device="cuda")
    scale[m - 1] = c.scale[0]
    rt.lora_add(c.y, c.x, rt.Adapters(a, b, scale), i32(c.starts), i32([m - 1, m - 1]))
    assert ((c.y.double() - want).abs() <= tol).all()


def test_captured_and_again(rt):
    """A graph gives the eager call's bits at every replay; so does another stream."""
    c = Case([1, 30, 2, 1], [0, 1, -1, 1], 2, 32, 1024, 520, seed=5)
    adapters = rt.Adapters(c.a, c.b, c.scale)
    rt.reserve_workspace(rt.lora_workspace_bytes(adapters, 4, 34))
    starts, adapter, start_y = i32(c.starts), i32(c.adapter), c.y.clone()
    first = rt.lora_add(c.y.clone(), c.x, adapters, starts, adapter)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.lora_add(c.y, c.x, adapters, starts, adapter)
    for i in range(4):
        c.y.copy_(start_y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.y, first), i
        assert torch.equal(rt.lora_add(start_y.clone(), c.x, adapters, starts, adapter), first)
    side = torch.cuda.Stream()
    y = start_y.clone()
    torch.cuda.synchronize()
    rt.lora_add(y, c.x, adapters, starts, adapter, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(y, first)


def test_beside_a_projection(rt):
    """linear_forward on shared Q4_K weights, then the requests' adapters, is each request's own product."""
    n, k, rows, rank = 256, 512, [1, 1, 6], 16
    w = torch.randn((n, k), device="cuda") * 0.05
    blocks = rt.quantize_q4k(w)
    c = Case(rows, [1, -1, 0], 2, rank, k, n, seed=7)
    dense = rt.dequant(rt.Q4K, blocks, n, k).double()
    y = rt.linear_forward(rt.Q4K, blocks, c.x, n, k)
    rt.lora_add(y, c.x, rt.Adapters(c.a, c.b, c.scale), i32(c.starts), i32(c.adapter))
    for s, i in enumerate(c.adapter):
        at = slice(int(c.starts[s]), int(c.starts[s + 1]))
        full = dense if i < 0 else dense + float(c.scale[i]) * c.b[i].double() @ c.a[i].double()
        size = c.x[at].double().abs() @ (dense.abs() + (0 if i < 0 else abs(float(c.scale[i])) * c.b[i].double().abs() @ c.a[i].double().abs())).T
        # (the projection's own contract: 1e-5 of the sizes, normwise)
        assert ((y[at].double() - c.x[at].double() @ full.T).abs() <= 1e-5 * size.amax(1, keepdim=True)).all()
