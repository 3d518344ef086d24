"""rt_hip_paged_attention over a 4-bit cache against its definition in float64.

Tolerances, from the roundings.  With A = sum_j p_j |v_j| for an output value
o = sum_j p_j v_j, S the largest scale * sum |q_i k_i| of the row and n keys:
 * a score is a sum of head_dim products in f32: at most head_dim roundings of
   2^-24 relative to a partial sum, of which a quarter may add up, an error of
   2^-24 head_dim S / 4; scaling, exponential and its argument (at most S +
   log2 n) add 2^-24 (S + 32).  f32 rows enter with 22 bits: 2^-22 S.  Each
   weight is off by that much, twice (itself and the sum it is divided by).
 * n additions of f32 to o and to the sum of weights: independent roundings, so
   sqrt(n / 3) standard deviations of 2^-24 A; six of them are 3.5 sqrt(n) 2^-24.
 * weights: of 16-bit rows rounded to f16, 2^-11 A; of f32 rows two limbs, 2^-22 A.
 * f16 ends at 2^-24: what a weight (its last limb) has below that is lost, half of
   it at most, 2^-25.  Weights are times 2^6 for the largest (more while the
   maximum lags), so 2^-31 of it, p_max <= 1: 2^-31 sum_j |v_j| over the keys seen.
   (Next to the terms above where the row's largest weights meet values near 0.)
 * 16-bit outputs are rounded by eps / 2 |o|.
"""
import math

import pytest
import torch

from helpers import say
from paged4 import filled, kept

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPES = list(DT)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Step:
    """Random requests (rows, keys) over a cache whose unused slots are NaN."""

    def __init__(self, rt, q, heads, kv_heads, dim, page, lens, seed=0, window=0, q_scale=1.0, joint=False, behind=0, byte=0xFF,
                 spoil=None):
        self.page, self.window, self.dim, self.kv_heads, self.group = page, window, dim, kv_heads, heads // kv_heads
        self.lens, self.scale = lens, 1.0 / math.sqrt(dim)
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows = sum(n for n, _ in lens) + behind
        self.starts = [0]
        for n, _ in lens:
            self.starts.append(self.starts[-1] + n)
        x = torch.randn((rows, heads + (2 if joint else 0), dim), generator=g, device="cuda") * q_scale
        self.q = x.to(DT[q])[:, :heads]
        self.out = torch.full((rows, heads + (1 if joint else 0), dim), -77.0, dtype=DT[q], device="cuda")[:, :heads]
        held = [-(-n // page) for _, n in lens]
        n_pages = sum(held) + 3
        ids = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        cols = max(held) + 2
        table, at = [], 0
        for h in held:
            table.append(ids[at:at + h] + [-1, 2**31 - 1][:1] * (cols - h))
            at += h
        self.table, self.n_pages = i32(table), n_pages
        self.kv = filled(rt, n_pages, page, kv_heads, dim, joint, byte)
        used = torch.zeros(n_pages * page, dtype=torch.bool, device="cuda")
        for row, (_, n) in zip(table, lens):
            for c in range(-(-n // page)):
                used[row[c] * page:row[c] * page + min(page, n - c * page)] = True
        k = torch.randn((n_pages * page, kv_heads, dim), generator=g, device="cuda") + 0.5
        v = torch.randn((n_pages * page, kv_heads, dim), generator=g, device="cuda")
        if spoil:
            spoil(self, k, v)
        slots = torch.nonzero(used)[:, 0].to(torch.int32)
        rt.paged_append(self.kv, k[used], v[used], slots)
        self.k, self.v = (torch.where(used[:, None, None], kept(x), torch.nan).view(n_pages, page, kv_heads, dim) for x in (k, v))

    def keys(self, s):
        """Keys and values of request s in float64, zeros on pages that are none."""
        n = self.lens[s][1]
        ids = self.table[s, :-(-n // self.page)].long()
        bad = (ids < 0) | (ids >= self.n_pages)
        out = []
        for t in (self.k, self.v):
            x = t[ids.clamp(0, self.n_pages - 1)].clone()
            x[bad] = 0.0
            out.append(x.reshape(-1, self.kv_heads, self.dim)[:n])
        return out

    def run(self, rt, out=None, max_fresh=0, stream=None):
        return rt.paged_attention(self.q, self.kv, self.table, i32(self.starts), i32([n for _, n in self.lens]), self.scale,
                                  window=self.window, max_fresh=max_fresh, out=self.out if out is None else out, stream=stream)

    def reference(self):
        """(expected, tolerance), float64, rows of all requests."""
        want = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(want)
        small = self.q.dtype != torch.float32
        eps = torch.finfo(self.q.dtype).eps / 2 if small else 2.0**-24
        for s, (n, length) in enumerate(self.lens):
            if n == 0 or length == 0:
                continue
            k, v = self.keys(s)
            at = torch.arange(length - n, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None]
            seen = j <= at
            if self.window:
                seen &= j > at - self.window
            rows = slice(self.starts[s], self.starts[s + 1])
            for h in range(self.kv_heads):
                for i in range(self.group):
                    head = h * self.group + i
                    q = self.q[rows, head].double()
                    # rows and keys apart, so that what a row does not see cannot reach it
                    score = torch.where(seen, (q @ k[:, h].T) * self.scale, -math.inf)
                    size = torch.where(seen, (q.abs() @ k[:, h].abs().T) * self.scale, 0.0)
                    p = torch.where(seen.any(1, keepdim=True), torch.softmax(score, 1), 0.0)
                    vh = v[:, h]
                    if torch.isfinite(vh).all():
                        o, a, all_ = p @ vh, p @ vh.abs(), seen.double() @ vh.abs()
                    else:
                        o = torch.stack([(r[m][:, None] * vh[m]).sum(0) for r, m in zip(p, seen)])
                        a = torch.stack([(r[m][:, None] * vh[m].abs()).sum(0) for r, m in zip(p, seen)])
                        all_ = torch.stack([vh[m].abs().sum(0) for m in seen])
                    big = size.amax(1, keepdim=True)
                    score_err = 2.0**-24 * (self.dim * big / 4 + big + 32) + (0.0 if small else 2.0**-22 * big)
                    err = 2 * score_err + 2.0**-24 * 3.5 * math.sqrt(length) + (2.0**-11 if small else 2.0**-22)
                    want[rows, head] = o
                    tol[rows, head] = err * a + 2.0**-31 * all_ + eps * o.abs() + 1e-30
                    if self.q.dtype == torch.float16:
                        tol[rows, head] += 2.0**-25  # below 2^-14 f16 has steps of 2^-24
        return want, tol

    def check(self, rt, max_fresh=0):
        got = self.run(rt, max_fresh=max_fresh).double()
        rows = self.starts[-1]
        want, tol = self.reference()
        both_nan = torch.isnan(got[:rows]) & torch.isnan(want[:rows])
        bad = ~(((got[:rows] - want[:rows]).abs() <= tol[:rows]) | both_nan)
        assert not bad.any(), (int(bad.sum()), (got[:rows] - want[:rows]).abs().max().item(), torch.nonzero(bad)[:3].tolist())
        assert (got[rows:] == -77.0).all()


RAGGED = [(1, 1), (1, 5), (3, 3), (7, 100), (1, 63), (1, 64), (1, 65), (2, 200), (0, 50), (33, 64), (64, 65), (1, 0), (5, 3),
          (9, 0), (0, 0), (130, 300), (1, 1000), (16, 16)]


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv_heads, group, page, window", [
    (1, 1, 16, 0), (2, 3, 8, 0), (1, 4, 64, 7), (3, 5, 32, 1), (2, 8, 128, 100), (1, 16, 16, 65), (8, 1, 1024, 0)])
def test_ragged(rt, q, dim, kv_heads, group, page, window):
    """Single tokens, drafts and chunks in one step, requests without rows or keys, fewer keys than rows, rows behind."""
    say("ragged4", q, dim, kv_heads, group, page, window)
    Step(rt, q, kv_heads * group, kv_heads, dim, page, RAGGED, seed=dim + group, window=window, behind=3,
         joint=page == 32).check(rt)


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("hint", [0, 1, 4, 1000])
def test_hint_is_only_a_hint(rt, q, hint):
    say("hint4", q, hint)
    Step(rt, q, 6, 2, 128, 16, [(1, 700), (40, 333), (1, 2), (4, 90)]).check(rt, max_fresh=hint)
    Step(rt, q, 6, 2, 64, 16, [(300, 700)], window=50).check(rt, max_fresh=hint)
    Step(rt, q, 4, 2, 256, 16, [(20, 700), (1, 9)], window=50).check(rt, max_fresh=hint)
    Step(rt, q, 6, 2, 64, 16, [(1, 3000)]).check(rt, max_fresh=hint)


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("kv_heads, group, dim, lens, window", [
    (1, 1, 128, [(1, 40000)], 0), (8, 3, 128, [(1, 9001), (1, 17)], 0), (1, 8, 256, [(3, 20000)], 0),
    (2, 2, 64, [(5, 30000), (1, 12000)], 5000), (2, 3, 128, [(700, 2100)], 0), (1, 2, 256, [(513, 1500), (1, 9)], 300),
    (4, 4, 64, [(1000, 1000), (200, 5000)], 0)])
def test_long(rt, q, kv_heads, group, dim, lens, window):
    """Long caches whose keys are cut between workgroups, chunks over long caches."""
    say("long4", q, kv_heads, group, dim, lens, window)
    Step(rt, q, kv_heads * group, kv_heads, dim, 16, lens, seed=7, window=window).check(rt)


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_requests(rt, q, dim):
    """More requests than a wave has lanes, chunks of several blocks among them."""
    say("many4", q, dim)
    lens = [(1 + 90 * (s % 37 == 5), 3 + 41 * s % 500 + 90) for s in range(150)]
    Step(rt, q, 4, 2, dim, 16, lens, seed=3).check(rt)


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 5, 200])
def test_values_that_are_no_numbers(rt, q, dim, n):
    """A NaN in v reaches the rows that see its key, in its group's dims, and no others; large and vanished weights."""
    say("nan values4", q, dim, n)

    def spoil(step, k, v):
        for s, (_, length) in enumerate(step.lens):
            for at, d in ((length - 1, 3), (length // 2, 40), (0, dim - 1), (max(0, length - 150), 33), (max(0, length - 3), 0)):
                page = int(step.table[s, at // step.page])
                v[page * step.page + at % step.page, s % step.kv_heads, d] = float("nan") if s % 2 else float("inf")

    Step(rt, q, 6, 2, dim, 16, [(n, 300), (n, 777), (n, 210), (n, 1500)], seed=5, spoil=spoil).check(rt)
    Step(rt, q, 6, 2, dim, 8, [(n, 300), (n, 777), (n, 210)], seed=6, window=64, spoil=spoil).check(rt)


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("n", [2, 60])
def test_keys_that_are_no_numbers(rt, q, n):
    """A NaN in a key leaves alone the rows that do not see it."""
    say("nan keys4", q, n)

    def spoil(step, k, v):
        page = int(step.table[0, 49 // step.page])
        k[page * step.page + 49 % step.page, 1, 5] = float("nan")

    step = Step(rt, q, 4, 2, 128, 16, [(n, 50), (n, 80)], seed=8, spoil=spoil)
    got, (want, tol) = step.run(rt).double(), step.reference()
    fine = torch.ones_like(got, dtype=torch.bool)
    fine[n - 1, 2:] = False  # the last row of request 0, heads of KV head 1
    assert ((got - want).abs() <= tol)[fine].all()


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("n", [1, 70])
def test_garbage(rt, q, n):
    """Pages that are none count as zeros; starts and lengths out of range touch nothing else."""
    say("garbage4", q, n)
    step = Step(rt, q, 4, 2, 128, 16, [(n, 200), (n, 333)], seed=9, byte=0)
    step.table[0, 3], step.table[1, 5], step.table[1, 20] = -1, step.n_pages, -(2**31)
    step.check(rt)
    before = step.out.clone()
    bad = [i32([5, 2, 10**9]), i32([-4, -3, 2**31 - 1])]
    for starts in bad:
        rt.paged_attention(step.q, step.kv, step.table, starts, i32([2**31 - 1, -5]), 0.1, out=step.out)
    torch.cuda.synchronize()
    assert torch.isfinite(before).all()


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("q_scale", [1e-30, 1e-4, 30.0, 1000.0])
def test_sizes_of_q(rt, q, q_scale):
    """Rows of very small and very large values (f16's range where it is f16)."""
    if q == "f16" and q_scale < 1e-6:
        q_scale = 1e-6
    say("q sizes4", q, q_scale)
    Step(rt, q, 6, 2, 128, 16, [(1, 500), (3, 70), (50, 90)], seed=4, q_scale=q_scale).check(rt)


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_same_bits_again(rt, q, dim):
    """Results do not depend on which workgroup joins a cut item; a graph gives the eager call's bits."""
    say("again4", q, dim)
    step = Step(rt, q, 4, 2, dim, 16, [(1, 20000), (1, 50), (4, 3000), (300, 900)], seed=2)
    rt.reserve_workspace(rt.paged_attention_workspace_bytes(step.kv, {"f32": rt.F32, "f16": rt.F16, "bf16": rt.BF16}[q], 4, 4, 306))
    first = step.run(rt).clone()
    starts, lens = i32(step.starts), i32([n for _, n in step.lens])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.paged_attention(step.q, step.kv, step.table, starts, lens, step.scale, out=step.out)
    for i in range(4):
        step.out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(step.out, first), i
        other = step.run(rt, out=torch.zeros_like(step.out))
        assert torch.equal(other, first), i


def test_streams(rt):
    """A result made on the call's own stream; two streams in turn."""
    step = Step(rt, "bf16", 4, 2, 128, 16, [(1, 2000), (1, 50)], seed=2)
    torch.cuda.synchronize()
    want = step.run(rt, out=torch.zeros_like(step.out))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, None, side):
        got = rt.paged_attention(step.q, step.kv, step.table, i32(step.starts), i32([n for _, n in step.lens]), step.scale,
                                 stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
