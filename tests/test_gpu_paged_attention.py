"""rt_hip_paged_attention against its definition in float64.

Tolerances, from the roundings.  With A = sum_j p_j |v_j| for an output value
o = sum_j p_j v_j, S the largest scale * sum |q_i k_i| of the row and n keys:
 * a score is a sum of head_dim products in f32: at most head_dim roundings of
   2^-24 relative to a partial sum, of which a quarter may add up, an error of
   2^-24 head_dim S / 4; scaling, exponential and its argument (at most S +
   log2 n) add 2^-24 (S + 32).  Each weight is off by that much, twice (itself
   and the sum it is divided by).
 * n additions of f32 to o and to the sum of weights: independent roundings, so
   sqrt(n / 3) standard deviations of 2^-24 A; six of them are 3.5 sqrt(n) 2^-24.
 * 16-bit types: each weight is rounded by eps / 2 of its type before it
   multiplies v, at most eps / 2 A in all; and o by eps / 2 |o|.
"""
import math

import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAIRS = [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "f16"), ("f32", "bf16")]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Step:
    """Random requests (rows, keys) over a cache whose unused slots hold NaN."""

    def __init__(self, q, kv, heads, kv_heads, dim, page, lens, seed=0, window=0, q_scale=1.0, joint=False, behind=0,
                 garbage=float("nan")):
        self.page, self.window, self.dim, self.kv_heads, self.group = page, window, dim, kv_heads, heads // kv_heads
        self.lens = lens
        self.scale = 1.0 / math.sqrt(dim)
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows = sum(n for n, _ in lens) + behind
        self.starts = [0]
        for n, _ in lens:
            self.starts.append(self.starts[-1] + n)
        x = torch.randn((rows, heads + (2 * kv_heads if joint else 0), dim), generator=g, device="cuda") * q_scale
        self.q = x.to(DT[q])[:, :heads]
        self.out = torch.full((rows, heads + (1 if joint else 0), dim), -77.0, dtype=DT[q], device="cuda")[:, :heads]
        held = [-(-n // page) for _, n in lens]
        n_pages = sum(held) + 3
        ids = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        cols = max(held) + 2
        table, at = [], 0
        for h in held:
            table.append(ids[at:at + h] + [-1, 2**31 - 1, 10**6][:1] * (cols - h))
            at += h
        self.table = i32(table)
        shape = (n_pages, 2, page, kv_heads, dim) if joint else (2, n_pages, page, kv_heads, dim)
        both = torch.randn(shape, generator=g, device="cuda").to(DT[kv])
        self.k, self.v = (both[:, 0], both[:, 1]) if joint else (both[0], both[1])
        used = torch.zeros((n_pages, page), dtype=torch.bool, device="cuda")
        for row, (_, n) in zip(table, lens):
            for c in range(-(-n // page)):
                used[row[c], :min(page, n - c * page)] = True
        for t in (self.k, self.v):
            t[~used] = garbage
        self.kv = None

    def keys(self, s):
        """Keys and values of request s in float64, zeros on pages that are none."""
        n = self.lens[s][1]
        ids = self.table[s, :-(-n // self.page)].long()
        bad = (ids < 0) | (ids >= self.k.shape[0])
        out = []
        for t in (self.k, self.v):
            x = t[ids.clamp(0, self.k.shape[0] - 1)].double()
            x[bad] = 0.0
            out.append(x.reshape(-1, self.kv_heads, self.dim)[:n])
        return out

    def run(self, rt, out=None, max_fresh=0, stream=None):
        self.kv = self.kv or rt.PagedKV(self.k, self.v)
        out = self.out if out is None else out
        return rt.paged_attention(self.q, self.kv, self.table, i32(self.starts), i32([n for _, n in self.lens]), self.scale,
                                  window=self.window, max_fresh=max_fresh, out=out, stream=stream)

    def reference(self):
        """(expected, tolerance), float64, rows of all requests."""
        want = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(want)
        small = self.q.dtype != torch.float32
        eps = torch.finfo(self.q.dtype).eps / 2 if small else 0.0
        for s, (n, length) in enumerate(self.lens):
            if n == 0:
                continue
            k, v = self.keys(s)
            at = torch.arange(length - n, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None]
            seen = j <= at
            if self.window:
                seen &= j > at - self.window
            for h in range(self.kv_heads):
                for i in range(self.group):
                    head = h * self.group + i
                    q = self.q[self.starts[s]:self.starts[s + 1], head].double()
                    # rows and keys apart, so that what a row does not see cannot reach it
                    score = torch.where(seen, (q @ k[:, h].T) * self.scale, -math.inf)
                    size = torch.where(seen, (q.abs() @ k[:, h].abs().T) * self.scale, 0.0)
                    rows = slice(self.starts[s], self.starts[s + 1])
                    if length == 0:
                        continue
                    p = torch.softmax(score, 1)
                    p = torch.where(seen.any(1, keepdim=True), p, 0.0)
                    vh = v[:, h]
                    if torch.isfinite(vh).all():
                        o, a = p @ vh, p @ vh.abs()
                    else:
                        o = torch.stack([(r[m][:, None] * vh[m]).sum(0) for r, m in zip(p, seen)])
                        a = torch.stack([(r[m][:, None] * vh[m].abs()).sum(0) for r, m in zip(p, seen)])
                    big = size.amax(1, keepdim=True) if length else size.sum(1, keepdim=True)
                    err = 2.0**-24 * (2 * (self.dim * big / 4 + big + 32) + 3.5 * math.sqrt(length)) + eps
                    want[rows, head] = o
                    tol[rows, head] = err * a + (torch.finfo(self.q.dtype).eps / 2) * o.abs() + 1e-30
                    if self.q.dtype == torch.float16:
                        tol[rows, head] += 2.0**-25  # below 2^-14 f16 has steps of 2^-24
        return want, tol

    def check(self, rt, max_fresh=0):
        got = self.run(rt, max_fresh=max_fresh).double()
        rows = self.starts[-1]
        want, tol = self.reference()
        bad = ~((got[:rows] - want[:rows]).abs() <= tol[:rows])
        assert not bad.any(), (int(bad.sum()), (got[:rows] - want[:rows]).abs().max().item(), torch.nonzero(bad)[:3].tolist())
        assert (got[rows:] == -77.0).all()


RAGGED = [(1, 1), (1, 5), (3, 3), (7, 100), (1, 63), (1, 64), (1, 65), (2, 200), (0, 50), (33, 64), (64, 65), (1, 0), (5, 3),
          (9, 0), (0, 0), (130, 300), (1, 1000), (16, 16)]


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv_heads, group, page, window", [
    (1, 1, 16, 0), (2, 3, 8, 0), (1, 4, 64, 7), (3, 5, 32, 1), (2, 8, 128, 100), (1, 16, 16, 65), (8, 1, 1024, 0)])
def test_ragged(rt, q, kv, dim, kv_heads, group, page, window):
    """Single tokens, drafts and chunks in one step, requests without rows or keys, fewer keys than rows, rows behind."""
    say("ragged", q, kv, dim, kv_heads, group, page, window)
    Step(q, kv, kv_heads * group, kv_heads, dim, page, RAGGED, seed=dim + group, window=window, behind=3,
         joint=page == 32).check(rt)


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("hint", [0, 1, 4, 1000])
def test_hint_is_only_a_hint(rt, q, kv, hint):
    """max_fresh right, wrong or missing: the same requests within the same tolerance."""
    say("hint", q, kv, hint)
    Step(q, kv, 6, 2, 128, 16, [(1, 700), (40, 333), (1, 2), (4, 90)], window=0).check(rt, max_fresh=hint)
    Step(q, kv, 6, 2, 64, 16, [(300, 700)], window=50).check(rt, max_fresh=hint)
    Step(q, kv, 6, 2, 64, 16, [(1, 3000)]).check(rt, max_fresh=hint)


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("kv_heads, group, dim, lens, window", [
    (1, 1, 128, [(1, 40000)], 0), (8, 3, 128, [(1, 9001), (1, 17)], 0), (1, 8, 256, [(3, 20000)], 0),
    (2, 2, 64, [(5, 30000), (1, 12000)], 5000), (2, 3, 128, [(700, 2100)], 0), (1, 2, 256, [(513, 1500), (1, 9)], 300),
    (4, 4, 64, [(1000, 1000), (200, 5000)], 0)])
def test_long(rt, q, kv, kv_heads, group, dim, lens, window):
    """Long caches whose keys are cut between workgroups, chunks over long caches."""
    say("long", q, kv, kv_heads, group, dim, lens, window)
    Step(q, kv, kv_heads * group, kv_heads, dim, 16, lens, seed=7, window=window).check(rt)


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("window", [0, 90])
def test_chunks_among_many_requests(rt, q, kv, window):
    """Chunks of several blocks at either end and inside of a batch that a wave has not lanes enough for."""
    say("chunks", q, kv, window)
    lens = [(1, 1 + 13 * s % 400) for s in range(131)]
    lens[0], lens[63], lens[64], lens[77], lens[130] = (700, 900), (300, 300), (0, 10), (513, 2000), (1030, 1030)
    Step(q, kv, 3, 1, 64, 32, lens, seed=3, window=window).check(rt)


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 300])
def test_rows_that_fill_the_card(rt, q, kv, dim, window):
    """Rows enough for the largest blocks, beside requests that have few."""
    say("full", q, kv, dim, window)
    Step(q, kv, 24, 8, dim, 16, [(900, 1500), (60, 700), (1, 500), (0, 4), (3, 2)], seed=dim, window=window).check(rt)


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_rows_of_full_blocks_do_not_see(rt, q, kv, dim, bad):
    """As below, with rows enough for the largest blocks; the same bits in every run, captured ones among them."""
    say("unseen full", q, kv, dim, bad)
    for n, length, window, at in ((450, 900, 0, 611), (440, 440, 120, 130)):
        st = Step(q, kv, 48, 2, dim, 16, [(n, length)], seed=5, window=window)
        pos = torch.arange(length - n, length, device="cuda")
        sees = (pos >= at) & ((pos < at + window) if window else True)
        page = st.table[0, at // 16]
        st.check(rt)
        clean = st.run(rt).clone()
        st.v[page, at % 16, 0, 3:dim:7] = bad
        got = st.run(rt).clone()
        # (the key's weight is 0 in those rows, so its products are zeros both times)
        assert torch.equal(got[~sees], clean[~sees])
        assert not torch.isfinite(got[sees][:, :24, 3:dim:7]).any() and torch.isfinite(got[sees][:, :24, 4:dim:7]).all()
        assert torch.isfinite(got[:, 24:]).all()
        starts, lens, out = i32(st.starts), i32([length]), torch.zeros_like(st.out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            rt.paged_attention(st.q, st.kv, st.table, starts, lens, st.scale, window=window, out=out)
        for _ in range(3):
            out.zero_()
            graph.replay()
            assert torch.equal(st.run(rt).nan_to_num(7.0), got.nan_to_num(7.0))
            assert torch.equal(out.nan_to_num(7.0), got.nan_to_num(7.0))


@pytest.mark.parametrize("q, kv", PAIRS)
def test_many_requests(rt, q, kv):
    """More requests than a workgroup has threads."""
    say("many", q, kv)
    lens = [(1 + i % 3, 3 + (i * 37) % 150) for i in range(1100)]
    Step(q, kv, 2, 1, 64, 8, lens, seed=3).check(rt)


@pytest.mark.parametrize("q, kv", PAIRS)
def test_sharp_scores(rt, q, kv):
    """Scores far apart: the maximum moves and the weights of most keys vanish."""
    say("sharp", q, kv)
    Step(q, kv, 4, 2, 128, 16, [(1, 3000), (90, 400), (6, 64)], seed=2, q_scale=12.0).check(rt)


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see(rt, q, kv, dim, bad):
    """Infinities and NaN in keys and values of positions that come later, or lie before the window: the rows that do
    not see them are as without them, those that do are NaN or infinite."""
    say("unseen", q, kv, dim, bad)
    for lens, window, at in (([(40, 90)], 0, 70), ([(8, 70)], 0, 66), ([(90, 200)], 16, 130), ([(3, 300)], 100, 199),
                             ([(1, 300)], 100, 199), ([(200, 400)], 33, 300)):
        st = Step(q, kv, 3, 1, dim, 16, lens, seed=5, window=window)
        n, length = lens[0]
        pos = torch.arange(length - n, length, device="cuda")
        sees = (pos >= at) & ((pos < at + window) if window else True)
        clean = st.run(rt).clone()
        page = st.table[0, at // 16]
        for t, name in ((st.v, "v"), (st.k, "k")):
            saved = t[page, at % 16].clone()
            t[page, at % 16, 0, 3:dim:7] = bad
            got = st.run(rt)
            # (a sum may be split otherwise than without them, by rounding)
            want, tol = st.reference()
            ok = ((got.double() - want).abs() <= tol) | (got.double() == want) | (torch.isnan(got) & torch.isnan(want))
            assert ok[~sees].all(), (name, lens)
            assert torch.equal(torch.isfinite(got[~sees]), torch.isfinite(clean[~sees]))
            if name == "v":
                assert not torch.isfinite(got[sees][..., 3:dim:7]).any()
                assert torch.isfinite(got[sees][..., 4:dim:7]).all()
            elif math.isnan(bad):
                assert torch.isnan(got[sees]).all()
            t[page, at % 16] = saved


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, lens, window, q_scale", [
    (2, [(1, 3000)], 0, 1.0), (2, [(1, 3000)], 0, 12.0), (3, [(5, 700), (1, 90)], 0, 1.0), (1, [(2, 5000)], 3000, 1.0),
    (2, [(60, 3000)], 0, 1.0), (2, [(60, 3000), (1, 17)], 0, 12.0), (48, [(440, 900)], 0, 1.0), (48, [(440, 900)], 300, 1.0)])
def test_values_that_are_not_finite(rt, q, kv, dim, heads, lens, window, q_scale):
    """Infinities of one sign, of both, and NaN in values, in keys that all rows of a request see, that some see, far
    from the last and next to it, with weights of every size down to those that vanish in 32 bits: what reaches a row
    is what the sum over the keys it sees has in 64 bits, to the sign."""
    say("not finite", q, kv, dim, heads, lens, window, q_scale)
    inf, nan = float("inf"), float("nan")
    st = Step(q, kv, heads, 1, dim, 16, lens, seed=11, window=window, q_scale=q_scale)
    n, length = lens[0]
    places = [3, length // 3, length // 2, length - n - 70, length - n - 1, length - 1 - n // 2, length - 1]
    pos = torch.arange(length - n, length, device="cuda")
    special = torch.zeros((n, dim), dtype=torch.float64, device="cuda")
    for i, at in enumerate(places):
        v = st.v[st.table[0, at // 16], at % 16, 0]
        v[2 * i + 1] = inf if i % 2 else -inf
        v[20] = inf
        v[22 + i % 2] = -inf if i % 4 < 2 else inf
        if i == 2:
            v[25] = nan
        # (every key that a row sees has a weight above 0)
        sees = (pos >= at) & ((pos < at + window) if window else True)
        special[sees] += torch.where(torch.isfinite(v), 0.0, v.double())
    got = st.run(rt).double()[:st.starts[-1]]
    st.v.nan_to_num_(0.0, 0.0, 0.0)  # (what is left of the sum where none of those is seen)
    want, tol = (x[:st.starts[-1]] for x in st.reference())
    special = torch.cat([special, special.new_zeros((st.starts[-1] - n, dim))])[:, None].expand(want.shape)
    assert torch.isnan(special).any() and (special == inf).any() and (special == -inf).any()
    right = torch.where(special == 0, (got - want).abs() <= tol, (got == special) | (torch.isnan(got) & torch.isnan(special)))
    assert right.all(), (int((~right).sum()), torch.nonzero(~right)[:4].tolist(), got[~right][:4].tolist(), special[~right][:4].tolist())


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("heads, dim, lens", [(1, 128, [(400, 395)]), (1, 64, [(9, 4), (120, 1), (300, 211)]),
                                              (48, 128, [(440, 300)]), (4, 256, [(4, 3), (1, 0), (1, 7)]), (16, 64, [(2, 1)])])
def test_windows_longer_than_any_request(rt, q, kv, heads, dim, lens):
    """The longest windows there are hide nothing, also from the rows of requests that have fewer keys than rows."""
    say("no window", q, kv, heads, dim, lens)
    st = Step(q, kv, heads, 1, dim, 16, lens, seed=8, behind=1)
    st.check(rt)
    want = st.run(rt).clone()
    for window in (2**31 - 1, 2**31 - 2, 2**31 - 200, 2**30, 1000):
        st.window = window
        st.out.fill_(-77.0)
        assert torch.equal(st.run(rt), want), window


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("size, scale", [(1e-36, 1e-10), (1e-30, 1e-30), (1.0, 1e-38), (0.0, 1.0)])
def test_scores_that_vanish(rt, q, kv, rows, size, scale):
    """Scores so small that every key has the same weight: the mean of the values, whose keys are cut between many
    workgroups.  (Errors: of n additions, and of the weights' rounding, which all share one value.)"""
    say("vanish", q, kv, rows, size, scale)
    n, dim, page = 20000, 128, 16
    k, v = torch.randn((2, n // page, page, 1, dim), device="cuda").to(DT[kv])
    x = (torch.ones((rows, 2, dim), device="cuda") * size).to(DT[q])
    table = torch.arange(n // page, dtype=torch.int32, device="cuda")[None]
    got = rt.paged_attention(x, rt.PagedKV(k, v), table, i32([0, rows]), i32([n]), scale)
    seen = torch.arange(n - rows + 1, n + 1, device="cuda")
    flat = v.double().reshape(n, dim)
    want = (flat.cumsum(0)[seen - 1] / seen[:, None])[:, None]
    size_ = (flat.abs().cumsum(0)[seen - 1] / seen[:, None])[:, None]
    eps = torch.finfo(DT[q]).eps / 2 if q != "f32" else 2.0**-24
    assert ((got.double() - want).abs() <= 2.0**-24 * (64 + 3.5 * math.sqrt(n)) * size_ + eps * want.abs() + 2.0**-25).all()


@pytest.mark.parametrize("q, kv", PAIRS)
def test_garbage_tables(rt, q, kv):
    """Pages that are none of the cache's count as zeros; starts and lengths that make no sense touch nothing else."""
    say("tables", q, kv)
    st = Step(q, kv, 4, 2, 128, 16, [(2, 90), (50, 200), (1, 33)], seed=4)
    st.table[0, 2], st.table[1, 0], st.table[1, 7], st.table[2, 2] = -1, st.k.shape[0], 2**31 - 1, -2**31
    st.check(rt)
    # lengths past the table's row are cut to it, starts to the rows there are
    st.table.clamp_(0, st.k.shape[0] - 1)
    st.k.nan_to_num_(0.5), st.v.nan_to_num_(0.5)
    kvs = rt.PagedKV(st.k, st.v)
    for starts, lens in (([0, 2, 52, 53], [90, 2**31 - 1, -5]), ([0, 1000, 20, 53], [90, 200, 33]),
                         ([-7, 2, 2**31 - 1, -2**31], [10**9, 10**9, 10**9])):
        out = rt.paged_attention(st.q, kvs, st.table, i32(starts), i32(lens), st.scale)
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("q, kv", PAIRS)
def test_same_bits(rt, q, kv):
    """The same call twice, and on another stream: the same bits."""
    say("bits", q, kv)
    st = Step(q, kv, 6, 2, 128, 16, [(1, 9000), (300, 900), (4, 77)], seed=9)
    a = st.run(rt, out=torch.zeros_like(st.out))
    b = st.run(rt, out=torch.zeros_like(st.out))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = st.run(rt, out=torch.zeros_like(st.out))
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("q, kv", PAIRS)
def test_on_another_stream(rt, q, kv):
    """Calls in turn on two streams that wait for each other: the workspace is shared, the results are the same."""
    say("streams", q, kv)
    step = Step(q, kv, 8, 2, 128, 16, [(1, 5000), (200, 900), (4, 77)])
    want = step.run(rt).clone()
    side, out = torch.cuda.Stream(), torch.empty_like(step.out)
    for _ in range(3):
        step.out.fill_(-77.0)
        out.fill_(-77.0)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step.run(rt, out=out)
        torch.cuda.current_stream().wait_stream(side)
        step.run(rt)
        assert torch.equal(out, want) and torch.equal(step.out, want)


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("lens", [[(1, 900)], [(200, 900), (1, 70)]])
def test_result_of_a_call_on_another_stream(rt, q, kv, lens):
    """No out, another stream's call, the current stream busy: nothing of that stream touches the result."""
    say("result on a stream", q, kv, lens)
    st = Step(q, kv, 6, 2, 128, 16, lens, behind=2)
    kvs, starts, keys = rt.PagedKV(st.k, st.v), i32(st.starts), i32([n for _, n in lens])
    want = rt.paged_attention(st.q, kvs, st.table, starts, keys, st.scale)
    busy, side = torch.zeros((64, 1 << 20), device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(40):
        busy.add_(1.0)
    got = rt.paged_attention(st.q, kvs, st.table, starts, keys, st.scale, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and (got[-2:] == 0).all() and got.abs().max() > 0


@pytest.mark.parametrize("q, kv", PAIRS)
def test_captured(rt, q, kv):
    """A captured call, replayed over other lengths, starts and tables between eager work: eager's bits each time."""
    say("captured", q, kv)
    rows, n = 64, 5
    st = Step(q, kv, 6, 2, 128, 16, [(20, 3000), (1, 500), (3, 3), (30, 64), (0, 9)], seed=1, behind=rows - 54)
    kvs = rt.PagedKV(st.k, st.v)
    dt = {"f32": rt.F32, "f16": rt.F16, "bf16": rt.BF16}[q]
    rt.reserve_workspace(rt.paged_attention_workspace_bytes(kvs, dt, 6, n, rows))
    starts, lens = i32(st.starts), i32([x for _, x in st.lens])
    out = torch.zeros_like(st.out)
    call = lambda o: rt.paged_attention(st.q, kvs, st.table, starts, lens, st.scale, out=o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for a, b in (([0, 20, 21, 24, 54, 54], [3000, 500, 3, 64, 9]), ([0, 1, 2, 3, 4, 5], [2900, 490, 2, 64, 9]),
                 ([0, 0, 60, 60, 61, 61], [3000, 200, 1, 33, 0])):
        starts.copy_(i32(a)), lens.copy_(i32(b))
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            eager = call(torch.zeros_like(out))
            assert torch.equal(out, eager)


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("rows", [40, 130])
def test_positions_past_30_bits(rt, q, kv, rows):
    """Chunks over 2^30 keys, all on one page but the last ones, whose weight is all there is: each row's result is the
    value of its own last key, which counts once.  (Scores of 0 for a billion keys, 60 for those: exp(-60) 2^30 < 1e-16.)"""
    say("far", q, kv, rows)
    page, dim, length = 1024, 64, 2**30 + 1500
    cols = -(-length // page)
    k, v = (torch.zeros((4, page, 1, dim), device="cuda", dtype=DT[kv]) for _ in range(2))
    v[0] = 100.0
    at = torch.arange(length - rows, length, device="cuda")
    table = torch.zeros((1, cols), dtype=torch.int32, device="cuda")
    table[0, -3:] = i32([1, 2, 3])
    place = (at - (cols - 3) * page)
    own, last = 1 + place // page, place % page
    # row i's key has its own two dims, and the row asks for them alone
    values = torch.randn((rows, dim), device="cuda").to(DT[kv])
    keys = torch.zeros((rows, dim), device="cuda")
    asks = torch.zeros((rows, 1, dim), device="cuda")
    for i in range(rows):
        a, b = i % dim, (i // dim + i + 1) % dim
        keys[i, a], keys[i, b] = 8.0, 8.0
        asks[i, 0, a], asks[i, 0, b] = 60.0, 60.0
    k[own, last, 0], v[own, last, 0] = keys.to(DT[kv]), values
    out = rt.paged_attention(asks.to(DT[q]), rt.PagedKV(k, v), table, i32([0, rows]), i32([length]), 1 / 16)
    # of the keys that a row sees, its own has the score 60, those that share a dim with it 30, the others 0
    score = asks[:, 0].double() @ keys.double().T / 16
    p = torch.exp(score.masked_fill_(at[None] > at[:, None], -math.inf) - 60)
    want = (p @ values.double()) / p.sum(1, keepdim=True)
    eps = torch.finfo(DT[q]).eps / 2 if q != "f32" else 2.0**-20
    tol = 2 * eps * (p @ values.double().abs()) / p.sum(1, keepdim=True) + 2**30 * math.exp(-60) * 100
    assert ((out[:, 0].double() - want).abs() <= tol).all(), (out[:, 0].double() - want).abs().max()


@pytest.mark.parametrize("q, kv", PAIRS)
@pytest.mark.parametrize("rows, dim", [(1, 128), (5, 64), (30, 256), (40, 64), (130, 128), (70, 256)])
def test_lengths_up_to_31_bits(rt, q, kv, rows, dim):
    """The longest request that a table can hold, 2^31 - 8 keys: the bits of one whose keys are the last 632 of it (as
    far into a tile), also where the length given is longer still."""
    say("longest", q, kv, rows, dim)
    page, near = 8, 632
    cols = 2**28 - 1
    k, v = torch.randn((2, near // page, page, 2, dim), device="cuda").to(DT[kv])
    x = torch.randn((rows, 4, dim), device="cuda").to(DT[q])
    ids = torch.randperm(near // page, device="cuda").to(torch.int32)
    table = torch.full((1, cols), -1, dtype=torch.int32, device="cuda")
    table[0, -(near // page):] = ids
    kvs, starts = rt.PagedKV(k, v), i32([0, rows])
    for window in (1, 300):
        want = rt.paged_attention(x, kvs, ids[None].contiguous(), starts, i32([near]), 0.1, window=window)
        assert want.abs().max() > 0
        for length in (page * cols, 2**31 - 1):
            assert torch.equal(rt.paged_attention(x, kvs, table, starts, i32([length]), 0.1, window=window), want)


def test_offsets_past_32_bits(rt):
    """A cache of more than 2^32 bytes, the request's pages at its end."""
    heads, dim, page = 8, 256, 128
    pages = (5 << 30) // (page * heads * dim * 2)
    k = torch.zeros((pages, page, heads, dim), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    ids = [pages - 1, 0, pages - 2]
    for t in (k, v):
        for i in ids:
            t[i] = torch.randn(t[i].shape, device="cuda").bfloat16()
    q = torch.randn((2, heads, dim), device="cuda").bfloat16()
    args = (i32([0, 2]), i32([300]), 0.06)
    far = rt.paged_attention(q, rt.PagedKV(k, v), i32([ids]), *args)
    near = rt.paged_attention(q, rt.PagedKV(k[ids].clone(), v[ids].clone()), i32([[0, 1, 2]]), *args)
    assert torch.equal(far, near) and far.abs().max() > 0


def test_another_head_layouts_refusals(rt):
    st = Step("bf16", "bf16", 4, 2, 64, 16, [(2, 20)])
    kvs = rt.PagedKV(st.k, st.v)
    args = (st.table, i32(st.starts), i32([20]), 0.1)
    with pytest.raises(rt.RtHipError):
        rt.paged_attention(st.q[:, :3].contiguous(), kvs, *args)
    with pytest.raises(rt.RtHipError):
        rt.paged_attention(st.q.half(), kvs, *args)
    with pytest.raises(ValueError):
        rt.paged_attention(st.q.transpose(0, 1), kvs, *args)
    with pytest.raises(ValueError):
        rt.paged_attention(st.q, kvs, st.table.long(), *args[1:])
    with pytest.raises(ValueError):
        rt.PagedKV(st.k, st.v[:, :8])
    with pytest.raises(ValueError):
        rt.PagedKV(st.k.transpose(1, 2), st.v.transpose(1, 2))
