"""rt_hip_verify_drafts against its definition in float64, request by request,
and against what the rule promises: tokens distributed as the target's."""
import numpy as np
import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu


def dist(row, t):
    """softmax(row / t) in float64; one of the first largest where t is 0."""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    p = np.zeros_like(x)
    top = x.max()
    if top == -np.inf:
        p[0] = 1.0
    elif not t > 0:
        p[int(np.argmax(x == top))] = 1.0
    elif top == np.inf:
        p[x == top] = 1.0 / (x == top).sum()
    else:
        p = np.exp((x - top) / np.float64(t))
        p /= p.sum()
    return p


def rules(logits, draft, tokens, starts, ua, us, temp, width):
    out, count = np.full((len(starts) - 1, width), -1), []
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        b = min(b, a + width)
        line = []
        for r in range(a, b):
            p = dist(logits[r], temp[s])
            w = p
            if r + 1 < b:
                d = int(tokens[r + 1])
                real = 0 <= d < p.size
                q = dist(draft[r], temp[s]) if draft is not None else np.eye(1, p.size, d)[0] if real else 0 * p
                if real and float(np.float32(ua[r])) * q[d] < p[d]:
                    line.append(d)
                    continue
                w = np.maximum(p - q, 0)
                w = w if w.sum() > 0 else p
            cum = np.cumsum(w)
            over = np.nonzero((cum > float(np.float32(us[s])) * cum[-1]) & (w > 0))[0]
            line.append(int(over[0]) if len(over) else int(np.nonzero(w)[0][-1]))
            break
        out[s, :len(line)] = line
        count.append(len(line))
    return out, np.array(count)


def call(rt, logits, draft, tokens, starts, ua, us, temp, max_draft, dtype=torch.float32, pad=0):
    def dev(x):
        if x is None:
            return None
        t = torch.zeros((x.shape[0], x.shape[1] + pad), dtype=dtype, device="cuda")[:, :x.shape[1]]
        return t.copy_(torch.from_numpy(x))
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    f32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.float32, device="cuda")
    a, b = rt.verify_drafts(dev(logits), i32(tokens), i32(starts), f32(ua), f32(us), max_draft,
                            draft_logits=dev(draft), temperature=None if temp is None else f32(temp))
    return a.cpu().numpy(), b.cpu().numpy()


def make(seed, n, vocab, lo, hi, bf16=False):
    rng = np.random.default_rng(seed)
    counts = rng.integers(lo, hi + 1, n) + 1
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1])
    logits = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    draft = (logits + rng.standard_normal((rows, vocab)).astype(np.float32)).astype(np.float32)
    if bf16:
        logits, draft = (torch.from_numpy(x).bfloat16().float().numpy() for x in (logits, draft))
    temp = np.where(rng.random(n) < 0.3, 0, rng.uniform(0.3, 2, n)).astype(np.float32)
    tokens = rng.integers(0, vocab, rows)
    for r in range(rows - 1):
        g = draft[r] + rng.gumbel(size=vocab)
        tokens[r + 1] = int(np.argmax(g if rng.random() < 0.8 else logits[r]))
    return logits, draft, tokens, starts, rng.random(rows, np.float32), rng.random(n, np.float32), temp


@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 1000, 4095, 4096, 4097, 32001])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("bf16", [False, True])
def test_verify(rt, vocab, with_draft, bf16):
    """Odd vocabularies, requests of 0 to 6 drafts, greedy ones among them, rows with a stride of their own."""
    for seed, (n, lo, hi) in enumerate([(1, 0, 0), (1, 6, 6), (9, 0, 4), (5, 2, 3)]):
        say("verify", vocab, with_draft, bf16, n)
        logits, draft, tokens, starts, ua, us, temp = make(seed, n, vocab, lo, hi, bf16)
        draft = draft if with_draft else None
        for limit in (hi, max(0, hi - 2), hi + 3):
            want = rules(logits, draft, tokens, starts, ua, us, temp, limit + 1)
            got = call(rt, logits, draft, tokens, starts, ua, us, temp, limit,
                       torch.bfloat16 if bf16 else torch.float32, pad=seed * 3)
            assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


def test_verify_a_vocabulary_of_a_million(rt):
    logits, draft, tokens, starts, ua, us, temp = make(3, 2, 1 << 20, 1, 2)
    temp[:] = 0.9
    want = rules(logits, draft, tokens, starts, ua, us, temp, 3)
    got = call(rt, logits, draft, tokens, starts, ua, us, temp, 2)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("n, lo, hi, vocab", [(3, 20, 70, 257), (600, 0, 3, 40), (2, 255, 255, 33), (2, 2, 4, 300001)])
@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_many(rt, n, lo, hi, vocab, with_draft):
    """More drafts than a workgroup has waves, many requests, more chunks of a row than a wave has lanes."""
    say("verify many", n, lo, hi, vocab, with_draft)
    logits, draft, tokens, starts, ua, us, temp = make(n, n, vocab, lo, hi)
    ua = (ua * 0.05).astype(np.float32)  # (most drafts accepted)
    draft = draft if with_draft else None
    want = rules(logits, draft, tokens, starts, ua, us, temp, hi + 1)
    got = call(rt, logits, draft, tokens, starts, ua, us, temp, hi)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


def test_verify_special_rows(rt):
    """Masked vocabularies, rows of nothing, infinities, NaN, equal distributions, ties, random numbers at 0 and next
    to 1, drafts without probability and outside the vocabulary."""
    v, inf, nan = 5000, np.inf, np.nan
    rng = np.random.default_rng(0)
    base = rng.standard_normal((2, v)).astype(np.float32)
    near1 = np.float32(1 - 2**-24)
    cases = []
    masked = np.full(v, -inf, np.float32)
    masked[[7, 4999]] = [1.0, 2.0]
    nothing, nans = np.full(v, -inf, np.float32), np.full(v, nan, np.float32)
    mixed = base[0].copy()
    mixed[::3] = nan
    infs = base[0].copy()
    infs[[11, 4500]] = inf
    ties = np.zeros(v, np.float32)
    low = np.full(v, np.finfo(np.float32).min, np.float32)
    low[4999] = -1.0
    for row in (masked, nothing, nans, mixed, infs, ties, low, base[0]):
        for drow in (row, base[1], masked, infs):
            for d in (7, 11, 4999, -1, v, 2**31 - 1, 0):
                cases.append((row, drow, d))
    n = len(cases)
    logits = np.stack([x for r, _, _ in cases for x in (r, r)])
    draft = np.stack([x for _, q, _ in cases for x in (q, q)])
    tokens = np.array([x for _, _, d in cases for x in (3, d)])
    starts = np.arange(n + 1) * 2
    for t in (0.0, 0.7, 1e-30, 1e30):
        for u1, u2 in ((0.0, 0.0), (near1, near1), (0.4, 0.6)):
            say("special", t, u1)
            for q in (draft, None):
                args = (logits, q, tokens, starts, np.full(2 * n, u1), np.full(n, u2), np.full(n, t, np.float32))
                want, got = rules(*args, 2), call(rt, *args, 1)
                assert np.array_equal(got[1], want[1])
                # (T = 1e30 leaves 5000 tokens of all but equal weight: the border at u2 lies between two of them
                # unless u2 is next to one of their sums)
                assert np.array_equal(got[0], want[0])


def test_verify_rows_of_requests(rt):
    """Requests without rows; starts past the rows are cut; a missing temperature is 1."""
    logits, draft, tokens, starts, ua, us, temp = make(1, 4, 300, 2, 2)
    odd = [0, 3, 3, 6, 12]
    want = rules(logits, draft, tokens, odd, ua, us, np.ones(4), 9)
    got = call(rt, logits, draft, tokens, odd, ua, us, None, 8)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0]) and got[1][1] == 0
    a, b = call(rt, logits, draft, tokens, [-4, 3, 2, 900, 2**31 - 1], ua, us, None, 8)
    assert (b >= 0).all() and (b <= 9).all() and a.max() < 300


def test_verify_is_the_targets_distribution(rt):
    """One draft of each of 60000 requests drawn from q: the first token comes out distributed as p.  5 standard
    deviations of a binomial count per token, 12 tokens."""
    n, v = 20000, 12
    rng = np.random.default_rng(8)
    p, q = rng.standard_normal(v) * 1.5, rng.standard_normal(v) * 1.5
    counts = np.zeros(v)
    for _ in range(3):
        d = rng.choice(v, n, p=dist(q, 1.0))
        tokens = np.stack([np.zeros(n, np.int64), d], 1).reshape(-1)
        logits, draft = np.tile(p.astype(np.float32), (2 * 4000, 1)), np.tile(q.astype(np.float32), (2 * 4000, 1))
        for i in range(0, n, 4000):
            out, _ = call(rt, logits, draft, tokens[2 * i:2 * i + 8000], np.arange(4001) * 2,
                          rng.random(8000, np.float32), rng.random(4000, np.float32), None, 1)
            counts += np.bincount(out[:, 0], minlength=v)
    want = dist(p.astype(np.float32), 1.0)
    total = counts.sum()
    assert (np.abs(counts - total * want) <= 5 * np.sqrt(total * want * (1 - want))).all()


def test_verify_captured(rt):
    """A captured call, replayed with other logits, drafts and lengths between eager work; the same bits each time."""
    v, rows, n = 40001, 24, 6
    dev = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device="cuda")
    buf = dict(logits=torch.zeros((rows, v), device="cuda"), draft=torch.zeros((rows, v), device="cuda"),
               tokens=dev([0] * rows, torch.int32), starts=dev([0] * (n + 1), torch.int32),
               ua=torch.zeros(rows, device="cuda"), us=torch.zeros(n, device="cuda"), temp=torch.zeros(n, device="cuda"))
    out = (torch.zeros((n, 5), dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"))

    def step():
        rt.verify_drafts(buf["logits"], buf["tokens"], buf["starts"], buf["ua"], buf["us"], 4, draft_logits=buf["draft"],
                         temperature=buf["temp"], out=out)
    rt.reserve_workspace(int(rt.library().lib.rt_hip_verify_drafts_workspace_bytes(v, n, rows, 4, 1)))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for seed in range(5):
        logits, draft, tokens, starts, ua, us, temp = make(seed, n, v, 0, 3)
        m = len(tokens)
        for name, x in (("logits", logits), ("draft", draft), ("tokens", tokens), ("ua", ua)):
            buf[name][:m].copy_(torch.from_numpy(np.asarray(x)))
        buf["starts"].copy_(torch.from_numpy(starts))
        buf["us"].copy_(torch.from_numpy(us))
        buf["temp"].copy_(torch.from_numpy(temp))
        want = rules(logits, draft, tokens, starts, ua, us, temp, 5)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert np.array_equal(out[0].cpu().numpy(), want[0]) and np.array_equal(out[1].cpu().numpy(), want[1])
            step()
            torch.cuda.synchronize()
            assert np.array_equal(out[0].cpu().numpy(), want[0])
