"""rt_hip_adjust_logits against its rules, token by token in float64.

Tolerances: each of the up to four operations on a logit (a product or quotient, a
product and two sums) rounds once in f32, 2^-24 of the largest number it meets, S =
|x| (1 + repetition) + frequency c + presence + |bias|; five such at most, and the
result to its type, eps / 2 of it.  What no rule changes has the same bits.
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
    def __init__(self, vocab, rows, dtype=torch.float32, history=50, prompt=0.4, bias=6, masks=3, seed=0, pad=0, spread=None):
        rng = np.random.default_rng(seed)
        self.vocab, self.rows, self.n = vocab, rows, len(rows)
        total = sum(rows)
        self.starts = np.concatenate([[0], np.cumsum(rows)])
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.store = (torch.randn((total + 2, vocab + pad), generator=g, device="cuda") * 3).to(dtype)
        self.logits = self.store[:total, :vocab]
        spread = spread or vocab
        self.history = rng.integers(0, spread, (self.n, history + 5))
        self.history_len = rng.integers(0, history + 1, self.n)
        self.prompt_len = (self.history_len * prompt).astype(int)
        self.tokens = rng.integers(0, spread, total)
        self.rep, self.pres, self.freq = rng.uniform(0.8, 1.5, self.n), rng.uniform(-1, 1, self.n), rng.uniform(-0.2, 0.5, self.n)
        counts = rng.integers(0, bias + 1, self.n)
        self.bias_start = np.concatenate([[0], np.cumsum(counts)])
        self.bias_token = rng.integers(0, max(1, spread // 4) if bias > 20 else spread, counts.sum())
        self.bias = rng.normal(size=counts.sum()) * 4
        words = (vocab + 31) // 32 + 1
        self.mask = rng.integers(0, 2, (max(masks, 1), 32 * words), dtype=np.int64)
        self.mask[0] = 0
        if masks > 2:
            self.mask[2] = rng.random(32 * words) < 0.02
        self.mask_row = rng.integers(-1, masks, total) if masks else np.full(total, -1)

    def rules(self, rt, **over):
        f = lambda x: torch.tensor(np.asarray(x, np.float32), device="cuda")  # noqa: E731
        bits = (self.mask.reshape(len(self.mask), -1, 32) << np.arange(32)).sum(-1)
        bits = np.where(bits >= 1 << 31, bits - (1 << 32), bits)
        a = dict(history=i32(self.history), history_len=i32(self.history_len), prompt_len=i32(self.prompt_len), repetition=f(self.rep),
                 presence=f(self.pres), frequency=f(self.freq), bias_start=i32(self.bias_start), bias_token=i32(self.bias_token),
                 bias=f(self.bias), mask=i32(bits), mask_row=i32(self.mask_row))
        a.update(over)
        self.given = a
        return rt.LogitRules(**a)

    def want(self, logits, drafts=True):
        """(expected in float64, tolerance, changed) by the rules that were given."""
        a, v = self.given, self.vocab
        x = logits.double().cpu().numpy().copy()
        tol = np.zeros_like(x)
        changed = np.zeros(x.shape, bool)
        get = lambda name, s, none: none if a[name] is None else float(a[name][s])  # noqa: E731
        for s in range(self.n):
            text = list(self.history[s, :min(max(self.history_len[s], 0), self.history.shape[1])]) if a["history"] is not None else []
            prompt = self.prompt_len[s] if a["prompt_len"] is not None else 0
            rep, pres, freq = get("repetition", s, 1.0), get("presence", s, 0.0), get("frequency", s, 0.0)
            rep = rep if rep > 0 else 1.0
            bias = {}
            if a["bias"] is not None:
                for i in range(self.bias_start[s], self.bias_start[s + 1]):
                    bias[int(self.bias_token[i])] = float(a["bias"][i])
            for i, r in enumerate(range(self.starts[s], self.starts[s + 1])):
                chosen = list(self.tokens[self.starts[s] + 1:r + 1]) if drafts else []
                t, made = text + chosen, text[max(prompt, 0):] + chosen
                for token in set(t):
                    if not 0 <= token < v:
                        continue
                    old, c = x[r, token], made.count(token)
                    size = abs(old) * (1 + rep + 1 / rep)
                    y = old / rep if old > 0 else old * rep
                    if c:
                        y = y - freq * c - pres
                        size += abs(freq) * c + abs(pres)
                    x[r, token] = y
                    tol[r, token] += size * 5 * 2.0**-24
                    changed[r, token] = True
                for token, b in bias.items():
                    if 0 <= token < v:
                        tol[r, token] += (abs(x[r, token]) + abs(b)) * 2.0**-24
                        x[r, token] += b
                        changed[r, token] = True
                m = self.mask_row[r] if a["mask_row"] is not None else r
                if a["mask"] is not None and 0 <= m < len(self.mask):
                    closed = self.mask[m, :v] == 0
                    x[r, closed] = -math.inf
                    changed[r, closed] = True
        return x, tol + np.where(np.isfinite(x), np.abs(x), 0) * torch.finfo(logits.dtype).eps / 2, changed

    def check(self, rt, drafts=True, **over):
        rules = self.rules(rt, **over)
        before = self.store.clone()
        want, tol, changed = self.want(self.logits, drafts)
        out = rt.adjust_logits(self.logits, i32(self.starts), rules, tokens=i32(self.tokens) if drafts else None)
        assert out is self.logits
        got = self.logits.double().cpu().numpy()
        bad = ~((got == want) | (np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)))
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])
        kept = torch.from_numpy(~changed).cuda()
        old = before[:len(got), :self.vocab]
        bits = torch.int32 if self.logits.dtype == torch.float32 else torch.int16
        assert torch.equal(self.logits.contiguous().view(bits)[kept], old.contiguous().view(bits)[kept])
        self.store[:len(got), :self.vocab] = 0
        before[:len(got), :self.vocab] = 0
        assert torch.equal(self.store, before)  # behind the rows and beside them


DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab, rows, pad", [
    (1, [1], 0), (31, [2, 0, 3], 1), (32, [1, 1], 0), (4096, [1, 4], 0), (4097, [3, 1], 7), (8191, [2], 1), (12289, [1] * 9, 3),
    (50000, [5, 1, 8, 0, 2], 0), (1003, [1] * 70 + [8], 5)])
def test_sizes(rt, dtype, vocab, rows, pad):
    say("adjust", dtype, vocab, rows, pad)
    Case(vocab, rows, dtype, pad=pad, seed=vocab).check(rt)
    Case(vocab, rows, dtype, pad=pad, seed=vocab + 1, spread=min(vocab, 12)).check(rt)  # tokens many times


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("none", [
    ["history", "history_len"], ["prompt_len"], ["repetition"], ["presence", "frequency"], ["bias", "bias_start", "bias_token"],
    ["mask", "mask_row"], ["mask_row"], ["repetition", "presence", "frequency"],
    ["history", "history_len", "prompt_len", "repetition", "presence", "frequency", "mask", "mask_row"],
    ["history", "history_len", "prompt_len", "repetition", "presence", "frequency", "bias", "bias_start", "bias_token"]])
def test_without(rt, dtype, none):
    """Rules of which some are not there; row r has mask r without mask_row."""
    say("adjust without", dtype, none)
    Case(5000, [2, 1, 3], dtype, masks=6, seed=3, spread=300).check(rt, **{x: None for x in none})
    Case(5000, [2, 1, 3], dtype, masks=6, seed=4, spread=300).check(rt, drafts=False, **{x: None for x in none})


def test_no_rules(rt):
    c = Case(3000, [2, 1])
    c.check(rt, **{x: None for x in ("history", "history_len", "prompt_len", "repetition", "presence", "frequency", "bias_start",
                                     "bias_token", "bias", "mask", "mask_row")})


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_histories(rt, dtype):
    """Histories longer than what is loaded at once, of few tokens and of many; entries of one token many times."""
    Case(9000, [1, 3, 2], dtype, history=30000, seed=5, bias=3000).check(rt)
    Case(9000, [1, 3, 2], dtype, history=7001, seed=6, spread=3).check(rt)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, bias", [([1, 90, 3], 6), ([40, 1], 300), ([2, 200], 33)])
def test_many_in_a_place(rt, dtype, rows, bias):
    """More drafts, and more biases, of one request in one part of the vocabulary than are kept in a list."""
    Case(9000, rows, dtype, history=300, seed=14, bias=bias, spread=200).check(rt)
    Case(4100, [2, 1], dtype, history=9000, seed=15, bias=bias, spread=4100).check(rt)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [94, 97])
def test_many_biases_in_a_place(rt, dtype, bias):
    """As many different biases in one part as its table takes, and more."""
    c = Case(4100, [2, 1, 3], dtype, seed=17, bias=bias)
    c.bias_start = np.array([0, bias, bias, 2 * bias])
    c.bias_token = np.concatenate([np.arange(bias), 100 - np.arange(bias)])
    c.bias = np.random.default_rng(0).normal(size=2 * bias)
    c.check(rt)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_requests(rt, dtype):
    """More parts than the card takes at once; among the requests some with long histories, many biases, many drafts."""
    rows = [1, 2, 1] * 66 + [40, 1, 2]
    c = Case(12100, rows, dtype, history=9000, seed=18, bias=4, spread=8000)
    long = c.history_len.copy()
    c.history_len = np.minimum(c.history_len, 40)
    c.history_len[[3, 150]] = long[[3, 150]] = 9000
    c.prompt_len = (c.history_len * 0.3).astype(int)
    c.tokens[c.starts[198]:c.starts[199]] = np.arange(40) % 36 + 4000
    start = c.bias_start[7]
    more = np.random.default_rng(1).integers(0, 300, 150)
    c.bias_token = np.concatenate([c.bias_token[:start], more, c.bias_token[start:]])
    c.bias = np.concatenate([c.bias[:start], np.random.default_rng(2).normal(size=150), c.bias[start:]])
    c.bias_start[8:] += 150
    c.check(rt)


@pytest.mark.parametrize("dtype", DTYPES)
def test_other_stream(rt, dtype):
    """On a stream that has work before it; rows that start anywhere."""
    c = Case(5000, [3, 1, 2], dtype, seed=16)
    stream = torch.cuda.Stream()
    for first in (1, 2, 3):
        c.store = torch.randn((8, 5011), device="cuda").to(dtype)
        c.logits = c.store[:6, :5000]
        shifted = torch.randn((7, 5003), device="cuda").to(dtype)[:6, first:first + 5000]
        rules, starts, tokens = c.rules(rt), i32(c.starts), i32(c.tokens)
        want = shifted.clone()
        rt.adjust_logits(want, starts, rules, tokens=tokens)
        later = torch.zeros_like(shifted)
        keep = torch.full((6, 5003), 7.0, device="cuda", dtype=dtype)
        odd = keep[:, first:first + 5000]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(20):
                later.add_(shifted)
                later.sub_(shifted)
            odd.copy_(shifted)
            rt.adjust_logits(odd, starts, rules, tokens=tokens)
        stream.synchronize()
        assert torch.equal(odd, want)
        assert (keep[:, :first] == 7).all() and (keep[:, first + 5000:] == 7).all()


def test_numbers_out_of_range(rt):
    """Lengths, starts, tokens and masks that are none: nothing outside is read or written."""
    c = Case(600, [2, 3, 1], seed=7, spread=600)
    c.history_len = np.array([-5, 10**9, 20])
    c.history[1, ::3] = -1
    c.history[2, :9] = 600
    c.prompt_len = np.array([-3, 10**9, 5])
    c.bias_start = np.array([0, 2, 2, 5])
    c.bias_token = np.array([-1, 600, 5, 2**31 - 1, 5])
    c.bias = np.array([1.0, 2.0, 3.0, 4.0, 5.0])
    c.tokens[1:4] = [-7, 600, 10**9]
    c.mask_row[:] = [-1, 3, 2, -(2**31), 2**31 - 1, 0]
    c.check(rt)
    for starts in ([-5, 2, 10**9, 6], [6, 6, 6, 6], [9, 9, 9, 12]):
        rt.adjust_logits(c.logits, i32(starts), c.rules(rt), tokens=i32(c.tokens))
    c.bias_start = np.array([-4, 10**9, 2, 3])
    rt.adjust_logits(c.logits, i32([0, 2, 5, 6]), c.rules(rt), tokens=i32(c.tokens))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_that_are_special(rt, dtype):
    """Infinities and NaN among logits, repetitions that are none."""
    c = Case(300, [2, 2, 1], dtype, seed=8, masks=0, bias=0)
    c.rep = np.array([0.0, -2.0, math.nan])
    c.logits[0, ::3], c.logits[1, ::5], c.logits[2, ::7] = math.inf, -math.inf, math.nan
    c.check(rt)


def test_captured(rt):
    """A captured call reads what its tensors hold at each replay."""
    c = Case(20000, [2, 1, 5], seed=9, history=200)
    rules = c.rules(rt)
    starts, tokens = i32(c.starts), i32(c.tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.adjust_logits(c.logits, starts, rules, tokens=tokens)
    for seed in (10, 11, 12):
        d = Case(20000, [2, 1, 5], seed=seed, history=200)
        d.bias_start, d.bias_token = c.bias_start, np.resize(d.bias_token, len(c.bias_token))
        d.bias = np.resize(d.bias, len(c.bias))
        fresh = d.rules(rt)
        for mine, other in zip(rules.tensors, fresh.tensors):
            mine.copy_(other)
        tokens.copy_(i32(d.tokens))
        c.logits.copy_(d.logits)
        graph.replay()
        torch.cuda.synchronize()
        rt.adjust_logits(d.logits, starts, fresh, tokens=tokens)
        assert torch.equal(c.logits, d.logits)


def test_then_verify(rt):
    """Greedy drafts verified on adjusted logits are what a draw token by token would take."""
    vocab, n, width = 400, 3, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    table = torch.randn((vocab, vocab), generator=g, device="cuda")  # logits of the token behind a token
    rep = torch.full((n,), 1.7, device="cuda")
    freq = torch.full((n,), 0.9, device="cuda")

    def step(texts, drafts):
        rows = [[t[-1]] + d for t, d in zip(texts, drafts)]
        tokens, starts = i32([x for r in rows for x in r]), i32(np.cumsum([0] + [len(r) for r in rows]))
        cols = max(len(t) for t in texts)
        rules = rt.LogitRules(history=i32([t + [-1] * (cols - len(t)) for t in texts]), history_len=i32([len(t) for t in texts]),
                              prompt_len=i32([1] * n), repetition=rep, frequency=freq)
        logits = rt.adjust_logits(table[tokens.long()].clone(), starts, rules, tokens=tokens)
        zeros = torch.zeros(len(tokens), device="cuda")
        out, count = rt.verify_drafts(logits, tokens, starts, zeros, zeros[:n], width, temperature=torch.zeros(n, device="cuda"))
        return [t + o[:c] for t, o, c in zip(texts, out.tolist(), count.tolist())]

    plain = [[5], [17], [99]]
    while len(plain[0]) < 40:
        plain = step(plain, [[]] * n)
    rng = np.random.default_rng(0)
    fast = [[5], [17], [99]]
    while min(len(t) for t in fast) < 30:
        guess = [[int(x) if rng.random() < 0.8 else int(rng.integers(vocab)) for x in p[len(t):len(t) + width]] for p, t in zip(plain, fast)]
        fast = step(fast, guess)
    for p, t in zip(plain, fast):
        assert p[:30] == t[:30]
