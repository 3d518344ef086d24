"""A server's step with a 4-bit cache, adapters and rules for the logits, as they are
used together: plan, projections with adapters, append, attention, adjusted logits,
verified drafts; eagerly and as one captured graph, against decoding token by token
in float64 by the definitions."""
import math

import numpy as np
import pytest
import torch

from helpers import say
from paged4 import kept

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE, VOCAB, RANK = 8, 2, 64, 16, 600, 16
HIDDEN = HEADS * DIM
SEQS, TOKENS, COLS, PAGES, WIDTH, LONGEST = 4, 28, 8, 30, 5, 100
ADAPTER = [1, -1, 0, 1]


def i32(x):
    return torch.tensor(np.asarray(x, np.int64), device="cuda").to(torch.int32)


class Weights:
    def __init__(self, rt):
        g = torch.Generator(device="cuda").manual_seed(11)
        randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
        self.emb = (randn(VOCAB, HIDDEN) * 0.5).to(torch.bfloat16).float()  # (what a product of many rows takes as it is)
        self.w = (randn(HIDDEN, HIDDEN) * 0.04).to(torch.bfloat16)
        self.head = randn(VOCAB, HIDDEN) * 0.5
        # (keys and values by token: the same bits in a step of any size)
        self.k, self.v = (randn(VOCAB, KV_HEADS, DIM) for _ in range(2))
        self.a = (randn(2, RANK, HIDDEN) / math.sqrt(HIDDEN)).to(torch.bfloat16)
        self.b = (randn(2, HIDDEN, RANK) / math.sqrt(RANK)).to(torch.bfloat16)
        self.scale = torch.tensor([1.5, 0.7], device="cuda")
        # the second request's answers avoid some tokens, the third's keep to a grammar
        self.bias_start, self.bias_token = i32([0, 0, 3, 3, 4]), i32([5, 77, 5, 9])
        self.bias = torch.tensor([3.0, -8.0, -2.0, 4.0], device="cuda")
        self.open = torch.rand((1, VOCAB), generator=g, device="cuda") < 0.3
        bits = torch.zeros((1, (VOCAB + 31) // 32 * 32), dtype=torch.int64, device="cuda")
        bits[:, :VOCAB] = self.open
        words = (bits.view(1, -1, 32) << torch.arange(32, device="cuda")).sum(-1)
        self.mask = torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)
        self.rep = torch.tensor([1.3, 1.0, 1.2, 1.6], device="cuda")
        self.pres = torch.tensor([0.0, 0.5, 0.0, 0.3], device="cuda")
        self.freq = torch.tensor([0.4, 0.2, 0.0, 0.1], device="cuda")
        self.adapters = rt.Adapters(self.a, self.b, self.scale)


class Server:
    """A step's arrays on the device."""

    def __init__(self, rt, weights):
        self.rt, self.w = rt, weights
        size = rt.paged_page_bytes(rt.Q4KV, PAGE, KV_HEADS, DIM)
        raw = torch.full((2, PAGES, size), 255, dtype=torch.uint8, device="cuda")
        self.kv = rt.PagedKV4(raw[0], raw[1], PAGE, KV_HEADS, DIM)
        self.table = torch.full((SEQS, COLS), -1, dtype=torch.int32, device="cuda")
        self.queue, self.state, self.held = i32(range(PAGES)), i32([0, PAGES]), i32([0] * SEQS)
        self.cached, self.fresh, self.tokens = i32([0] * SEQS), i32([0] * SEQS), i32([0] * TOKENS)
        self.plan = rt.PagedPlan(SEQS, TOKENS, "cuda", self.held, self.state)
        self.history, self.history_len, self.prompt_len = i32(np.full((SEQS, LONGEST), -1)), i32([0] * SEQS), i32([0] * SEQS)
        self.mask_row = i32([-1] * TOKENS)
        self.rules = rt.LogitRules(history=self.history, history_len=self.history_len, prompt_len=self.prompt_len,
                                   repetition=weights.rep, presence=weights.pres, frequency=weights.freq,
                                   bias_start=weights.bias_start, bias_token=weights.bias_token, bias=weights.bias,
                                   mask=weights.mask, mask_row=self.mask_row)
        self.adapter = i32(ADAPTER)
        self.out = torch.zeros((TOKENS, HEADS, DIM), device="cuda")
        self.zeros = torch.zeros(TOKENS, device="cuda")
        self.chosen = (torch.zeros((SEQS, WIDTH + 1), dtype=torch.int32, device="cuda"), i32([0] * SEQS))

    def device_step(self):
        rt, w = self.rt, self.w
        rt.paged_plan(self.cached, self.fresh, self.held, self.table, self.queue, self.state, PAGE, TOKENS, plan=self.plan)
        rows = self.tokens.long()
        x = w.emb[rows]
        q = rt.linear_forward(rt.BF16, w.w, x, HIDDEN, HIDDEN)
        rt.lora_add(q, x, w.adapters, self.plan.q_start, self.adapter)
        rt.paged_append(self.kv, w.k[rows], w.v[rows], self.plan.slots)
        rt.paged_attention(q.view(TOKENS, HEADS, DIM), self.kv, self.table, self.plan.q_start, self.plan.kv_len, 1 / math.sqrt(DIM),
                           out=self.out)
        self.logits = (x + 3 * self.out.view(TOKENS, HIDDEN)) @ w.head.T
        rt.adjust_logits(self.logits, self.plan.q_start, self.rules, tokens=self.tokens)
        rt.verify_drafts(self.logits, self.tokens, self.plan.q_start, self.zeros, self.zeros[:SEQS], WIDTH,
                         temperature=self.zeros[:SEQS], out=self.chosen)

    def decode(self, texts, draft, steps, run):
        """Tokens behind the prompts, greedily, with drafts; the prompt's chunk first."""
        prompts = [len(t) for t in texts]
        texts, done = [list(t) for t in texts], [0] * SEQS
        self.prompt_len.copy_(i32(prompts))
        while min(len(t) - p for t, p in zip(texts, prompts)) < steps:
            # a prompt but for its last token in chunks; then the last token, with drafts behind it
            chunks = [t[done[s]:min(done[s] + 7, len(t) - 1)] or [t[-1]] + draft(s, t) for s, t in enumerate(texts)]
            assert sum(map(len, chunks)) <= TOKENS
            flat = [x for c in chunks for x in c]
            self.tokens.copy_(i32(flat + [0] * (TOKENS - len(flat))))
            self.cached.copy_(i32(done)), self.fresh.copy_(i32([len(c) for c in chunks]))
            rows = np.full((SEQS, LONGEST), -1)
            for s, t in enumerate(texts):
                rows[s, :len(t)] = t
            self.history.copy_(i32(rows)), self.history_len.copy_(i32([len(t) for t in texts]))
            of_row = [0 if s == 2 else -1 for s, c in enumerate(chunks) for _ in c]
            self.mask_row.copy_(i32(of_row + [-1] * (TOKENS - len(flat))))
            run()
            torch.cuda.synchronize()
            for s, (line, count) in enumerate(zip(*(x.tolist() for x in self.chosen))):
                if done[s] < len(texts[s]) - 1:
                    done[s] += len(chunks[s])
                else:
                    texts[s] += line[:count]
                    done[s] += count
        return [t[:p + steps] for t, p in zip(texts, prompts)]


def by_definition(w, texts, steps):
    """The same tokens one by one in float64."""
    out = []
    for s, prompt in enumerate(texts):
        text = list(prompt)
        for _ in range(steps):
            at = torch.tensor(text, device="cuda")
            x = w.emb[at[-1]].double()
            q = w.w.double() @ x
            if ADAPTER[s] >= 0:
                i = ADAPTER[s]
                q = q + w.scale[i].double() * (w.b[i].double() @ (w.a[i].double() @ x))
            keys, values = kept(w.k[at]), kept(w.v[at])
            q = q.view(KV_HEADS, HEADS // KV_HEADS, DIM)
            p = torch.softmax((q[None] * keys[:, :, None]).sum(-1) / math.sqrt(DIM), 0)
            o = (p[..., None] * values[:, :, None]).sum(0).reshape(HIDDEN)
            y = w.head.double() @ (x + 3 * o)
            made = text[len(prompt):]
            for t in set(text):
                y[t] = y[t] / w.rep[s].double() if y[t] > 0 else y[t] * w.rep[s].double()
                if t in made:
                    y[t] -= w.freq[s].double() * made.count(t) + w.pres[s].double()
            last = dict(zip(w.bias_token[w.bias_start[s]:w.bias_start[s + 1]].tolist(),
                            w.bias[w.bias_start[s]:w.bias_start[s + 1]].double().tolist()))
            for t, b in last.items():
                y[t] += b
            if s == 2:
                y[~w.open[0]] = -math.inf
            text.append(int(y.argmax()))
        out.append(text)
    return out


@pytest.mark.parametrize("captured", [False, True])
def test_a_server_with_adapters_and_rules(rt, captured):
    say("server4", captured)
    w = Weights(rt)
    rng = np.random.default_rng(5)
    texts = [rng.integers(0, VOCAB, n).tolist() for n in (23, 1, 9, 40)]
    steps = 30
    want = by_definition(w, texts, steps)

    def serve(draft):
        sv = Server(rt, w)
        run = sv.device_step
        if captured:
            rt.reserve_workspace(max(rt.paged_attention_workspace_bytes(sv.kv, rt.F32, HEADS, SEQS, TOKENS),
                                     rt.lora_workspace_bytes(w.adapters, SEQS, TOKENS)))
            sv.device_step()  # (with no fresh tokens: nothing happens)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                sv.device_step()
            run = graph.replay
        return sv.decode(texts, draft, steps, run)

    assert serve(lambda s, t: []) == want
    # drafts that are right for some tokens and then wrong
    guess = lambda s, t: [int(x) if rng.random() < 0.8 else int(rng.integers(VOCAB)) for x in want[s][len(t):len(t) + WIDTH]]  # noqa: E731
    assert serve(guess) == want
    assert all(len(set(t[-steps:])) > 5 for t in want)


def test_two_graphs_share_the_workspace(rt):
    """A graph of single tokens and one of chunks, replayed in turn with eager calls between: each as the eager call."""
    g = torch.Generator(device="cuda").manual_seed(21)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    pages, page = 40, 16
    size = rt.paged_page_bytes(rt.Q4KV, page, KV_HEADS, DIM)
    raw = torch.full((2, pages, size), 255, dtype=torch.uint8, device="cuda")
    kv = rt.PagedKV4(raw[0], raw[1], page, KV_HEADS, DIM)
    rt.paged_append(kv, randn(pages * page, KV_HEADS, DIM), randn(pages * page, KV_HEADS, DIM),
                    torch.arange(pages * page, dtype=torch.int32, device="cuda"))
    adapters = rt.Adapters(randn(3, RANK, HIDDEN).to(torch.bfloat16), randn(3, HIDDEN, RANK).to(torch.bfloat16), randn(3))

    class Calls:
        def __init__(self, rows, lens):
            self.starts, self.lens = i32(np.cumsum([0] + rows)), i32(lens)
            self.adapter = i32(np.arange(len(rows)) % 4 - 1)
            self.table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).repeat(len(rows), 1)
            self.x, self.q, self.y = (randn(sum(rows), HIDDEN) for _ in range(3))
            self.out = torch.zeros((sum(rows), HEADS, DIM), device="cuda")

        def run(self):
            self.y.copy_(self.q)
            rt.lora_add(self.y, self.x, adapters, self.starts, self.adapter)
            rt.paged_attention(self.y.view(-1, HEADS, DIM), kv, self.table, self.starts, self.lens, 1 / math.sqrt(DIM), out=self.out)

        def want(self):
            self.run()
            torch.cuda.synchronize()
            return self.out.clone()

    few, many, other = Calls([1] * 9, [600, 1, 33, 640, 17, 16, 15, 500, 64]), Calls([70, 1, 130], [70, 300, 640]), Calls([5] * 6, [400] * 6)
    rt.reserve_workspace(max(rt.paged_attention_workspace_bytes(kv, rt.F32, HEADS, 9, 201), rt.lora_workspace_bytes(adapters, 9, 201)))
    graphs = []
    for c in (few, many):
        c.want()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.run()
        graphs.append(graph)
    for i in range(3):
        for c in (few, many):
            c.x.copy_(randn(*c.x.shape)), c.q.copy_(randn(*c.q.shape))
        want = [c.want() for c in (few, many)]
        for c in (few, many):
            c.out.fill_(9.0)
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        if i:
            other.run()
        graphs[0].replay()
        torch.cuda.synchronize()
        for c, w in zip((few, many), want):
            assert torch.equal(c.out, w), i
