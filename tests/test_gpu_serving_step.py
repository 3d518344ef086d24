"""The serving calls as they are used together: prompts in chunks, decoding and
verified drafts over one paged cache, against attention over each request's own
keys and values kept aside; eagerly and as one captured graph."""
import math

import numpy as np
import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE, VOCAB = 6, 2, 64, 16, 700


def i32(x):
    return torch.tensor(np.asarray(x, np.int64), device="cuda").to(torch.int32)


class Server:
    """Pages, queue and requests' lengths on the device; the keys and values of each request kept on the host too."""

    def __init__(self, rt, n_seq, pages, cols, tokens, dtype):
        self.rt, self.n, self.tokens, self.dtype = rt, n_seq, tokens, dtype
        self.kv = rt.PagedKV(*torch.full((2, pages, PAGE, KV_HEADS, DIM), float("nan"), dtype=dtype, device="cuda"))
        self.table = torch.full((n_seq, cols), -1, dtype=torch.int32, device="cuda")
        self.queue, self.state = i32(np.random.default_rng(0).permutation(pages)), i32([5, pages])
        self.cached, self.fresh = i32([0] * n_seq), i32([0] * n_seq)
        self.held = i32([0] * n_seq)
        self.plan = rt.PagedPlan(n_seq, tokens, "cuda", self.held, self.state)
        self.q = torch.zeros((tokens, HEADS, DIM), device="cuda", dtype=dtype)
        self.joint = torch.zeros((tokens, 2 * KV_HEADS, DIM), device="cuda")
        self.out = torch.zeros_like(self.q)

    def device_step(self):
        rt = self.rt
        rt.paged_plan(self.cached, self.fresh, self.held, self.table, self.queue, self.state, PAGE, self.tokens, plan=self.plan)
        rt.paged_append(self.kv, self.joint[:, :KV_HEADS], self.joint[:, KV_HEADS:], self.plan.slots)
        rt.paged_attention(self.q, self.kv, self.table, self.plan.q_start, self.plan.kv_len, 1 / math.sqrt(DIM), out=self.out)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_server(rt, captured, dtype):
    say("server", captured, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    rng = np.random.default_rng(2)
    n, tokens = 9, 160
    pages = 26  # (few: some steps find the queue empty)
    sv = Server(rt, n, pages, 12, tokens, dtype)
    kinds = {torch.bfloat16: rt.BF16, torch.float32: rt.F32}
    rt.reserve_workspace(rt.paged_attention_workspace_bytes(sv.kv, kinds[dtype], HEADS, n, tokens))
    graph = None
    if captured:
        sv.device_step()  # (with no fresh tokens: nothing happens)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            sv.device_step()
    kept = [(torch.zeros((0, KV_HEADS, DIM), device="cuda"),) * 2 for _ in range(n)]
    served = refused = ended = 0
    for step in range(60):
        # prompts in chunks, single tokens, chunks of drafts; now and then a request ends
        lens = np.array([k.shape[0] for k, _ in kept])
        fresh = np.where(lens == 0, rng.integers(1, 60, n), rng.choice([0, 1, 1, 1, 4, 6], n))
        fresh[(rng.random(n) < 0.06) | (lens + fresh > 12 * PAGE)] = -1
        while np.maximum(fresh, 0).sum() > tokens:
            fresh[int(np.argmax(fresh))] //= 2
        sv.cached.copy_(i32(lens)), sv.fresh.copy_(i32(fresh))
        sv.q.copy_(torch.randn(sv.q.shape, generator=g, device="cuda"))
        sv.joint.copy_(torch.randn(sv.joint.shape, generator=g, device="cuda"))
        sv.out.fill_(-5.0)
        if graph:
            graph.replay()
        else:
            sv.device_step()
        torch.cuda.synchronize()
        start, kv_len = sv.plan.q_start.tolist(), sv.plan.kv_len.tolist()
        assert (sv.out[start[-1]:] == -5.0).all()
        for s in range(n):
            rows = slice(start[s], start[s + 1])
            if fresh[s] < 0:
                kept[s] = (torch.zeros((0, KV_HEADS, DIM), device="cuda"),) * 2
                ended += 1
                continue
            if kv_len[s] == 0:
                refused += fresh[s] > 0
                assert (sv.out[rows] == 0).all()
                continue
            served += 1
            k, v = (torch.cat([old, new[rows]]) for old, new in zip(kept[s], (sv.joint[:, :KV_HEADS], sv.joint[:, KV_HEADS:])))
            assert kv_len[s] == len(k)
            m = int(fresh[s])
            if m:
                q = sv.q[rows].double().reshape(m, KV_HEADS, HEADS // KV_HEADS, DIM)
                kd, vd = k.to(dtype).double(), v.to(dtype).double()
                score = torch.einsum("mhgd,nhd->hgmn", q, kd) / math.sqrt(DIM)
                hidden = torch.arange(len(k), device="cuda")[None] > torch.arange(len(k) - m, len(k), device="cuda")[:, None]
                p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                want = torch.einsum("hgmn,nhd->mhgd", p, vd).reshape(m, HEADS, DIM)
                size = torch.einsum("hgmn,nhd->mhgd", p, vd.abs()).reshape(m, HEADS, DIM)
                # as in the attention's own test: weights and outputs rounded to 16 bits, f32 sums of 64 products
                # (scores up to 40) and at most 192 keys
                eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
                tol = (eps + 2.0**-24 * (2 * (64 * 40 / 4 + 40 + 32) + 50)) * size + torch.finfo(dtype).eps / 2 * want.abs()
                assert ((sv.out[rows].double() - want).abs() <= tol).all(), (step, s)
            # drafts: all but one of a chunk may be refused, the cache keeps the accepted ones
            keep = len(k) if m < 2 or lens[s] == 0 else len(k) - int(rng.integers(0, m))
            kept[s] = (k[:keep], v[:keep])
        # every page is in the queue or held by one request
        head, free = sv.state.tolist()
        held = sv.held.tolist()
        queue = sv.queue.tolist()
        there = [queue[(head + i) % pages] for i in range(free)]
        there += [p for s in range(n) for p in sv.table[s, :held[s]].tolist()]
        assert sorted(there) == list(range(pages)), step
    assert served > 200 and refused > 5 and ended > 10


def test_drafts_over_a_paged_cache(rt):
    """Greedy drafts of a tiny model verified in chunks give the tokens of decoding one by one."""
    torch.manual_seed(3)
    emb = torch.randn((VOCAB, HEADS * DIM), device="cuda") * 0.5
    wk, wv = (torch.randn((HEADS * DIM, KV_HEADS * DIM), device="cuda") * 0.08 for _ in range(2))
    n, steps, width = 3, 24, 5

    def model(kv, plan, table, tokens):
        """One layer of attention over the embeddings, f32 throughout; logits by the embedding."""
        x = emb[tokens.long()]
        k, v = ((x @ w).view(-1, KV_HEADS, DIM) for w in (wk, wv))
        rt.paged_append(kv, k, v, plan.slots)
        o = rt.paged_attention(x.view(-1, HEADS, DIM), kv, table, plan.q_start, plan.kv_len, 1 / math.sqrt(DIM))
        return (x + 3 * o.reshape(-1, HEADS * DIM)) @ emb.T

    def decode(draft):
        cache = torch.zeros((2, 40, PAGE, KV_HEADS, DIM), device="cuda")
        kv = rt.PagedKV(cache[0], cache[1])
        table, queue, state, held = torch.full((n, 8), -1, dtype=torch.int32, device="cuda"), i32(range(40)), i32([0, 40]), i32([0] * n)
        text = [[7 + 11 * s] for s in range(n)]
        done = [0] * n
        while min(len(t) for t in text) <= steps:
            chunks = [[t[-1]] + draft(s, t) for s, t in enumerate(text)]
            tokens = i32([x for c in chunks for x in c])
            plan = rt.paged_plan(i32(done), i32([len(c) for c in chunks]), held, table, queue, state, PAGE, len(tokens))
            held, state = plan.held, plan.queue_state
            logits = model(kv, plan, table, tokens)
            zeros = torch.zeros(len(tokens), device="cuda")
            out, count = rt.verify_drafts(logits, tokens, plan.q_start, zeros, zeros[:n], width, temperature=torch.zeros(n, device="cuda"))
            for s, (line, c) in enumerate(zip(out.tolist(), count.tolist())):
                text[s] += line[:c]
                done[s] += c
        return [t[:steps] for t in text]

    plain = decode(lambda s, t: [])
    # drafts that are right for some tokens and then wrong
    rng = np.random.default_rng(4)
    guess = lambda s, t: [int(x) if rng.random() < 0.8 else int(rng.integers(VOCAB)) for x in plain[s][len(t):len(t) + width]]
    assert decode(guess) == plain
    assert len({x for t in plain for x in t}) > 3
