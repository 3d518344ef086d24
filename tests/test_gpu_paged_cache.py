"""rt_hip_paged_plan against its rules request by request, rt_hip_paged_append
against the rounding of torch's casts."""
import numpy as np
import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x, np.int64).astype(np.int32).reshape(-1), device="cuda")


def plan_rules(cached, fresh, held, table, queue, head, free, page, tokens):
    """The documented rules, one request after the other."""
    table, queue = table.copy(), queue.copy()
    n, cols = table.shape
    cap = len(queue)
    slots, positions = np.full(tokens, -1), np.full(tokens, -1)
    q_start, kv_len, held_out = [0], [], []
    rows, wanted, back = 0, 0, 0
    taken, stuck, given = 0, False, []
    for s in range(n):
        new = max(int(fresh[s]), 0)
        rows += new
        start = q_start[-1]
        q_start.append(min(rows, tokens))
        if fresh[s] < 0:
            given += list(table[s, :min(max(held[s], 0), cols)])
            held_out.append(0)
            kv_len.append(0)
            continue
        pages = -(-(int(cached[s]) + new) // page)
        want = max(0, pages - int(held[s]))
        ok = cached[s] >= 0 and 0 <= held[s] <= cols and rows <= tokens and pages <= cols
        if ok and want:
            wanted += want
            ok = wanted <= free
        if not ok:
            held_out.append(held[s])
            kv_len.append(0)
            continue
        for c in range(want):
            table[s, held[s] + c] = queue[(head + taken) % cap]
            taken += 1
        held_out.append(held[s] + want)
        kv_len.append(cached[s] + new)
        for i in range(new):
            pos = cached[s] + i
            positions[start + i] = pos
            slots[start + i] = table[s, pos // page] * page + pos % page
    for p in given:
        queue[(head + free + back) % cap] = p
        back += 1
    return dict(q_start=q_start, kv_len=kv_len, slots=slots, positions=positions, held=held_out,
                queue_state=[(head + taken) % cap, free - taken + back], table=table, queue=queue)


def make(seed, n, page, cols, tokens_room, spare, ended=0.1, chunk=40, slack=0.3):
    rng = np.random.default_rng(seed)
    fresh = rng.integers(0, chunk + 1, n)
    fresh[rng.random(n) < ended] = -1
    most = max(1, cols * page - chunk)
    cached = rng.integers(0, most + 1, n)
    held = -(-cached // page)
    held = np.where(rng.random(n) < slack, np.minimum(held + rng.integers(0, 3, n), cols), held)
    n_pages = int(held.sum()) + spare
    ids = rng.permutation(n_pages)
    table = np.full((n, cols), -1)
    at = 0
    for s in range(n):
        table[s, :held[s]] = ids[at:at + held[s]]
        at += held[s]
    head = int(rng.integers(n_pages))
    queue = np.full(n_pages, -7)
    queue[(head + np.arange(spare)) % n_pages] = ids[at:]
    return cached, fresh, held, table, queue, head, spare, page, int(np.maximum(fresh, 0).sum()) + tokens_room


def check(rt, cached, fresh, held, table, queue, head, free, page, tokens, in_place=False):
    want = plan_rules(cached, fresh, held, table, queue, head, free, page, tokens)
    d = dict(cached=i32(cached), fresh=i32(fresh), held=i32(held), queue=i32(queue), state=i32([head, free]))
    t = i32(table).reshape(table.shape)
    plan = rt.PagedPlan(len(cached), tokens, "cuda", d["held"], d["state"]) if in_place else None
    plan = rt.paged_plan(d["cached"], d["fresh"], d["held"], t, d["queue"], d["state"], page, tokens, plan=plan)
    got = dict(q_start=plan.q_start, kv_len=plan.kv_len, slots=plan.slots, positions=plan.positions, held=plan.held,
               queue_state=plan.queue_state, table=t, queue=d["queue"])
    for name, v in want.items():
        assert np.array_equal(got[name].cpu().numpy(), np.asarray(v)), name


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n, page, cols, room, spare, chunk", [
    (1, 16, 4, 0, 40, 1), (1, 8, 1, 3, 9, 8), (3, 16, 5, 0, 2, 40), (64, 16, 33, 7, 64, 1), (65, 128, 9, 1, 12, 300),
    (256, 32, 17, 0, 200, 60), (257, 8, 65, 100, 300, 9), (1000, 16, 40, 5, 1500, 100), (1025, 64, 6, 0, 300, 70),
    (4096, 16, 8, 33, 900, 30)])
def test_plan(rt, n, page, cols, room, spare, chunk, in_place):
    """Odd sizes, requests in one and several rounds of the scans, pages that run out, ended requests, pages in hand."""
    say("plan", n, page, cols)
    for seed in range(3):
        check(rt, *make(seed, n, page, cols, room, spare, chunk=chunk), in_place=in_place)


def test_plan_many_tokens(rt):
    """More than one workgroup, and requests that are very unequal; in place too."""
    for seed, in_place in ((0, False), (1, True)):
        c, f, h, t, q, head, free, page, _ = make(seed, 40, 16, 4000, 0, 9000, chunk=5)
        f[7], c[7] = 50000, 3
        c[11], f[11] = 0, 4097
        h[7], h[11] = 1, 0
        check(rt, c, f, h, t, q, head, free, page, int(np.maximum(f, 0).sum()) + 5000, in_place=in_place)


def test_plan_refused_requests(rt):
    """No room in the table's row, in the rows, or bad numbers: not served, the others are."""
    c, f, h = np.array([10, 60, 5, -3, 20, 0, 9]), np.array([6, 9, 0, 2, 1, 30, 1]), np.array([1, 4, 1, 0, 9, 0, 1])
    table = np.arange(7 * 4).reshape(7, 4)
    queue = np.arange(40)
    for tokens in (100, 49, 48, 20, 6, 0):
        check(rt, c, f, h, table, queue, 30, 10, 16, tokens)
    for free in (0, 1, 2, 3):
        check(rt, c, f, h, table, queue, 39, free, 16, 60)


def test_plan_empty_steps(rt):
    z = np.zeros(0, np.int64)
    check(rt, z, z, z, np.zeros((0, 3), np.int64), np.arange(4), 1, 2, 16, 5)
    check(rt, np.array([0, 7]), np.array([0, 0]), np.array([0, 1]), np.array([[-1], [2]]), np.arange(4), 3, 1, 8, 0)
    check(rt, np.array([16, 7]), np.array([-1, -1]), np.array([2, 0]), np.array([[5, 4], [-1, -1]]), np.arange(9), 8, 1, 8, 3)


def test_plan_survives_a_broken_state(rt):
    """A queue state and table that make no sense: nothing outside the buffers, slots only of the cache's pages."""
    n, tokens, page = 5, 60, 16
    big = 2**31 - 1
    held, table = i32([1, 2, 0, 3, 1]), i32(np.array([[big, -5, 7]] * n)).reshape(n, 3)
    for state in ([-9, 50], [big, big], [-2**31, -1], [3, 4]):
        q = i32([big, -1, 2, 900, -2**31, 1])
        plan = rt.paged_plan(i32([3, 20, 0, big, 16]), i32([4, 9, 17, 5, 10]), held, table, q, i32(state), page, tokens)
        slots = plan.slots.cpu().numpy()
        assert ((slots >= -1) & (slots < 6 * page)).all()
        assert (plan.q_start.cpu().numpy() == [0, 4, 13, 30, 35, 45]).all()


def test_plan_step_captured(rt):
    """A captured plan with its state in place: every replay is the next step."""
    n, page, cols, tokens = 37, 16, 12, 37 * 3
    rng = np.random.default_rng(5)
    cached, held = np.zeros(n, np.int64), np.zeros(n, np.int64)
    table, queue, head, free = np.full((n, cols), -1), rng.permutation(400), 17, 400
    d = dict(cached=i32(cached), fresh=i32(np.zeros(n)), held=i32(held), queue=i32(queue), state=i32([head, free]))
    t = i32(table).reshape(n, cols)
    plan = rt.PagedPlan(n, tokens, "cuda", d["held"], d["state"])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        rt.paged_plan(d["cached"], d["fresh"], d["held"], t, d["queue"], d["state"], page, tokens, plan=plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.paged_plan(d["cached"], d["fresh"], d["held"], t, d["queue"], d["state"], page, tokens, plan=plan)
    for step in range(40):
        fresh = rng.integers(0, 4, n)
        fresh[cached + fresh > cols * page] = -1
        fresh[rng.random(n) < 0.05] = -1
        want = plan_rules(cached, fresh, held, table, queue, head, free, page, tokens)
        d["cached"].copy_(i32(cached))
        d["fresh"].copy_(i32(fresh))
        graph.replay()
        torch.cuda.synchronize()
        got = dict(q_start=plan.q_start, kv_len=plan.kv_len, slots=plan.slots, positions=plan.positions, held=plan.held,
                   queue_state=plan.queue_state, table=t, queue=d["queue"])
        for name, v in want.items():
            assert np.array_equal(got[name].cpu().numpy(), np.asarray(v)), (step, name)
        cached = np.where(fresh < 0, 0, np.asarray(want["kv_len"]))
        held, table, queue = np.asarray(want["held"]), want["table"], want["queue"]
        head, free = want["queue_state"]


DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("src", list(DT))
@pytest.mark.parametrize("dst", list(DT))
@pytest.mark.parametrize("tokens, heads, dim, page, joint", [
    (1, 1, 64, 8, False), (7, 3, 128, 16, True), (40, 8, 128, 16, False), (129, 5, 64, 32, True), (33, 2, 256, 8, True)])
def test_append(rt, src, dst, tokens, heads, dim, page, joint):
    """Every pair of types: the values of torch's casts, bit for bit; rows of a joint projection; k and v pages in
    one tensor; rows without a slot, or with one outside the cache, leave it as it was."""
    say("append", src, dst, tokens)
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn((tokens, (4 if joint else 2) * heads, dim), generator=g) * 3
    x[0, 0, :6] = torch.tensor([0.0, -0.0, 1e-7, 70000.0, 6e-8, -1e38])
    x[-1, -1, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    x = x.to(DT[src]).cuda()
    k, v = x[:, -2 * heads:-heads], x[:, -heads:]
    pages = tokens // page + 3
    both = torch.randn((pages, 2, page, heads, dim), generator=g).to(DT[dst]).cuda()
    want = both.clone()
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    if tokens > 6:
        slots[1], slots[4], slots[5] = -1, pages * page, -2**31
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want[s // page, 0, s % page] = k[t].to(DT[dst])
            want[s // page, 1, s % page] = v[t].to(DT[dst])
    rt.paged_append(rt.PagedKV(both[:, 0], both[:, 1]), k, v, slots.cuda())
    bits = torch.int32 if dst == "f32" else torch.int16
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(both), nan)
    assert torch.equal(both.view(bits)[~nan], want.view(bits)[~nan])


def test_append_far_pages(rt):
    """Pages whose offsets pass 32 bits: 2.2 GiB of f32 keys, the last page and one past the 2^31st byte."""
    heads, dim, page = 8, 256, 128
    pages = (9 << 28) // (page * heads * dim * 4)
    k = torch.zeros((pages, page, heads, dim), device="cuda")
    v = torch.zeros_like(k)
    x = torch.randn((3, heads, dim), device="cuda")
    slots = [pages * page - 1, (1 << 31) // (heads * dim * 4) + 5, 0]
    rt.paged_append(rt.PagedKV(k, v), x, -x, i32(slots))
    for i, s in enumerate(slots):
        assert torch.equal(k[s // page, s % page], x[i]) and torch.equal(v[s // page, s % page], -x[i])
    assert int((k != 0).sum()) == int((x != 0).sum())
