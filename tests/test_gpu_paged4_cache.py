"""The 4-bit cache: append against the definition, value for value, and paged_read of every kind of cache."""
import pytest
import torch

from helpers import say
from paged4 import filled, kept

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=12345.0), torch.nan_to_num(b.double(), nan=12345.0))


@pytest.mark.parametrize("src", list(DT))
@pytest.mark.parametrize("dim, heads, page, tokens, joint", [
    (128, 8, 16, 1, False), (128, 2, 8, 7, True), (64, 1, 16, 129, False), (64, 5, 64, 40, True), (256, 3, 32, 100, False),
    (256, 1, 1024, 1500, True), (128, 8, 16, 4096, False)])
def test_append_and_read(rt, src, dim, heads, page, tokens, joint):
    say("append4", src, dim, heads, page, tokens, joint)
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    n_pages = -(-tokens // page) + 3
    kv = filled(rt, n_pages, page, heads, dim, joint)
    scale = torch.exp(torch.randn((tokens, 1, 1), generator=g, device="cuda") * 2)
    rows = (torch.randn((tokens, 3 * heads, dim), generator=g, device="cuda") * scale + 0.3).to(DT[src])
    k, v = rows[:, heads:2 * heads], rows[:, 2 * heads:]  # part of a joint projection
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
    if tokens > 3:
        slots[1], slots[2] = -1, n_pages * page
    rt.paged_append(kv, k, v, slots)
    ok = (slots >= 0) & (slots < n_pages * page)
    got_k, got_v = rt.paged_read(kv, slots)
    assert got_k.dtype == torch.float16
    for got, x in ((got_k, k), (got_v, v)):
        assert same(got, torch.where(ok[:, None, None], kept(x), 0.0))
    # the other slots are as they were, and no code touches a neighbour's
    other = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    other[slots[ok].long()] = False
    for x in rt.paged_read(kv, torch.nonzero(other)[:, 0].to(torch.int32)):
        assert torch.isnan(x).all()


def test_a_token_again(rt):
    """A slot that is written again holds what came last, its neighbours what they had."""
    kv = filled(rt, 2, 16, 2, 64)
    x = torch.randn((32, 2, 64), device="cuda")
    all_ = torch.arange(32, dtype=torch.int32, device="cuda")
    rt.paged_append(kv, x, -x, all_)
    y = torch.randn((3, 2, 64), device="cuda") * 9
    at = torch.tensor([5, 17, 6], dtype=torch.int32, device="cuda")
    rt.paged_append(kv, y, y + 1, at)
    want_k, want_v = kept(x), kept(-x)
    want_k[at.long()], want_v[at.long()] = kept(y), kept(y + 1)
    k, v = rt.paged_read(kv, all_, dtype=torch.float32)
    assert same(k, want_k) and same(v, want_v)


def test_special_groups(rt):
    """Groups of one value, of zeros, of values that f16 hardly holds, at the limit and past it, not finite; ties."""
    say("special groups")
    rows = torch.randn((16, 1, 128), device="cuda")
    rows[0] = 0.0
    rows[1] = 3.14159
    rows[2] *= 1e-8
    rows[3] *= 1e-6
    rows[4, 0, :32] = torch.linspace(-16384, 16384, 32, device="cuda")
    rows[5, 0, 40] = 16400.0
    rows[6, 0, 70] = float("inf")
    rows[7, 0, 127] = float("nan")
    rows[8, 0, 0] = -float("inf")
    rows[9, 0, :64] = torch.arange(64, device="cuda") / 4 + 0.125  # a is a power of two times 31 / 30: many ties
    rows[10, 0, :32] = torch.arange(32, device="cuda") * 15 / 64   # steps of exactly half a code
    rows[11] = rows[11] * 1e-3 + 1000
    rows[12] = -0.0
    rows[13, 0, 1:32] = 0.0
    rows[14] = 3e38
    rows[15] = 1e-42
    kv = filled(rt, 2, 8, 1, 128)
    slots = torch.arange(16, dtype=torch.int32, device="cuda")
    rt.paged_append(kv, rows, rows.flip(0).contiguous(), slots)
    k, v = rt.paged_read(kv, slots)
    assert same(k, kept(rows)) and same(v, kept(rows.flip(0)))
    nan = torch.isnan(k[:, 0]).view(16, 4, 32)
    assert torch.equal(nan.any(-1), nan.all(-1))
    want = torch.zeros((16, 4), dtype=torch.bool, device="cuda")
    want[5, 1] = want[6, 2] = want[7, 3] = want[8, 0] = True
    want[14] = True
    assert torch.equal(nan.all(-1), want)


@pytest.mark.parametrize("cache", list(DT))
@pytest.mark.parametrize("dst", list(DT))
def test_read_of_other_caches(rt, cache, dst):
    say("read", cache, dst)
    raw = torch.randn((9, 2, 16, 3, 64), device="cuda").to(DT[cache])
    kv = rt.PagedKV(raw[:, 0], raw[:, 1])
    slots = torch.tensor([0, 143, 7, -1, 144, 7, 100, -(2**31)], dtype=torch.int32, device="cuda")
    joint = torch.full((8, 6, 64), 5.0, dtype=DT[dst], device="cuda")
    rt.paged_read(kv, slots, out=(joint[:, :3], joint[:, 3:]))
    ok = (slots >= 0) & (slots < 144)
    at = torch.where(ok, slots, 0).long()
    for i in range(2):
        want = raw[:, i].reshape(144, 3, 64)[at].to(DT[dst])
        assert torch.equal(joint[:, 3 * i:3 * i + 3], torch.where(ok[:, None, None], want, 0.0))
    a, b = rt.paged_read(kv, slots[:0])
    assert a.shape == b.shape == (0, 3, 64) and a.dtype == DT[cache]


def test_far_pages(rt):
    """Offsets past 2^32 bytes: the pages of a cache of 5 GB."""
    page, heads, dim = 1024, 16, 128
    size = rt.paged_page_bytes(rt.Q4KV, page, heads, dim)
    n_pages = 5 * 2**30 // size
    raw = torch.zeros((2, n_pages, size), dtype=torch.uint8, device="cuda")
    kv = rt.PagedKV4(raw[0], raw[1], page, heads, dim)
    slots = torch.tensor([0, 3, n_pages * page - 1, n_pages * page - 9, n_pages // 2 * page], dtype=torch.int32, device="cuda")
    x = torch.randn((5, heads, dim), device="cuda")
    rt.paged_append(kv, x, 2 * x, slots)
    k, v = rt.paged_read(kv, slots)
    assert same(k, kept(x)) and same(v, kept(2 * x))
    q = torch.randn((1, heads, dim), device="cuda")
    table = torch.full((1, 1), n_pages - 1, dtype=torch.int32, device="cuda")
    start, n = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([page], dtype=torch.int32, device="cuda")
    out = rt.paged_attention(q, kv, table, start, n, 0.1)
    keys, values = (t.double() for t in rt.paged_read(kv, torch.arange(page, device="cuda", dtype=torch.int32) + (n_pages - 1) * page))
    p = torch.softmax(0.1 * (keys * q[0].double()).sum(-1), 0)
    want = (p[:, :, None] * values).sum(0)
    assert (out[0] - want).abs().max() < 2e-6  # (f32 rows: sums of 1024 values below 6, of which two are not 0)


def test_captured(rt):
    kv = filled(rt, 4, 16, 2, 128, byte=0)
    x = torch.randn((20, 2, 128), device="cuda")
    slots = torch.arange(20, dtype=torch.int32, device="cuda")
    out = torch.zeros((2, 20, 2, 128), device="cuda")
    graph = torch.cuda.CUDAGraph()
    rt.paged_append(kv, x, x, slots)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        rt.paged_append(kv, x, x, slots)
        rt.paged_read(kv, slots, out=(out[0], out[1]))
    for i in range(3):
        x.copy_(torch.randn(x.shape, device="cuda"))
        slots.copy_(torch.randperm(64, device="cuda")[:20])
        graph.replay()
        torch.cuda.synchronize()
        assert same(out[0], kept(x)) and same(out[1], kept(x)), i


def many_slots(order, tokens, n_slots):
    """Slots of many tokens: from the first on, from an odd one on, in pieces of every length, in any order."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    n = torch.arange(tokens, device="cuda")
    if order == "first":
        slots = n
    elif order == "odd":
        slots = n + 1
    elif order == "pieces":  # (-1 now and then, then a hole)
        slots = n + n // 7
        slots[::61] = -1
    else:
        slots = torch.randperm(n_slots, generator=g, device="cuda")[:tokens]
    slots = slots.to(torch.int32)
    if order != "any":
        slots[tokens // 2 // 4 * 4 + 3] = n_slots  # (one of four in a row is none)
    return slots


@pytest.mark.parametrize("order", ["first", "odd", "pieces", "any"])
@pytest.mark.parametrize("src, dim, heads, page, tokens", [("bf16", 256, 8, 32, 2051), ("f32", 128, 8, 8, 4099),
                                                           ("f16", 64, 24, 512, 2742)])
def test_many_tokens(rt, src, dim, heads, page, tokens, order):
    say("many", src, dim, heads, page, tokens, order)
    g = torch.Generator(device="cuda").manual_seed(dim)
    n_pages = -(-(tokens + tokens // 7 + 2) // page)
    n_slots = n_pages * page
    kv = filled(rt, n_pages, page, heads, dim)
    rows = (torch.randn((tokens, 2 * heads, dim), generator=g, device="cuda") * 3).to(DT[src])
    k, v = rows[:, :heads], rows[:, heads:]
    slots = many_slots(order, tokens, n_slots)
    rt.paged_append(kv, k, v, slots)
    ok = (slots >= 0) & (slots < n_slots)
    got = rt.paged_read(kv, slots)
    one = [rt.paged_read(kv, part) for part in slots.split(500)]  # (few at a time)
    for i, x in enumerate((k, v)):
        assert same(got[i], torch.where(ok[:, None, None], kept(x), 0.0))
        assert same(got[i], torch.cat([o[i] for o in one]))
    other = torch.ones(n_slots, dtype=torch.bool, device="cuda")
    other[slots[ok].long()] = False
    for x in rt.paged_read(kv, torch.nonzero(other)[:, 0].to(torch.int32)):
        assert torch.isnan(x).all()


@pytest.mark.parametrize("cache", list(DT))
def test_many_tokens_of_other_caches(rt, cache):
    raw = torch.randn((2, 300, 16, 8, 128), device="cuda").to(DT[cache])
    kv = rt.PagedKV(raw[0], raw[1])
    slots = torch.randint(-3, 4810, (4101,), device="cuda", dtype=torch.int32)
    ok = (slots >= 0) & (slots < 4800)
    for i, got in enumerate(rt.paged_read(kv, slots)):
        want = raw[i].reshape(4800, 8, 128)[torch.where(ok, slots, 0).long()]
        assert torch.equal(got, torch.where(ok[:, None, None], want, 0.0))
