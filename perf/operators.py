"""Operators of batched serving over a paged KV cache: their cases, inputs, plain forms and 64-bit results.

Each case is a dict of plain values; `kind` selects the operator:

  plan       pages, block table, slots and positions of a step's new tokens, from the requests' lengths
  append     the step's keys and values into the pages, at those slots
  attention  the step's queries over the pages: single tokens, drafts to verify, chunks of prompts
  verify     drafted tokens accepted or replaced by the target model's distributions

A step of a serving loop is plan, append (each layer), attention (each layer), verify.
"""
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _rt():
    name = "rich_triplet_cpp_amd"
    if name not in sys.modules:
        path = os.path.join(ROOT, "rich-triplet-cpp_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location(name, path, submodule_search_locations=[os.path.dirname(path)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
        mod.rt_hip.init(0)
    return sys.modules[name].rt_hip


# ---------------------------------------------------------------- cases --

def listed():
    return [
        # the bookkeeping before a decode step of 64 requests: one new token each, a page for one in sixteen
        {"name": "plan_decode_64", "kind": "plan", "n_seq": 64, "decode": 1.0, "chunk": 1, "ctx_lo": 20, "ctx_hi": 8192,
         "page": 16, "released": 0, "layout": 1},
        # a busy server's step: a thousand requests, some prompts in chunks, some ended since the last step
        {"name": "plan_mixed_1000", "kind": "plan", "n_seq": 1000, "decode": 0.9, "chunk": 512, "ctx_lo": 1,
         "ctx_hi": 32768, "page": 16, "released": 37, "layout": 2},
        # drafts of 8 requests, 5 tokens each: f32 projections of the library's GEMM into an f16 cache
        {"name": "append_verify_f16", "kind": "append", "tokens": 40, "kv_heads": 8, "head_dim": 128, "src": "f32",
         "dst": "f16", "page": 16, "pages": 512, "layout": 3},
        # a prompt's chunk, bf16 rows of a joint q/k/v projection
        {"name": "append_chunk_bf16", "kind": "append", "tokens": 8192, "kv_heads": 8, "head_dim": 128, "src": "bf16",
         "dst": "bf16", "page": 16, "pages": 1024, "layout": 4},
        # one request, one token, Llama-3.2-3B's heads, the engine's f16 cache and f32 activations
        {"name": "attention_token_f32_f16", "kind": "attention", "q": "f32", "kv": "f16", "heads": 24, "kv_heads": 8,
         "head_dim": 128, "window": 0, "page": 16, "n_seq": 1, "decode": 1.0, "chunk": 1, "ctx_lo": 777, "ctx_hi": 777,
         "layout": 5},
        # a decode step of 64 requests of very different lengths
        {"name": "attention_decode_64_bf16", "kind": "attention", "q": "bf16", "kv": "bf16", "heads": 24,
         "kv_heads": 8, "head_dim": 128, "window": 0, "page": 16, "n_seq": 64, "decode": 1.0, "chunk": 1,
         "ctx_lo": 100, "ctx_hi": 16000, "layout": 6},
        # speculative verify, 16 requests of 5 tokens: a local layer of Gemma-3-4B (head_dim 256, 1024 keys back)
        {"name": "attention_verify_f16_window", "kind": "attention", "q": "f16", "kv": "f16", "heads": 8,
         "kv_heads": 4, "head_dim": 256, "window": 1024, "page": 32, "n_seq": 16, "decode": 0.0, "chunk": 5,
         "ctx_lo": 300, "ctx_hi": 9000, "layout": 7},
        # f32 throughout, as the engine's default cache: a chunk of a prompt over what came before
        {"name": "attention_chunk_f32", "kind": "attention", "q": "f32", "kv": "f32", "heads": 24, "kv_heads": 8,
         "head_dim": 128, "window": 0, "page": 16, "n_seq": 1, "decode": 0.0, "chunk": 517, "ctx_lo": 1100,
         "ctx_hi": 1100, "layout": 8},
        # a step that mixes chunks of prompts with decoding requests, narrow heads
        {"name": "attention_mixed_bf16", "kind": "attention", "q": "bf16", "kv": "bf16", "heads": 32, "kv_heads": 8,
         "head_dim": 64, "window": 0, "page": 64, "n_seq": 35, "decode": 0.9, "chunk": 900, "ctx_lo": 50,
         "ctx_hi": 6000, "layout": 9},
        # the largest: 4096 tokens of a long prompt over 8192 before them
        {"name": "attention_chunk_4096_bf16", "kind": "attention", "q": "bf16", "kv": "bf16", "heads": 24,
         "kv_heads": 8, "head_dim": 128, "window": 0, "page": 16, "n_seq": 1, "decode": 0.0, "chunk": 4096,
         "ctx_lo": 8192, "ctx_hi": 8192, "layout": 10},
        # the engine's largest batch: one request, 7 drafts, drawn from a draft model's distributions
        {"name": "verify_one_7", "kind": "verify", "n_seq": 1, "draft_lo": 7, "draft_hi": 7, "vocab": 128256,
         "dtype": "f32", "draft": True, "greedy": 0.0, "layout": 11},
        # 64 requests with up to 4 drafts, some of them greedy
        {"name": "verify_64", "kind": "verify", "n_seq": 64, "draft_lo": 0, "draft_hi": 4, "vocab": 128256,
         "dtype": "f32", "draft": True, "greedy": 0.25, "layout": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attention", "attention", "attention", "verify"])
    layout = rng.randrange(1 << 30)
    if kind == "plan":
        return {"kind": kind, "n_seq": _log_int(rng, 1, 2000), "decode": rng.choice([0.5, 0.9, 1.0]),
                "chunk": _log_int(rng, 1, 512), "ctx_lo": 1, "ctx_hi": _log_int(rng, 2, 32768),
                "page": rng.choice([8, 16, 32, 64, 128]), "released": rng.choice([0, 0, 1, 5]), "layout": layout}
    if kind == "append":
        src = rng.choice(["f32", "f16", "bf16"])
        page = rng.choice([8, 16, 32, 64, 128])
        tokens = _log_int(rng, 1, 8192)
        return {"kind": kind, "tokens": tokens, "kv_heads": rng.randint(1, 8), "head_dim": rng.choice([64, 128, 256]),
                "src": src, "dst": src if rng.random() < 0.5 else rng.choice(["f32", "f16", "bf16"]), "page": page,
                "pages": (tokens + page - 1) // page + rng.randint(1, 64), "layout": layout}
    if kind == "verify":
        lo = rng.randint(0, 4)
        hi, vocab = lo + rng.randint(0, 3), _log_int(rng, 1000, 262144)
        return {"kind": kind, "n_seq": _log_int(rng, 1, max(1, min(64, int(3e7 / (hi + 1) / vocab)))), "draft_lo": lo,
                "draft_hi": hi, "vocab": vocab, "dtype": rng.choice(["f32", "f32", "bf16"]),
                "draft": rng.random() < 0.7, "greedy": rng.choice([0.0, 0.3, 1.0]), "layout": layout}
    q = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv = q if q != "f32" else rng.choice(["f32", "f16", "bf16"])
    form = rng.choice(["token", "decode", "verify", "chunk", "mixed"])
    case = {"kind": kind, "q": q, "kv": kv, "kv_heads": rng.randint(1, 8), "head_dim": rng.choice([64, 128, 256]),
            "window": _log_int(rng, 1, 4096) if rng.random() < 0.3 else 0, "page": rng.choice([8, 16, 32, 64, 128]),
            "layout": layout}
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 8])
    if form == "token":
        case.update(n_seq=1, decode=1.0, chunk=1, ctx_lo=1, ctx_hi=_log_int(rng, 2, 65536))
    elif form == "decode":
        case.update(n_seq=_log_int(rng, 2, 64), decode=1.0, chunk=1, ctx_lo=1, ctx_hi=_log_int(rng, 2, 8192))
    elif form == "verify":
        case.update(n_seq=_log_int(rng, 1, 32), decode=0.0, chunk=rng.randint(2, 9), ctx_lo=1,
                    ctx_hi=_log_int(rng, 2, 8192))
    elif form == "chunk":
        case.update(n_seq=1, decode=0.0, chunk=_log_int(rng, 16, 1024 if q == "f32" else 2048), ctx_lo=1,
                    ctx_hi=_log_int(rng, 2, 4096))
    else:
        case.update(n_seq=_log_int(rng, 2, 32), decode=0.8, chunk=_log_int(rng, 10, 512), ctx_lo=1,
                    ctx_hi=_log_int(rng, 2, 4096))
    while True:  # no more than the largest listed ones (f32 products cost several times the others)
        w = work(case)
        if w["bytes"] <= 8e8 and w["flops"] <= (6e10 if q == "f32" else 4e11):
            return case
        case["ctx_hi"] = max(2, case["ctx_hi"] * 2 // 3)
        case["chunk"] = max(1, case["chunk"] * 4 // 5)


def _lengths(case):
    """Cached and new tokens of each request: a share `decode` of them one token, the others about `chunk`."""
    rng = random.Random(case["layout"])
    cached = [_log_int(rng, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["n_seq"])]
    if case["ctx_lo"] == case["ctx_hi"]:
        fresh = [case["chunk"]] * case["n_seq"]
    else:
        fresh = [1 if i % 10 < round(10 * case["decode"]) else max(1, case["chunk"] - rng.randint(0, case["chunk"] // 8))
                 for i in range(case["n_seq"])]
    return cached, fresh


def _drafts(case):
    rng = random.Random(case["layout"])
    return [rng.randint(case["draft_lo"], case["draft_hi"]) for _ in range(case["n_seq"])]


def _pages(n, page):
    return (n + page - 1) // page


def _keys(case, c, f):
    """(query, key) pairs of a request and the first key it needs: query i sees keys (c + i - window, c + i]."""
    w = case["window"]
    if not w:
        return f * c + f * (f + 1) // 2, 0
    return sum(min(c + i + 1, w) for i in range(f)), max(0, c - w + 1)


def work(case):
    kind = case["kind"]
    if kind == "plan":
        cached, fresh = _lengths(case)
        tokens, n = sum(fresh), case["n_seq"]
        taken = sum(_pages(c + f, case["page"]) - _pages(c, case["page"]) for c, f in zip(cached, fresh))
        back = sum(_pages(c, case["page"]) for c in cached[:case["released"]])
        # per request three numbers in and three out, per page one read and one written, per token slot and position
        return {"bytes": 4 * (6 * n + 2 * taken + 2 * back + 2 * tokens), "flops": 4 * tokens + 8 * n}
    if kind == "append":
        n = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": n * (BYTES[case["src"]] + BYTES[case["dst"]]) + 4 * case["tokens"], "flops": n}
    if kind == "attention":
        cached, fresh = _lengths(case)
        hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
        size = flops = 0
        for c, f in zip(cached, fresh):
            pairs, first = _keys(case, c, f)
            size += 2 * f * hq * d * BYTES[case["q"]] + 2 * (c + f - first) * hk * d * BYTES[case["kv"]]
            flops += 4 * pairs * hq * d
        return {"bytes": size, "flops": flops}
    drafts, b, v = _drafts(case), BYTES[case["dtype"]], case["vocab"]
    rows = sum(drafts) + case["n_seq"]
    return {"bytes": b * v * (rows + (sum(drafts) if case["draft"] else 0)), "flops": 4 * v * rows}


# --------------------------------------------------------------- inputs --

def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(held, page_ids, cols):
    """Block table whose request i holds the next held[i] of page_ids; what lies behind is -1."""
    t = np.full((len(held), cols), -1, np.int32)
    at = 0
    for i, h in enumerate(held):
        t[i, :h] = page_ids[at:at + h]
        at += h
    return t


def _prepare_plan(case, seed):
    rng = np.random.default_rng(seed)
    page = case["page"]
    cached, fresh = _lengths(case)
    for i in range(min(case["released"], case["n_seq"])):
        fresh[i] = -1
    held = [_pages(c, page) for c in cached]
    need = [max(0, _pages(c + f, page) - h) if f >= 0 else 0 for c, f, h in zip(cached, fresh, held)]
    n_pages = sum(held) + sum(need) + 64
    ids = rng.permutation(n_pages).astype(np.int32)
    cols = max(max(h + n for h, n in zip(held, need)), 1)
    free = n_pages - sum(held)
    head = int(rng.integers(n_pages))
    queue = np.full(n_pages, -1, np.int32)
    queue[(head + np.arange(free)) % n_pages] = ids[sum(held):]
    tokens = sum(max(f, 0) for f in fresh)
    return {"case": case, "tokens": tokens, "cached": _i32(cached), "fresh": _i32(fresh), "held": _i32(held),
            "table": torch.from_numpy(_table(held, ids, cols)).cuda(), "queue": torch.from_numpy(queue).cuda(),
            "queue_state": _i32([head, free])}


def _prepare_append(case, seed):
    g = _gen(seed)
    hk, d, n, page = case["kv_heads"], case["head_dim"], case["tokens"], case["page"]
    # rows of a joint projection: 2 hk heads of queries before the keys and values
    joint = torch.randn((n, 4 * hk, d), generator=g, device="cuda").to(DTYPES[case["src"]])
    cache = torch.zeros((2, case["pages"], page, hk, d), dtype=DTYPES[case["dst"]], device="cuda")
    slots = torch.randperm(case["pages"], generator=g, device="cuda")[:_pages(n, page)]
    slots = (slots[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n].to(torch.int32)
    if n > 8:
        slots[n // 2] = -1  # padding
    state = {"case": case, "k": joint[:, 2 * hk:3 * hk], "v": joint[:, 3 * hk:], "k_pages": cache[0],
             "v_pages": cache[1], "slots": slots}
    return _with_cache(state)


def _prepare_attention(case, seed):
    g = _gen(seed)
    hq, hk, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    cached, fresh = _lengths(case)
    lens = [c + f for c, f in zip(cached, fresh)]
    held = [_pages(n, page) for n in lens]
    n_pages = sum(held) + 8
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu().numpy()
    kv = DTYPES[case["kv"]]
    k = torch.empty((n_pages, page, hk, d), dtype=kv, device="cuda")
    v = torch.empty((n_pages, page, hk, d), dtype=kv, device="cuda")
    for t in (k, v):
        for p in range(0, n_pages, 4096):  # (randn in pieces: f32 of a large cache at once is not needed)
            t[p:p + 4096] = torch.randn(t[p:p + 4096].shape, generator=g, device="cuda").to(kv)
    q = (torch.randn((sum(fresh), hq, d), generator=g, device="cuda") * 1.5).to(DTYPES[case["q"]])
    starts = [0]
    for f in fresh:
        starts.append(starts[-1] + f)
    state = {"case": case, "q": q, "k_pages": k, "v_pages": v, "scale": 1.0 / math.sqrt(d), "lens": lens,
             "fresh": fresh, "starts": starts, "table": torch.from_numpy(_table(held, ids, max(held))).cuda(),
             "q_start": _i32(starts), "kv_len": _i32(lens), "out": torch.zeros_like(q)}
    return _with_cache(state)


def _with_cache(state):
    if own:
        state["kv"] = _rt().PagedKV(state["k_pages"], state["v_pages"])
    return state


def _prepare_verify(case, seed):
    g = _gen(seed)
    drafts, v, n = _drafts(case), case["vocab"], case["n_seq"]
    starts = [0]
    for c in drafts:
        starts.append(starts[-1] + c + 1)
    rows = starts[-1]
    dt = DTYPES[case["dtype"]]
    # a target with a few likely tokens and a draft model near it; each row predicts the token after it
    base = torch.randn((rows, v), generator=g, device="cuda") * 2.5
    target = base.to(dt)
    draft = (base + torch.randn((rows, v), generator=g, device="cuda") * 0.7).to(dt) if case["draft"] else None
    rng = random.Random(seed)
    temp = [0.0 if rng.random() < case["greedy"] else rng.uniform(0.5, 1.2) for _ in range(n)]
    row_temp = torch.tensor([t for t, c in zip(temp, drafts) for _ in range(c + 1)], device="cuda")[:, None]
    near = (draft if draft is not None else target).float()
    noise = -torch.log(-torch.log(torch.rand((rows, v), generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)))
    drawn = torch.argmax(near + noise * row_temp, dim=1).to(torch.int32)  # the draft of a row's successor
    tokens = torch.randint(0, v, (rows,), generator=g, device="cuda", dtype=torch.int32)
    later = [s + i for s, c in zip(starts, drafts) for i in range(1, c + 1)]
    if later:
        at = torch.tensor(later, device="cuda")
        tokens[at] = drawn[at - 1]
    return {"case": case, "logits": target, "draft_logits": draft, "tokens": tokens, "row_start": _i32(starts),
            "starts": starts, "max_draft": max(max(drafts), 1),
            "accept_u": torch.rand((rows,), generator=g, device="cuda"),
            "sample_u": torch.rand((n,), generator=g, device="cuda"),
            "temperature": torch.tensor(temp, dtype=torch.float32, device="cuda")}


# ----------------------------------------------------------- one pass --

def run(state):
    kind = state["case"]["kind"]
    return globals()[("_own_" if own else "_plain_") + kind](state)


def _own_plan(st):
    plan = _rt().paged_plan(st["cached"], st["fresh"], st["held"], st["table"], st["queue"], st["queue_state"],
                            st["case"]["page"], st["tokens"])
    return {"q_start": plan.q_start, "kv_len": plan.kv_len, "slots": plan.slots, "positions": plan.positions,
            "held": plan.held, "queue_state": plan.queue_state, "table": st["table"], "queue": st["queue"]}


def _plain_plan(st):
    cached, fresh, held = (st[x].long() for x in ("cached", "fresh", "held"))
    table, queue, page, tokens = st["table"], st["queue"], st["case"]["page"], st["tokens"]
    n, cols = table.shape
    cap = queue.numel()
    head, free = st["queue_state"].long().unbind()
    new = fresh.clamp(min=0)
    need = ((cached + new + page - 1) // page - held).clamp(min=0)
    need = torch.where(fresh >= 0, need, torch.zeros_like(need))
    fits = held + need <= cols
    want = torch.where(fits, need, torch.zeros_like(need))
    upto = torch.cumsum(want, 0)
    served = fits & ((want == 0) | (upto <= free))
    take = torch.where(served, want, torch.zeros_like(want))
    first = upto - want
    # pages of the queue's front into the tables, ended requests' pages to its end
    col = torch.arange(cols, device=table.device)[None]
    j = col - held[:, None]
    page_id = queue[(head + first[:, None] + j.clamp(min=0)) % cap]
    table.copy_(torch.where((j >= 0) & (j < take[:, None]), page_id, table))
    gone = torch.where(fresh < 0, held, torch.zeros_like(held))
    behind = torch.cumsum(gone, 0) - gone
    dest = torch.where(col < gone[:, None], (head + free + behind[:, None] + col) % cap, torch.full_like(j, cap))
    longer = torch.cat([queue, queue.new_zeros(1)])
    longer.scatter_(0, dest.reshape(-1), table.reshape(-1))
    queue.copy_(longer[:cap])
    q_start = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    kv_len = torch.where(served & (fresh >= 0), cached + new, torch.zeros_like(new))
    t = torch.arange(tokens, device=table.device)
    s = torch.searchsorted(q_start[1:].contiguous(), t, right=True).clamp(max=n - 1)
    pos = cached[s] + t - q_start[s]
    ok = (t < q_start[n]) & served[s]
    slot = table[s, (pos // page).clamp(0, cols - 1)].long() * page + pos % page
    none = torch.full_like(pos, -1)
    held_out = torch.where(fresh < 0, torch.zeros_like(held), held + take)
    state_out = torch.stack([(head + take.sum()) % cap, free - take.sum() + gone.sum()])
    i32 = torch.int32
    return {"q_start": q_start.to(i32), "kv_len": kv_len.to(i32), "slots": torch.where(ok, slot, none).to(i32),
            "positions": torch.where(ok, pos, none).to(i32), "held": held_out.to(i32),
            "queue_state": state_out.to(i32), "table": table, "queue": queue}


def _own_append(st):
    _rt().paged_append(st["kv"], st["k"], st["v"], st["slots"])
    return {"k": st["k_pages"], "v": st["v_pages"]}


def _plain_append(st):
    for src, pages in ((st["k"], st["k_pages"]), (st["v"], st["v_pages"])):
        n_pages, page, hk, d = pages.shape
        flat = pages.view(n_pages * page, hk, d)
        slots = st["slots"].long()
        at = slots.clamp(min=0)
        # a token without a slot writes back the row of token 0, which has one
        rows = torch.where((slots >= 0)[:, None, None], src.float(), src[:1].float()).to(pages.dtype)
        flat[torch.where(slots >= 0, at, at[:1])] = rows
    return {"k": st["k_pages"], "v": st["v_pages"]}


def _own_attention(st):
    return _rt().paged_attention(st["q"], st["kv"], st["table"], st["q_start"], st["kv_len"], st["scale"],
                                 window=st["case"]["window"], max_fresh=max(st["fresh"]), out=st["out"])


def _plain_attention(st):
    """Requests with as many new tokens go together, their keys padded to the longest, as memory allows."""
    case = st["case"]
    page, window = case["page"], case["window"]
    q, k_pages, v_pages, out = st["q"], st["k_pages"], st["v_pages"], st["out"]
    hk, d = k_pages.shape[2:]
    group = q.shape[1] // hk
    order = sorted(range(case["n_seq"]), key=lambda s: (st["fresh"][s], st["lens"][s]))
    batches = []
    for s in order:
        f, longest = st["fresh"][s], st["lens"][s]
        last = batches[-1] if batches else None
        if last and st["fresh"][last[0]] == f and (len(last) + 1) * longest * (hk * d + hk * group * min(f, 1024)) < 1 << 29:
            last.append(s)
        else:
            batches.append([s])
    for batch in batches:
        f, longest, b = st["fresh"][batch[0]], max(st["lens"][s] for s in batch), len(batch)
        if f == 0:
            continue
        seqs = torch.tensor(batch, device=q.device)
        ids = st["table"][seqs, :_pages(longest, page)].clamp(min=0).long()
        keys = ids.shape[1] * page
        lens = st["kv_len"][seqs].long()
        key_at = torch.arange(keys, device=q.device)
        live = key_at[None] < lens[:, None]
        k = k_pages[ids].reshape(b, keys, hk, d).float()
        v = v_pages[ids].reshape(b, keys, hk, d).float()
        k = torch.where(live[:, :, None, None], k, torch.zeros_like(k)).permute(0, 2, 3, 1).contiguous()
        v = torch.where(live[:, :, None, None], v, torch.zeros_like(v)).permute(0, 2, 1, 3).contiguous()
        for i in range(0, f, 1024):
            n = min(1024, f - i)
            rows = (st["q_start"][seqs].long()[:, None] + torch.arange(i, i + n, device=q.device)).reshape(-1)
            x = q[rows].float().reshape(b, n, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * n, d)
            s = torch.matmul(x, k) * st["scale"]
            at = lens[:, None] - f + i + torch.arange(n, device=q.device)[None]
            seen = key_at[None, None] <= at[:, :, None]
            if window:
                seen = seen & (key_at[None, None] > at[:, :, None] - window)
            s = s.reshape(b, hk, group, n, keys).masked_fill_(~seen[:, None, None], float("-inf"))
            s = torch.exp(s - s.amax(-1, keepdim=True))
            s = (s / s.sum(-1, keepdim=True)).reshape(b, hk, group * n, keys)
            o = torch.matmul(s, v).reshape(b, hk, group, n, d).permute(0, 3, 1, 2, 4).reshape(b * n, hk * group, d)
            out[rows] = o.to(out.dtype)
    return out


def _own_verify(st):
    tokens, count = _rt().verify_drafts(st["logits"], st["tokens"], st["row_start"], st["accept_u"], st["sample_u"],
                                        max_draft=st["max_draft"], draft_logits=st["draft_logits"],
                                        temperature=st["temperature"])
    return {"tokens": tokens, "count": count}


def _weights(x, temperature):
    """Rows of probabilities, 64 bits: softmax(x / temperature), the first largest token where that is 0."""
    x = x.double()
    top = x.amax(1, keepdim=True)
    t = temperature.double()[:, None]
    w = torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t)))
    greedy = torch.zeros_like(w).scatter_(1, torch.argmax((x == top).int(), dim=1, keepdim=True), 1.0)
    w = torch.where(t > 0, w, greedy)
    return w / w.sum(1, keepdim=True)


def _plain_verify(st):
    starts, logits, tokens = st["starts"], st["logits"], st["tokens"].long()
    n, width = len(starts) - 1, st["max_draft"] + 1
    rows, vocab = logits.shape
    seq = torch.repeat_interleave(torch.arange(n, device=logits.device), st["row_start"].diff(), output_size=rows)
    p = _weights(logits, st["temperature"][seq])
    row = torch.arange(rows, device=logits.device)
    first = st["row_start"].long()[seq]
    count = st["row_start"].diff().long()
    drafted = row - first + 1 < count[seq]  # this row judges the draft behind it
    after = tokens[(row + 1).clamp(max=rows - 1)]
    if st["draft_logits"] is not None:
        q = _weights(st["draft_logits"], st["temperature"][seq])
    else:
        q = torch.zeros_like(p).scatter_(1, after[:, None], 1.0)
    p_d, q_d = (x.gather(1, after[:, None])[:, 0] for x in (p, q))
    refused = drafted & ~(st["accept_u"].double() * q_d < p_d)
    # the first refused row of each request, or its last row
    stop = torch.where(refused | ~drafted, row, torch.full_like(row, rows))
    stop = torch.full((n,), rows, device=row.device).scatter_reduce_(0, seq, stop, "amin")
    p_s, q_s = p[stop], q[stop]
    rest = (p_s - q_s).clamp(min=0)
    rest = torch.where(refused[stop][:, None] & (rest.sum(1, keepdim=True) > 0), rest, p_s)
    cum = torch.cumsum(rest, 1)
    u = st["sample_u"].double()[:, None] * cum[:, -1:]
    chosen = torch.searchsorted(cum, u, right=True)[:, 0]
    last = vocab - 1 - torch.argmax((rest > 0).int().flip(1), dim=1)
    chosen = torch.minimum(chosen, last)
    accepted = stop - st["row_start"][:-1].long()
    at = torch.arange(width, device=row.device)[None]
    src = (st["row_start"][:-1].long()[:, None] + 1 + at).clamp(max=rows - 1)
    out = torch.where(at < accepted[:, None], tokens[src], torch.full_like(src, -1))
    out = torch.where(at == accepted[:, None], chosen[:, None], out)
    return {"tokens": out.to(torch.int32), "count": (accepted + 1).to(torch.int32)}


# ------------------------------------------------------- 64-bit results --

def exact(case, seed):
    """What run returns, from the definitions, request by request."""
    st = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(st)
    if case["kind"] == "verify":
        return _exact_verify(st)
    if case["kind"] == "append":
        out = {}
        for name in ("k", "v"):
            pages = st[name + "_pages"].double()
            hk, d = pages.shape[2:]
            flat = pages.view(-1, hk, d)
            for t, slot in enumerate(st["slots"].tolist()):
                if slot >= 0:
                    flat[slot] = st[name][t].double()
            out[name] = pages
        return out
    hk, d, page, window = case["kv_heads"], case["head_dim"], case["page"], case["window"]
    group = case["heads"] // hk
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s, (n, length, start) in enumerate(zip(st["fresh"], st["lens"], st["starts"])):
        base = 0 if not window else max(0, length - n - window + 1) // page
        ids = st["table"][s, base:_pages(length, page)].long()
        key = torch.arange(base * page, length, device="cuda")
        for h in range(hk):
            k = st["k_pages"][ids, :, h].reshape(-1, d)[:len(key)].double()
            v = st["v_pages"][ids, :, h].reshape(-1, d)[:len(key)].double()
            for g in range(h * group, (h + 1) * group):
                for i in range(0, n, 2048):
                    m = min(2048, n - i)
                    x = st["q"][start + i:start + i + m, g].double()
                    at = torch.arange(length - n + i, length - n + i + m, device="cuda")[:, None]
                    hidden = key[None] > at
                    if window:
                        hidden |= key[None] <= at - window
                    e = (x @ k.T) * st["scale"]
                    e[hidden] = -math.inf
                    out[start + i:start + i + m, g] = torch.softmax(e, dim=1) @ v
    return out


def _exact_plan(st):
    case, page = st["case"], st["case"]["page"]
    cached, fresh, held = (st[x].tolist() for x in ("cached", "fresh", "held"))
    table, queue = st["table"].cpu().numpy().copy(), st["queue"].cpu().numpy().copy()
    head, free = st["queue_state"].tolist()
    cap, end = len(queue), head + free
    slots, positions = np.full(st["tokens"], -1, np.int64), np.full(st["tokens"], -1, np.int64)
    q_start, kv_len, asked, taken, back = [0], [], 0, 0, 0
    for s in range(case["n_seq"]):
        n, start = max(fresh[s], 0), q_start[-1]
        q_start.append(start + n)
        if fresh[s] < 0:
            for c in range(held[s]):
                queue[(end + back) % cap] = table[s, c]
                back += 1
            held[s] = 0
            kv_len.append(0)
            continue
        need = max(0, _pages(cached[s] + n, page) - held[s])
        if held[s] + need > table.shape[1] or (need and asked + need > free):
            asked += need if held[s] + need <= table.shape[1] else 0
            kv_len.append(0)
            continue
        for c in range(need):
            table[s, held[s] + c] = queue[(head + asked + c) % cap]
        asked += need
        taken += need
        held[s] += need
        kv_len.append(cached[s] + n)
        pos = np.arange(cached[s], cached[s] + n)
        positions[start:start + n] = pos
        slots[start:start + n] = table[s, pos // page].astype(np.int64) * page + pos % page
    return {"q_start": np.array(q_start), "kv_len": np.array(kv_len), "slots": slots, "positions": positions,
            "held": np.array(held), "queue_state": np.array([(head + taken) % cap, free - taken + back]),
            "table": table, "queue": queue}


def _exact_verify(st):
    def distribution(row, t):
        x = row.double()
        if t == 0.0:
            p = torch.zeros_like(x)
            p[int(torch.argmax((x == x.max()).int()))] = 1.0
            return p
        return torch.softmax(x / t, dim=0)

    width = st["max_draft"] + 1
    tokens, temp = st["tokens"].tolist(), st["temperature"].double().tolist()
    accept_u, sample_u = st["accept_u"].double().tolist(), st["sample_u"].double().tolist()
    out, count = [], []
    for s, (a, b) in enumerate(zip(st["starts"], st["starts"][1:])):
        line = []
        for r in range(a, b):
            p = distribution(st["logits"][r], temp[s])
            if r + 1 < b:
                d = tokens[r + 1]
                if st["draft_logits"] is not None:
                    q = distribution(st["draft_logits"][r], temp[s])
                else:
                    q = torch.zeros_like(p)
                    q[d] = 1.0
                if accept_u[r] * float(q[d]) < float(p[d]):
                    line.append(d)
                    continue
                if float((p - q).clamp(min=0).sum()) > 0:
                    p = (p - q).clamp(min=0)
            cum = torch.cumsum(p, 0)
            line.append(int(torch.argmax((cum > sample_u[s] * float(cum[-1])).int())))
            break
        out.append(line + [-1] * (width - len(line)))
        count.append(len(line))
    return {"tokens": np.array(out), "count": np.array(count)}
