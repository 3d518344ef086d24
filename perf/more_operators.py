"""Operators of a serving step with a 4-bit KV cache, adapters and constrained sampling: cases, inputs, plain forms and
64-bit results.

Each case is a dict of plain values; `kind` selects the operator:

  append     new keys and values into pages of 4 bits, and read back as the values that these stand for
  attention  the step's queries over such pages: single tokens, drafts to verify, chunks of prompts
  adjust     logits with penalties for repeated tokens, biases and grammar masks, before tokens are drawn or verified
  lora       low-rank adapters of many requests, added to a shared projection's output

Of 32 neighbouring values of a head the 4-bit cache keeps f16 numbers a and b and codes c of 0 .. 15; a code stands for
the f16 number nearest a * (1 + c / 16) + b.  With lo and hi the group's least and greatest value, every step rounded to
f32: a = f16((hi - lo) * (16 / 15)), b = f16(lo - a), c = rint((x - b) * (16 / a)) - 16 within 0 .. 15 (0 where a is 0).
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
        # a decode step of 64 requests: f32 rows of the projection, one token each
        {"name": "append_decode_f32", "kind": "append", "tokens": 64, "kv_heads": 8, "head_dim": 128, "src": "f32",
         "page": 16, "pages": 512, "layout": 1},
        # a prompt's chunk, bf16 rows of a joint q/k/v projection
        {"name": "append_chunk_bf16", "kind": "append", "tokens": 8192, "kv_heads": 8, "head_dim": 128, "src": "bf16",
         "page": 32, "pages": 600, "layout": 2},
        # one request, one token, f32 rows: the latency of a short answer
        {"name": "attention_token_f32", "kind": "attention", "q": "f32", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "window": 0, "page": 16, "n_seq": 1, "decode": 1.0, "chunk": 1, "ctx_lo": 777, "ctx_hi": 777, "layout": 3},
        # a decode step of 64 requests of very different lengths: what the 4-bit cache is for
        {"name": "attention_decode_64_bf16", "kind": "attention", "q": "bf16", "heads": 32, "kv_heads": 8,
         "head_dim": 128, "window": 0, "page": 16, "n_seq": 64, "decode": 1.0, "chunk": 1, "ctx_lo": 100,
         "ctx_hi": 16000, "layout": 4},
        # speculative verify, 16 requests of 5 tokens, heads of 256 and a window of 1024 keys: a local layer of Gemma-3-4B
        {"name": "attention_verify_f16_window", "kind": "attention", "q": "f16", "heads": 8, "kv_heads": 4,
         "head_dim": 256, "window": 1024, "page": 32, "n_seq": 16, "decode": 0.0, "chunk": 5, "ctx_lo": 300,
         "ctx_hi": 9000, "layout": 5},
        # the largest: 2048 tokens of a long prompt over 6000 before them
        {"name": "attention_chunk_bf16", "kind": "attention", "q": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "window": 0, "page": 16, "n_seq": 1, "decode": 0.0, "chunk": 2048, "ctx_lo": 6000, "ctx_hi": 6000, "layout": 6},
        # one request that samples with penalties, no drafts
        {"name": "adjust_one", "kind": "adjust", "n_seq": 1, "draft_lo": 0, "draft_hi": 0, "vocab": 128256, "dtype": "f32",
         "history": 800, "bias": 20, "masked": 0.0, "layout": 7},
        # a step of 64 requests, half of them held to a grammar
        {"name": "adjust_64_grammar", "kind": "adjust", "n_seq": 64, "draft_lo": 0, "draft_hi": 0, "vocab": 128256,
         "dtype": "f32", "history": 4000, "bias": 50, "masked": 0.5, "layout": 8},
        # drafts to verify: 40 requests of up to 5 rows, Gemma 3's vocabulary in bf16, every row under a mask
        {"name": "adjust_drafts_bf16", "kind": "adjust", "n_seq": 40, "draft_lo": 2, "draft_hi": 4, "vocab": 262144,
         "dtype": "bf16", "history": 2000, "bias": 5, "masked": 1.0, "layout": 9},
        # one request's token through one adapter
        {"name": "lora_token", "kind": "lora", "n_seq": 1, "rows_lo": 1, "rows_hi": 1, "adapters": 1, "rank": 16, "k": 2560,
         "n": 2560, "x": "f32", "pool": "bf16", "none": 0.0, "layout": 10},
        # a decode step of 64 requests over 32 adapters, some requests without: Gemma-3-4B's gate projection
        {"name": "lora_decode_64", "kind": "lora", "n_seq": 64, "rows_lo": 1, "rows_hi": 1, "adapters": 32, "rank": 32,
         "k": 2560, "n": 10240, "x": "f32", "pool": "bf16", "none": 0.1, "layout": 11},
        # chunks of prompts of six requests beside decoding ones, f16 adapters of rank 64
        {"name": "lora_prompts", "kind": "lora", "n_seq": 6, "rows_lo": 200, "rows_hi": 700, "adapters": 4, "rank": 64,
         "k": 2560, "n": 4096, "x": "f32", "pool": "f16", "none": 0.0, "layout": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "adjust", "adjust", "lora", "lora"])
    layout = rng.randrange(1 << 30)
    if kind == "append":
        page = rng.choice([8, 16, 32, 64, 128])
        tokens = _log_int(rng, 1, 8192)
        return {"kind": kind, "tokens": tokens, "kv_heads": rng.randint(1, 8), "head_dim": rng.choice([64, 128, 256]),
                "src": rng.choice(["f32", "f16", "bf16"]), "page": page,
                "pages": (tokens + page - 1) // page + rng.randint(1, 64), "layout": layout}
    if kind == "adjust":
        lo, vocab = rng.randint(0, 4), _log_int(rng, 1000, 262144)
        hi = lo + rng.randint(0, 3)
        return {"kind": kind, "n_seq": _log_int(rng, 1, max(1, min(64, int(4e7 / (hi + 1) / vocab)))), "draft_lo": lo,
                "draft_hi": hi, "vocab": vocab, "dtype": rng.choice(["f32", "f32", "bf16"]),
                "history": _log_int(rng, 1, 20000), "bias": rng.choice([0, 3, 100]),
                "masked": rng.choice([0.0, 0.3, 1.0]), "layout": layout}
    if kind == "lora":
        form = rng.choice(["token", "decode", "prompts"])
        case = {"kind": kind, "rank": rng.choice([8, 16, 32, 64, 128]), "k": 64 * _log_int(rng, 4, 160),
                "n": _log_int(rng, 64, 10240), "x": rng.choice(["f32", "f32", "bf16"]),
                "pool": rng.choice(["bf16", "f16"]), "none": rng.choice([0.0, 0.2]), "layout": layout}
        if form == "token":
            case.update(n_seq=1, rows_lo=1, rows_hi=rng.randint(1, 8), adapters=1, none=0.0)
        elif form == "decode":
            case.update(n_seq=_log_int(rng, 2, 64), rows_lo=1, rows_hi=rng.choice([1, 1, 5]), adapters=_log_int(rng, 1, 64))
        else:
            case.update(n_seq=_log_int(rng, 1, 16), rows_lo=1, rows_hi=_log_int(rng, 10, 500), adapters=_log_int(rng, 1, 8))
        while work(case)["bytes"] > 1e8:  # no more than the largest listed one
            case["n"] = max(64, case["n"] * 2 // 3)
            case["k"] = max(256, case["k"] * 2 // 3 // 64 * 64)
            case["rank"] = max(8, case["rank"] // 2)
        return case
    case = {"kind": kind, "q": rng.choice(["bf16", "bf16", "f16", "f32"]), "kv_heads": rng.randint(1, 8),
            "head_dim": rng.choice([64, 128, 256]), "window": _log_int(rng, 1, 4096) if rng.random() < 0.3 else 0,
            "page": rng.choice([8, 16, 32, 64, 128]), "layout": layout}
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 8])
    form = rng.choice(["token", "decode", "decode", "verify", "chunk", "mixed"])
    if form == "token":
        case.update(n_seq=1, decode=1.0, chunk=1, ctx_lo=1, ctx_hi=_log_int(rng, 2, 65536))
    elif form == "decode":
        case.update(n_seq=_log_int(rng, 2, 64), decode=1.0, chunk=1, ctx_lo=1, ctx_hi=_log_int(rng, 2, 16384))
    elif form == "verify":
        case.update(n_seq=_log_int(rng, 1, 32), decode=0.0, chunk=rng.randint(2, 9), ctx_lo=1,
                    ctx_hi=_log_int(rng, 2, 8192))
    elif form == "chunk":
        case.update(n_seq=1, decode=0.0, chunk=_log_int(rng, 16, 512 if case["q"] == "f32" else 1024), ctx_lo=1,
                    ctx_hi=_log_int(rng, 2, 4096))
    else:
        case.update(n_seq=_log_int(rng, 2, 32), decode=0.8, chunk=_log_int(rng, 10, 512), ctx_lo=1,
                    ctx_hi=_log_int(rng, 2, 4096))
    while True:  # no more than the largest listed ones (f32 rows cost twice the others)
        w = work(case)
        if w["bytes"] <= 2.5e8 and w["flops"] <= (1e11 if case["q"] == "f32" else 2.3e11):
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


def _pages(n, page):
    return (n + page - 1) // page


def _starts(counts):
    return [0] + np.cumsum(counts).tolist()


def _adjust_layout(case):
    """Rows, tokens of history, biases and mask (-1: none) of each request; about one mask for three that have one."""
    rng = random.Random(case["layout"])
    n = case["n_seq"]
    rows = [1 + rng.randint(case["draft_lo"], case["draft_hi"]) for _ in range(n)]
    history = [max(1, int(case["history"] * rng.uniform(0.2, 1.0))) for _ in range(n)]
    bias = [rng.randint(0, case["bias"]) for _ in range(n)]
    held = [rng.random() < case["masked"] for _ in range(n)]
    # each row of a request has a mask of its own: a grammar's state moves with the drafts
    masks = max(1, _pages(sum(r for r, h in zip(rows, held) if h), 3))
    of_row = [rng.randrange(masks) if h else -1 for r, h in zip(rows, held) for _ in range(r)]
    allowed = [rng.choice([0.0005, 0.01, 0.6]) for _ in range(masks)]
    return rows, history, bias, of_row, allowed


def _lora_layout(case):
    rng = random.Random(case["layout"])
    rows = [rng.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["n_seq"])]
    adapter = [-1 if rng.random() < case["none"] else rng.randrange(case["adapters"]) for _ in rows]
    return rows, adapter


def work(case):
    kind = case["kind"]
    if kind == "append":
        n = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": int(n * (BYTES[case["src"]] + 0.625 + 2)) + 8 * case["tokens"], "flops": 4 * n}
    if kind == "attention":
        cached, fresh = _lengths(case)
        hq, hk, d, w = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
        size = flops = 0
        for c, f in zip(cached, fresh):
            pairs = sum(min(c + i + 1, w) for i in range(f)) if w else f * c + f * (f + 1) // 2
            first = max(0, c - w + 1) if w else 0
            size += 2 * f * hq * d * BYTES[case["q"]] + int(2 * (c + f - first) * hk * d * 0.625)
            flops += 4 * pairs * hq * d
        return {"bytes": size, "flops": flops}
    if kind == "adjust":
        rows, history, bias, of_row, allowed = _adjust_layout(case)
        v, b = case["vocab"], BYTES[case["dtype"]]
        masks = sorted({m for m in of_row if m >= 0})
        # masks once, what they close written, what a history or a bias touches read and written
        size = sum(v // 8 for _ in masks) + sum(int(v * b * (1 - allowed[m])) for m in of_row if m >= 0)
        touched = sum(r * (min(h // 2, v) + k) for r, h, k in zip(rows, history, bias))
        return {"bytes": size + 2 * b * touched + 4 * sum(history) + 8 * sum(bias), "flops": 4 * touched + len(of_row)}
    rows, adapter = _lora_layout(case)
    k, n, r = case["k"], case["n"], case["rank"]
    used = len({a for a in adapter if a >= 0})
    t = sum(m for m, a in zip(rows, adapter) if a >= 0)
    return {"bytes": used * r * (k + n) * 2 + t * (k * BYTES[case["x"]] + 8 * n) + 64, "flops": 2 * t * r * (k + n) + 1}


# --------------------------------------------------------------- inputs --

def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _channels(g, hk, d):
    """A head's channels: most alike, some far larger and off zero, as keys have them."""
    size = torch.exp(torch.randn((hk, d), generator=g, device="cuda") * 0.5)
    off = torch.randn((hk, d), generator=g, device="cuda") * (torch.rand((hk, d), generator=g, device="cuda") < 0.05) * 4
    return size, off


def _prepare_append(case, seed):
    g = _gen(seed)
    hk, d, n, page = case["kv_heads"], case["head_dim"], case["tokens"], case["page"]
    size, off = _channels(g, hk, d)
    # rows of a joint projection: 2 hk heads of queries before the keys and values
    joint = torch.randn((n, 4 * hk, d), generator=g, device="cuda")
    joint[:, 2 * hk:3 * hk] = joint[:, 2 * hk:3 * hk] * size + off
    joint = joint.to(DTYPES[case["src"]])
    slots = torch.randperm(case["pages"], generator=g, device="cuda")[:_pages(n, page)]
    slots = (slots[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n].to(torch.int32)
    if n > 8:
        slots[n // 2] = -1  # padding
    state = {"case": case, "k": joint[:, 2 * hk:3 * hk], "v": joint[:, 3 * hk:], "slots": slots}
    return _with_cache(state, case["pages"])


def _with_cache(state, n_pages):
    """A cache of zeros: the framework's, or codes and group numbers in arrays of their own."""
    case = state["case"]
    page, hk, d = case["page"], case["kv_heads"], case["head_dim"]
    if own:
        rt = _rt()
        size = rt.paged_page_bytes(rt.Q4KV, page, hk, d)
        pages = torch.zeros((2, n_pages, size), dtype=torch.uint8, device="cuda")
        state["kv"] = rt.PagedKV4(pages[0], pages[1], page, hk, d)
    else:
        for x in ("k", "v"):
            state[x + "_codes"] = torch.zeros((n_pages * page, hk, d // 2), dtype=torch.uint8, device="cuda")
            state[x + "_groups"] = torch.zeros((n_pages * page, hk, d // 32, 2), dtype=torch.float16, device="cuda")
    return state


def _prepare_attention(case, seed):
    g = _gen(seed)
    hq, hk, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    cached, fresh = _lengths(case)
    lens = [c + f for c, f in zip(cached, fresh)]
    held = [_pages(n, page) for n in lens]
    n_pages = sum(held) + 8
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu().numpy()
    table = np.full((len(held), max(held)), -1, np.int32)
    for i, (h, at) in enumerate(zip(held, _starts(held))):
        table[i, :h] = ids[at:at + h]
    state = {"case": case, "scale": 1.0 / math.sqrt(d), "lens": lens, "fresh": fresh, "starts": _starts(fresh),
             "q_start": _i32(_starts(fresh)), "kv_len": _i32(lens), "table": torch.from_numpy(table).cuda(),
             "n_pages": n_pages, "seed": seed}
    state = _with_cache(state, n_pages)
    for at, k, v in _pieces(case, seed, n_pages):  # what earlier steps have put there
        slots = torch.arange(at, at + k.shape[0], device="cuda")
        if own:
            _rt().paged_append(state["kv"], k, v, slots.to(torch.int32))
        else:
            for x, rows in (("k", k), ("v", v)):
                state[x + "_codes"][slots], state[x + "_groups"][slots] = _plain_quantize(rows)
    state["q"] = (torch.randn((sum(fresh), hq, d), generator=g, device="cuda") * 0.7).to(DTYPES[case["q"]])
    state["out"] = torch.zeros_like(state["q"])
    return state


def _pieces(case, seed, n_pages):
    """(first slot, keys, values): the rows of all slots in f32, some thousand at a time."""
    g = _gen(seed + 1)
    hk, d, n = case["kv_heads"], case["head_dim"], n_pages * case["page"]
    size, off = _channels(g, hk, d)
    for at in range(0, n, 32768):
        shape = (min(32768, n - at), hk, d)
        yield (at, torch.randn(shape, generator=g, device="cuda") * size + off,
               torch.randn(shape, generator=g, device="cuda"))


def _prepare_adjust(case, seed):
    g = _gen(seed)
    rows, history, bias, of_row, allowed = _adjust_layout(case)
    n, v, words = case["n_seq"], case["vocab"], (case["vocab"] + 31) // 32
    logits = (torch.randn((sum(rows), v), generator=g, device="cuda") * 2.5).to(DTYPES[case["dtype"]])
    # texts repeat themselves: frequent tokens of a few thousand, and any others
    common = torch.randint(0, v, (2000,), generator=g, device="cuda")

    def text(shape):
        often = common[(2000 * torch.rand(shape, generator=g, device="cuda") ** 3).long().clamp(max=1999)]
        any_ = torch.randint(0, v, shape, generator=g, device="cuda")
        return torch.where(torch.rand(shape, generator=g, device="cuda") < 0.6, often, any_).to(torch.int32)

    bits = [(torch.rand((words, 32), generator=g, device="cuda") < a).long() for a in allowed]
    mask = (torch.stack(bits) << torch.arange(32, device="cuda")).sum(-1)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
    u = lambda lo, hi: torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo  # noqa: E731
    state = {"case": case, "logits": logits, "tokens": text((sum(rows),)), "row_start": _i32(_starts(rows)),
             "starts": _starts(rows), "history": text((n, max(history) + 16)), "history_len": _i32(history),
             "prompt_len": _i32([h // 3 for h in history]), "repetition": u(1.0, 1.3), "presence": u(0.0, 1.0),
             "frequency": u(0.0, 0.5), "bias_start": _i32(_starts(bias)), "bias_token": text((sum(bias),)),
             "bias": torch.randn(sum(bias), generator=g, device="cuda") * 5, "mask": mask, "mask_row": _i32(of_row)}
    if own:
        state["rules"] = _rt().LogitRules(**{x: state[x] for x in (
            "history", "history_len", "prompt_len", "repetition", "presence", "frequency", "bias_start", "bias_token",
            "bias", "mask", "mask_row")})
    return state


def _prepare_lora(case, seed):
    g = _gen(seed)
    rows, adapter = _lora_layout(case)
    m, k, n, r, dt = case["adapters"], case["k"], case["n"], case["rank"], DTYPES[case["pool"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    state = {"case": case, "x": randn(sum(rows), k).to(DTYPES[case["x"]]), "a": (randn(m, r, k) / math.sqrt(k)).to(dt),
             "b": (randn(m, n, r) / math.sqrt(r)).to(dt), "scale": torch.rand(m, generator=g, device="cuda") + 0.5,
             "row_start": _i32(_starts(rows)), "starts": _starts(rows), "adapter": _i32(adapter),
             "y": randn(sum(rows), n)}  # (what the shared projection has left)
    if own:
        state["adapters"] = _rt().Adapters(state["a"], state["b"], state["scale"])
    return state


# ----------------------------------------------------------- one pass --

def run(state):
    kind = state["case"]["kind"]
    return globals()[("_own_" if own else "_plain_") + kind](state)


def _own_append(st):
    rt = _rt()
    rt.paged_append(st["kv"], st["k"], st["v"], st["slots"])
    k, v = rt.paged_read(st["kv"], st["slots"])
    return {"k": k, "v": v}


def _plain_quantize(rows):
    """Codes, two to a byte, and (a, b) of groups of 32 of rows [n, heads, dim]."""
    x = rows.float().unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1), x.amax(-1)
    a = ((hi - lo) * (16.0 / 15.0)).to(torch.float16)
    b = (lo - a.float()).to(torch.float16)
    step = torch.where(a > 0, 16.0 / a.float(), torch.zeros_like(lo))
    c = torch.round((x - b.float()[..., None]) * step[..., None]) - 16
    c = c.clamp(0, 15).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.stack([a, b], -1)


def _plain_values(codes, groups):
    """What codes [..., dim / 2] and groups [..., dim / 32, 2] stand for, f16 numbers held in f32."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).float()
    a, b = groups.float().unbind(-1)
    return (a[..., None] * (1 + c / 16) + b[..., None]).to(torch.float16).float().flatten(-2)


def _plain_append(st):
    slots = st["slots"].long()
    ok = slots >= 0
    out = {}
    for x in ("k", "v"):
        codes, groups = st[x + "_codes"], st[x + "_groups"]
        new_codes, new_groups = _plain_quantize(st[x])
        # a token without a slot writes back the row of token 0, which has one
        to = torch.where(ok, slots, slots[:1])
        codes[to] = torch.where(ok[:, None, None], new_codes, new_codes[:1])
        groups[to] = torch.where(ok[:, None, None, None], new_groups, new_groups[:1])
        values = _plain_values(codes[to], groups[to])
        out[x] = torch.where(ok[:, None, None], values, torch.zeros_like(values)).to(torch.float16)
    return out


def _own_attention(st):
    return _rt().paged_attention(st["q"], st["kv"], st["table"], st["q_start"], st["kv_len"], st["scale"],
                                 window=st["case"]["window"], max_fresh=max(st["fresh"]), out=st["out"])


def _plain_attention(st):
    """Requests with as many new tokens go together, their keys padded to the longest, as memory allows."""
    case = st["case"]
    page, window, hk, d = case["page"], case["window"], case["kv_heads"], case["head_dim"]
    q, out = st["q"], st["out"]
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
        f, longest, n = st["fresh"][batch[0]], max(st["lens"][s] for s in batch), len(batch)
        seqs = torch.tensor(batch, device=q.device)
        ids = st["table"][seqs, :_pages(longest, page)].clamp(min=0).long()
        slots = (ids[:, :, None] * page + torch.arange(page, device=q.device)).flatten(1)
        keys = slots.shape[1]
        lens = st["kv_len"][seqs].long()
        key_at = torch.arange(keys, device=q.device)
        live = (key_at[None] < lens[:, None])[:, :, None, None]
        k, v = (_plain_values(st[x + "_codes"][slots], st[x + "_groups"][slots]) for x in ("k", "v"))
        k = torch.where(live, k, torch.zeros_like(k)).permute(0, 2, 3, 1).contiguous()
        v = torch.where(live, v, torch.zeros_like(v)).permute(0, 2, 1, 3).contiguous()
        for i in range(0, f, 1024):
            m = min(1024, f - i)
            rows = (st["q_start"][seqs].long()[:, None] + torch.arange(i, i + m, device=q.device)).reshape(-1)
            x = q[rows].float().reshape(n, m, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * m, d)
            s = torch.matmul(x, k) * st["scale"]
            at = lens[:, None] - f + i + torch.arange(m, device=q.device)[None]
            seen = key_at[None, None] <= at[:, :, None]
            if window:
                seen = seen & (key_at[None, None] > at[:, :, None] - window)
            s = s.reshape(n, hk, group, m, keys).masked_fill_(~seen[:, None, None], float("-inf"))
            s = torch.exp(s - s.amax(-1, keepdim=True))
            s = (s / s.sum(-1, keepdim=True)).reshape(n, hk, group * m, keys)
            o = torch.matmul(s, v).reshape(n, hk, group, m, d).permute(0, 3, 1, 2, 4).reshape(n * m, hk * group, d)
            out[rows] = o.to(out.dtype)
    return out


def _own_adjust(st):
    return _rt().adjust_logits(st["logits"], st["row_start"], st["rules"], tokens=st["tokens"])


def _plain_adjust(st):
    logits = st["logits"]
    rows, v = logits.shape
    n, cols = st["history"].shape
    dev = logits.device
    seq = torch.repeat_interleave(torch.arange(n, device=dev), st["row_start"].diff(), output_size=rows)
    at = torch.arange(cols, device=dev)[None]
    # how often each request's history has a token, and how often behind its prompt
    live = at < st["history_len"][:, None]
    made = live & (at >= st["prompt_len"][:, None])
    base = [torch.zeros((n, v), dtype=torch.int32, device=dev).scatter_add_(1, st["history"].long(), m.to(torch.int32))
            for m in (live, made)]
    there, count = (c[seq] for c in base)
    # the drafts up to each row
    row = torch.arange(rows, device=dev)
    first = st["row_start"].long()[seq]
    width = st["case"]["draft_hi"] + 1
    drafts = row[:, None] - torch.arange(width, device=dev)[None]
    is_draft = drafts > first[:, None]
    tokens = st["tokens"].long()[drafts.clamp(min=0)]
    there.scatter_add_(1, tokens, is_draft.to(torch.int32))
    count.scatter_add_(1, tokens, is_draft.to(torch.int32))
    x = logits.float()
    rep, pres, freq = (st[name][seq][:, None] for name in ("repetition", "presence", "frequency"))
    x = torch.where(there > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(count > 0, x - freq * count - pres, x)
    # of the entries for one token the last counts
    m = st["bias"].numel()
    if m:
        entry = torch.arange(m, device=dev)
        owner = torch.searchsorted(st["bias_start"][1:].long().contiguous(), entry, right=True)
        place = owner * v + st["bias_token"].long()
        last = torch.full((n * v,), -1, dtype=torch.int64, device=dev).scatter_reduce_(0, place, entry, "amax")
        last = last.view(n, v)[seq]
        x = torch.where(last >= 0, x + st["bias"][last.clamp(min=0)], x)
    word = torch.arange(v, device=dev)
    bits = (st["mask"][:, word // 32] >> (word % 32)) & 1
    closed = (st["mask_row"] >= 0)[:, None] & (bits[st["mask_row"].long().clamp(min=0)] == 0)
    logits.copy_(x.masked_fill_(closed, float("-inf")))
    return logits


def _own_lora(st):
    return _rt().lora_add(st["y"], st["x"], st["adapters"], st["row_start"], st["adapter"])


def _plain_lora(st):
    """Every row through every adapter, the others' parts made 0 in between."""
    m, r, k = st["a"].shape
    x, y, dev = st["x"].float(), st["y"], st["y"].device
    t = (x @ st["a"].float().view(m * r, k).T).view(-1, m, r)
    of_row = torch.repeat_interleave(st["adapter"], st["row_start"].diff(), output_size=x.shape[0])
    mine = of_row[:, None] == torch.arange(m, device=dev)[None]
    t = torch.where(mine[:, :, None], t * st["scale"][:, None], torch.zeros_like(t))
    y += t.flatten(1) @ st["b"].float().permute(0, 2, 1).reshape(m * r, -1)
    return y


# ------------------------------------------------------- 64-bit results --

def exact(case, seed):
    """What run returns, from the definitions, request by request."""
    st = prepare(case, seed)
    return globals()["_exact_" + case["kind"]](st)


def _f32(x):
    return x.float().double()


def _f16(x):
    return x.float().half().double()


def _exact_values(x):
    """The values that a 4-bit cache keeps of x [..., dim], float64: each rounding of the definition by itself."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    a = _f16(_f32(_f32(hi - lo) * _f32(torch.tensor(16.0 / 15.0, dtype=torch.float64, device=x.device))))
    b = _f16(_f32(lo - a))
    steps = _f32(_f32(g - b) * _f32(16.0 / a))
    code = torch.where(a == 0, 0.0, (steps.round() - 16).clamp(0, 15))
    return _f16(a + a * code / 16 + b).reshape(x.shape)


def _exact_append(st):
    gone = (st["slots"] < 0)[:, None, None]
    return {x: _exact_values(st[x]).masked_fill(gone, 0.0) for x in ("k", "v")}


def _exact_attention(st):
    case = st["case"]
    hk, d, page, window = case["kv_heads"], case["head_dim"], case["page"], case["window"]
    group = case["heads"] // hk
    keys, values = (torch.empty((st["n_pages"], page, hk, d), dtype=torch.float16, device="cuda") for _ in range(2))
    for at, k, v in _pieces(case, st["seed"], st["n_pages"]):
        for all_, x in ((keys, k), (values, v)):  # (f16 numbers: nothing is lost in between)
            all_.view(-1, hk, d)[at:at + len(x)] = _exact_values(x).half()
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s, (n, length, start) in enumerate(zip(st["fresh"], st["lens"], st["starts"])):
        base = 0 if not window else max(0, length - n - window + 1) // page
        ids = st["table"][s, base:_pages(length, page)].long()
        key = torch.arange(base * page, length, device="cuda")
        for h in range(hk):
            k, v = (x[ids, :, h].reshape(-1, d)[:len(key)].double() for x in (keys, values))
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


def _exact_adjust(st):
    out = st["logits"].double()
    v = out.shape[1]
    hist_len, prompt_len = st["history_len"].tolist(), st["prompt_len"].tolist()
    rep, pres, freq = (st[x].double().tolist() for x in ("repetition", "presence", "frequency"))
    bias_at, mask_row = st["bias_start"].tolist(), st["mask_row"].tolist()
    entries = list(zip(st["bias_token"].tolist(), st["bias"].double().tolist()))
    bit = torch.arange(32, device="cuda")
    for s, (a, b) in enumerate(zip(st["starts"], st["starts"][1:])):
        history = st["history"][s, :hist_len[s]].long()
        bias = dict(entries[bias_at[s]:bias_at[s + 1]])  # (the last of a token's entries)
        for r in range(a, b):
            drafts = st["tokens"][a + 1:r + 1].long()
            there = torch.cat([history, drafts]).unique()
            made = torch.bincount(torch.cat([history[prompt_len[s]:], drafts]), minlength=v).double()
            x = out[r]
            x[there] = torch.where(x[there] > 0, x[there] / rep[s], x[there] * rep[s])
            x -= freq[s] * made + pres[s] * (made > 0)
            for token, value in bias.items():
                x[token] += value
            if mask_row[r] >= 0:
                open_ = (st["mask"][mask_row[r]][:, None] >> bit) & 1
                x[open_.reshape(-1)[:v] == 0] = -math.inf
    return out


def _exact_lora(st):
    out = st["y"].double()
    for s, a in enumerate(st["adapter"].tolist()):
        if a >= 0:
            rows = slice(st["starts"][s], st["starts"][s + 1])
            t = st["x"][rows].double() @ st["a"][a].double().T
            out[rows] += float(st["scale"][a]) * (t @ st["b"][a].double().T)
    return out
