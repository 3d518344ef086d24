"""The 4-bit KV cache by its definition, for the tests: what append keeps of values."""
import torch

GROUP = 32


def kept(x):
    """What a 4-bit cache keeps of x [..., head_dim] (f32, f16 or bf16), in float64: the definition's steps, each
    rounded where it says so."""
    f32, f16 = (lambda v: v.float().double()), (lambda v: v.float().half().double())
    g = x.double().unflatten(-1, (-1, GROUP))
    none = ~(g.abs() <= 16384).all(-1, keepdim=True)
    g = torch.where(none, 0.0, g)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    a = f16(f32(f32(hi - lo) * f32(torch.tensor(16 / 15, dtype=torch.float64, device=x.device))))
    b = f16(f32(lo - a))
    code = (f32(f32(g - b) * f32(16 / a)).round() - 16).clamp(0, 15)
    code = torch.where(a > 0, code, 0.0)
    return torch.where(none, torch.nan, f16(a * (1 + code / 16) + b)).flatten(-2)


def filled(rt, n_pages, page, heads, dim, joint=False, byte=0xFF):
    """A cache whose bytes are all `byte` (0xFF: every group is NaN); joint: pages of keys and values in turn."""
    size = rt.paged_page_bytes(rt.Q4KV, page, heads, dim)
    raw = torch.full((n_pages, 2, size) if joint else (2, n_pages, size), byte, dtype=torch.uint8, device="cuda")
    k, v = (raw[:, 0], raw[:, 1]) if joint else (raw[0], raw[1])
    return rt.PagedKV4(k, v, page, heads, dim)
