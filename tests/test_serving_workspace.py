"""Workspace sizes of the serving calls never fall as a step grows: a server reserves for its
largest step and captures smaller ones too (no GPU needed)."""
import ctypes as C
import itertools

import pytest

from conftest import load_package


@pytest.fixture(scope="module")
def rt():
    return load_package().rt_hip


def grows(size, *axes):
    """size of every point is no more than that of the next one along each axis."""
    for at in itertools.product(*(range(len(a)) for a in axes)):
        here = size(*(a[i] for a, i in zip(axes, at)))
        assert here > 0
        for d in range(len(axes)):
            if at[d] + 1 < len(axes[d]):
                more = [a[i + (j == d)] for j, (a, i) in enumerate(zip(axes, at))]
                assert size(*more) >= here, (*(a[i] for a, i in zip(axes, at)), more)


REQUESTS = [1, 2, 12, 23, 64, 100, 1000, 4096]
ROWS = [1, 2, 12, 16, 31, 32, 33, 64, 65, 200, 400, 511, 512, 513, 4000, 5000, 100000, 1 << 24]


@pytest.mark.parametrize("rank", [8, 32, 64, 72, 128])
@pytest.mark.parametrize("k", [8, 512, 520, 2560, 10240, 1 << 20])
def test_lora(rt, rank, k):
    lora = C.byref(rt.LoraStruct(a=16, b=16, scale=16, dtype=rt.BF16, n_adapters=2, rank=rank, k=k, n=64))
    grows(lambda n_seq, rows: rt.library().lib.rt_hip_lora_workspace_bytes(lora, n_seq, rows), REQUESTS, ROWS)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (6, 2), (32, 8), (16, 1)])
@pytest.mark.parametrize("cache, q", [("Q4KV", "F32"), ("Q4KV", "BF16"), ("F16", "F32"), ("BF16", "BF16"), ("F32", "F32")])
def test_attention(rt, dim, heads, kv_heads, cache, q):
    """Over 4-bit pages, and over the others; by rows of the step and by the most of a request."""
    kv = C.byref(rt.PagedKvStruct(k=1 << 20, v=1 << 40, dtype=getattr(rt, cache), n_pages=2, page_size=16, n_kv_heads=kv_heads,
                                  head_dim=dim, page_stride=0))
    need = rt.library().lib.rt_hip_paged_attention_workspace_bytes
    grows(lambda n_seq, rows: need(kv, getattr(rt, q), heads, n_seq, rows, 0), REQUESTS, ROWS[:-1])
    grows(lambda n_seq, rows, most: need(kv, getattr(rt, q), heads, n_seq, rows, most), REQUESTS[:4], ROWS[:12], ROWS[:12])
