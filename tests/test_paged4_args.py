"""Arguments that the calls over a 4-bit cache refuse, and paged_read (no GPU needed)."""
import ctypes as C

import pytest

from conftest import load_package

ARG, SHAPE, ALIGN, UNSUPPORTED = 1, 2, 3, 6


@pytest.fixture(scope="module")
def rt():
    return load_package().rt_hip


@pytest.fixture(scope="module")
def mem():
    """Addresses of 24 separate, 16-byte aligned pieces of 4096 bytes."""
    buf = C.create_string_buffer(24 * 4096 + 64)
    base = (C.addressof(buf) + 63) & ~63
    yield [base + 4096 * i for i in range(24)]
    del buf


def cache(rt, mem, **over):
    args = dict(k=mem[20], v=mem[22], dtype=rt.Q4KV, n_pages=2, page_size=8, n_kv_heads=1, head_dim=64, page_stride=0)
    args.update(over)
    return C.byref(rt.PagedKvStruct(**args))


def append(rt, m, **over):
    a = dict(kv=cache(rt, m), k=m[0], v=m[1], dtype=rt.F32, stride=64, slots=m[2], n=4)
    a.update(over)
    return rt.library().status("rt_hip_paged_append", *a.values(), None)


def read(rt, m, **over):
    a = dict(kv=cache(rt, m), slots=m[2], n=4, k=m[0], v=m[1], dtype=rt.F32, stride=64)
    a.update(over)
    return rt.library().status("rt_hip_paged_read", *a.values(), None)


def attention(rt, m, **over):
    a = dict(q=m[0], dtype=rt.F16, q_stride=128, heads=2, kv=cache(rt, m), table=m[1], cols=2, q_start=m[2], kv_len=m[3],
             n_seq=2, n_tokens=4, max_fresh=0, scale=C.c_float(0.1), window=0, out=m[4], out_stride=128)
    a.update(over)
    return rt.library().status("rt_hip_paged_attention", *a.values(), None)


def test_page_bytes(rt):
    assert rt.paged_page_bytes(rt.Q4KV, 16, 8, 128) == 16 * 8 * 128 * 5 // 8
    assert rt.paged_page_bytes(rt.Q4KV, 8, 1, 64) == 320
    assert rt.paged_page_bytes(rt.F16, 16, 8, 128) == 16 * 8 * 128 * 2
    assert rt.paged_page_bytes(rt.F32, 1024, 256, 256) == 1024 * 256 * 256 * 4
    for bad in ((rt.Q4K, 16, 8, 128), (rt.Q4KV, 24, 8, 128), (rt.Q4KV, 16, 0, 128), (rt.Q4KV, 16, 8, 96), (rt.Q4KV, 16, 257, 64)):
        assert rt.paged_page_bytes(*bad) == -1
    with pytest.raises(ValueError):
        rt.paged_page_bytes(rt.Q4KV, 1 << 40, 8, 128)


@pytest.mark.parametrize("over, code", [
    (dict(k=None), ARG), (dict(page_size=24), SHAPE), (dict(head_dim=96), SHAPE), (dict(n_kv_heads=0), SHAPE),
    (dict(n_pages=0), SHAPE), (dict(page_stride=319), ARG), (dict(page_stride=328), ALIGN), (dict(page_stride=1 << 32), SHAPE),
    (dict(n_pages=1 << 28), SHAPE), (dict(dtype=8), UNSUPPORTED)])
def test_cache_refused_everywhere(rt, mem, over, code):
    for call in (append, read, attention):
        assert call(rt, mem, kv=cache(rt, mem, **over)) == code
        assert call(rt, mem, kv=None) == ARG
        assert call(rt, mem, kv=cache(rt, mem, v=mem[22] + 8)) == ALIGN


def test_keys_and_values_that_share_memory(rt, mem):
    assert append(rt, mem, kv=cache(rt, mem, v=mem[20])) == ARG
    assert append(rt, mem, kv=cache(rt, mem, v=mem[20] + 304, page_stride=640)) == ARG
    assert append(rt, mem, k=mem[20] + 320) == ARG  # rows inside the cache
    assert append(rt, mem, dtype=rt.Q4KV) == UNSUPPORTED


@pytest.mark.parametrize("over, code", [
    (dict(dtype=2), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED), (dict(n=-1), ARG), (dict(k=None), ARG), (dict(v=None), ARG),
    (dict(slots=None), ARG), (dict(stride=63), ARG), (dict(stride=66), ALIGN), (dict(n=1 << 30), SHAPE),
    (dict(stride=1 << 46), SHAPE)])
def test_read_refuses(rt, mem, over, code):
    assert read(rt, mem, **over) == code
    assert b"rt_hip_paged_read" in rt.library().lib.rt_hip_last_error()


def test_read_refuses_overlap(rt, mem):
    assert read(rt, mem, v=mem[0]) == ARG
    assert read(rt, mem, v=mem[0] + 128, stride=96) == ARG  # rows of the two that cut into each other
    assert read(rt, mem, k=mem[20]) == ARG
    assert read(rt, mem, v=mem[22] + 320) == ARG
    assert read(rt, mem, v=mem[2] - 1008) == ARG            # over slots
    assert read(rt, mem, n=0, k=None, v=None, slots=None) == 0


@pytest.mark.parametrize("over, code", [
    (dict(dtype=2), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED), (dict(heads=0), SHAPE), (dict(scale=C.c_float(0.0)), ARG),
    (dict(q_stride=127), ARG), (dict(out=None), ARG), (dict(window=-1), ARG), (dict(n_seq=4097), SHAPE)])
def test_attention_refuses(rt, mem, over, code):
    assert attention(rt, mem, **over) == code
    assert attention(rt, mem, out=mem[22]) == ARG
    assert attention(rt, mem, n_tokens=0) == 0


def test_workspace_of_every_type(rt, mem):
    lib = rt.library().lib
    for dtype in (rt.F32, rt.F16, rt.BF16):
        assert lib.rt_hip_paged_attention_workspace_bytes(cache(rt, mem), dtype, 2, 1, 1, 1) > 0
    assert lib.rt_hip_paged_attention_workspace_bytes(cache(rt, mem), rt.Q4KV, 2, 1, 1, 1) == -1
    assert lib.rt_hip_paged_attention_workspace_bytes(cache(rt, mem), rt.F16, 2, 0, 0, 0) == 0


def test_binding_checks_before_it_calls(rt):
    torch = pytest.importorskip("torch")
    k = torch.zeros(2, 320, dtype=torch.uint8)
    with pytest.raises(ValueError, match="GPU"):
        rt.PagedKV4(k, k.clone(), 8, 1, 64)
