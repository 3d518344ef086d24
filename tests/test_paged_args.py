"""Arguments that the calls of batched serving refuse: a status and a message,
before anything reaches the device (no GPU needed)."""
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
    args = dict(k=mem[20], v=mem[22], dtype=rt.F16, n_pages=2, page_size=8, n_kv_heads=1, head_dim=64, page_stride=0)
    args.update(over)
    return C.byref(rt.PagedKvStruct(**args))


def plan(rt, m, **over):
    a = dict(cached=m[0], fresh=m[1], held=m[2], held_out=m[3], table=m[4], cols=4, queue=m[5], state=m[6], state_out=m[7],
             n_pages=8, page=16, n_seq=3, n_tokens=5, q_start=m[8], kv_len=m[9], slots=m[10], positions=m[11])
    a.update(over)
    return rt.library().status("rt_hip_paged_plan", *a.values(), None)


def append(rt, m, **over):
    a = dict(kv=cache(rt, m), k=m[0], v=m[1], dtype=rt.F32, stride=64, slots=m[2], n=4)
    a.update(over)
    return rt.library().status("rt_hip_paged_append", *a.values(), None)


def attention(rt, m, **over):
    a = dict(q=m[0], dtype=rt.F16, q_stride=128, heads=2, kv=cache(rt, m), table=m[1], cols=2, q_start=m[2], kv_len=m[3],
             n_seq=2, n_tokens=4, max_fresh=0, scale=C.c_float(0.1), window=0, out=m[4], out_stride=128)
    a.update(over)
    return rt.library().status("rt_hip_paged_attention", *a.values(), None)


def verify(rt, m, **over):
    a = dict(logits=m[0], stride=50, draft=m[1], draft_stride=50, dtype=rt.F32, vocab=50, tokens=m[2], row_start=m[3],
             accept=m[4], sample=m[5], temp=m[6], n_seq=2, n_rows=6, max_draft=2, out=m[7], count=m[8])
    a.update(over)
    return rt.library().status("rt_hip_verify_drafts", *a.values(), None)


@pytest.mark.parametrize("over, code", [
    (dict(n_seq=-1), ARG), (dict(n_tokens=-1), ARG), (dict(n_seq=4097), SHAPE), (dict(cached=None), ARG),
    (dict(slots=None), ARG), (dict(queue=None), ARG), (dict(page=12), SHAPE), (dict(page=4), SHAPE),
    (dict(page=2048), SHAPE), (dict(n_pages=0), ARG | SHAPE), (dict(n_pages=1 << 27), SHAPE), (dict(cols=0), ARG),
    (dict(cols=1 << 30), SHAPE), (dict(table=None), ARG)])
def test_plan_refuses(rt, mem, over, code):
    assert plan(rt, mem, **over) in ((ARG, SHAPE) if code == ARG | SHAPE else (code,))
    assert b"rt_hip_paged_plan" in rt.library().lib.rt_hip_last_error()


@pytest.mark.parametrize("a, b", [("held_out", "cached"), ("slots", "positions"), ("table", "queue"), ("kv_len", "fresh"),
                                  ("state_out", "held"), ("q_start", "kv_len")])
def test_plan_refuses_overlap(rt, mem, a, b):
    names = dict(cached=0, fresh=1, held=2, held_out=3, table=4, queue=5, state=6, state_out=7, q_start=8, kv_len=9,
                 slots=10, positions=11)
    assert plan(rt, mem, **{a: mem[names[b]]}) == ARG


@pytest.mark.parametrize("over, code", [
    (dict(dtype=2), UNSUPPORTED), (dict(n=-1), ARG), (dict(k=None), ARG), (dict(slots=None), ARG), (dict(stride=63), ARG),
    (dict(stride=66), ALIGN), (dict(n=1 << 30), SHAPE)])
def test_append_refuses(rt, mem, over, code):
    assert append(rt, mem, **over) == code
    assert append(rt, mem, k=mem[0] + 8) == ALIGN
    assert append(rt, mem, v=mem[20]) == ARG  # rows inside the cache


@pytest.mark.parametrize("over, code", [
    (dict(k=None), ARG), (dict(dtype=2), UNSUPPORTED), (dict(page_size=24), SHAPE), (dict(head_dim=96), SHAPE),
    (dict(n_kv_heads=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(page_stride=511), ARG), (dict(page_stride=516), ALIGN),
    (dict(n_pages=1 << 28), SHAPE)])
def test_cache_refused_everywhere(rt, mem, over, code):
    assert append(rt, mem, kv=cache(rt, mem, **over)) == code
    assert attention(rt, mem, kv=cache(rt, mem, **over)) == code
    assert append(rt, mem, kv=None) == ARG
    assert attention(rt, mem, kv=cache(rt, mem, v=mem[22] + 2)) == ALIGN


@pytest.mark.parametrize("over, code", [
    (dict(q=None), ARG), (dict(dtype=1), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED), (dict(heads=0), SHAPE),
    (dict(heads=1025), SHAPE), (dict(n_seq=4097), SHAPE), (dict(n_seq=-1), ARG), (dict(n_tokens=-2), ARG),
    (dict(max_fresh=-1), ARG), (dict(scale=C.c_float(0.0)), ARG), (dict(scale=C.c_float(-1.0)), ARG),
    (dict(scale=C.c_float(float("nan"))), ARG), (dict(scale=C.c_float(float("inf"))), ARG), (dict(window=-1), ARG),
    (dict(q_stride=127), ARG), (dict(out_stride=64), ARG), (dict(q_stride=129), ALIGN), (dict(cols=0), ARG),
    (dict(table=None), ARG), (dict(kv_len=None), ARG), (dict(n_tokens=0x7fffffff), SHAPE)])
def test_attention_refuses(rt, mem, over, code):
    assert attention(rt, mem, **over) == code
    assert b"rt_hip_paged_attention" in rt.library().lib.rt_hip_last_error()


def test_attention_refuses_overlap_and_heads(rt, mem):
    assert attention(rt, mem, out=mem[0] + 16) == ARG
    assert attention(rt, mem, out=mem[22]) == ARG
    assert attention(rt, mem, kv=cache(rt, mem, n_kv_heads=2, n_pages=1), heads=3, q_stride=192, out_stride=192) == SHAPE
    assert attention(rt, mem, q=mem[0] + 4) == ALIGN
    lib = rt.library().lib
    assert lib.rt_hip_paged_attention_workspace_bytes(cache(rt, mem), rt.BF16, 2, 1, 1, 1) == -1
    assert lib.rt_hip_paged_attention_workspace_bytes(cache(rt, mem), rt.F16, 2, 0, 0, 0) == 0


@pytest.mark.parametrize("over, code", [
    (dict(dtype=6), UNSUPPORTED), (dict(vocab=0), ARG), (dict(vocab=(1 << 20) + 1, stride=1 << 21), SHAPE),
    (dict(n_seq=-1), ARG), (dict(n_rows=-1), ARG), (dict(max_draft=-1), ARG), (dict(max_draft=256), SHAPE),
    (dict(n_seq=4000, max_draft=20), SHAPE), (dict(logits=None), ARG), (dict(tokens=None), ARG), (dict(out=None), ARG),
    (dict(sample=None), ARG), (dict(stride=49), ARG), (dict(draft_stride=49), ARG)])
def test_verify_refuses(rt, mem, over, code):
    assert verify(rt, mem, **over) == code
    assert verify(rt, mem, logits=mem[0] + 2) == ALIGN
    assert verify(rt, mem, out=mem[2]) == ARG
    assert verify(rt, mem, count=mem[7] + 4) == ARG
    assert rt.library().lib.rt_hip_verify_drafts_workspace_bytes(0, 1, 1, 1, 0) == -1


def test_nothing_to_do(rt, mem):
    """No rows or no requests: accepted without a launch."""
    assert append(rt, mem, n=0, k=None, v=None, slots=None) == 0
    assert attention(rt, mem, n_tokens=0) == 0
    assert attention(rt, mem, n_seq=0) == 0
    assert verify(rt, mem, n_seq=0) == 0


def test_binding_checks_before_it_calls(rt):
    """The Python binding refuses what the C call could not see: CPU tensors, dtypes, shapes, strides."""
    import torch
    k = torch.zeros(2, 8, 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        rt.PagedKV(k, k)
    with pytest.raises(ValueError, match="int32"):
        rt.paged_plan(torch.zeros(2), torch.zeros(2), torch.zeros(2), None, None, None, 16, 4)
    with pytest.raises(ValueError, match="GPU"):
        rt.verify_drafts(torch.zeros(3, 9), None, None, None, torch.zeros(1), 1)


@pytest.fixture
def no_library(rt, monkeypatch):
    """The binding with a library that is never to be called."""
    class Never:
        def call(self, name, *args):
            raise AssertionError(f"{name} was called")
    monkeypatch.setattr(rt, "library", lambda: Never())
    return rt


@pytest.mark.parametrize("n, tokens", [(2, 4), (0, 3), (1, 0)])
@pytest.mark.parametrize("given", [False, True])
def test_plan_refuses_cpu_tensors(no_library, n, tokens, given):
    """Tensors of the right types and shapes, all of them on the CPU: none of their addresses reaches the kernel."""
    import torch
    rt = no_library
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    plan = rt.PagedPlan(n, tokens, "cpu") if given else None
    with pytest.raises(ValueError, match="GPU"):
        rt.paged_plan(z(n), z(n), z(n), z(n, 3), z(8), z(2), 16, tokens, plan=plan)


class OnGpu:
    """A CPU tensor that says it lives on GPU 0."""
    is_cuda = True

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return 0


@pytest.mark.parametrize("pages", [2, 8])
@pytest.mark.parametrize("stride", [0, 64, 1016])
def test_cache_whose_pages_overlap(rt, pages, stride):
    """Pages that share memory: one page expanded (a stride of 0, which is the C call's word for dense), or pages that
    start inside the one before."""
    import torch
    k = OnGpu(torch.zeros(pages * 1024).as_strided((pages, 16, 1, 64), (stride, 64, 64, 1)))
    with pytest.raises(ValueError, match="overlap"):
        rt.PagedKV(k, k)
    # one page has no next one, and pages further apart than dense are a layout like any other
    one = OnGpu(torch.zeros(1024).as_strided((1, 16, 1, 64), (stride, 64, 64, 1)))
    assert rt.PagedKV(one, one).struct.page_stride == 1024
    far = OnGpu(torch.zeros(pages * 2048).as_strided((pages, 16, 1, 64), (2048, 64, 64, 1)))
    assert rt.PagedKV(far, far).struct.page_stride == 2048


@pytest.fixture
def streams(rt, monkeypatch):
    """The binding over CPU tensors that say they live on GPU 0, with a torch that keeps a current stream; what was
    allocated and what was called on which stream, in order, by name."""
    import contextlib
    import torch
    seen, now = [], ["current"]

    class Stream:
        cuda_stream = "side"

    class Cuda:
        @staticmethod
        @contextlib.contextmanager
        def stream(s):
            before, now[0] = now[0], s.cuda_stream
            yield
            now[0] = before

    class Torch:
        cuda = Cuda

        class _C:
            _cuda_getDevice = staticmethod(lambda: 0)
            _cuda_getCurrentRawStream = staticmethod(lambda device: now[0])

        def __getattr__(self, name):
            return getattr(torch, name)

        def _made(name):
            def make(self, *args, **kw):
                seen.append((name, now[0]))
                return OnGpu(getattr(torch, name)(*args, **kw))
            return make
        empty, zeros, full = _made("empty"), _made("zeros"), _made("full")

    class Lib:
        def call(self, name, *args):
            seen.append((name, args[-1]))

    monkeypatch.setattr(rt, "_torch", lambda: Torch())
    monkeypatch.setattr(rt, "library", lambda: Lib())
    return Stream(), seen


@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("what", ["plan", "attention", "verify"])
def test_results_are_made_on_the_stream_of_the_call(rt, streams, side, what):
    """What a call allocates, and fills, belongs to the stream it runs on: a fill of the current stream's could come
    after the kernel, and memory that stream has just given back could still be in use there."""
    import torch
    stream, seen = streams
    i32 = lambda *shape: OnGpu(torch.zeros(shape, dtype=torch.int32))
    f32 = lambda *shape: OnGpu(torch.zeros(shape))
    kw = dict(stream=stream) if side else {}
    if what == "plan":
        rt.paged_plan(i32(2), i32(2), i32(2), i32(2, 3), i32(8), i32(2), 16, 5, **kw)
    elif what == "attention":
        rt.paged_attention(f32(5, 2, 64), rt.PagedKV(f32(8, 16, 1, 64), f32(8, 16, 1, 64)), i32(2, 3), i32(3), i32(2), 0.1, **kw)
    else:
        rt.verify_drafts(f32(5, 9), i32(5), i32(3), f32(5), f32(2), 3, **kw)
    assert len(seen) >= 2 and seen[-1][0].startswith("rt_hip_")
    assert {on for _, on in seen} == {"side" if side else "current"}, seen


@pytest.mark.parametrize("scale", [1.7014121e38, 2.4e38, 3.4028234e38])
def test_attention_refuses_scales_whose_exponents_overflow(rt, mem, scale):
    """Scores are weighed as powers of two, so scale * log2(e) has to be finite too: no more than 2^127."""
    assert attention(rt, mem, scale=C.c_float(scale)) == ARG
    assert attention(rt, mem, scale=C.c_float(scale), n_tokens=0) == ARG
    assert attention(rt, mem, scale=C.c_float(2.0**127), n_tokens=0) == 0


@pytest.mark.parametrize("far", [2**31, 2**32, 2**32 + 16, 2**63, -2**31 - 1, -2**32 + 16])
def test_numbers_that_do_not_fit(no_library, far):
    """Numbers that the C call takes in 32 bits: larger ones would arrive as others."""
    import torch
    rt = no_library
    i32 = lambda *shape: OnGpu(torch.zeros(shape, dtype=torch.int32))
    f32 = lambda *shape: OnGpu(torch.zeros(shape))
    kv = rt.PagedKV(f32(8, 16, 1, 64), f32(8, 16, 1, 64))
    for name in ("window", "max_fresh"):
        with pytest.raises(ValueError, match=name):
            rt.paged_attention(f32(5, 2, 64), kv, i32(2, 3), i32(3), i32(2), 0.1, out=f32(5, 2, 64), **{name: far})
    for at, name in enumerate(("n_q_heads", "n_seq", "tokens", "max_fresh")):
        with pytest.raises(ValueError, match=name):
            rt.paged_attention_workspace_bytes(kv, rt.F32, *[far if i == at else 2 for i in range(4)])
    with pytest.raises(ValueError, match="page_size"):
        rt.paged_plan(i32(2), i32(2), i32(2), i32(2, 3), i32(8), i32(2), far, 5, plan=rt.PagedPlan(2, 5, "cpu"))


@pytest.mark.parametrize("apart, stride, pages, one", [
    (0, 0, 2, True), (512, 0, 2, True), (512, 0, 1, False), (1024, 0, 2, False), (512, 1024, 4, False), (512, 1024, 1, False),
    (1024, 1024, 4, True), (256, 1024, 4, True), (768, 1024, 4, True), (1536, 1024, 2, False), (1536, 1024, 4, False),
    (2048, 1024, 2, False)])
def test_append_refuses_keys_over_values(rt, mem, apart, stride, pages, one):
    """Keys and values of one memory (values apart, of 512 to a page): both would be written there.  Either order; pages
    of the two in turn are no such case, nor is it one to read."""
    base = mem[12]
    for k, v in ((base, base + 2 * apart), (base + 2 * apart, base)):
        kv = cache(rt, mem, k=k, v=v, page_stride=stride, n_pages=pages)
        assert append(rt, mem, kv=kv, n=0, k=None, v=None, slots=None) == (ARG if one else 0)
        assert attention(rt, mem, kv=kv, n_tokens=0) == 0
