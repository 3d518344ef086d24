"""Bytes of a 4-bit cache's pages that append never wrote reach no row, whatever they are.

Finite numbers a and b of a group can stand for infinities (a = b = 61280, bytes of 0x7b, for every
code; two in a hundred values of bits at random), and a weight of 0 times one of those is a
NaN.  Tolerances: those of test_gpu_paged4_attention, whose steps these are."""
import pytest
import torch

from helpers import say
from test_gpu_paged4_attention import TYPES, Step

pytestmark = pytest.mark.gpu


def poison(raw, byte, seed):
    if byte == "any":
        g = torch.Generator(device="cuda").manual_seed(seed)
        raw.copy_(torch.randint(0, 256, raw.shape, generator=g, device="cuda").to(torch.uint8))
    else:
        raw.fill_(byte)


class Unwritten(Step):
    """A step over pages that held `byte` ("any": bits at random) before, whose pages in front of
    the first key that a request's rows see hold it again."""

    def __init__(self, rt, byte, *args, **kw):
        def before(step, k, v):
            for i, raw in enumerate((step.kv.k, step.kv.v)):
                poison(raw, byte, 10 + i)

        super().__init__(rt, *args, spoil=before, **kw)
        self.stale = 0
        for s, (n, length) in enumerate(self.lens):
            first = length - n - self.window + 1 if self.window else 0
            for c in range(max(0, first) // self.page):
                for i, raw in enumerate((self.kv.k, self.kv.v)):
                    poison(raw[int(self.table[s, c])], byte, 20 + i)
                self.stale += 1


BYTES = [0x7B, 0xFB, "any"]
# keys that end inside a group of 8, a tile of 32 or 64, a page; few rows, many, both
MIXED = [(1, 1), (1, 43), (5, 301), (40, 43), (130, 333), (64, 65), (33, 39), (3, 1000), (2, 2), (300, 307)]


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("byte", BYTES)
def test_behind_the_last_key(rt, q, dim, byte):
    say("unwritten4", q, dim, byte)
    Unwritten(rt, byte, q, 6, 2, dim, 16, MIXED, seed=dim).check(rt)
    Unwritten(rt, byte, q, 2, 2, dim, 64, [(200, 459)], seed=dim + 1).check(rt)
    Unwritten(rt, byte, q, 8, 1, dim, 8, [(1, 700), (1, 9)], seed=dim + 2, joint=True).check(rt)


@pytest.mark.parametrize("q", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("byte", BYTES)
@pytest.mark.parametrize("page, window", [(8, 10), (16, 100), (8, 1)])
def test_in_front_of_the_window(rt, q, dim, byte, page, window):
    say("unwritten4 window", q, dim, byte, page, window)
    step = Unwritten(rt, byte, q, 6, 2, dim, page, MIXED, seed=dim, window=window)
    assert step.stale > 20
    step.check(rt)
    # keys that end with a tile: only those in front of the window were not written
    for lens in ([(70, 448)], [(1, 256), (5, 640), (3, 1024), (2, 128)]):
        Unwritten(rt, byte, q, 4, 2, dim, page, lens, seed=dim + 1, window=window).check(rt)


def test_few_and_many_rows_alike(rt):
    """A row alone, and among many, over pages of any bytes."""
    for byte in BYTES:
        many = Unwritten(rt, byte, "f32", 4, 2, 128, 16, [(40, 77)], seed=3)
        got = many.run(rt).clone()
        assert torch.isfinite(got).all()
        last = Unwritten(rt, byte, "f32", 4, 2, 128, 16, [(1, 77)], seed=3)
        last.kv, last.table = many.kv, many.table
        last.q.copy_(many.q[-1:])
        want, tol = many.reference()
        assert ((last.run(rt)[0] - want[-1]).abs() <= tol[-1]).all()
