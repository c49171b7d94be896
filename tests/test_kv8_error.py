"""How far what a page holds may be from what came, as `ops.kv8` states it: within 2^-4 of the value or 2^-10 of the page's scale; where
the scale has grown since, within 2^-4 of the value or 2^-9 of the scale."""
import pytest
import torch

from plain import kv8_plain as plain

HD = 256
# The sum behind the second: a number that becomes subnormal when the scale is S was off by half a step of the binade below 2^-6 S, 2^-11 S,
# and is rounded by 2^-10 of that scale and of every later one, each at least twice the one before: below 2^-9 of the last.


def rows_of(factor, seed):
    """Rows of one page whose largest magnitudes grow by `factor` from row to row; small values between steps of all kinds."""
    g = torch.Generator().manual_seed(seed)
    n = 14 if factor < 5 else 8                                            # (larger ones pass 448 * 2^40 before the 14th)
    x = torch.zeros((n, 1, HD))
    for i in range(n):
        top = 300.0 * factor ** i
        x[i, 0] = top * 2.0 ** (-18 * torch.rand(HD, generator=g)) * torch.where(torch.rand(HD, generator=g) < 0.5, -1.0, 1.0)
        x[i, 0, 0] = top
    return x


def off(held, x, scale):
    """The largest error, as a part of what is allowed below 2^-4 of the value: in units of 2^-10 of the scale."""
    e = (held - x.double()).abs()
    return float(torch.where(e <= 2.0 ** -4 * x.double().abs(), torch.zeros_like(e), e / (2.0 ** -10 * scale)).max())


def empty():
    return plain.PlainCache(torch.zeros((2, 1, plain.PAGE, HD), dtype=torch.uint8), torch.zeros((2, 1, plain.PAGE, HD), dtype=torch.uint8),
                            torch.ones(2, 1), torch.ones(2, 1))


@pytest.mark.parametrize("factor", [1.3, 2.0, 3.1, 4.0, 30.0])
def test_the_definition(factor):
    worst = 0.0
    for seed in range(8):
        x, cache = rows_of(factor, seed), empty()
        for i in range(x.shape[0]):
            cache.append(x[i:i + 1], 0, torch.tensor([1]), i)
            scale = float(cache.scale[0][1, 0])
            held = cache.read(0, [1], 0, i + 1)
            assert off(held[i:], x[i], scale) <= 1.0                       # (the row that came last was rounded once)
            assert off(held, x[:i + 1, 0], scale) <= 2.0
            worst = max(worst, off(held, x[:i + 1, 0], scale))
    assert factor > 2 or worst > 1.0                                       # numbers of a page that grows step by step do pass 2^-10


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("factor", [1.3, 2.0, 3.1, 30.0])
def test_the_device(factor, dtype):
    from picolm_b200 import ops
    from test_gpu_kv8 import DEV, DTYPES, Setup, i32
    s = Setup([plain.PAGE], 1, HD, seed=1).device()
    x = rows_of(factor, 3).to(DTYPES[dtype])
    rows, page = x.to(DEV), int(s.table[0, 0])
    for i in range(x.shape[0]):
        ops.store_kv8(rows[i:i + 1], rows[i:i + 1], s.dk, s.dv, s.dks, s.dvs, i32([0, 1]), i32([i + 1]), s.dt, 1)
        for held, scale in ((s.dk, s.dks), (s.dv, s.dvs)):
            now = float(scale[page, 0])
            got = plain.VALUES[held[page, 0, :i + 1].view(torch.uint8).cpu().long()] * now
            assert off(got[i:], x[i], now) <= 1.0 and off(got, x[:i + 1, 0], now) <= 2.0
