"""Attention over the 8-bit cache where one key has almost all of a row's weight: what the others give still counts, as it does
in long contexts whose first token draws the weight and holds next to nothing."""
import math

import pytest
import torch

from plain import kv8_plain as plain
from test_gpu_kv8 import DEV, PAGE, Setup, i32

pytestmark = pytest.mark.gpu


def one_key_above(n, new, H, G, hd, octaves, spread, seed):
    """A sequence of n keys: the first one's weight is 2^octaves of the others', which are equal, and its value is zero; the others' values
    are positive, in pages whose scales lie up to 2^spread apart."""
    s = Setup([n], G, hd, seed).fill([n], G, hd)
    scale = hd ** -0.5
    s.k &= 0
    s.ks[:] = 1.0
    s.k[int(s.table[0, 0]), :, 0, 0] = 0x38                            # 1.0 in the first component
    s.v &= 0x7f
    s.v[s.v == 0x7f] = 0x38
    s.v[int(s.table[0, 0]), :, 0] = 0
    s.vs[:] = 2.0 ** torch.randint(0, spread + 1, s.vs.shape, generator=s.g)
    q = torch.zeros((new, H, hd))
    q[:, :, 0] = octaves * math.log(2) / scale
    return s.device(), q.bfloat16(), scale


def check(got, s, q, positions, G, scale, spread):
    """Weights are halves times a power of two a row, 2^6 at the largest or more: 2^-11 of a weight down to 2^-20 of the largest, below
    that 2^-31 of the largest (2^-28 where pages' units differ: a weight then stands for up to 2^3 of its page's); scores, exp2, sums
    and the result as everywhere."""
    cache = s.plain()
    H, hd = q.shape[1:]
    for t, p in positions:
        o, w, size = plain.attend(q[t].double(), p, cache, s.table[0], G, scale)
        n = p + 1
        v = torch.stack([cache.read(1, s.table[0], h // (H // G), n).abs().sum(0) for h in range(H)])
        rel = 2 * (hd + 8) * 2.0 ** -24 * size[:, None] * 1.5 + 2.0 ** -20 + (n + 8) * 2.0 ** -24 + 2.0 ** -11 * 1.01
        bound = torch.finfo(torch.bfloat16).eps / 2 * o.abs() + rel * w + v * 2.0 ** (-28 if spread else -31)
        off = ((got[t].double().cpu().reshape(H, hd) - o).abs() / bound)
        assert float(off.max()) <= 1.0001, f"row {t} at {p}: off {float(off.max()):.3g} times the bound, {float(o.mean()):.3g} expected"


@pytest.mark.parametrize("spread", [0, 3])
@pytest.mark.parametrize("octaves", [14.0, 20.3, 24.6, 27.0])
@pytest.mark.parametrize("H,G,hd", [(4, 2, 64), (8, 1, 128), (6, 2, 96), (20, 1, 64), (4, 2, 256)])
def test_single_tokens(H, G, hd, octaves, spread):
    from picolm_b200 import ops
    n = 3000
    s, q, scale = one_key_above(n, 3, H, G, hd, octaves, spread, seed=hd)
    pos = [n - 1, 1000, 200]
    for splits in (None, 0, 1, 8):
        got = ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(pos), i32([0, 0, 0]), s.dt, n, G, scale, n_splits=splits)
        check(got, s, q, list(enumerate(pos)), G, scale, spread)


@pytest.mark.parametrize("spread", [0, 3])
@pytest.mark.parametrize("octaves", [14.0, 20.3, 24.6, 27.0])
@pytest.mark.parametrize("H,G,hd,new", [(4, 2, 64, 300), (4, 2, 128, 70), (6, 2, 96, 100), (4, 2, 64, 5), (4, 1, 128, 7), (4, 2, 256, 90)])
def test_prompts(H, G, hd, new, octaves, spread):
    from picolm_b200 import ops
    n = 2500
    s, q, scale = one_key_above(n, new, H, G, hd, octaves, spread, seed=hd + new)
    for more in (dict(), dict(keep_first=1, window=2 * n)):              # (the second walks from the newest page to the oldest)
        got = ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, new]), i32([n]), s.dt, new, n, G, scale, **more)
        check(got, s, q, [(t, n - new + t) for t in sorted({0, 1, new // 2, new - 1})], G, scale, spread)
    ops.check_status(DEV)


@pytest.mark.parametrize("low", [-40, -60])
@pytest.mark.parametrize("H,G,hd,new", [(4, 2, 64, 1), (8, 1, 128, 1), (4, 2, 64, 300), (4, 1, 128, 7), (4, 2, 128, 70), (8, 2, 96, 100)])
def test_units_as_far_apart_as_the_format_has_them(H, G, hd, new, low):
    """Pages of values around 2^low and 2^40 in turn, with equal scores and with unequal ones: sums stay finite in either unit."""
    from picolm_b200 import ops
    n, scale = 2500, hd ** -0.5
    s = Setup([n], G, hd, seed=hd).fill([n], G, hd)
    for i in range(s.table.shape[1]):
        s.vs[int(s.table[0, i])] = 2.0 ** (40 if i % 2 else low)
    s.device()
    for size in (0.0, 1.0):
        q = (torch.randn((new, H, hd), generator=s.g) * size).bfloat16()
        pos = [n - new + t for t in range(new)]
        if new == 1:
            outs = [ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(pos), i32([0]), s.dt, n, G, scale, n_splits=k) for k in (None, 0, 1, 8)]
        else:
            outs = [ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, new]), i32([n]), s.dt, new, n, G, scale, **more)
                    for more in (dict(), dict(keep_first=1, window=2 * n))]
        for got in outs:
            check(got, s, q, [(t, pos[t]) for t in sorted({0, new // 2, new - 1})], G, scale, 3)
