"""A value that is NaN reaches every row that sees its place, also one whose weight there is nothing, whatever the kernel and however
the keys are cut; places that a row does not see do not."""
import math

import pytest
import torch

from test_gpu_kv8 import DEV, DTYPES, PAGE, Setup, check_attention, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("H,G,hd", [(4, 2, 64), (20, 2, 128), (3, 1, 24), (4, 4, 96)])
def test_a_value_without_weight(H, G, hd, dtype):
    """Its key's score is some 300 octaves below the others'."""
    from picolm_b200 import ops
    n = 260
    s = Setup([n], G, hd, seed=hd).fill([n], G, hd)
    s.k[:, :, :, 0] = 0x38                                            # 1.0
    for pos, comp in ((50, 3), (130, 7), (n - 3, 11)):
        page, place = int(s.table[0, pos // PAGE]), pos % PAGE
        s.k[page, :, place, 0] = 0xe0                                 # -64.0
        s.v[page, 0, place, comp] = 0x7f
    s.ks[:] = 2.0 ** -2
    s.device()
    scale = hd ** -0.5
    q = torch.randn((40, H, hd), generator=s.g) * 0.1
    q[:, :, 0] = 13.0 / scale
    q = q.to(DTYPES[dtype])
    for window in (None, 180):
        pos = [n - 1, n - 2, n - 4, 129, 49]
        for splits in (None, 0, 1, 3, 8):
            got = ops.attention_kv8_decode(q[:5].contiguous().to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(pos), i32([0] * 5), s.dt, n, G, scale, window=window,
                                           n_splits=splits)
            check_attention(got, s, q, [(t, 0, p) for t, p in enumerate(pos)], G, scale, dtype, window=window)
        for new in (3, 40):
            got = ops.attention_kv8_prefill(q[:new].contiguous().to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, new]), i32([n]), s.dt, new, n, G, scale, window=window)
            check_attention(got, s, q, [(t, 0, n - new + t) for t in range(0, new, 3)], G, scale, dtype, window=window)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("H,G,hd", [(4, 2, 64), (2, 1, 128), (3, 1, 24)])
def test_a_value_where_all_scores_are_minus_infinity(H, G, hd, dtype):
    """Beside a sink such a row is zero but for the components whose value is NaN somewhere."""
    from picolm_b200 import ops
    n = 700
    s = Setup([n], G, hd, seed=hd).fill([n], G, hd)
    s.k[:, :, :, 1] = 0x38
    for pos, comp in ((2, 0), (330, 5), (n - 2, 9)):
        s.v[int(s.table[0, pos // PAGE]), 0, pos % PAGE, comp] = 0xff
    s.device()
    sink = torch.randn(H, generator=s.g)
    q = torch.randn((40, H, hd), generator=s.g).to(DTYPES[dtype])
    q[0, 0, 1], q[2, H - 1, 1] = -math.inf, -math.inf
    pos = [n - 1, n - 3, 400]
    for splits in (None, 0, 1, 3, 8):
        got = ops.attention_kv8_decode(q[:3].contiguous().to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(pos), i32([0] * 3), s.dt, n, G, hd ** -0.5, n_splits=splits,
                                       sink=sink.to(DEV))
        check_attention(got, s, q, [(t, 0, p) for t, p in enumerate(pos)], G, hd ** -0.5, dtype, sink=sink)
    for new in (3, 40):
        got = ops.attention_kv8_prefill(q[:new].contiguous().to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, new]), i32([n]), s.dt, new, n, G, hd ** -0.5,
                                        sink=sink.to(DEV))
        check_attention(got, s, q, [(t, 0, n - new + t) for t in (0, 1, 2, new - 1)], G, hd ** -0.5, dtype, sink=sink)
