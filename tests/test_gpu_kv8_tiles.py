"""Long prompts over the 8-bit cache of head sizes other than 64 and 128: more rows than the streaming kernel is given."""
import pytest
import torch

from test_gpu_kv8 import DEV, i32, check_attention
from test_gpu_kv8_scales import arguments, unequal

pytestmark = pytest.mark.gpu

CASES = [  # H, G, hd, (new, before), more
    (8, 2, 80, [(100, 30), (2, 3), (70, 64)], {}), (6, 2, 96, [(150, 0)], dict(window=20)), (4, 1, 256, [(66, 10), (0, 5)], {}), (8, 2, 112, [(129, 77)], dict(slopes=True)),
    (4, 1, 32, [(140, 77), (90, 1)], dict(window=40, keep_first=70)), (8, 2, 48, [(150, 0)], dict(window=-32)), (4, 1, 16, [(200, 5)], dict(sink=True)),
    (8, 2, 96, [(90, 200)], dict(sink=True, slopes=True, window=60, keep_first=3)), (4, 1, 160, [(80, 300)], dict(window=64)),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_tiles(case):
    from picolm_b200 import ops
    from picolm_b200.ops.kv8 import kv8_streams
    H, G, hd, seqs, more = CASES[case]
    lens, max_new = [n + b for n, b in seqs], max(n for n, _ in seqs)
    assert not kv8_streams(len(seqs) * G, max_new * H // G, max(lens), hd)
    s = unequal(lens, G, hd, 300 + case)
    s.v[int(s.table[0, 1]), 0, 3, 5] = 0x7f                             # a value that is NaN, which some rows see
    s.device()
    offs = [0]
    for n, _ in seqs:
        offs.append(offs[-1] + n)
    T = offs[-1]
    q = (torch.randn((T + 2, H, hd), generator=s.g) * 0.25).bfloat16()
    args, on = arguments(more, H, s.g)
    for bound in (max_new, max_new + 70):
        out = torch.full((T + 2, H * hd), 5.0, dtype=q.dtype, device=DEV)
        ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(offs), i32(lens), s.dt, bound, max(lens), G, hd ** -0.5, out=out, **on)
        assert bool((out[T:] == 5.0).all()), "rows of no sequence"
        check_attention(out, s, q, [(offs[b] + i, b, before + i) for b, (n, before) in enumerate(seqs) for i in sorted({*range(0, n, 13), n - 1} - {-1})],
                        G, hd ** -0.5, "bfloat16", **args)
