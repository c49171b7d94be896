"""The checked build reports a page's scale that is no power of two, or one out of bounds, at every kernel that reads it."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import sys; sys.path[:0] = [{root!r}, {tests!r}]
import torch
from picolm_b200 import ops
from test_gpu_kv8 import DEV, DTYPES, Setup, i32
assert ops._lib.CHECKED
H, G = 4, 2
for hd, new, dtype in ((64, 100, "bfloat16"), (64, 3, "bfloat16"), (80, 40, "bfloat16"), (24, 5, "bfloat16"), (64, 1, "float32")):
    s = Setup([150], G, hd, seed=1).fill([150], G, hd).device()
    q = torch.randn((new, H, hd), generator=s.g).to(DTYPES[dtype]).to(DEV)
    cache = (s.dk, s.dv, s.dks, s.dvs)
    rows = torch.randn((1, G, hd), generator=s.g).to(q.dtype).to(DEV)
    calls = [lambda: ops.attention_kv8_prefill(q, *cache, i32([0, new]), i32([150]), s.dt, new, 150, G, 0.1),
             lambda: ops.attention_kv8_decode(q[:1], *cache, i32([149]), i32([0]), s.dt, 150, G, 0.1),
             lambda: ops.store_kv8(rows, rows, *cache, i32([0, 1]), i32([150]), s.dt, 1)]
    for call in calls:
        call()
        ops.check_status(DEV)
        for scales in (s.dks, s.dvs):
            for bad in (3.0, 0.0, -2.0, 2.0 ** 41, 2.0 ** -61, float("nan"), float("inf")):
                page = int(s.dt[0, 2])
                good = scales[page, 1].clone()
                scales[page, 1] = bad
                call()
                scales[page, 1] = good
                try:
                    ops.check_status(DEV)
                except ops.KernelError as e:
                    assert "scale of a page" in str(e)
                else:
                    raise AssertionError(f"{{hd}} {{new}} {{dtype}}: {{bad}} passed")
print("checked")
"""


def test_scales_that_the_format_does_not_have():
    tests = os.path.dirname(os.path.abspath(__file__))
    code = CHILD.format(root=os.path.dirname(tests), tests=tests)
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PICOLM_B200_CHECK="1"), capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and "checked" in r.stdout, r.stderr[-2000:]
