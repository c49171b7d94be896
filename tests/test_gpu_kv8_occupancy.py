"""The streaming kernel of 8-bit attention deals work out to as many CTAs as it says run at once: an SM has room for them.  What a launch
takes comes from the profiler, in a process of its own that has compiled every head size before the profiler starts."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SM_SMEM, SM_REGISTERS, SYSTEM_SMEM = 228 * 1024, 64 * 1024, 1024
CASES = [(64, 8), (64, 16), (64, 32), (96, 8), (112, 8), (112, 16), (128, 8), (128, 16), (128, 32), (240, 8), (240, 16), (256, 8), (256, 16)]

CHILD = """
import sys; sys.path[:0] = [{root!r}, {tests!r}]
import json, torch
from torch.profiler import ProfilerActivity, profile
from picolm_b200 import ops
from picolm_b200.ops import kv8
from test_gpu_kv8 import DEV, Setup, i32
calls = []
for hd, rows in {cases!r}:
    s = Setup([300], 1, hd, seed=1).fill([300], 1, hd).device()
    q = torch.randn((1, rows, hd), generator=s.g).bfloat16().to(DEV)
    for splits in (0, 2):
        calls.append((hd, rows, splits, lambda s=s, q=q, splits=splits: ops.attention_kv8_decode(
            q, s.dk, s.dv, s.dks, s.dvs, i32([299]), i32([0]), s.dt, 300, 1, 0.1, n_splits=splits)))
        calls[-1][3]()
torch.cuda.synchronize()
for hd, rows, splits, call in calls:
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    p.export_chrome_trace({trace!r})
    a, = [e["args"] for e in json.load(open({trace!r}))["traceEvents"] if "kv8_stream_kernel" in e.get("name", "") and "args" in e]
    print(json.dumps(["launch", hd, rows, splits, a["block"][0], a["registers per thread"], a["shared memory"], *kv8.kv8_few_plan(hd, rows)[:2], kv8.SM_COUNT]))
"""


def test_as_many_ctas_as_it_says(tmp_path):
    tests = os.path.dirname(os.path.abspath(__file__))
    code = CHILD.format(root=os.path.dirname(tests), tests=tests, cases=CASES, trace=str(tmp_path / "trace.json"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    found = [json.loads(line)[1:] for line in r.stdout.splitlines() if line.startswith('["launch"')]
    assert len(found) == 2 * len(CASES)
    short = []
    for hd, rows, splits, threads, registers, smem, tile, at_once, sms in found:
        room = min(SM_SMEM // (smem + SYSTEM_SMEM), SM_REGISTERS // (-(-registers * 32 // 256) * 256 * (threads // 32)))
        assert tile >= min(rows, 16)
        if at_once > room * sms:
            short.append((hd, rows, splits, smem, registers, at_once, room))
    assert not short, "more CTAs than run at once: " + str(short)
