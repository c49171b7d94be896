"""The 8-bit cache's operators as programs call them: captured and replayed, on two streams at once, twice, through the checked
build, with sequences that the table does not hold, and with a wait that runs out."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_kv8 import DEV, PAGE, Setup, check_attention, i32, run_append, same_cache, tables

pytestmark = pytest.mark.gpu


def setup(lens, H=8, G=2, hd=64, seed=3, per_seq=None):
    s = Setup(lens, G, hd, seed, per_seq=per_seq).fill(lens, G, hd).device()
    return s, torch.randn((len(lens), H, hd), generator=s.g).bfloat16()


@pytest.mark.parametrize("n_splits", [0, 4])
def test_decode_in_a_graph_follows_the_buffers(n_splits):
    """One capture, replayed for other positions, sequences and queries, and the same bits every time."""
    from picolm_b200 import ops
    lens = [700, 64, 129, 300]
    s, q = setup(lens)
    pos, seq, dq = i32([0] * 4), i32([0] * 4), torch.zeros_like(q, device=DEV)
    call = lambda: ops.attention_kv8_decode(dq, s.dk, s.dv, s.dks, s.dvs, pos, seq, s.dt, 700, 2, 0.125, n_splits=n_splits)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for order, back in (([0, 1, 2, 3], 0), ([3, 0, 2, 1], 5), ([1, 1, 0, 0], 1)):
        p = [lens[b] - 1 - back for b in order]
        pos.copy_(i32(p)), seq.copy_(i32(order)), dq.copy_(q)
        g.replay()
        first = out.clone()
        check_attention(first, s, q, list(zip(range(4), order, p)), 2, 0.125, "bfloat16")
        g.replay()
        assert torch.equal(out, first)


@pytest.mark.parametrize("hd,new", [(64, 100), (128, 80), (96, 70), (64, 6)])
def test_two_streams_at_once(hd, new):
    """Appends and attention of two caches on two streams: the same bits as one after the other."""
    from picolm_b200 import ops
    H, G = 8, 2
    both = []
    for k in range(2):
        s = Setup([900 + new], G, hd, seed=k).fill([900], G, hd).device()
        qkv = torch.randn((new, (H + 2 * G) * hd), generator=s.g).bfloat16().to(DEV)
        both.append((s, qkv))

    def work(s, qkv):
        q = torch.empty((new, H, hd), dtype=torch.bfloat16, device=DEV)
        outs = []
        for _ in range(4):
            ops.rope_store_kv8(qkv, q, s.dk, s.dv, s.dks, s.dvs, None, None, i32([0, new]), i32([900 + new]), s.dt, new, H, G, hd, 0, "half")
            outs.append(ops.attention_kv8_prefill(q, s.dk, s.dv, s.dks, s.dvs, i32([0, new]), i32([900 + new]), s.dt, new, 900 + new, G, hd ** -0.5))
            outs.append(ops.attention_kv8_decode(q, s.dk, s.dv, s.dks, s.dvs, i32([900 + new - 1] * new), i32([0] * new), s.dt, 900 + new, G, hd ** -0.5, n_splits=0))
        return outs

    alone = [[o.clone() for o in work(*x)] for x in both]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in both]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    together = []
    for st, x in zip(streams, both):
        with torch.cuda.stream(st):
            together.append(work(*x))
    torch.cuda.synchronize()
    for a, b in zip(alone, together):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    ops.check_status(DEV)


def test_steps_one_after_another_without_a_pause():
    """An append and the attention that reads it, launched back to back over page borders: every kernel may begin while the one before
    still runs, and none may read what that one has not written."""
    from picolm_b200 import ops
    H, G, hd, n = 8, 2, 128, 70
    s = Setup([60 + n] * 3, G, hd, seed=11).fill([60] * 3, G, hd).device()
    rows = torch.randn((n, 3, (H + 2 * G) * hd), generator=s.g).bfloat16()
    dev = rows.to(DEV)
    q = [torch.empty((3, H, hd), dtype=torch.bfloat16, device=DEV) for _ in range(n)]
    start, seq = i32([0, 1, 2, 3]), i32([0, 1, 2])
    lens, pos = [i32([61 + j] * 3) for j in range(n)], [i32([60 + j] * 3) for j in range(n)]
    torch.cuda.synchronize()
    outs = []
    for j in range(n):
        ops.rope_store_kv8(dev[j], q[j], s.dk, s.dv, s.dks, s.dvs, None, None, start, lens[j], s.dt, 1, H, G, hd, 0, "half")
        outs.append(ops.attention_kv8_decode(q[j], s.dk, s.dv, s.dks, s.dvs, pos[j], seq, s.dt, 61 + j, G, hd ** -0.5))
    torch.cuda.synchronize()
    want = s.plain()
    for j in range(n):
        x = rows[j].float().view(3, H + 2 * G, hd)
        for b in range(3):
            want.append(x[b:b + 1, H:H + G], 0, s.table[b], 60 + j)
            want.append(x[b:b + 1, H + G:], 1, s.table[b], 60 + j)
        if j % 23 == 4 or j == n - 1:
            class Now:
                table, plain = s.table, staticmethod(lambda: want)
            check_attention(outs[j], Now, rows[j].view(3, H + 2 * G, hd)[:, :H], [(b, b, 60 + j) for b in range(3)], G, hd ** -0.5, "bfloat16")
    same_cache(s, want, None)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_sequences_that_the_table_does_not_hold_are_left_out(dtype):
    """Positions behind the table's row, and more new tokens than a sequence has: those have no rows, the others are as ever."""
    from picolm_b200 import ops
    H, G, hd = 4, 2, 64
    s = Setup([100, 128, 90], G, hd, seed=4, per_seq=2).fill([100, 128, 90], G, hd).device()
    q = torch.randn((9, H, hd), generator=s.g).to(torch.bfloat16 if dtype == "bfloat16" else torch.float32)
    out = torch.full((9, H * hd), 3.0, dtype=q.dtype, device=DEV)
    ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, 3, 6, 9]), i32([100, 130, 2]), s.dt, 3, 128, G, 0.125, out=out)
    check_attention(out, s, q, [(i, 0, 97 + i) for i in range(3)], G, 0.125, dtype)
    assert bool((out[3:] == 3.0).all())
    got = ops.attention_kv8_decode(q[:3].contiguous().to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([99, 128, 50]), i32([0, 1, 2]), s.dt, 128, G, 0.125, n_splits=0)
    check_attention(got, s, q, [(0, 0, 99), (2, 2, 50)], G, 0.125, dtype)


def test_more_heads_rows_and_pages_than_one_of_anything():
    """Many sequences (more than a warp's lanes hold at once), most of them short, one long; many heads a kv head."""
    from picolm_b200 import ops
    lens = [1 + (7 * i) % 90 for i in range(150)]
    lens[77] = 3000
    s, q = setup(lens, H=4, G=1, hd=64)
    got = ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([n - 1 for n in lens]), i32(list(range(150))), s.dt, 3000, 1, 0.125, n_splits=0)
    check_attention(got, s, q, [(b, b, lens[b] - 1) for b in (0, 1, 31, 32, 76, 77, 78, 127, 128, 149)], 1, 0.125, "bfloat16")
    s, q = setup([200, 65], H=80, G=1, hd=128)
    got = ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([199, 64]), i32([0, 1]), s.dt, 200, 1, 0.1)
    check_attention(got, s, q, [(0, 0, 199), (1, 1, 64)], 1, 0.1, "bfloat16")


def test_a_page_that_does_not_come_is_reported_not_hung():
    """A test build of the prompts' kernel that announces more bytes of a page than it asks for: no page ever counts as there, the
    kernel gives up and returns, and the next call is right."""
    from picolm_b200 import ops
    from picolm_b200.csrc.build import load_library
    from picolm_b200.ops import _lib
    H, G, hd, n = 8, 2, 64, 100
    lib = load_library("attention_kv8_tc@stall", ["-DPLM_HD=64", "-DPLM_WAIT_LIMIT=20000", "-DPLM_TEST_STALL"])
    f = lib.plm_kv8_attention_tc
    f.argtypes, f.restype = _lib._SIGNATURES["plm_kv8_attention_tc"], ctypes.c_int
    lib.plm_test_stall.argtypes = [ctypes.c_int, ctypes.c_void_p]
    s = Setup([300], G, hd, seed=8).fill([300], G, hd).device()
    q = torch.randn((n, H, hd), generator=s.g).bfloat16()
    dq, start, kv_len, status = q.to(DEV), i32([0, n]), i32([300]), ops.status_word(DEV)
    ops.check_status(DEV)
    stream = torch.cuda.current_stream().cuda_stream

    def call():
        out = torch.zeros((n, H * hd), dtype=torch.bfloat16, device=DEV)
        assert f(dq.data_ptr(), s.dk.data_ptr(), s.dv.data_ptr(), s.dks.data_ptr(), s.dvs.data_ptr(), out.data_ptr(), start.data_ptr(), kv_len.data_ptr(),
                 s.dt.data_ptr(), s.dt.shape[1], 1, n, H, G, 0.125, 0, status.data_ptr(), None, 0, None, stream) == 0
        torch.cuda.synchronize()
        return out

    assert lib.plm_test_stall(1, stream) == 0
    call()
    assert int(status.item()) in (70, 71, 72, 73)
    with pytest.raises(ops.KernelError, match="gave up waiting"):
        ops.check_status(DEV)
    assert lib.plm_test_stall(0, stream) == 0
    check_attention(call(), s, q, [(i, 0, 200 + i) for i in range(0, n, 9)], G, 0.125, "bfloat16")
    ops.check_status(DEV)


CHECKED = """
import sys; sys.path[:0] = [{root!r}, {tests!r}]
import torch
from picolm_b200 import ops
from test_gpu_kv8 import DEV, Setup, i32, check_attention
assert ops._lib.CHECKED
H, G = 4, 2
for hd, n in ((64, 100), (64, 3), (80, 40), (24, 5)):
    s = Setup([150], G, hd, seed=1).fill([150], G, hd).device()
    q = torch.randn((n, H, hd), generator=s.g).bfloat16()
    call = lambda: ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, n]), i32([150]), s.dt, n, 150, G, 0.1)
    check_attention(call(), s, q, [(i, 0, 150 - n + i) for i in range(0, n, 11)], G, 0.1, "bfloat16")
    rows = torch.randn((n, H + 2 * G, hd), generator=s.g).bfloat16().reshape(n, -1).to(DEV)
    store = lambda: ops.rope_store_kv8(rows, torch.empty_like(q, device=DEV), s.dk, s.dv, s.dks, s.dvs, None, None, i32([0, n]), i32([150]), s.dt, n, H, G, hd, 0, "half")
    store()
    ops.check_status(DEV)
    s.dt[0, 2] = 4000                                          # a page that the cache does not have
    for f in (call, store):
        f()
        try:
            ops.check_status(DEV)
        except ops.KernelError as e:
            assert "page number" in str(e)
        else:
            raise AssertionError("nothing was reported")
print("checked")
"""


def test_the_checked_build_reports_a_page_that_is_not_there():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = CHECKED.format(root=root, tests=os.path.join(root, "tests"))
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PICOLM_B200_CHECK="1"), capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "checked" in r.stdout, r.stderr[-2000:]


def test_a_cache_whose_offsets_pass_32_bits():
    """Pages behind the first 4 GB of keys and of values: the same bits as in a small cache."""
    from picolm_b200 import ops
    H, G, hd, n = 8, 8, 128, 70
    far, lens = 66_000, [400, 300]
    s, _ = setup(lens, H=H, G=G, hd=hd)
    big = [torch.zeros((far + s.n_pages, G, PAGE, hd), dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2)]
    scales = [torch.ones((far + s.n_pages, G), device=DEV) for _ in range(2)]
    assert big[0].numel() > 2 ** 32
    for x, y in zip(big + scales, (s.dk, s.dv, s.dks, s.dvs)):
        (x.view(torch.uint8) if x.dim() == 4 else x)[far:] = y.view(torch.uint8) if y.dim() == 4 else y
    table = torch.where(s.dt > 0, s.dt + far, 0).to(torch.int32)
    rows = torch.randn((2 * n, (H + 2 * G) * hd), generator=s.g)
    for dtype in (torch.bfloat16, torch.float32):
        x = rows.to(dtype).to(DEV)
        outs = []
        for cache, t in (((s.dk, s.dv, s.dks, s.dvs), s.dt), ((*big, *scales), table)):
            q = torch.empty((2 * n, H, hd), dtype=dtype, device=DEV)
            start, kv_len = i32([0, n, 2 * n]), i32(lens)
            ops.rope_store_kv8(x, q, *cache, None, None, start, kv_len, t, n, H, G, hd, 0, "half")
            a = ops.attention_kv8_prefill(q, *cache, start, kv_len, t, n, 400, G, 0.09)
            q2 = q[:2].contiguous()
            outs.append([a] + [ops.attention_kv8_decode(q2, *cache, i32([399, 299]), i32([0, 1]), t, 400, G, 0.09, n_splits=k) for k in (0, 2)])
            few = ops.attention_kv8_prefill(q2, *cache, i32([0, 1, 2]), kv_len, t, 1, 400, G, 0.09)
            outs[-1].append(few)
        assert all(torch.equal(a, b) for a, b in zip(*outs))
    for x, y in zip(big, (s.dk, s.dv)):
        assert torch.equal(x[far:].view(torch.uint8), y.view(torch.uint8)) and not bool(x[:far].view(torch.uint8).any())
