"""The 8-bit cache on the device against its definition (tests/plain/kv8_plain.py): what pages hold, bit for bit, and
attention over them against 64 bits."""
import math

import pytest
import torch

from plain import kv8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def tables(n, rot, theta=10000.0):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)[None]
    return ang.cos().float(), ang.sin().float()


class Setup:
    """Pages of several sequences in a shuffled pool whose every byte was NaN, with scales of 2^30, before anybody wrote."""

    def __init__(self, lens, G, hd, seed, more_pages=3, per_seq=None):
        g = torch.Generator().manual_seed(seed)
        need = [(n + PAGE - 1) // PAGE for n in lens]
        self.n_pages = sum(need) + 1 + more_pages
        order = (torch.randperm(self.n_pages - 1, generator=g) + 1).tolist()
        self.table = torch.zeros((len(lens), per_seq or max(max(need), 1)), dtype=torch.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        shape = (self.n_pages, G, PAGE, hd)
        self.k, self.v = (torch.full(shape, 0x7f, dtype=torch.uint8) for _ in range(2))
        self.ks, self.vs = (torch.full((self.n_pages, G), 2.0 ** 30) for _ in range(2))
        self.g = g

    def device(self):
        self.dk, self.dv = self.k.to(DEV).view(torch.float8_e4m3fn), self.v.to(DEV).view(torch.float8_e4m3fn)
        self.dks, self.dvs, self.dt = self.ks.to(DEV), self.vs.to(DEV), self.table.to(DEV)
        return self

    def fill(self, lens, G, hd, spread=0.0, nans=0):
        """Random contents for positions 0 .. n of every sequence, pages of unequal magnitude (2^+-spread)."""
        for b, n in enumerate(lens):
            for i in range((n + PAGE - 1) // PAGE):
                p, rows = int(self.table[b, i]), min(PAGE, n - i * PAGE)
                for held, scale in ((self.k, self.ks), (self.v, self.vs)):
                    x = torch.randn((G, rows, hd), generator=self.g, dtype=torch.float64)
                    x *= 2.0 ** (spread * (2 * torch.rand((G, 1, 1), generator=self.g, dtype=torch.float64) - 1))
                    for g in range(G):
                        e = plain.exponent(float(x[g].abs().max()))
                        held[p, g, :rows] = plain.to_bytes(x[g] / 2.0 ** e)
                        scale[p, g] = 2.0 ** e
        return self

    def plain(self):
        return plain.PlainCache(self.k, self.v, self.ks, self.vs)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def same_cache(s, want, pages, where=""):
    """Bytes and scales of `pages` (page -> places written) equal, all others untouched."""
    for name, got, scale, held, w_scale in (("k", s.dk, s.dks, want.bytes[0], want.scale[0]), ("v", s.dv, s.dvs, want.bytes[1], want.scale[1])):
        got = got.view(torch.uint8).cpu()
        nan = plain.VALUES[got.long()].isnan() & plain.VALUES[held.long()].isnan()
        assert bool(((got == held) | nan).all()), f"{where}{name}: {int(((got != held) & ~nan).sum())} bytes differ"
        assert torch.equal(scale.cpu().double(), w_scale), f"{where}{name}_scale"


def run_append(s, rows, starts, lens, H, G, hd, rot, pairing, dtype, cos, sin, max_new=None, want=None):
    """One step: rows[b] float [n_b, H + 2G, hd], to the device and to the plain cache."""
    from picolm_b200 import ops
    want = want or s.plain()
    x = torch.cat([r for r in rows]) if rows else torch.zeros((0, H + 2 * G, hd))
    x = x.to(DTYPES[dtype])
    T = x.shape[0]
    qkv = x.reshape(T, -1).to(DEV).contiguous()
    q = torch.full((T, H, hd), 7.0, dtype=qkv.dtype, device=DEV)
    offs = [0]
    for r in rows:
        offs.append(offs[-1] + r.shape[0])
    ops.rope_store_kv8(qkv, q, s.dk, s.dv, s.dks, s.dvs, None if cos is None else cos.to(DEV), None if sin is None else sin.to(DEV),
                       i32(offs), i32(lens), s.dt, max_new or max([r.shape[0] for r in rows] + [1]), H, G, hd, rot, pairing)
    t, want_q = 0, torch.zeros((T, H, hd))
    for b, r in enumerate(rows):
        n = r.shape[0]
        f = x[t:t + n].float()
        turned = torch.stack([plain.rotate(f[i, :H + G], starts[b] + i, cos, sin, rot, pairing) for i in range(n)]) if n else f[:, :H + G]
        want_q[t:t + n] = turned[:, :H]
        want.append(turned[:, H:], 0, s.table[b], starts[b])
        want.append(f[:, H + G:], 1, s.table[b], starts[b])
        t += n
    got_q = q.cpu()
    w = want_q.to(q.dtype)
    assert torch.equal(torch.nan_to_num(got_q, nan=-12345.0), torch.nan_to_num(w, nan=-12345.0)), "rotated queries"
    return want


APPENDS = [  # (new, before) of every sequence
    [(1, 0)], [(64, 0)], [(65, 0)], [(63, 0), (1, 0), (200, 0)], [(1, 63), (1, 64), (1, 100), (1, 1)],
    [(70, 40), (3, 62), (5, 64), (130, 127)], [(0, 5), (4, 0), (0, 0), (2, 63)], [(4, 61)] * 9,
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("H,G,hd,rot,pairing", [(4, 2, 64, 64, "half"), (3, 1, 128, 64, "adjacent"), (5, 5, 80, 40, "half"),
                                                 (2, 1, 24, 6, "half"), (8, 2, 256, 256, "adjacent"), (6, 2, 8, 0, "half")])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_holds_what_the_format_says(case, H, G, hd, rot, pairing, dtype):
    seqs = APPENDS[case]
    lens = [n + b for n, b in seqs]
    s = Setup([n + 64 for n in lens], G, hd, seed=case * 100 + hd).fill([b for _, b in seqs], G, hd).device()
    cos, sin = tables(max(lens) + 1, rot) if rot else (None, None)
    rows = [torch.randn((n, H + 2 * G, hd), generator=s.g) * (1 + 3 * torch.rand((n, 1, 1), generator=s.g)) for n, _ in seqs]
    want = run_append(s, rows, [b for _, b in seqs], lens, H, G, hd, rot, pairing, dtype, cos, sin)
    same_cache(s, want, None)


@pytest.mark.parametrize("n", [1, 3, 40])
def test_a_page_whose_scale_grows_keeps_what_it_holds(n):
    """Magnitudes that grow from step to step, up to the point where what was there becomes subnormal, and zero."""
    H, G, hd = 2, 2, 64
    s = Setup([64 * 3], G, hd, seed=n).device()
    want, pos = None, 0
    for level in (2.0 ** -70, 1e-6, 1.0, 0.5, 300.0, 1e5, 1e9, 2.0 ** 45):
        if pos + n > 64 * 3:
            break
        rows = torch.randn((n, H + 2 * G, hd), generator=s.g) * level
        want = run_append(s, [rows], [pos], [pos + n], H, G, hd, 0, "half", "float32", None, None, want=want)
        same_cache(s, want, None, f"at {pos}: ")
        pos += n


def test_zeros_what_is_not_finite_and_what_is_too_large():
    H, G, hd = 1, 1, 64
    s = Setup([64 * 2], G, hd, seed=1).device()
    rows = torch.zeros((6, 3, hd))
    rows[1, :, 3], rows[1, :, 4], rows[1, :, 5] = math.inf, -math.inf, math.nan
    rows[2, :, 7] = 3.0e38
    rows[3, :, 8] = 2.0 ** -149
    rows[4, :, 9], rows[5, :, 9] = 448.0 * 2.0 ** 40, 449.0 * 2.0 ** 40
    want = None
    for i in range(6):
        want = run_append(s, [rows[i:i + 1]], [i], [i + 1], H, G, hd, 0, "half", "float32", None, None, want=want)
        same_cache(s, want, None, f"row {i}: ")
    s2 = Setup([64 * 2], G, hd, seed=1).device()
    same_cache(s2, run_append(s2, [rows], [0], [6], H, G, hd, 0, "half", "float32", None, None), None, "at once: ")


def test_values_at_the_borders_of_the_scale_and_of_rounding():
    """Largest magnitudes at, below and above 448 * 2^e, and every midpoint between two e4m3 numbers."""
    H, G, hd = 1, 1, 256
    for e in (-60, -59, -3, 0, 5, 39, 40):
        s = Setup([64], G, hd, seed=2).device()
        rows = torch.zeros((3, 3, hd))
        pos = plain.VALUES[:0x7f]
        mid = ((pos[1:] + pos[:-1]) / 2).float()
        rows[0, :, :126] = mid * 2.0 ** e
        rows[0, :, 126:252] = -mid * 2.0 ** e
        rows[0, :, 252] = 448.0 * 2.0 ** e
        rows[1, :, 0] = float(torch.nextafter(torch.tensor(448.0), torch.tensor(0.0))) * 2.0 ** e
        want = run_append(s, [rows[:2]], [0], [2], H, G, hd, 0, "half", "float32", None, None)
        same_cache(s, want, None, f"e {e}: ")
        assert e in (-60,) or float(s.dks[int(s.table[0, 0]), 0]) == 2.0 ** e
        rows[2, :, 0] = float(torch.nextafter(torch.tensor(448.0), torch.tensor(500.0))) * 2.0 ** e
        want = run_append(s, [rows[2:]], [2], [3], H, G, hd, 0, "half", "float32", None, None, want=want)
        same_cache(s, want, None, f"e {e}, one more: ")


def test_rows_that_are_not_grouped_and_rows_of_no_sequence():
    """Keys and values of their own (no queries), rows that lie apart, rows behind the last sequence, pages nobody owns."""
    from picolm_b200 import ops
    G, hd = 2, 48
    lens, starts = [70, 5], [0, 3]
    s = Setup([128, 64], G, hd, seed=9).fill(starts, G, hd).device()
    n = [70, 2]
    T = sum(n) + 11
    x = torch.randn((T, 2, G, hd), generator=s.g)
    k, v = x[:, 0].contiguous().to(DEV), x[:, 1].contiguous().to(DEV)
    ops.store_kv8(k, v, s.dk, s.dv, s.dks, s.dvs, i32([0, 70, 72]), i32(lens), s.dt, 70)
    want = s.plain()
    t = 0
    for b in range(2):
        want.append(x[t:t + n[b], 0], 0, s.table[b], starts[b])
        want.append(x[t:t + n[b], 1], 1, s.table[b], starts[b])
        t += n[b]
    same_cache(s, want, None)
    # a table of zeros: nothing is written, queries are rotated
    before = s.dk.view(torch.uint8).clone(), s.dks.clone()
    qkv = torch.randn((3, 5 * hd), generator=s.g).to(DEV)
    q = torch.zeros((3, 1, hd), device=DEV)
    ops.rope_store_kv8(qkv, q, s.dk, s.dv, s.dks, s.dvs, None, None, i32([0, 3]), i32([3]), torch.zeros((1, 2), dtype=torch.int32, device=DEV),
                       3, 1, G, hd, 0, "half")
    assert torch.equal(s.dk.view(torch.uint8), before[0]) and torch.equal(s.dks, before[1])
    assert torch.equal(q.reshape(3, hd), qkv[:, :hd])


# ------------------------------------------------------------------ attention
def check_attention(got, s, q, tokens, G, scale, dtype, **more):
    """tokens: (row of q, sequence, position).  The bound, for one component o of a head: what is rounded is
      out: half a step of its type, eps / 2 relative;
      the scores: sums of hd products in fp32, (hd + 8) 2^-24 of sum |q k| scale, twice (score and maximum), a relative error of
        every weight; exp2 2^-21; float32 ends here but for the sums over n keys, (n + 8) 2^-24 relative to sum w |v|;
      bfloat16: weights as halves, 2^-11 relative or, below 2^-14, 2^-24 of the largest value a key."""
    cache = s.plain()
    H, hd = q.shape[1:]
    for t, b, p in tokens:
        o, w, size = plain.attend(q[t].double(), p, cache, s.table[b], G, scale, **more)
        x = got[t].double().cpu().reshape(H, hd)
        n = p + 1
        assert torch.equal(x.isnan(), o.isnan()), f"row {t}: NaN in other places"
        rel = 2 * (hd + 8) * 2.0 ** -24 * size[:, None] * 1.5 + 2.0 ** -20 + (n + 8) * 2.0 ** -24
        bound = torch.finfo(DTYPES[dtype]).eps / 2 * o.abs() + rel * w
        if dtype == "bfloat16":
            top = max(float(torch.nan_to_num(cache.read(1, s.table[b], g, n)).abs().max()) for g in range(G))
            bound = bound + 2.0 ** -11 * w * 1.01 + n * 2.0 ** -24 * top * min(1.0, 64.0 / n)
        bad = ((x - o).abs() > bound * 1.0001) & ~o.isnan()
        assert not bool(bad.any()), f"row {t} at {p}: off {float(((x - o).abs() / bound.clamp_min(1e-300))[bad].max()):.3g} times the bound"


DECODES = [  # H, G, hd, positions, more
    (4, 2, 64, [0], {}), (8, 2, 128, [0, 1, 62, 63, 64, 65, 500], {}), (4, 1, 64, [2000, 0, 129], {}), (16, 1, 128, [77, 640], {}),
    (40, 2, 64, [130, 40], {}), (6, 2, 96, [300, 5, 64], dict(window=100)), (3, 3, 80, [200, 128], dict(window=1)), (4, 4, 256, [130, 70], {}),
    (9, 1, 256, [333], {}), (4, 2, 16, [90, 7], {}), (4, 2, 48, [190, 63], {}), (2, 1, 32, [64, 700], dict(window=64)),
    (8, 2, 64, [511, 30], dict(window=-128)), (8, 2, 128, [900, 20, 399], dict(window=70, keep_first=5)), (4, 2, 64, [800], dict(window=64, keep_first=130)),
    (4, 2, 112, [100, 333], dict(slopes=True)), (8, 4, 64, [0, 64, 300], dict(sink=True)), (5, 5, 24, [100, 64, 3], dict(sink=True, window=50)),
    (4, 2, 40, [150], dict(slopes=True, sink=True, window=60, keep_first=3)), (12, 2, 8, [70, 300], {}),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("spread", [0.0, 20.0])
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode(case, spread, dtype):
    from picolm_b200 import ops
    H, G, hd, positions, more = DECODES[case]
    lens = [p + 1 for p in positions]
    s = Setup(lens, G, hd, seed=case).fill(lens, G, hd).device()
    if spread:                                                        # values in units far apart, page by page
        s.vs *= 2.0 ** torch.randint(-int(spread), int(spread) + 1, s.vs.shape, generator=s.g)
        s.vs.clamp_(2.0 ** -60, 2.0 ** 40)
        s.device()
    q = torch.randn((len(lens), H, hd), generator=s.g).to(DTYPES[dtype])
    args = dict(more)
    if args.pop("sink", None):
        args["sink"] = torch.randn(H, generator=s.g) * 2
    if args.pop("slopes", None):
        args["slopes"] = torch.rand(H, generator=s.g) * 0.1
    on = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    order = torch.randperm(len(lens), generator=s.g).tolist()        # rows in another order than the table's
    for splits in (None, 0, 1, 3, 8):
        got = ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([positions[b] for b in order]), i32(order), s.dt, max(lens), G,
                                       hd ** -0.5, n_splits=splits, **on)
        check_attention(got, s, q, [(t, b, positions[b]) for t, b in enumerate(order)], G, hd ** -0.5, dtype, **args)


PREFILLS = [  # H, G, hd, (new, before), more
    (4, 2, 64, [(5, 0)], {}), (8, 2, 128, [(130, 0), (1, 63), (64, 64)], {}), (4, 1, 64, [(7, 100), (3, 0), (0, 9), (8, 56)], {}),
    (4, 2, 80, [(100, 30), (2, 3)], {}), (6, 3, 96, [(70, 0)], dict(window=20)), (2, 2, 256, [(66, 10)], {}), (10, 2, 64, [(129, 0), (40, 40)], dict(window=50)),
    (4, 2, 128, [(140, 77)], dict(window=40, keep_first=70)), (4, 2, 64, [(150, 0)], dict(window=-32)), (4, 4, 64, [(90, 5), (6, 0)], dict(slopes=True)),
    (8, 2, 128, [(200, 0)], dict(sink=True)), (3, 1, 24, [(50, 20), (9, 0)], {}), (4, 2, 32, [(33, 64)], dict(sink=True, slopes=True)),
    (8, 2, 128, [(4, 300), (4, 3), (3, 61)], dict(window=64)), (16, 1, 64, [(4, 128), (2, 1)], {}), (4, 2, 16, [(80, 0)], {}),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("spread", [0.0, 20.0])
@pytest.mark.parametrize("case", range(len(PREFILLS)))
def test_prefill(case, spread, dtype):
    from picolm_b200 import ops
    H, G, hd, seqs, more = PREFILLS[case]
    lens = [n + b for n, b in seqs]
    s = Setup(lens, G, hd, seed=case).fill(lens, G, hd).device()
    if spread:
        s.vs *= 2.0 ** torch.randint(-int(spread), int(spread) + 1, s.vs.shape, generator=s.g)
        s.vs.clamp_(2.0 ** -60, 2.0 ** 40)
        s.device()
    offs = [0]
    for n, _ in seqs:
        offs.append(offs[-1] + n)
    T = offs[-1]
    q = torch.randn((T + 4, H, hd), generator=s.g).to(DTYPES[dtype])
    args = dict(more)
    if args.pop("sink", None):
        args["sink"] = torch.randn(H, generator=s.g) * 2
    if args.pop("slopes", None):
        args["slopes"] = torch.rand(H, generator=s.g) * 0.1
    on = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    max_new = max(n for n, _ in seqs)
    for bound, splits in ((max_new, None), (max_new + 70, None), (max_new, 0), (max_new, 5)):          # an upper bound serves too
        out = torch.full((T + 4, H * hd), 5.0, dtype=q.dtype, device=DEV)
        got = ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(offs), i32(lens), s.dt, bound, max(lens), G, hd ** -0.5,
                                        out=out, n_splits=splits, **on)
        assert got is out and bool((out[T:] == 5.0).all()), "rows of no sequence"
        check_attention(got, s, q, [(offs[b] + i, b, before + i) for b, (n, before) in enumerate(seqs) for i in sorted({*range(0, n, 7), n - 1} - {-1})],
                        G, hd ** -0.5, dtype, **args)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("H,G,hd,n", [(4, 2, 64, 4), (4, 2, 64, 100), (4, 2, 128, 90), (4, 2, 80, 40), (2, 2, 24, 9)])
def test_a_nan_reaches_the_rows_that_see_it_and_no_others(H, G, hd, n, dtype):
    """Keys and values that are NaN, early, in the last page, behind the window."""
    from picolm_b200 import ops
    before, window = 130, 75
    s = Setup([before + n], G, hd, seed=n).fill([before + n], G, hd)
    for pos, comp in ((50, 3), (before + 1, 5), (before + n - 1, 7), (before - window + 3, 9)):
        page, place = int(s.table[0, pos // PAGE]), pos % PAGE
        s.v[page, 0, place, comp] = 0x7f
        s.v[page, 0, place, (comp + 8) % hd] = 0xff
    pos = before + n - 2
    s.k[int(s.table[0, pos // PAGE]), G - 1, pos % PAGE, 1] = 0xff
    s.device()
    q = torch.randn((n, H, hd), generator=s.g).to(DTYPES[dtype])
    got = ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, n]), i32([before + n]), s.dt, n, before + n, G, hd ** -0.5, window=window)
    check_attention(got, s, q, [(i, 0, before + i) for i in range(n)], G, hd ** -0.5, dtype, window=window)
    pos = [before + n - 1] * n
    got = ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(pos), i32([0] * n), s.dt, before + n, G, hd ** -0.5, window=window)
    check_attention(got, s, q, [(i, 0, pos[i]) for i in range(0, n, 3)], G, hd ** -0.5, dtype, window=window)


@pytest.mark.parametrize("level", [1e-30, 1e-6, 1.0, 1e6, 1e20])
def test_queries_of_any_magnitude(level):
    from picolm_b200 import ops
    H, G, hd, n = 4, 2, 64, 3
    s = Setup([100] * n, G, hd, seed=5).fill([100] * n, G, hd).device()
    q = torch.randn((n, H, hd), generator=s.g)
    q[1] *= 2.0 ** (20 * torch.rand((H, hd), generator=s.g) - 20)
    q[2, 1] = 0
    q = (q * level).bfloat16()
    scale = hd ** -0.5 / level
    got = ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([99, 80, 64]), i32([0, 1, 2]), s.dt, 100, G, scale)
    check_attention(got, s, q, [(0, 0, 99), (1, 1, 80), (2, 2, 64)], G, scale, "bfloat16")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("H,G,hd", [(8, 2, 64), (16, 1, 128), (4, 2, 80), (2, 2, 24)])
def test_rows_whose_scores_are_all_nan_or_all_minus_infinity(H, G, hd, dtype):
    """A range of keys that has nothing but a NaN must not pass for an empty one, and a softmax of minus infinities is NaN, or nothing
    beside a sink."""
    from picolm_b200 import ops
    n = 65                                                            # one key on the second page, and that one is NaN
    s = Setup([n, 300, 3], G, hd, seed=2).fill([n, 300, 3], G, hd)
    s.k[int(s.table[0, 1]), :, 0, 0] = 0x7f
    s.k[:, :, :, 1] = 0x38                                            # (1.0)
    s.device()
    q = torch.randn((4, H, hd), generator=s.g).to(DTYPES[dtype])
    q[1, 0, 2] = math.nan                                             # a query that is NaN
    q[2, 1, 1] = -math.inf                                            # scores that are -inf
    sink = torch.randn(H, generator=s.g)
    pos, seq = [64, 299, 299, 2], [0, 1, 1, 2]
    for more in (None, sink):
        on = None if more is None else more.to(DEV)
        for splits in (None, 0, 1, 3, 8):
            got = ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(pos), i32(seq), s.dt, 300, G, hd ** -0.5, n_splits=splits, sink=on)
            check_attention(got, s, q, [(t, seq[t], pos[t]) for t in range(4)], G, hd ** -0.5, dtype, sink=more)
            assert bool(got[0].isnan().all()) and bool((got.view(4, H, hd)[2, 1] == 0).all()) == (more is not None)
    # prompts: the same keys and queries among others, few rows and many
    for new in (4, 60):
        s = Setup([130 + new], G, hd, seed=new).fill([130 + new], G, hd)
        s.k[:, :, :, 1] = 0x38
        s.k[int(s.table[0, (129 + new) // PAGE]), :, (129 + new) % PAGE, 0] = 0xff
        s.device()
        q = torch.randn((new, H, hd), generator=s.g).to(DTYPES[dtype])
        q[1, 0, 2], q[2, 1, 1] = math.nan, -math.inf
        for more in (None, sink):
            for window in (None, 1):
                got = ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, new]), i32([130 + new]), s.dt, new, 130 + new, G, hd ** -0.5,
                                                window=window, sink=None if more is None else more.to(DEV))
                check_attention(got, s, q, [(i, 0, 130 + i) for i in range(new)], G, hd ** -0.5, dtype, sink=more, window=window)


def test_bounds_far_beyond_what_a_table_holds():
    """keep_first, window, max_new and max_kv_len that pass 32 bits mean all that there is."""
    from picolm_b200 import ops
    H, G, hd, n, far = 4, 2, 64, 70, 1 << 40
    s = Setup([100 + n], G, hd, seed=1).fill([100 + n], G, hd).device()
    q = torch.randn((n, H, hd), generator=s.g)
    for dtype in ("bfloat16", "float32"):
        x = q.to(DTYPES[dtype])
        for new in (2, n):
            start, kv = i32([0, new]), i32([100 + new])
            for more in (dict(window=far), dict(window=-far), dict(window=9, keep_first=far), dict(keep_first=2 ** 31 - 1, window=2 ** 31 - 1)):
                got = ops.attention_kv8_prefill(x[:new].to(DEV), s.dk, s.dv, s.dks, s.dvs, start, kv, s.dt, far, far, G, 0.125, **more)
                check_attention(got, s, x, [(i, 0, 100 + i) for i in range(0, new, 11)], G, 0.125, dtype)
        got = ops.attention_kv8_decode(x[:3].to(DEV), s.dk, s.dv, s.dks, s.dvs, i32([0, 99, 169]), i32([0, 0, 0]), s.dt, far, G, 0.125, window=far)
        check_attention(got, s, x, [(0, 0, 0), (1, 0, 99), (2, 0, 169)], G, 0.125, dtype)


def test_more_new_tokens_than_the_sequence_is_long():
    """Nothing is written for it, wherever its first position would be."""
    from picolm_b200 import ops
    H, G, hd = 2, 1, 64
    s = Setup([100, 100], G, hd, seed=6).fill([100, 100], G, hd).device()
    before = [x.clone() for x in (s.dk.view(torch.uint8), s.dv.view(torch.uint8), s.dks, s.dvs)]
    for kv in (0, 1, 20, 70):
        qkv = torch.randn((80, (H + 2 * G) * hd), generator=s.g).bfloat16().to(DEV)
        q = torch.full((80, H, hd), 7.0, dtype=torch.bfloat16, device=DEV)
        ops.rope_store_kv8(qkv, q, s.dk, s.dv, s.dks, s.dvs, None, None, i32([0, 0, 80]), i32([100, kv]), s.dt, 80, H, G, hd, 0, "half")
        assert bool((q == 7.0).all())
    assert all(torch.equal(a, b) for a, b in zip(before, (s.dk.view(torch.uint8), s.dv.view(torch.uint8), s.dks, s.dvs)))


@pytest.mark.parametrize("more", [{}, dict(window=50), dict(window=40, keep_first=70), dict(window=-32), dict(slopes=True, keep_first=3, window=90), dict(sink=True)],
                         ids=["causal", "window", "kept", "chunks", "slopes", "sink"])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_of_more_tiles_than_run_at_once(hd, more):
    """Enough sequences that a tile of 256 rows is one CTA's (fewer take 128 rows a CTA), of unequal lengths, one without new tokens; a NaN
    in one value and one key."""
    from picolm_b200 import ops
    H, G = 4, 2
    seqs = [(70 + j % 5, 13 * j % 130) for j in range(38)] + [(0, 9), (129, 70)]
    lens = [n + b for n, b in seqs]
    s = Setup(lens, G, hd, seed=hd).fill(lens, G, hd)
    s.v[int(s.table[3, 1]), 1, 10, 7], s.k[int(s.table[5, 1]), 0, 20, 2] = 0x7f, 0xff
    s.vs *= 2.0 ** torch.randint(-12, 13, s.vs.shape, generator=s.g)
    s.vs.clamp_(2.0 ** -60, 2.0 ** 40)
    s.device()
    offs = [0]
    for n, _ in seqs:
        offs.append(offs[-1] + n)
    q = torch.randn((offs[-1] + 3, H, hd), generator=s.g).bfloat16()
    args = dict(more)
    if args.pop("sink", None):
        args["sink"] = torch.randn(H, generator=s.g) * 2
    if args.pop("slopes", None):
        args["slopes"] = torch.rand(H, generator=s.g) * 0.1
    on = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    out = torch.full((offs[-1] + 3, H * hd), 5.0, dtype=q.dtype, device=DEV)
    ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(offs), i32(lens), s.dt, 129, max(lens), G, hd ** -0.5, out=out, **on)
    assert bool((out[offs[-1]:] == 5.0).all()), "rows of no sequence"
    check_attention(out, s, q, [(offs[b] + i, b, before + i) for b, (n, before) in enumerate(seqs) for i in sorted({0, n // 3, 64, n - 1} & set(range(n)))],
                    G, hd ** -0.5, "bfloat16", **args)
    ops.check_status(DEV)
