"""The 8-bit cache where it is used: layers and whole models over it.  What every attention call gives is checked against its
definition over what the device's cache holds at that moment; what the cache holds against the same run's keys and values in
the run's own type."""
import math

import pytest
import torch

from plain import kv8_plain as plain
from test_gpu_kv8 import DTYPES, check_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64


class Held:
    """A device cache layer as `check_attention` wants one (its `plain`, its `table`)."""

    def __init__(self, kv):
        self.kv, self.table = kv, kv.block_table.cpu()

    def plain(self):
        b = [t.view(torch.uint8).cpu() for t in (self.kv.k, self.kv.v)]
        return plain.PlainCache(b[0], b[1], self.kv.k_scale.cpu(), self.kv.v_scale.cpu())


class Watch:
    """Stands in for `ops.attention` and checks rows of every call over an 8-bit cache."""

    def __init__(self, monkeypatch, dtype, every=17):
        from picolm_b200 import ops
        self.real, self.dtype, self.every, self.calls = ops.attention, dtype, every, 0
        monkeypatch.setattr(ops, "attention", self)

    def __call__(self, q, kv, step, num_kv_heads, scale, chunk=None, sink=None, slopes=None):
        out = self.real(q, kv, step, num_kv_heads, scale, chunk=chunk, sink=sink, slopes=slopes)
        assert kv.k.dtype == torch.float8_e4m3fn and kv.v.dtype == torch.float8_e4m3fn
        seq, pos = step.tok_seq.tolist(), step.tok_pos.tolist()
        T = q.shape[0]
        rows = sorted({*range(0, T, self.every), T - 1})
        more = dict(window=-int(chunk) if chunk else kv.window, keep_first=kv.keep_first if not chunk else 0,
                    sink=None if sink is None else sink.cpu(), slopes=None if slopes is None else slopes.cpu())
        check_attention(out, Held(kv), q.cpu(), [(t, seq[t], pos[t]) for t in rows], num_kv_heads, scale, self.dtype, **more)
        self.calls += 1
        return out


def cache_of(specs, dtype, in_8_bits):
    from picolm_b200.cache import SequenceCache
    return SequenceCache(specs, max_tokens=64 * 24, max_seqs=5, kv_dtype=torch.float8_e4m3fn if in_8_bits else DTYPES[dtype], device=DEV,
                         row_dtype=DTYPES[dtype])


def step_of(cache, entries):
    from picolm_b200.engine.step_batch import build_step_batch
    cache.reserve([(s, len(t)) for s, t in entries])
    return build_step_batch(entries, [[len(t) - 1] for _, t in entries], cache, torch.device(DEV))


def views(cache, spec_numbers, step):
    from picolm_b200.engine.model import Model
    return Model._views([(c, True) for c in spec_numbers], cache, step)


LAYERS = {
    "plain": dict(num_heads=4, num_kv_heads=2, head_dim=32, rope=(32, "half")),
    "adjacent, part of a head": dict(num_heads=6, num_kv_heads=3, head_dim=64, rope=(32, "adjacent")),
    "no position, window": dict(num_heads=4, num_kv_heads=1, head_dim=128, window=50),
    "heads of 24": dict(num_heads=3, num_kv_heads=1, head_dim=24, rope=(24, "half")),
    "norm, bias, sink": dict(num_heads=4, num_kv_heads=2, head_dim=64, rope=(64, "half"), bias=True, sink_name="sink",
                             qk_norm={"eps": 1e-5, "q_name": "qn", "k_name": "kn"}),
    "wide values, chunks": dict(num_heads=4, num_kv_heads=2, head_dim=24, value_dim=40, chunk=33, rope=(16, "adjacent")),
    "keys as values, gate": dict(num_heads=4, num_kv_heads=4, head_dim=32, values_from_keys=True, gate_name="gate", rope=(32, "half")),
    "kept first, slopes": dict(num_heads=4, num_kv_heads=2, head_dim=64, window=40, keep_first=9, slopes=[0.5, 0.1, 0.02, 0.0]),
    "convolution": dict(num_heads=4, num_kv_heads=2, head_dim=32, conv={"taps": 3}, rope=(32, "half"), head_scale_name="hs"),
}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", sorted(LAYERS))
def test_attention_layer_over_steps(monkeypatch, name, dtype):
    """Prompts, pieces behind them and single tokens, with sequences that end and pages that go to others."""
    from picolm_b200.config import PartSpec
    from picolm_b200.parts import build_part
    from picolm_b200.runtime import Runtime
    p = dict(LAYERS[name])
    rope = p.pop("rope", None)
    if rope:
        p["position"] = PartSpec("rope", dict(head_dim=p["head_dim"], rotary_dim=rope[0], theta=1000.0, scaling=None, pairing=rope[1],
                                              max_positions=512))
    d = 48
    rt = Runtime.create(dtype, DEV)
    p.update(hidden_size=d, q_name="q", k_name="k", v_name="v", o_name="o")
    part = build_part("mixer", PartSpec("attention", p), rt)
    assert part.takes_kv8
    g = torch.Generator().manual_seed(len(name))
    part.load({n: (torch.randn(ws.shape, generator=g) * (0.3 if len(ws.shape) > 1 else 1.0)).to(DTYPES[dtype]).to(DEV)
               for n, ws in part.weight_specs().items()})
    part.prepare(512)
    specs = part.cache_specs()
    eight, plain16 = cache_of(specs, dtype, True), cache_of(specs, dtype, False)
    watch = Watch(monkeypatch, dtype, every=23)
    want = None
    exact = dtype == "float32" or part.general               # (bfloat16 rows that are not rounded before they are held: see below)
    slots = [[c.allocate() for _ in range(3)] for c in (eight, plain16)]
    started = [0, 0, 0]
    steps = [[70, 3, 130], [5, 64, 1], [1, 1, 1], [None, 1, 2], [40, 30, None]]
    for number, lens in enumerate(steps):
        if number == 4:                                       # sequence 0 begins anew on pages that others had
            for c, s in zip((eight, plain16), slots):
                c.release(s[0])
                s[0] = c.allocate()
            started[0] = 0
        live = [i for i, n in enumerate(lens) if n]
        h = torch.randn((sum(lens[i] for i in live), d), generator=g).to(DTYPES[dtype]).to(DEV)
        held = []
        for which, (c, s) in enumerate(zip((eight, plain16), slots)):
            step = step_of(c, [(s[i], list(range(lens[i]))) for i in live])
            kv = views(c, range(len(specs)), step)
            if which == 0:
                part.forward(h, step, kv if len(kv) > 1 else kv[0])
            else:
                monkeypatch.setattr("picolm_b200.ops.attention", watch.real)
                part.forward(h, step, kv if len(kv) > 1 else kv[0])
                monkeypatch.setattr("picolm_b200.ops.attention", watch)
            held.append(kv[0])
        if want is None:
            want = plain.PlainCache(torch.zeros(held[0].k.shape, dtype=torch.uint8), torch.zeros(held[0].v.shape, dtype=torch.uint8),
                                    torch.ones(held[0].k_scale.shape), torch.ones(held[0].v_scale.shape))
        tables = [x.block_table.cpu() for x in held]
        for row, i in enumerate(live):
            n, at = lens[i], started[i]
            pos = torch.arange(at, at + n)
            page = tables[1][row][pos // PAGE].long()
            for which, x16 in enumerate((held[1].k, held[1].v)):
                want.append(x16.cpu()[page, :, pos % PAGE].float(), which, tables[0][row], at)
        for i in live:
            started[i] += lens[i]
            for c, s in zip((eight, plain16), slots):
                c.advance(s[i], lens[i])
        for which, (got, scale) in enumerate(((held[0].k, held[0].k_scale), (held[0].v, held[0].v_scale))):
            got, scale = got.view(torch.uint8).cpu(), scale.cpu().double()
            for row, i in enumerate(live):
                for b in range((started[i] + PAGE - 1) // PAGE):
                    page, rows = int(tables[0][row][b]), min(PAGE, started[i] - b * PAGE)
                    if page == 0:
                        continue                              # a page that has left the window
                    if exact:
                        assert torch.equal(scale[page], want.scale[which][page])
                        assert torch.equal(got[page, :, :rows], want.bytes[which][page, :, :rows])
                    else:
                        # what is held here was rounded once, from float32; the other to bfloat16 first: each within half a step
                        a = plain.VALUES[got[page, :, :rows].long()] * scale[page][:, None, None]
                        b2 = plain.VALUES[want.bytes[which][page, :, :rows].long()] * want.scale[which][page][:, None, None]
                        tol = (2.0 ** -3 + 2.0 ** -7) * torch.maximum(a.abs(), b2.abs()) + 2.0 ** -9 * torch.maximum(scale[page], want.scale[which][page])[:, None, None]
                        assert bool(((a - b2).abs() <= tol).all())
    assert watch.calls == len(steps)
    eight.check()


def test_cache_in_8_bits_counts_its_bytes_and_is_refused_where_it_does_not_fit(model_dirs):
    from picolm_b200.engine import Engine
    a, b = (Engine.from_folder(model_dirs["A"], max_tokens=256, cache_type=t) for t in (None, "e4m3"))
    assert 2 * b.cache.kv_bytes_per_token() == a.cache.kv_bytes_per_token()
    assert b.cache.kv_groups[0].k.dtype == torch.float8_e4m3fn and a.cache.kv_groups[0].k_scale is None
    with pytest.raises(ValueError, match="cache type"):
        Engine.from_folder(model_dirs["A"], max_tokens=256, cache_type="int8")
    part = next(p for blk in a.model.blocks for _, p in blk.parts() if getattr(p, "kind", "") == "attention")
    part.position.takes_kv8 = False
    with pytest.raises(ValueError, match="takes_kv8"):
        Engine(a.model, 256, cache_type="e4m3")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B_sharp"])
def test_models_over_8_bits(monkeypatch, model_dirs, name, dtype):
    """Whole models kernel by kernel with every attention call checked; then replayed graphs against that; then how far the
    logits are from the run's own cache: keys and values are off by 2.6 % (the root mean square of a relative error that is
    even within 2^-4 of a number's leading power of two), three times that is allowed for a few layers."""
    from picolm_b200.engine import Engine
    from util import random_tokens
    d = model_dirs[name]
    vocab = 256 if name[0] == "A" else 384
    reqs = [random_tokens(n, vocab, n) for n in (5, 70, 33)]
    later = [random_tokens(12, vocab, 100 + i) for i in range(3)]
    logits = {}
    for kind in ("checked", "graphs", "own"):
        eng = Engine.from_folder(d, dtype=dtype, max_tokens=64 * 12, use_graphs=kind == "graphs", cache_type=None if kind == "own" else "e4m3")
        if kind == "checked":
            watch = Watch(monkeypatch, dtype)
        slots = [eng.new_sequence() for _ in reqs]
        out = [eng.step([(s, r) for s, r in zip(slots, reqs)]).clone()]
        for j in range(12):
            out.append(eng.step([(s, [t[j]]) for s, t in zip(slots, later)]).clone())
        logits[kind] = torch.cat(out).double().cpu()
        if kind == "checked":
            assert watch.calls > 0
            monkeypatch.setattr("picolm_b200.ops.attention", watch.real)
        for s in slots:
            eng.end_sequence(s)
        eng.cache.check()
    rms = logits["own"].pow(2).mean().sqrt()
    assert float((logits["checked"] - logits["own"]).pow(2).mean().sqrt() / rms) <= 0.08
    assert float((logits["checked"] - logits["own"]).abs().max()) > 0
    assert float((logits["checked"] - logits["graphs"]).pow(2).mean().sqrt() / rms) <= (1e-5 if dtype == "float32" else 0.02)


def test_the_cut_of_a_prompt_hardly_shows(model_dirs):
    """float32: the same tokens whole, in pieces and one by one hold the same values but for numbers that were rounded again when
    their page's scale grew: those are subnormal, within a step of 2^-9 of the scale."""
    from picolm_b200.engine import Engine
    from util import random_tokens
    toks = random_tokens(100, 384, 3)
    held = []
    for cut in ([100], [30, 1, 40, 29], [1] * 100):
        eng = Engine.from_folder(model_dirs["B"], dtype="float32", max_tokens=256, cache_type="e4m3", use_graphs=False)
        s, at = eng.new_sequence(), 0
        for n in cut:
            eng.step([(s, toks[at:at + n])], [[]])
            at += n
        g = eng.cache.kv_groups[0]
        pages = [int(p) for p in g.table[s][:2]]
        # the first layer's: what later layers see differs by what was held before them
        held.append([(plain.VALUES[x[0][pages].view(torch.uint8).cpu().long()], sc[0][pages].cpu().double()[:, :, None, None])
                     for x, sc in ((g.k, g.k_scale), (g.v, g.v_scale))])
    for other in held[1:]:
        for (a, sa), (b, sb) in zip(held[0], other):
            assert torch.equal(sa, sb)
            n = 100 - PAGE
            for page, rows in ((0, PAGE), (1, n)):
                x, y = a[page, :, :rows], b[page, :, :rows]
                differ = x != y
                assert bool(((x - y).abs()[differ] <= 2.0 ** -9).all()) and bool((x.abs()[differ] < 2.0 ** -6 + 2.0 ** -9).all())


def test_generation_and_the_command_line(model_dirs, capsys):
    """`generate` in batches over a cache in 8 bits whose pages go from batch to batch: greedy tokens of a request do not depend on
    the others', and the command line takes the option."""
    from picolm_b200.api import generate, model_load
    from picolm_b200.cli import main
    from util import random_tokens
    prompts = [random_tokens(n, 256, n) for n in (9, 40, 70, 3, 61)]
    eng = model_load(model_dirs["A_sharp"], dtype="float32", context=128, max_batch=2, cache_type="e4m3")
    both = generate(eng, prompts, max_tokens=20, temperature=0.0, stop_ids=[])
    alone = [generate(eng, [p], max_tokens=20, temperature=0.0, stop_ids=[])[0] for p in prompts]
    assert both == alone
    assert main([model_dirs["A_sharp"], "-p", ",".join(map(str, prompts[0])), "-n", "20", "-t", "0", "--dtype", "float32", "--cache-type", "e4m3",
                 "--stop-id", "999"]) == 0
    assert [int(t) for t in capsys.readouterr().out.split()] == both[0]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("design", ["laperax", "fupapel"])
def test_other_designs_over_8_bits(monkeypatch, tmp_path, design, dtype):
    """Attention in other forms beside recurrences, latents and borrowed caches: every call over 8 bits is checked, rows of a latent
    cache stay in the run's type."""
    if design == "laperax":
        import test_gpu_laperax as m
        layers = [m._att(), m._ret(), m._att(size=None, dim=32, vdim=32, rot=None), m._del()]
    else:
        import test_gpu_fupapel as m
        layers = [m._attn(), m._attn2(), m._latent(), m._attn2(kv_from=1)]
    d = m._make(tmp_path, design, m._config(layers), 7)[0]
    from picolm_b200.engine import Engine
    from util import random_tokens
    eng = Engine.from_folder(d, dtype=dtype, max_tokens=64 * 16, cache_type="e4m3", use_graphs=False)
    real = None
    from picolm_b200 import ops
    watch = Watch(monkeypatch, dtype, every=41)
    latents = [0]
    real = watch.__call__

    def only_8_bits(q, kv, *args, **more):                    # (a latent's rows are keys and values in the run's type)
        if kv.k.dtype != torch.float8_e4m3fn:
            latents[0] += 1
            return watch.real(q, kv, *args, **more)
        return real(q, kv, *args, **more)

    monkeypatch.setattr(ops, "attention", only_8_bits)
    slots = [eng.new_sequence() for _ in range(2)]
    out = eng.step([(slots[0], random_tokens(90, m.VOCAB, 1)), (slots[1], random_tokens(20, m.VOCAB, 2))])
    for j in range(4):
        out = eng.step([(s, random_tokens(1, m.VOCAB, 10 + j)) for s in slots])
    assert bool(torch.isfinite(out).all()) and watch.calls >= 10
    assert (latents[0] > 0) == (design == "fupapel")
