"""A paged cache that holds keys and values in 8 bits, with one scale for each page of 64 tokens and kv head: appending
a step's keys and values to it (with the rotary encoding on the way), and the attention that reads it, for single
tokens and for prompts.  `run` is one pass through one of these operators: in plain torch (`own` false) or by the
framework's calls.

What the cache holds: e4m3 numbers times a power of two, `k_scale` / `v_scale` [pages, kv heads]: the smallest 2^e with
448 * 2^e at or above the page's largest magnitude (-60 <= e <= 40).  Page 0 is nobody's.  A page that is open when a step
begins keeps its rows and its scale, unless the new rows need a larger one: its rows are then held against that.

The sizes are those of the benchmark (heads of 64, 32 over 8, prompts of 2,048, batches of 8 to 64), of the attention
layers of width 4,096 (heads of 128), and ragged and odd ones between."""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
MOST = 448.0                     # the largest e4m3 number


def listed():
    return [
        # One request generating: the step's key and value go into the cache, its queries are rotated.
        dict(name="append one", kind="append", dtype="bfloat16", heads=32, kv_heads=8, head_dim=64, rotary=64, pairing="half",
             seqs=1, new=1, context=1000),
        # A full batch generating: 64 open pages a head, some of which need a larger scale.
        dict(name="append 64", kind="append", dtype="bfloat16", heads=32, kv_heads=8, head_dim=128, rotary=128, pairing="half",
             seqs=64, new=1, context=4096),
        # The benchmark's prompt, read in one step into fresh pages.
        dict(name="append prompt", kind="append", dtype="bfloat16", heads=32, kv_heads=8, head_dim=64, rotary=64, pairing="half",
             seqs=1, new=2048, context=0),
        # Pieces of prompts behind what is there, in the 32-bit run, a part of a head of odd size rotated in adjacent pairs.
        dict(name="append ragged float32", kind="append", dtype="float32", heads=15, kv_heads=5, head_dim=80, rotary=40,
             pairing="adjacent", seqs=7, new=1011, context=777),
        # One request generating behind a medium context: latency.
        dict(name="decode one", kind="decode", dtype="bfloat16", heads=32, kv_heads=8, head_dim=64, seqs=1, new=1, context=2000,
             window=0, sink=False),
        # Eight long documents: the cache's bytes are everything.
        dict(name="decode long", kind="decode", dtype="bfloat16", heads=32, kv_heads=8, head_dim=128, seqs=8, new=1, context=32767,
             window=0, sink=False),
        # A full batch over unequal contexts.
        dict(name="decode 64", kind="decode", dtype="bfloat16", heads=32, kv_heads=8, head_dim=64, seqs=64, new=1, context=4095,
             window=0, sink=False),
        # Layers with a sliding window and a sink, heads of an odd size in groups of three.
        dict(name="decode window", kind="decode", dtype="bfloat16", heads=24, kv_heads=8, head_dim=96, seqs=19, new=1, context=5000,
             window=1024, sink=True),
        # The benchmark's prompt over its own keys.
        dict(name="prompt", kind="prompt", dtype="bfloat16", heads=32, kv_heads=8, head_dim=64, seqs=1, new=2048, context=0,
             window=0, sink=False),
        # A piece of a long prompt behind the pieces before it.
        dict(name="prompt piece", kind="prompt", dtype="bfloat16", heads=32, kv_heads=8, head_dim=128, seqs=1, new=1000,
             context=15000, window=0, sink=False),
        # A few tokens each behind their conversations (the next turn, or guesses to be checked).
        dict(name="prompt few", kind="prompt", dtype="bfloat16", heads=32, kv_heads=8, head_dim=128, seqs=16, new=9, context=3001,
             window=0, sink=False),
        # The 32-bit run that results are checked against: two prompts of odd lengths.
        dict(name="prompt float32", kind="prompt", dtype="float32", heads=32, kv_heads=8, head_dim=64, seqs=2, new=301, context=0,
             window=0, sink=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "prompt"))
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 7, 8))
    head_dim = rng.choice((64, 64, 128, 128, 32, 80, 96, 112, 256))
    dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    case = dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim)
    if kind == "append":
        case.update(rotary=rng.choice((head_dim, head_dim // 2)), pairing=rng.choice(("half", "adjacent")),
                    seqs=_log(rng, 1, 64), context=rng.choice((0, _log(rng, 1, 4000))))
        case["new"] = rng.choice((1, _log(rng, 1, 2048 if case["seqs"] < 3 else 200)))
        if not case["context"] and case["new"] == 1:
            case["context"] = 63
        return case
    window = rng.choice((0, 0, 0, _log(rng, 1, 4000)))
    sink = rng.random() < 0.25
    if kind == "decode":
        # (no more bytes than the largest listed case; the 32-bit run is the small one)
        most = 200_000_000 // (2 * kv_heads * head_dim) if dtype == "bfloat16" else 12_000_000 // (heads * head_dim)
        seqs = _log(rng, 1, 64)
        case.update(seqs=seqs, new=1, context=_log(rng, 1, max(2, min(32767, most // seqs))))
    else:
        seqs = _log(rng, 1, 16)
        new = _log(rng, 2, max(3, min(2048 if dtype == "bfloat16" else 400, 3000 // seqs)))
        context = rng.choice((0, _log(rng, 1, max(2, min(8000, 60_000_000 // (seqs * new * heads))))))
        case.update(seqs=seqs, new=new, context=context)
    case.update(window=window, sink=sink)
    return case


def _lengths(case):
    """(new tokens, tokens held before) of each sequence: the first has the case's, the others less."""
    new = [max(1, case["new"] * (16 - (5 * i) % 13) // 16) for i in range(case["seqs"])]
    held = [max(0, case["context"] * (16 - (7 * i) % 13) // 16 - i % 3) if i else case["context"] for i in range(case["seqs"])]
    return new, held


def _scale_of(most):
    """The scale of pages whose largest magnitudes are `most`: 2^e, the smallest with 448 * 2^e >= most."""
    m, e = torch.frexp(most)
    e = e - torch.where(m <= 0.875, 9, 8)                     # most = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(most > 0, e, -60).clamp(-60, 40)
    return torch.ldexp(torch.ones_like(most), e)


def _to_8_bits(x):
    return x.clamp(-MOST, MOST).to(torch.float8_e4m3fn)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    H, G, hd, B = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    new, held = _lengths(case)
    lens = [n + h for n, h in zip(new, held)]
    per_seq = max((n + PAGE - 1) // PAGE for n in lens)
    n_pages = sum((n + PAGE - 1) // PAGE for n in lens) + 1

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    # which page each block of 64 tokens lies on: anywhere
    order = torch.randperm(n_pages - 1, generator=g, device=DEVICE).to(torch.int32) + 1
    table = torch.zeros((B, per_seq), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(lens):
        p = (n + PAGE - 1) // PAGE
        table[b, :p] = order[at:at + p]
        at += p
    # what the cache holds: keys with a few large channels, pages of unequal magnitude
    channel = 1.0 + 6.0 * (torch.rand((1, G, 1, hd), generator=g, device=DEVICE) > 0.95).float()
    cache = {}
    for name in ("k", "v"):
        level = torch.exp(0.4 * normal(n_pages, G, 1, 1))
        x = normal(n_pages, G, PAGE, hd) * level
        if name == "k":
            x *= channel * 0.7
        s = _scale_of(x.abs().amax(dim=(2, 3)))
        cache[name], cache[name + "_scale"] = _to_8_bits(x / s[:, :, None, None]), s
        del x
    T = sum(new)
    s = dict(case=dict(case), k=cache["k"], v=cache["v"], k_scale=cache["k_scale"], v_scale=cache["v_scale"], table=table)
    i32 = dict(dtype=torch.int32, device=DEVICE)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s.update(seq_start=torch.tensor(starts, **i32), seq_kv_len=torch.tensor(lens, **i32), max_new=max(new), max_kv=max(lens), T=T,
             tok_seq=torch.tensor([b for b, n in enumerate(new) for _ in range(n)], **i32),
             tok_pos=torch.tensor([h + j for n, h in zip(new, held) for j in range(n)], **i32))
    if case["kind"] == "append":
        rot = case["rotary"]
        x = normal(T, H + 2 * G, hd) * torch.exp(0.5 * normal(T, 1, 1))
        x[:, H:H + G] *= channel[:, :, 0] * 0.7
        s["qkv"] = x.to(dtype).reshape(T, (H + 2 * G) * hd)
        angle = torch.arange(max(lens), dtype=torch.float64, device=DEVICE)[:, None] * \
            500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)[None]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        # pages that go on: the first place that this step writes on each page (64: none)
        first = torch.full((n_pages,), PAGE, dtype=torch.int64, device=DEVICE)
        page = table.long()[s["tok_seq"].long(), s["tok_pos"].long() // PAGE]
        s["first_place"] = first.scatter_reduce(0, page, s["tok_pos"].long() % PAGE, "amin")
    else:
        s["q"] = normal(T, H, hd).to(dtype)
        s["sink"] = normal(H) if case["sink"] else None
        s["scale"] = 1.0 / math.sqrt(hd)
    return s


# ------------------------------------------------------------------ the plain forms
def _rotated(x, cos, sin, rot, pairing):
    """x float32 [T, heads, hd], cos and sin [T, 1, rot / 2]."""
    y = x.clone()
    if pairing == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_append(s):
    c = s["case"]
    H, G, hd, T = c["heads"], c["kv_heads"], c["head_dim"], s["T"]
    x = s["qkv"].float().reshape(T, H + 2 * G, hd)
    pos = s["tok_pos"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qk = _rotated(x[:, :H + G], cos, sin, c["rotary"], c["pairing"])
    page, place = s["table"].long()[s["tok_seq"].long(), pos // PAGE], pos % PAGE

    def store(rows, held, scale):
        most = torch.zeros_like(scale).scatter_reduce(0, page[:, None].expand(-1, G), rows.abs().amax(dim=2), "amax")
        goes_on = (s["first_place"] > 0)[:, None]
        fresh = torch.where(goes_on, torch.maximum(scale, _scale_of(most)), _scale_of(most))
        fresh = torch.where((s["first_place"] < PAGE)[:, None], fresh, scale)
        before = torch.arange(PAGE, device=held.device)[None] < s["first_place"][:, None]          # rows that are there
        again = _to_8_bits(held.float() * (scale / fresh)[:, :, None, None])
        # (8-bit numbers are chosen and placed as bytes: not every torch operation takes them)
        held_bytes = torch.where(before[:, None, :, None], again.view(torch.uint8), held.view(torch.uint8))
        held_bytes[page, :, place] = _to_8_bits(rows / fresh[page][:, :, None]).view(torch.uint8)
        held.view(torch.uint8).copy_(held_bytes)
        scale.copy_(fresh)

    store(qk[:, H:], s["k"], s["k_scale"])
    store(x[:, H + G:], s["v"], s["v_scale"])
    return qk[:, :H].to(s["qkv"].dtype), s["k"], s["v"], s["k_scale"], s["v_scale"]


def _plain_attention(s):
    """Every sequence's queries, padded to the longest, over all its pages at once."""
    c = s["case"]
    H, G, hd, T, B = c["heads"], c["kv_heads"], c["head_dim"], s["T"], c["seqs"]
    R, M = H // G, s["max_new"]
    table = s["table"].long()
    L = table.shape[1] * PAGE
    tok_seq, pos = s["tok_seq"].long(), s["tok_pos"].long()
    row = torch.arange(T, device=DEVICE) - s["seq_start"].long()[tok_seq]
    q = torch.zeros((B, M, H, hd), device=DEVICE)
    q[tok_seq, row] = s["q"].float()
    at = torch.full((B, M), -1, dtype=torch.long, device=DEVICE)
    at[tok_seq, row] = pos
    key = torch.arange(L, device=DEVICE)
    seen = key <= at[:, :, None]                                                                  # [B, M, L]
    if c["window"]:
        seen &= key > at[:, :, None] - c["window"]

    def read(held, scale):
        x = held[table].float() * scale[table][:, :, :, None, None]                               # [B, P, G, 64, hd]
        return x.permute(0, 2, 1, 3, 4).reshape(B, G, L, hd)

    # [B, G, M * R, hd] x [B, G, hd, L]
    q = q.reshape(B, M, G, R, hd).permute(0, 2, 1, 3, 4).reshape(B, G, M * R, hd)
    score = (q @ read(s["k"], s["k_scale"]).transpose(2, 3) * s["scale"]).reshape(B, G, M, R, L)
    score = score.masked_fill_(~seen[:, None, :, None], -math.inf)
    most = score.amax(dim=-1, keepdim=True).clamp_min(-3e38)
    if s["sink"] is not None:
        sink = s["sink"].reshape(1, G, 1, R, 1)
        most = torch.maximum(most, sink)
    p = score.sub_(most).exp_()
    total = p.sum(dim=-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - most)
    out = p.reshape(B, G, M * R, L) @ read(s["v"], s["v_scale"])
    out = out.reshape(B, G, M, R, hd) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(B, M, H * hd)
    return out[tok_seq, row].to(s["q"].dtype)


def run(s):
    c = s["case"]
    if own:
        from picolm_b200 import ops
        H, G, hd = c["heads"], c["kv_heads"], c["head_dim"]
        if c["kind"] == "append":
            q = torch.empty((s["T"], H, hd), dtype=s["qkv"].dtype, device=s["qkv"].device)
            ops.rope_store_kv8(s["qkv"], q, s["k"], s["v"], s["k_scale"], s["v_scale"], s["cos"], s["sin"], s["seq_start"],
                               s["seq_kv_len"], s["table"], s["max_new"], H, G, hd, c["rotary"], c["pairing"])
            return q, s["k"], s["v"], s["k_scale"], s["v_scale"]
        more = dict(window=c["window"] or None, sink=s["sink"])
        if c["kind"] == "decode":
            return ops.attention_kv8_decode(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["tok_pos"], s["tok_seq"],
                                            s["table"], s["max_kv"], G, s["scale"], **more)
        return ops.attention_kv8_prefill(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["seq_start"], s["seq_kv_len"],
                                         s["table"], s["max_new"], s["max_kv"], G, s["scale"], **more)
    return _plain_append(s) if c["kind"] == "append" else _plain_attention(s)


def _seen_pairs(new, held, window):
    """(query, key) pairs of one sequence, and how many of its keys any query sees."""
    pairs = sum(min(window or p + 1, p + 1) for p in range(held, held + new))
    keys = held + new if not window else min(held + new, window + new - 1)
    return pairs, keys


def work(case):
    H, G, hd = case["heads"], case["kv_heads"], case["head_dim"]
    item = 4 if case["dtype"] == "float32" else 2
    new, held = _lengths(case)
    T = sum(new)
    if case["kind"] == "append":
        pages = sum((h + n - 1) // PAGE - h // PAGE + 1 for n, h in zip(new, held))
        return {"bytes": T * (2 * H + 2 * G) * hd * item + T * 2 * G * hd + T * case["rotary"] * 4 + pages * G * 16 + T * 8,
                "flops": 3 * T * (H + G) * case["rotary"] + 4 * T * G * hd}
    pairs = keys = 0
    for n, h in zip(new, held):
        a, b = _seen_pairs(n, h, case["window"])
        pairs, keys = pairs + a, keys + b
    return {"bytes": 2 * keys * G * hd + 2 * (keys // PAGE + len(new)) * G * 4 + 2 * T * H * hd * item, "flops": 4 * pairs * H * hd}


# ------------------------------------------------------------------ the same from the definition, in 64 bits
def _nearest_8_bits(x):
    """The e4m3 numbers (as float64) nearest to x, ties to the even one, magnitudes beyond 448 held there."""
    e = torch.frexp(x.abs().clamp_min(2.0 ** -7))[1] - 1                     # 2^e <= |x|, and no step below the smallest normal's
    step = torch.ldexp(torch.ones_like(x), e.clamp_min(-6) - 3)
    return (torch.round(x / step) * step).clamp(-MOST, MOST)


def _exact_append(s):
    c = s["case"]
    H, G, hd, rot = c["heads"], c["kv_heads"], c["head_dim"], c["rotary"]
    x = s["qkv"].double().reshape(-1, H + 2 * G, hd)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["tok_pos"].long()][:, None]      # e^(i angle)
    z = x[:, :H + G, :rot]
    z = z.unflatten(-1, (rot // 2, 2)) if c["pairing"] == "adjacent" else z.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    z = z.flatten(-2) if c["pairing"] == "adjacent" else z.transpose(-1, -2).flatten(-2)
    x[:, :H + G, :rot] = z
    out = []
    tok_seq, tok_pos, table = s["tok_seq"].tolist(), s["tok_pos"].tolist(), s["table"].tolist()
    rows_of = {}
    for t, (b, p) in enumerate(zip(tok_seq, tok_pos)):
        rows_of.setdefault(table[b][p // PAGE], []).append((p % PAGE, t))
    for name, lo in (("k", H), ("v", H + G)):
        held, scale = s[name].double(), s[name + "_scale"].double()
        for page, places in rows_of.items():
            place = places[0][0]                                             # the step's rows of a page follow one another
            rows = x[places[0][1]:places[-1][1] + 1, lo:lo + G].transpose(0, 1)          # [G, rows, hd]
            most = rows.abs().amax(dim=(1, 2))
            e = torch.ceil(torch.log2(most / MOST))
            e = torch.where(torch.exp2(e - 1) * MOST >= most, e - 1, e).clamp(-60, 40)
            new = torch.exp2(e)
            if place:
                new = torch.maximum(new, scale[page])
                held[page, :, :place] = _nearest_8_bits(held[page, :, :place] * (scale[page] / new)[:, None, None])
            held[page, :, place:place + len(places)] = _nearest_8_bits(rows / new[:, None, None])
            scale[page] = new
        out.append((held, scale))
    return x[:, :H], out[0][0], out[1][0], out[0][1], out[1][1]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    H, G, hd = case["heads"], case["kv_heads"], case["head_dim"]
    R = H // G
    new, held = _lengths(case)
    out = torch.empty((s["T"], H, hd), dtype=torch.float64, device=DEVICE)
    t0 = 0
    for b, (n, h) in enumerate(zip(new, held)):
        length = n + h
        pages = s["table"][b, :(length + PAGE - 1) // PAGE].long()
        p = torch.arange(h, length, device=DEVICE)[:, None]
        j = torch.arange(length, device=DEVICE)[None]
        hidden = (j > p) | (j <= p - case["window"]) if case["window"] else j > p
        for g in range(G):
            k = (s["k"][pages, g].double() * s["k_scale"][pages, g].double()[:, None, None]).reshape(-1, hd)[:length]
            v = (s["v"][pages, g].double() * s["v_scale"][pages, g].double()[:, None, None]).reshape(-1, hd)[:length]
            for h0 in range(g * R, (g + 1) * R):
                a = (s["q"][t0:t0 + n, h0].double() @ k.T) * s["scale"]
                a[hidden] = -math.inf
                if s["sink"] is not None:
                    a = torch.cat([a, s["sink"][h0].double().expand(n, 1)], dim=1)
                w = torch.softmax(a, dim=1)[:, :length]
                out[t0:t0 + n, h0] = w @ v
        t0 += n
    return out.reshape(s["T"], H * hd)
