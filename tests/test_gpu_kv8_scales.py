"""Attention over pages whose keys' scales differ by page and kv head: a scale that is taken from another page, or another head,
shows in the scores."""
import pytest
import torch

from test_gpu_kv8 import DECODES, DEV, DTYPES, PREFILLS, Setup, check_attention, i32

pytestmark = pytest.mark.gpu


def unequal(lens, G, hd, seed):
    """Contents as they come, keys' scales then spread over 2^-4 .. 2^4 and values' over 2^-20 .. 2^20, page by page and head by head."""
    s = Setup(lens, G, hd, seed=seed).fill(lens, G, hd)
    s.ks *= 2.0 ** torch.randint(-4, 5, s.ks.shape, generator=s.g)
    s.vs *= 2.0 ** torch.randint(-20, 21, s.vs.shape, generator=s.g)
    s.ks.clamp_(2.0 ** -60, 2.0 ** 40)
    s.vs.clamp_(2.0 ** -60, 2.0 ** 40)
    return s.device()


def arguments(more, H, g):
    args = dict(more)
    if args.pop("sink", None):
        args["sink"] = torch.randn(H, generator=g) * 2
    if args.pop("slopes", None):
        args["slopes"] = torch.rand(H, generator=g) * 0.1
    return args, {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in args.items()}


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode(case, dtype):
    from picolm_b200 import ops
    H, G, hd, positions, more = DECODES[case]
    lens = [p + 1 for p in positions]
    s = unequal(lens, G, hd, 100 + case)
    q = (torch.randn((len(lens), H, hd), generator=s.g) * 0.25).to(DTYPES[dtype])
    args, on = arguments(more, H, s.g)
    for splits in (None, 0, 1, 3, 8):
        got = ops.attention_kv8_decode(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(positions), i32(list(range(len(lens)))), s.dt, max(lens), G, hd ** -0.5,
                                       n_splits=splits, **on)
        check_attention(got, s, q, [(b, b, p) for b, p in enumerate(positions)], G, hd ** -0.5, dtype, **args)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("case", range(len(PREFILLS) + 3))
def test_prefill(case, dtype):
    from picolm_b200 import ops
    # (beside the cases there: kept first positions with a sink, over few tiles and over more than run at once)
    more_cases = [(8, 2, 128, [(150, 200), (70, 0)], dict(window=90, keep_first=70, sink=True)), (4, 2, 64, [(140, 300)], dict(window=50, keep_first=5, sink=True)),
                  (4, 2, 64, [(140 + i, 7 * i) for i in range(40)], dict(window=80, keep_first=66, sink=True))]
    H, G, hd, seqs, more = (PREFILLS + more_cases)[case]
    lens = [n + b for n, b in seqs]
    s = unequal(lens, G, hd, 200 + case)
    offs = [0]
    for n, _ in seqs:
        offs.append(offs[-1] + n)
    q = (torch.randn((offs[-1], H, hd), generator=s.g) * 0.25).to(DTYPES[dtype])
    args, on = arguments(more, H, s.g)
    max_new = max(n for n, _ in seqs)
    for splits in (None, 0, 5):
        got = ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(offs), i32(lens), s.dt, max_new, max(lens), G, hd ** -0.5, n_splits=splits, **on)
        check_attention(got, s, q, [(offs[b] + i, b, before + i) for b, (n, before) in enumerate(seqs) for i in sorted({0, n // 3, n // 2, n - 1} & set(range(n)))],
                        G, hd ** -0.5, dtype, **args)
    from picolm_b200.ops import check_status
    check_status(DEV)


def test_many_sequences_dealt_out_with_more_tiles_than_one():
    """More sequences than a warp's lanes ask for at once, several tiles of rows each, of unequal lengths, some without new tokens."""
    from picolm_b200 import ops
    H, G, hd = 12, 2, 64
    seqs = [((3 + i % 13) % 16, (37 * i) % 150) for i in range(170)]
    seqs[90] = (15, 2500)
    lens = [n + b for n, b in seqs]
    s = unequal(lens, G, hd, 7)
    offs = [0]
    for n, _ in seqs:
        offs.append(offs[-1] + n)
    q = (torch.randn((offs[-1], H, hd), generator=s.g) * 0.25).bfloat16()
    for splits in (0, 2):
        got = ops.attention_kv8_prefill(q.to(DEV), s.dk, s.dv, s.dks, s.dvs, i32(offs), i32(lens), s.dt, 15, max(lens), G, hd ** -0.5, n_splits=splits)
        check_attention(got, s, q, [(offs[b] + i, b, before + i) for b, (n, before) in enumerate(seqs) if b % 9 == 0 or 88 <= b <= 130
                                    for i in sorted({0, n - 1} & set(range(n)))], G, hd ** -0.5, "bfloat16")
