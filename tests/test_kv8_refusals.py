"""Arguments that the 8-bit cache's entry points refuse before any launch (C, without a device), and that its Python faces refuse."""
import ctypes

import pytest
import torch

SHAPE, ALIGN, UNSUPPORTED, DTYPE = -2, -3, -4, -1


def _entry(library, name, flags=()):
    from picolm_b200.csrc.build import load_library
    from picolm_b200.ops import _lib
    f = getattr(load_library(library, flags), name)
    f.argtypes, f.restype = _lib._SIGNATURES[name], ctypes.c_int
    return f


class Args(dict):
    """The arguments of an entry by name, in order; `some` is an address behind which nothing is read."""

    def call(self, f, **changes):
        assert not set(changes) - set(self)
        return f(*{**self, **changes}.values())


some = ctypes.addressof(ctypes.create_string_buffer(256)) & ~63

APPEND = Args(q=some, k=some, v=some, dtype=1, ldq=512, ldk=512, ldv=512, q_out=some, kc=some, vc=some, ks=some, vs=some, cos=some, sin=some,
              n_table=64, seq_start=some, seq_kv_len=some, table=some, max_pages=1, n_seqs=1, max_new=1, H=4, G=2, hd=64, rot=64, pairing=0, stream=None)
ROWS = Args(q=some, dtype=0, kc=some, vc=some, ks=some, vs=some, out=some, ws=None, tok_pos=some, tok_seq=some, seq_start=None, seq_kv_len=None,
            table=some, max_pages=1, n_rows=1, n_seqs=1, max_new=1, H=4, G=2, hd=64, scale=0.1, window=0, n_splits=1, sink=None, keep=0, slopes=None,
            stream=None)
FEW = Args(q=some, kc=some, vc=some, ks=some, vs=some, out=some, ws=None, tok_pos=some, tok_seq=some, seq_start=None, seq_kv_len=None, table=some,
           max_pages=1, n_rows=1, n_seqs=1, max_new=1, H=4, G=2, scale=0.1, window=0, n_splits=1, n_ctas=0, sink=None, keep=0, slopes=None, stream=None)
TILES = Args(q=some, kc=some, vc=some, ks=some, vs=some, out=some, seq_start=some, seq_kv_len=some, table=some, max_pages=1, n_seqs=1, max_new=9, H=4,
             G=2, scale=0.1, window=0, sink=None, keep=0, slopes=None, stream=None)
TC = Args(q=some, kc=some, vc=some, ks=some, vs=some, out=some, seq_start=some, seq_kv_len=some, table=some, max_pages=1, n_seqs=1, max_new=9, H=4,
          G=2, scale=0.1, window=0, status=some, sink=None, keep=0, slopes=None, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(hd=12), SHAPE), (dict(hd=264), SHAPE), (dict(hd=0), SHAPE), (dict(rot=66), SHAPE), (dict(rot=7), SHAPE), (dict(rot=0), SHAPE),
    (dict(G=0), SHAPE), (dict(H=-1), SHAPE), (dict(q=None), SHAPE), (dict(q_out=None), SHAPE), (dict(n_table=0), SHAPE), (dict(max_pages=0), SHAPE),
    (dict(n_seqs=65536), SHAPE), (dict(H=65535), SHAPE), (dict(pairing=2), UNSUPPORTED), (dict(kc=some + 4), ALIGN), (dict(dtype=3), DTYPE),
    (dict(n_seqs=0), 0), (dict(max_new=0), 0)])
def test_append_refuses(change, code):
    assert APPEND.call(_entry("kv8", "plm_kv8_append"), **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(hd=12), SHAPE), (dict(hd=264), SHAPE), (dict(G=3), SHAPE), (dict(n_splits=0), SHAPE), (dict(n_splits=2), SHAPE), (dict(keep=-1), SHAPE),
    (dict(G=0), SHAPE), (dict(tok_seq=None), UNSUPPORTED), (dict(tok_pos=None, tok_seq=None), UNSUPPORTED), (dict(seq_start=some), UNSUPPORTED),
    (dict(tok_pos=None, tok_seq=None, seq_start=some), UNSUPPORTED), (dict(q=some + 8), ALIGN), (dict(dtype=2), DTYPE), (dict(n_rows=0), 0)])
def test_attention_rows_refuses(change, code):
    assert ROWS.call(_entry("kv8", "plm_kv8_attention_rows"), **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(G=3), SHAPE), (dict(n_splits=0), SHAPE), (dict(n_splits=9), SHAPE), (dict(ws=some, n_ctas=0), SHAPE), (dict(ws=some, n_ctas=100000), SHAPE),
    (dict(keep=-1), SHAPE), (dict(n_seqs=65536), SHAPE), (dict(tok_pos=None), UNSUPPORTED), (dict(seq_start=some, seq_kv_len=some), UNSUPPORTED),
    (dict(kc=some + 8), ALIGN), (dict(max_new=0), 0)])
def test_attention_few_refuses(change, code):
    assert FEW.call(_entry("attention_kv8@hd64", "plm_kv8_attention_few", ["-DPLM_HD=64"]), **change) == code


@pytest.mark.parametrize("change,code", [(dict(G=3), SHAPE), (dict(H=0), SHAPE), (dict(n_seqs=65536), SHAPE), (dict(keep=-1), SHAPE), (dict(vc=some + 8), ALIGN),
                                         (dict(n_seqs=0), 0)])
def test_attention_of_prompts_refuses(change, code):
    assert TILES.call(_entry("attention_kv8@hd80", "plm_kv8_attention_tiles", ["-DPLM_HD=80"]), **change) == code
    f = _entry("attention_kv8_tc@hd64", "plm_kv8_attention_tc", ["-DPLM_HD=64"])
    assert TC.call(f, **change) == code
    assert TC.call(f, status=None) == SHAPE and TC.call(f, out=some + 8) == ALIGN


def _tensors(device, H=4, G=2, hd=64, T=3, B=2, dtype=torch.bfloat16):
    i32 = dict(dtype=torch.int32, device=device)
    z = lambda *s, **k: torch.zeros(*s, device=device, **k)
    cache = dict(k_cache=z(5, G, 64, hd).to(torch.float8_e4m3fn), v_cache=z(5, G, 64, hd).to(torch.float8_e4m3fn), k_scale=z(5, G) + 1, v_scale=z(5, G) + 1)
    step = dict(seq_start=torch.tensor([0, 1, 3], **i32), seq_kv_len=torch.tensor([1, 2], **i32), block_table=torch.tensor([[1], [2]], **i32))
    append = dict(qkv=z(T, (H + 2 * G) * hd, dtype=dtype), q_out=z(T, H, hd, dtype=dtype), **cache, cos=z(64, hd // 2), sin=z(64, hd // 2), **step, max_new=2,
                  num_heads=H, num_kv_heads=G, head_dim=hd, rotary_dim=hd, pairing="half")
    decode = dict(q=z(T, H, hd, dtype=dtype), **cache, tok_pos=torch.tensor([0, 0, 1][:T], **i32), tok_seq=torch.tensor([0, 1, 1][:T], **i32),
                  block_table=step["block_table"], max_kv_len=2, num_kv_heads=G, scale=0.1)
    prefill = dict(q=z(T, H, hd, dtype=dtype), **cache, **step, max_new=2, max_kv_len=2, num_kv_heads=G, scale=0.1)
    return dict(rope_store_kv8=append, attention_kv8_decode=decode, attention_kv8_prefill=prefill,
                store_kv8=dict(k=z(T, G, hd, dtype=dtype), v=z(T, G, hd, dtype=dtype), **cache, **step, max_new=2))


def test_faces_refuse_tensors_on_the_host():
    from picolm_b200 import ops
    for name, args in _tensors("cpu").items():
        with pytest.raises(ops.KernelError, match="cpu"):
            getattr(ops, name)(**args)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rope_store_kv8", "store_kv8", "attention_kv8_decode", "attention_kv8_prefill"])
def test_faces_refuse_and_say_why(name):
    from picolm_b200 import ops
    f, good = getattr(ops, name), _tensors("cuda:0")[name]
    f(**good)
    cache = [("k_cache", good["k_cache"].float()), ("k_cache", good["k_cache"].view(torch.uint8)), ("v_cache", good["v_cache"][:4].contiguous()),
             ("k_cache", good["k_cache"][:, :, :32].contiguous()), ("v_cache", good["v_cache"].cpu()), ("k_scale", good["k_scale"].half()),
             ("v_scale", good["v_scale"][:, :1].contiguous()), ("k_scale", good["k_scale"].t()), ("block_table", good["block_table"].long()),
             ("block_table", good["block_table"][0]), ("block_table", good["block_table"][:, :0]), ("block_table", good["block_table"].cpu())]
    if "seq_start" in good:
        cache += [("seq_start", good["seq_start"][:2]), ("seq_kv_len", good["seq_kv_len"].long()), ("max_new", 0), ("block_table", good["block_table"][:1])]
    if name == "rope_store_kv8":
        cache += [("qkv", good["qkv"][:, :-8]), ("q_out", good["q_out"].float()), ("q_out", good["q_out"][:2]), ("cos", None), ("cos", good["cos"].double()),
                  ("sin", good["sin"][:5].contiguous()), ("rotary_dim", 3), ("rotary_dim", 66), ("pairing", "other"), ("num_heads", 3)]
    elif name == "store_kv8":
        cache += [("k", good["k"].float()), ("v", good["v"][:2]), ("k", good["k"][0])]
    else:
        cache += [("q", good["q"].half()), ("q", good["q"][0]), ("q", good["q"].transpose(0, 1)), ("num_kv_heads", 3), ("num_kv_heads", 0), ("scale", 0.0),
                  ("scale", float("nan")), ("n_splits", 9), ("n_splits", -1), ("out", torch.zeros(3, 5, device="cuda:0")),
                  ("sink", torch.zeros(3, device="cuda:0")), ("slopes", torch.zeros(4)), ("keep_first", -1)]
    if name == "attention_kv8_decode":
        cache += [("tok_pos", good["tok_pos"][:2]), ("tok_seq", good["tok_seq"].long())]
    for key, value in cache:
        with pytest.raises(ops.KernelError):
            f(**{**good, key: value})
    empty = _tensors("cuda:0", T=0)[name]
    f(**empty)


@pytest.mark.parametrize("tile", [8, 16, 32])
@pytest.mark.parametrize("head_dim,at_once", [(64, 592), (128, 444), (256, 296)])
def test_the_number_of_ranges_is_one_that_the_kernel_takes(head_dim, at_once, tile):
    """0 to 8 ranges for any step, and no more than one for two pages."""
    from picolm_b200.ops.kv8 import KV8_CLUSTER_SPLITS, kv8_cluster_splits
    for ctas in (1, 3, 8, 64, 500, 2048, 65535 * 128):
        for keys in (1, 64, 65, 129, 1000, 4096, 33000, 2 ** 21, 2 ** 31 - 1):
            n = kv8_cluster_splits(ctas, at_once, -(-keys // 64), head_dim, tile)
            assert 0 <= n <= KV8_CLUSTER_SPLITS and n <= max(1, -(-keys // 64) // 2), (ctas, keys, n)
