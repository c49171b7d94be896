"""The paged cache in 8 bits: e4m3 numbers [pages, G, PAGE_TOKENS, hd] with a scale for each page and kv head, float32
[pages, G], a power of two.  Appending a step's keys and values (with the rotary encoding on the way) and attention over
what is held, for single tokens and for prompts.

What a place holds is its number times its page's scale.  A scale is the smallest 2^e, -60 <= e <= 40, with 448 * 2^e at or above the
largest magnitude that its page holds (values beyond 448 * 2^40 are held as that, values that are not finite as NaN).  A
page whose scale has to grow because of a later token keeps what it holds: its numbers' exponents shift, and only what
becomes subnormal is rounded again.  Page 0 is nobody's and is never written.

Errors.  A number held is within 2^-4 of the value, relative to it, or within 2^-10 of its page's scale for values below
2^-6 of that.  Attention works in fp32 over exactly what is held (float32 queries), or with queries and weights as halves
and fp32 sums (bfloat16 queries)."""
from __future__ import annotations

from typing import Optional

import torch

from ..csrc.build import attention_variant
from ._lib import PAGE_TOKENS, SM_COUNT, KernelError, _check, _dev, _dt, _fn, _i32, _p, _stream, set_bounds, status_word
from .attention import _bias_check, _sink_check

KV8_DTYPE = torch.float8_e4m3fn
KV8_MAX_HEAD_DIM = 256


def kv8_supported(head_dim: int) -> bool:
    """Head sizes the 8-bit cache takes: multiples of 8 up to 256."""
    return head_dim % 8 == 0 and 8 <= head_dim <= KV8_MAX_HEAD_DIM


def _cache_check(what, k_cache, v_cache, k_scale, v_scale, G, hd, device):
    if not kv8_supported(hd):
        raise KernelError(f"{what}: head_dim {hd} is not supported (a multiple of 8 up to {KV8_MAX_HEAD_DIM})")
    for c, s, n in ((k_cache, k_scale, "k"), (v_cache, v_scale, "v")):
        _dev(c, n + "_cache"), _dev(s, n + "_scale")
        if c.dtype != KV8_DTYPE or c.dim() != 4 or c.shape[1:] != (G, PAGE_TOKENS, hd):
            raise KernelError(f"{what}: {n}_cache must be [pages, {G}, {PAGE_TOKENS}, {hd}] of {KV8_DTYPE}, got {c.dtype} {tuple(c.shape)}")
        if s.dtype != torch.float32 or s.shape != c.shape[:2]:
            raise KernelError(f"{what}: {n}_scale must be float32 [pages, {G}], got {s.dtype} {tuple(s.shape)}")
        if c.device != device or s.device != device:
            raise KernelError(f"{what}: the rows are on {device}, {n}_cache on {c.device}, {n}_scale on {s.device}")
    if k_cache.shape != v_cache.shape:
        raise KernelError(f"{what}: k_cache has {k_cache.shape[0]} pages, v_cache {v_cache.shape[0]}")


def _step_check(what, device, table, *ints):
    for t, n in ints + ((table, "block_table"),):
        _i32(t, n)
        if t.device != device:
            raise KernelError(f"{what}: the rows are on {device}, {n} on {t.device}")
    if table.dim() != 2 or table.shape[1] == 0:
        raise KernelError(f"{what}: block_table must be [sequences, pages a sequence], got {tuple(table.shape)}")


def _sequences_check(what, seq_start, seq_kv_len, table, rows: int, max_new: int) -> int:
    B = seq_kv_len.numel()
    if seq_start.dim() != 1 or seq_kv_len.dim() != 1 or seq_start.numel() != B + 1 or table.shape[0] < B:
        raise KernelError(f"{what}: seq_start must be [sequences + 1], seq_kv_len [sequences], block_table [sequences, pages]; got "
                          f"{tuple(seq_start.shape)}, {tuple(seq_kv_len.shape)}, {tuple(table.shape)}")
    if rows and max_new <= 0:
        raise KernelError(f"{what}: max_new must be positive, got {max_new}")
    return B


def _on(device) -> None:
    if device.index is not None and device.index != torch.cuda.current_device():
        raise KernelError(f"the tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")


def _bounds(library, flags, k_cache, table, device, n_table: int = 0) -> None:
    positions = table.shape[1] * PAGE_TOKENS
    set_bounds(library, flags, n_pages=k_cache.shape[0], n_seqs=table.shape[0],
               n_positions=min(positions, n_table) if n_table else positions, device=device)


def _append(what, q, k, v, q_out, k_cache, v_cache, k_scale, v_scale, cos, sin, seq_start, seq_kv_len, block_table, max_new,
            H, G, hd, rotary_dim, pairing) -> None:
    device, T = k.device, k.shape[0]
    _on(device)
    _cache_check(what, k_cache, v_cache, k_scale, v_scale, G, hd, device)
    _step_check(what, device, block_table, (seq_start, "seq_start"), (seq_kv_len, "seq_kv_len"))
    B = _sequences_check(what, seq_start, seq_kv_len, block_table, T, max_new)
    if pairing not in ("half", "adjacent"):
        raise KernelError(f"{what}: unknown pairing {pairing!r}")
    if (cos is None) != (sin is None):
        raise KernelError(f"{what}: cos and sin come together")
    if cos is not None:
        _dev(cos, "cos"), _dev(sin, "sin")
        if not 0 < rotary_dim <= hd or rotary_dim % 2:
            raise KernelError(f"{what}: rotary_dim {rotary_dim} must be even, positive and at most head_dim {hd}")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape[0] == 0 or \
                cos.shape[1] != rotary_dim // 2 or sin.shape != cos.shape:
            raise KernelError(f"{what}: cos / sin tables must be float32 [positions, rotary_dim / 2]")
        if cos.device != device or sin.device != device:
            raise KernelError(f"{what}: the rows are on {device}, the tables on {cos.device} and {sin.device}")
    if T == 0:
        return
    _bounds("kv8", (), k_cache, block_table, device, cos.shape[0] if cos is not None else 0)
    item = k.element_size()
    _check(_fn("kv8", "plm_kv8_append")(
        _p(q), _p(k), _p(v), _dt(k, "rows"), 0 if q is None else q.stride(0), k.stride(0), v.stride(0), _p(q_out), _p(k_cache), _p(v_cache),
        _p(k_scale), _p(v_scale), _p(cos), _p(sin), 0 if cos is None else cos.shape[0], _p(seq_start), _p(seq_kv_len), _p(block_table),
        block_table.shape[1], B, int(max_new), H, G, hd, rotary_dim if cos is not None else 0, 0 if pairing == "half" else 1, _stream()),
        f"{what} T={T} H={H} G={G} hd={hd}", nbytes=T * ((2 * H + 2 * G) * hd * item + 2 * G * hd))


def rope_store_kv8(qkv: torch.Tensor, q_out: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], seq_start: torch.Tensor,
                   seq_kv_len: torch.Tensor, block_table: torch.Tensor, max_new: int, num_heads: int, num_kv_heads: int,
                   head_dim: int, rotary_dim: int, pairing: str) -> None:
    """Rotate the query and key heads of `qkv` [T, (H + 2G) * hd] by their tokens' positions (cos / sin None: no rotation);
    write queries to `q_out` [T, H, hd], keys and values to the 8-bit cache.  Sequence b brings rows seq_start[b] ..
    seq_start[b + 1], at most `max_new`, and ends at position seq_kv_len[b] - 1; its pages are row b of `block_table`.  A token at the
    first place of a page begins it: whatever the page held is forgotten.  Rows of no sequence are left alone, and so are their
    rows of q_out.  No page may belong to two sequences."""
    _dev(qkv, "qkv"), _dev(q_out, "q_out")
    T, H, G, hd = qkv.shape[0], num_heads, num_kv_heads, head_dim
    if H <= 0 or G <= 0 or qkv.dim() != 2 or qkv.shape[1] != (H + 2 * G) * hd or q_out.shape != (T, H, hd) or q_out.dtype != qkv.dtype:
        raise KernelError("rope_store_kv8: qkv / q_out shapes do not match the head counts")
    if q_out.device != qkv.device:
        raise KernelError(f"rope_store_kv8: qkv is on {qkv.device}, q_out on {q_out.device}")
    _append("rope_store_kv8", qkv, qkv[:, H * hd:], qkv[:, (H + G) * hd:], q_out, k_cache, v_cache, k_scale, v_scale, cos, sin,
            seq_start, seq_kv_len, block_table, max_new, H, G, hd, rotary_dim, pairing)


def store_kv8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, seq_start: torch.Tensor, seq_kv_len: torch.Tensor, block_table: torch.Tensor,
              max_new: int) -> None:
    """Keys and values [T, G, hd] as they are (normed and rotated before) to the 8-bit cache; the rest as in `rope_store_kv8`."""
    _dev(k, "k"), _dev(v, "v")
    if k.dim() != 3 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise KernelError("store_kv8: k and v must be [T, G, head_dim] of one type on one device")
    T, G, hd = k.shape
    _append("store_kv8", None, k, v, None, k_cache, v_cache, k_scale, v_scale, None, None, seq_start, seq_kv_len, block_table,
            max_new, 0, G, hd, 0, "half")


# ------------------------------------------------------------------ attention
def attention_kv8_mma_supported(q: torch.Tensor) -> bool:
    """The tensor-core kernels take bfloat16 and head sizes that are multiples of 16 up to 256; the others run in fp32."""
    return q.dtype == torch.bfloat16 and q.shape[-1] % 16 == 0 and 16 <= q.shape[-1] <= KV8_MAX_HEAD_DIM


KV8_CLUSTER_SPLITS = 8          # up to this many ranges of keys meet inside a thread-block cluster, without scratch
KV8_FEW_ROWS, KV8_FEW_ROWS_MOST = 64, 256          # (token, head) rows a sequence and kv head up to which keys may be streamed

_few = {}


def kv8_few_plan(head_dim: int, rows: int):
    """(rows a CTA of the streaming kernel takes at a time, CTAs that run at once, floats of workspace for a CTA) for at most
    `rows` (token, head) rows of a sequence and kv head."""
    plan = _few.get((head_dim, rows))
    if plan is None:
        lib, flags = attention_variant(head_dim, "attention_kv8")
        plan = tuple(_fn(lib, "plm_kv8_few_" + what, flags)(rows) for what in ("tile", "ctas", "floats"))
        _few[head_dim, rows] = plan
    return plan


def kv8_cluster_splits(ctas: int, at_once: int, max_kv_len: int) -> int:
    """Into how many ranges, the CTAs of a cluster, the streaming kernel cuts the keys of each sequence, for `ctas` CTAs without
    cutting and `at_once` that run at once; 0: the keys of the step are dealt out over one wave of CTAs.  Dealing out costs a second
    kernel and a longer start, some 6 us, and pays where the ranges would be longer than 16 pages or the CTAs more than run at once
    (us, clusters / dealt out, 32 heads over 8: one sequence of 8,000 keys of 64 8.1 / 14.0, one of 32,000 of 128 26.6 / 24.8; 16 of 2,000
    of 64 9.9 / 16.3, 64 of 1,000 of 128 30.1 / 27.5)."""
    pages = -(-max_kv_len // PAGE_TOKENS)
    splits = min(KV8_CLUSTER_SPLITS, at_once // ctas, max(1, pages // 2))
    return splits if splits >= 1 and pages <= 16 * splits else 0


def kv8_streams(walks: int, rows: int, max_kv_len: int, head_dim: int) -> bool:
    """Whether prompts of at most `rows` (token, head) rows a sequence and kv head, `walks` of those, have their keys streamed (32 rows
    at a time, the keys cut among CTAs) or take a CTA for 256 rows that walks all of them.  By what the two take a page: the tcgen05
    kernel about 1 us whatever the rows, the streaming one 0.9 us of an SM for 32 rows of heads of 128 (0.4 of 64) and 10 more to begin
    and join.  us, streamed / not, 32 heads over 8 of 128: 16 sequences of 9 tokens behind 3,000 75 / 49; one of 4, 16 and 40 behind
    8,000 16 / 106, 53 / 106, 79 / 144."""
    if head_dim not in (64, 128):
        return rows <= KV8_FEW_ROWS
    if rows > KV8_FEW_ROWS_MOST:
        return False
    pages = -(-max_kv_len // PAGE_TOKENS)
    streamed = 10 + walks * -(-rows // 32) * pages * (0.9 if head_dim == 128 else 0.4) / SM_COUNT
    return streamed < -(-walks // SM_COUNT) * pages


def _attend(what, q, k_cache, v_cache, k_scale, v_scale, block_table, ints, max_new, max_kv_len, num_kv_heads, scale, window, out,
            sink, keep_first, slopes, n_splits):
    _dev(q, "q")
    if q.dim() != 3:
        raise KernelError(f"{what}: q must be [T, heads, head_dim], got {tuple(q.shape)}")
    device = q.device
    T, H, hd = q.shape
    G = num_kv_heads
    _on(device)
    if G <= 0 or H % G:
        raise KernelError(f"{what}: the number of heads is not a multiple of the number of KV heads")
    _dt(q, "q")
    _cache_check(what, k_cache, v_cache, k_scale, v_scale, G, hd, device)
    _sink_check(sink, H), _bias_check(keep_first, window, slopes, H)
    for t, n in ((sink, "sink"), (slopes, "slopes")):
        if t is not None and t.device != device:
            raise KernelError(f"{what}: q is on {device}, {n} on {t.device}")
    if not scale > 0:
        raise KernelError(f"{what}: the scale must be positive, got {scale}")
    if n_splits is not None and not 0 <= n_splits <= KV8_CLUSTER_SPLITS:
        raise KernelError(f"{what}: n_splits must lie in 0 .. {KV8_CLUSTER_SPLITS}, got {n_splits}")
    decode = ints[0][1] == "tok_pos"
    _step_check(what, device, block_table, *ints)
    if decode:
        if ints[0][0].shape != (T,) or ints[1][0].shape != (T,):
            raise KernelError(f"{what}: tok_pos and tok_seq must be [{T}], got {tuple(ints[0][0].shape)} and {tuple(ints[1][0].shape)}")
        B = T
    else:
        B = _sequences_check(what, ints[0][0], ints[1][0], block_table, T, max_new)
    if out is None:
        out = torch.empty((T, H * hd), dtype=q.dtype, device=device)
    elif out.dtype != q.dtype or out.shape != (T, H * hd) or out.device != device or not out.is_contiguous():
        raise KernelError(f"{what}: out must be a contiguous {q.dtype} [{T}, {H * hd}] tensor on {device}")
    if T == 0 or B == 0:
        return out
    step = (_p(ints[0][0]), _p(ints[1][0]), None, None) if decode else (None, None, _p(ints[0][0]), _p(ints[1][0]))
    cache = (_p(k_cache), _p(v_cache), _p(k_scale), _p(v_scale))
    tail = (float(scale), int(window or 0))
    rest = (_p(sink), int(keep_first), _p(slopes), _stream())
    rows = max_new * (H // G)
    seen = max_kv_len if not window or window < 0 else min(max_kv_len, window + keep_first + max_new + 2 * PAGE_TOKENS)
    need = dict(nbytes=B * seen * 2 * G * hd + 2 * T * H * hd * q.element_size(), flops=4 * T * H * hd * seen)
    say = f"{what} T={T} H={H} G={G} hd={hd}"
    if not attention_kv8_mma_supported(q):
        ctas = B * G * (-(-rows // 32) if rows > 4 else 1)
        splits = n_splits or max(1, min(4 * SM_COUNT // max(ctas, 1), seen // 64, 256, 65535 // G))
        ws = torch.empty((T * H * splits * (hd + 2),), dtype=torch.float32, device=device) if splits > 1 else None
        _bounds("kv8", (), k_cache, block_table, device)
        _check(_fn("kv8", "plm_kv8_attention_rows")(
            _p(q), _dt(q, "q"), *cache, _p(out), _p(ws), *step, _p(block_table), block_table.shape[1], T, B, int(max_new), H, G, hd, *tail,
            splits, *rest), f"{say} rows splits={splits}", kernels=2 if ws is not None else 1, **need)
        return out
    lib, flags = attention_variant(hd, "attention_kv8")
    _bounds(lib, flags, k_cache, block_table, device)
    if decode or kv8_streams(B * G, rows, seen, hd):
        tile, at_once, floats = kv8_few_plan(hd, rows)
        walks = B * G * -(-rows // tile)
        splits = kv8_cluster_splits(walks, at_once, seen) if n_splits is None else n_splits
        ws = None if splits else torch.empty((at_once * floats + 2 * walks,), dtype=torch.float32, device=device)
        _check(_fn(lib, "plm_kv8_attention_few", flags)(
            _p(q), *cache, _p(out), _p(ws), *step, _p(block_table), block_table.shape[1], T, B, int(max_new), H, G, *tail, splits, at_once, *rest),
            f"{say} few splits={splits}", kernels=1 if splits else 2, **need)
        return out
    if hd in (64, 128):
        lib, flags = attention_variant(hd, "attention_kv8_tc")
        _bounds(lib, flags, k_cache, block_table, device)
        _check(_fn(lib, "plm_kv8_attention_tc", flags)(
            _p(q), *cache, _p(out), *step[2:], _p(block_table), block_table.shape[1], B, int(max_new), H, G, *tail, _p(status_word(device)),
            *rest), f"{say} tc", **need)
        return out
    _check(_fn(lib, "plm_kv8_attention_tiles", flags)(
        _p(q), *cache, _p(out), *step[2:], _p(block_table), block_table.shape[1], B, int(max_new), H, G, *tail, *rest), f"{say} tiles", **need)
    return out


def attention_kv8_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, tok_pos: torch.Tensor, tok_seq: torch.Tensor, block_table: torch.Tensor,
                         max_kv_len: int, num_kv_heads: int, scale: float, window: Optional[int] = None,
                         out: Optional[torch.Tensor] = None, sink: Optional[torch.Tensor] = None, keep_first: int = 0,
                         slopes: Optional[torch.Tensor] = None, n_splits: Optional[int] = None) -> torch.Tensor:
    """Attention of single query tokens (one per row of q [T, H, hd], at position tok_pos[t] of sequence tok_seq[t]) over the 8-bit
    cache; returns [T, H * hd].  `max_kv_len`: an upper bound of tok_pos + 1, for the choice of how many ranges the keys are cut
    into (`n_splits` sets it: 1 to 8 ranges, or 0, all keys of the step dealt out over one wave of CTAs).  `window`, `sink`, `keep_first`, `slopes`: see `attention_rows`."""
    return _attend("attention_kv8_decode", q, k_cache, v_cache, k_scale, v_scale, block_table, ((tok_pos, "tok_pos"), (tok_seq, "tok_seq")),
                   1, max_kv_len, num_kv_heads, scale, window, out, sink, keep_first, slopes, n_splits)


def attention_kv8_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                          v_scale: torch.Tensor, seq_start: torch.Tensor, seq_kv_len: torch.Tensor, block_table: torch.Tensor,
                          max_new: int, max_kv_len: int, num_kv_heads: int, scale: float, window: Optional[int] = None,
                          out: Optional[torch.Tensor] = None, sink: Optional[torch.Tensor] = None, keep_first: int = 0,
                          slopes: Optional[torch.Tensor] = None, n_splits: Optional[int] = None) -> torch.Tensor:
    """Causal attention of every sequence's new tokens (rows seq_start[b] .. seq_start[b + 1] of q [T, H, hd], at most `max_new`) over
    its keys 0 .. seq_kv_len[b] - 1 (at most `max_kv_len`) in the 8-bit cache; returns [T, H * hd].  Rows of no sequence are left as they
    are in `out`.  The rest as in `attention_kv8_decode`."""
    return _attend("attention_kv8_prefill", q, k_cache, v_cache, k_scale, v_scale, block_table,
                   ((seq_start, "seq_start"), (seq_kv_len, "seq_kv_len")), max_new, max_kv_len, num_kv_heads, scale, window, out, sink,
                   keep_first, slopes, n_splits)
