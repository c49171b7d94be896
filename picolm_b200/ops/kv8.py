"""The paged cache in 8 bits: e4m3 numbers [pages, G, PAGE_TOKENS, hd] with a scale for each page and kv head, float32
[pages, G], a power of two.  Appending a step's keys and values (with the rotary encoding on the way) and attention over
what is held, for single tokens and for prompts.

What a place holds is its number times its page's scale.  A scale is the smallest 2^e, -60 <= e <= 40, with 448 * 2^e at or above the
largest magnitude that its page holds (values beyond 448 * 2^40 are held as that, values that are not finite as NaN).  A
page whose scale has to grow because of a later token keeps what it holds: its numbers' exponents shift, and only what
becomes subnormal is rounded again.  Page 0 is nobody's and is never written.  A cache made elsewhere must
hold such scales too, no others: the kernels go by their exponents (the checked build reports one that is not).

Errors.  A number held is within 2^-4 of the value, relative to it, or within 2^-10 of its page's scale for values below
2^-6 of that; of a page whose scale has grown since it came, within 2^-9 of the scale (every growth rounds what is subnormal
once more, and the scale at least doubles: 2^-10 (1 + 1/2 + ..)).  Keys and values that `qk_norm_rope_store` hands over (heads that
are normed, biased or convolved) are rows of the run's type: in a bfloat16 run rounded to that, 2^-9, before.  Attention works in fp32 over exactly what is held (float32 queries), or with queries and weights as halves
and fp32 sums (bfloat16 queries): weights to 2^-11 down to 2^-20 of a row's largest, below that to 2^-31 of the largest."""
from __future__ import annotations

import functools
from typing import Optional

import torch

from ..csrc.build import attention_variant
from ._lib import (CHECKED, PAGE_TOKENS, SM_COUNT, TRACED, KernelError, _check, _dev, _dt, _fn, _i32, _p, _stream, set_bounds,
                   status_word)
from .attention import _bias_check, _sink_check

KV8_DTYPE = torch.float8_e4m3fn
KV8_MAX_HEAD_DIM = 256


def kv8_supported(head_dim: int) -> bool:
    """Head sizes the 8-bit cache takes: multiples of 8 up to 256."""
    return head_dim % 8 == 0 and 8 <= head_dim <= KV8_MAX_HEAD_DIM


# The checks run on every launch of a decode step, so they are written to be quick: a tensor's device is one integer (-1: not on a
# CUDA device), and what a message says is put together where it is raised.
def _misplaced(what: str, dev: int, named) -> None:
    """Raises for the first of the tensors that is not on device `dev` or not contiguous."""
    for t, name in named:
        _dev(t, name)
        if t.get_device() != dev:
            raise KernelError(f"{what}: the rows are on cuda:{dev}, {name} on {t.device}")


def _current(dev: int) -> None:
    if dev != torch.cuda.current_device():
        raise KernelError(f"the tensors are on cuda:{dev}, the current device is cuda:{torch.cuda.current_device()}")


def _cache_check(what, k_cache, v_cache, k_scale, v_scale, G, hd, dev):
    if k_cache.get_device() != dev or v_cache.get_device() != dev or k_scale.get_device() != dev or v_scale.get_device() != dev or not (
            k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        _misplaced(what, dev, ((k_cache, "k_cache"), (v_cache, "v_cache"), (k_scale, "k_scale"), (v_scale, "v_scale")))
    if not kv8_supported(hd):
        raise KernelError(f"{what}: head_dim {hd} is not supported (a multiple of 8 up to {KV8_MAX_HEAD_DIM})")
    shape = k_cache.shape
    held = (shape[0] if shape else 0, G)
    if k_cache.dtype is not KV8_DTYPE or v_cache.dtype is not KV8_DTYPE or shape != (held[0], G, PAGE_TOKENS, hd) or v_cache.shape != shape:
        raise KernelError(f"{what}: k_cache and v_cache must be [pages, {G}, {PAGE_TOKENS}, {hd}] of {KV8_DTYPE}, got {k_cache.dtype} {tuple(shape)} and "
                          f"{v_cache.dtype} {tuple(v_cache.shape)}")
    if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32 or k_scale.shape != held or v_scale.shape != held:
        raise KernelError(f"{what}: k_scale and v_scale must be float32 [{shape[0]}, {G}], got {k_scale.dtype} {tuple(k_scale.shape)} and "
                          f"{v_scale.dtype} {tuple(v_scale.shape)}")


def _step_check(what, dev, table, first, second, names):
    if first.get_device() != dev or second.get_device() != dev or table.get_device() != dev or first.dtype is not torch.int32 or \
            second.dtype is not torch.int32 or table.dtype is not torch.int32 or not (first.is_contiguous() and second.is_contiguous() and
                                                                                      table.is_contiguous()):
        named = ((first, names[0]), (second, names[1]), (table, "block_table"))
        _misplaced(what, dev, named)
        for t, name in named:
            _i32(t, name)
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


def _bounds(library, flags, k_cache, table, n_table: int = 0) -> None:
    positions = table.shape[1] * PAGE_TOKENS
    set_bounds(library, flags, n_pages=k_cache.shape[0], n_seqs=table.shape[0],
               n_positions=min(positions, n_table) if n_table else positions, device=k_cache.device)


def _launched(code: int, say, kernels: int = 1, nbytes: int = 0, flops: int = 0) -> None:
    """`_check` with a name that is put together only where it is looked at."""
    _check(code, say() if code or TRACED else "", kernels, nbytes, flops)


def _append(what, dev, T, q_at, k_at, v_at, dtype, item, lds, q_out, k_cache, v_cache, k_scale, v_scale, cos, sin, seq_start, seq_kv_len,
            block_table, max_new, H, G, hd, rotary_dim, pairing) -> None:
    """`q_at`, `k_at`, `v_at`: addresses of the rows, `lds` elements apart."""
    _cache_check(what, k_cache, v_cache, k_scale, v_scale, G, hd, dev)
    _current(dev)
    _step_check(what, dev, block_table, seq_start, seq_kv_len, ("seq_start", "seq_kv_len"))
    B = _sequences_check(what, seq_start, seq_kv_len, block_table, T, max_new)
    if pairing != "half" and pairing != "adjacent":
        raise KernelError(f"{what}: unknown pairing {pairing!r}")
    n_table = 0
    if cos is not None or sin is not None:
        if cos is None or sin is None:
            raise KernelError(f"{what}: cos and sin come together")
        if cos.get_device() != dev or sin.get_device() != dev or not (cos.is_contiguous() and sin.is_contiguous()):
            _misplaced(what, dev, ((cos, "cos"), (sin, "sin")))
        if not 0 < rotary_dim <= hd or rotary_dim % 2:
            raise KernelError(f"{what}: rotary_dim {rotary_dim} must be even, positive and at most head_dim {hd}")
        shape = cos.shape
        if cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or len(shape) != 2 or shape[0] == 0 or shape[1] != rotary_dim // 2 or \
                sin.shape != shape:
            raise KernelError(f"{what}: cos / sin tables must be float32 [positions, rotary_dim / 2]")
        n_table = shape[0]
    if T == 0:
        return
    if max_new > T:
        max_new = T
    if CHECKED:
        _bounds("kv8", (), k_cache, block_table, n_table)
    code = _fn("kv8", "plm_kv8_append")(
        q_at, k_at, v_at, dtype, *lds, None if q_out is None else q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
        v_scale.data_ptr(), _p(cos), _p(sin), n_table, seq_start.data_ptr(), seq_kv_len.data_ptr(), block_table.data_ptr(), block_table.shape[1], B,
        max_new, H, G, hd, rotary_dim if n_table else 0, 0 if pairing == "half" else 1, _stream())
    _launched(code, lambda: f"{what} T={T} H={H} G={G} hd={hd}", 1, T * ((2 * H + 2 * G) * hd * item + 2 * G * hd))


def rope_store_kv8(qkv: torch.Tensor, q_out: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], seq_start: torch.Tensor,
                   seq_kv_len: torch.Tensor, block_table: torch.Tensor, max_new: int, num_heads: int, num_kv_heads: int,
                   head_dim: int, rotary_dim: int, pairing: str) -> None:
    """Rotate the query and key heads of `qkv` [T, (H + 2G) * hd] by their tokens' positions (cos / sin None: no rotation);
    write queries to `q_out` [T, H, hd], keys and values to the 8-bit cache.  Sequence b brings rows seq_start[b] ..
    seq_start[b + 1], at most `max_new`, and ends at position seq_kv_len[b] - 1; its pages are row b of `block_table`
    (what lies behind that row's last page is not kept).  A token at the first place of a page begins it: whatever the page held is
    forgotten.  One at an earlier place than the last follows what lies before it, and the page's scale stays at least as large as it
    was.  Rows of no sequence are left alone, and so are their rows of q_out.  No page may belong to two sequences."""
    dev, H, G, hd = qkv.get_device(), num_heads, num_kv_heads, head_dim
    if dev < 0 or q_out.get_device() != dev or not (qkv.is_contiguous() and q_out.is_contiguous()):
        _misplaced("rope_store_kv8", dev, ((qkv, "qkv"), (q_out, "q_out")))
    shape, width = qkv.shape, (H + 2 * G) * hd
    if H <= 0 or G <= 0 or len(shape) != 2 or shape[1] != width or q_out.shape != (shape[0], H, hd) or q_out.dtype is not qkv.dtype:
        raise KernelError("rope_store_kv8: qkv / q_out shapes do not match the head counts")
    item, at = qkv.element_size(), qkv.data_ptr()
    _append("rope_store_kv8", dev, shape[0], at, at + H * hd * item, at + (H + G) * hd * item, _dt(qkv, "qkv"), item, (width, width, width), q_out,
            k_cache, v_cache, k_scale, v_scale, cos, sin, seq_start, seq_kv_len, block_table, int(max_new), H, G, hd, rotary_dim, pairing)


def store_kv8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, seq_start: torch.Tensor, seq_kv_len: torch.Tensor, block_table: torch.Tensor,
              max_new: int) -> None:
    """Keys and values [T, G, hd] as they are (normed and rotated before) to the 8-bit cache; the rest as in `rope_store_kv8`."""
    dev = k.get_device()
    if dev < 0 or v.get_device() != dev or not (k.is_contiguous() and v.is_contiguous()):
        _misplaced("store_kv8", dev, ((k, "k"), (v, "v")))
    if k.dim() != 3 or v.shape != k.shape or v.dtype is not k.dtype:
        raise KernelError("store_kv8: k and v must be [T, G, head_dim] of one type")
    T, G, hd = k.shape
    _append("store_kv8", dev, T, None, k.data_ptr(), v.data_ptr(), _dt(k, "k"), k.element_size(), (0, G * hd, G * hd), None, k_cache, v_cache, k_scale,
            v_scale, None, None, seq_start, seq_kv_len, block_table, int(max_new), 0, G, hd, 0, "half")


# ------------------------------------------------------------------ attention
def attention_kv8_mma_supported(q: torch.Tensor) -> bool:
    """The tensor-core kernels take bfloat16 and head sizes that are multiples of 16 up to 256; the others run in fp32."""
    return q.dtype == torch.bfloat16 and q.shape[-1] % 16 == 0 and 16 <= q.shape[-1] <= KV8_MAX_HEAD_DIM


KV8_CLUSTER_SPLITS = 8          # up to this many ranges of keys meet inside a thread-block cluster, without scratch
KV8_FEW_ROWS, KV8_FEW_ROWS_MOST = 64, 256          # (token, head) rows a sequence and kv head up to which keys are streamed in any case, or may be

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


@functools.lru_cache(maxsize=4096)
def kv8_cluster_splits(ctas: int, at_once: int, pages: int, head_dim: int, tile: int = 8) -> int:
    """Into how many ranges, the CTAs of a cluster, the streaming kernel cuts the `pages` of each sequence, for `ctas` CTAs without
    cutting, of `tile` rows, and `at_once` that run at once; 0: the keys of the step are dealt out over one wave of CTAs, which costs a
    second kernel and a longer start, some 6 us.  As many ranges as run at once, where that leaves up to 64 pages to each; else, a CTA
    costing some 1 us of an SM and the last ones' ranges the step's end, the square root of pages over CTAs (with the factor that was
    best at 256 to 1,024 CTAs).  Dealt out where few walks leave most SMs without work for longer than the 6 us, and where CTAs of
    more than 8 rows, which cost 2 to 4 us, do not run at once and have walks that are long enough (40 sequences of 4 tokens, 32 heads over 8,
    behind 2,000 keys of 128 42 / 47, of 64 31 / 28; 64 of 8 behind 1,000 of 64 55 / 43).
    us, dealt out / in 1, 2, 4, 8 ranges, 32 heads over 8, single tokens, unequal lengths up to the number: 64 sequences of 4,096 keys
    of 64 41 / 39, 38, 45, 63; of 16,384 121 / 135, 118, 109, 117; 256 of 2,048 79 / 61, 80, 120, 190; 8 of 16,384 27 / 62, 35, 25, 24;
    64 of 4,096 of 128 68 / 64, 62, 69, 102; 32 of 8,192 68 / 76, 71, 64, 73; one of 32,000 23 / 166, 87, 47, 27.  Of 112: 64 of 4,096 61 / 58, 57, 66,
    99; 8 of 32,768 64 / 163, 86, 71, 67.  Other heads (8 over 1, 16 over 2, 64 and 128 over 8, 32 over 32, 6 over 6), 1 to 200 sequences of
    1,000 to 60,000: what is chosen takes at most 1.13 of the best."""
    most, runs = max(1, min(KV8_CLUSTER_SPLITS, pages // 2)), at_once // ctas
    splits = min(most, runs)
    if tile > 8:
        if splits < 2 and pages * head_dim > 2500:
            return 0
        splits = max(1, splits)
    elif splits < 2 or pages > 64 * splits:
        splits = min(most, max(1, round((31 * pages / ctas) ** 0.5)))
    page = head_dim / 330                                 # us a CTA that has an SM to itself
    return 0 if ctas * splits < at_once and pages / splits * page > 6.5 + pages * ctas / at_once * page else splits


def kv8_streams(walks: int, rows: int, max_kv_len: int, head_dim: int) -> bool:
    """Whether prompts of at most `rows` (token, head) rows a sequence and kv head, `walks` of those, have their keys streamed (16 or 32
    rows at a time, the keys cut among CTAs) or take a CTA for 128 or 256 rows that walks all of them.  By what the two take, in us: the
    tcgen05 kernel 7 to begin and end and 0.6 a page for 128 rows (heads of 64: 0.54), 1.0 for 256; the streaming one 10 and 0.5 of an
    SM (0.25) a page for up to 16 rows, for 32 20 and 0.72 (12 and 0.5).  us, streamed / not, 32 heads over 8 of 128: 16 sequences
    of 4 tokens behind 3,000 31 / 36, of 8 51 / 37, 64 of 8 behind 1,000 67 / 55; one of 16 behind 8,000 34 / 81, of 8 behind 1,000 18 / 17; of 64: 4 of 8 behind
    4,000 18 / 41, 16 of 8 behind 3,000 33 / 33, of 16 46 / 34; 16 heads over 2 of 128, 16 of 4 behind 3,000 23 / 35, 40 behind 2,000 40 / 27.
    Other head sizes, whose tiles are 64 rows and leave the keys whole: up to KV8_FEW_ROWS rows always, above while there are at most 16
    tiles a page (then both keep the SMs busy, and the streaming kernel's CTAs cost more to begin and to end).  us, streamed / not, 32 heads over 8
    of 96: one of 32 behind 1,000 18 / 47, behind 8,000 32 / 279, of 64 47 / 280; 16 of 32 behind 3,000 87 / 140, behind 500 45 / 35; 64 of 64 behind
    1,000 270 / 225; of 256: one of 32 behind 8,000 56 / 901, 64 behind 1,000 332 / 334; 16 heads over 2 of 80: 16 of 32 behind 3,000 51 / 114, 64 behind
    1,000 71 / 60."""
    if rows > KV8_FEW_ROWS_MOST:
        return False
    pages = -(-max_kv_len // PAGE_TOKENS)
    if head_dim not in (64, 128):
        return rows <= KV8_FEW_ROWS or walks * -(-rows // 64) <= 16 * pages
    start, page = ((10, 0.5) if rows <= 16 else (20, 0.72)) if head_dim == 128 else ((10, 0.25) if rows <= 16 else (12, 0.5))
    streamed = start + walks * -(-rows // 32) * pages * page / SM_COUNT
    ctas, a_page = walks * -(-rows // 128), 0.6 if head_dim == 128 else 0.54
    if rows > 128 and ctas > SM_COUNT:
        ctas, a_page = walks, 1.0
    return streamed < max(1.0, ctas / SM_COUNT) * (7 + pages * a_page)


_variants = {}


def _variant(head_dim: int, family: str):
    v = _variants.get((head_dim, family))
    if v is None:
        v = _variants[head_dim, family] = attention_variant(head_dim, family)
    return v


def _attend(what, q, k_cache, v_cache, k_scale, v_scale, block_table, first, second, decode, max_new, max_kv_len, num_kv_heads, scale,
            window, out, sink, keep_first, slopes, n_splits):
    dev, G = q.get_device(), num_kv_heads
    if dev < 0 or not q.is_contiguous():
        _dev(q, "q")
    if q.dim() != 3:
        raise KernelError(f"{what}: q must be [T, heads, head_dim], got {tuple(q.shape)}")
    T, H, hd = q.shape
    if G <= 0 or H % G:
        raise KernelError(f"{what}: the number of heads is not a multiple of the number of KV heads")
    dtype = _dt(q, "q")
    _cache_check(what, k_cache, v_cache, k_scale, v_scale, G, hd, dev)
    _current(dev)
    if sink is not None or slopes is not None or keep_first:
        _sink_check(sink, H), _bias_check(keep_first, window, slopes, H)
        for t, n in ((sink, "sink"), (slopes, "slopes")):
            if t is not None and t.get_device() != dev:
                raise KernelError(f"{what}: q is on {q.device}, {n} on {t.device}")
    if not scale > 0:
        raise KernelError(f"{what}: the scale must be positive, got {scale}")
    if n_splits is not None and not 0 <= n_splits <= KV8_CLUSTER_SPLITS:
        raise KernelError(f"{what}: n_splits must lie in 0 .. {KV8_CLUSTER_SPLITS}, got {n_splits}")
    if decode:
        _step_check(what, dev, block_table, first, second, ("tok_pos", "tok_seq"))
        if first.shape != (T,) or second.shape != (T,):
            raise KernelError(f"{what}: tok_pos and tok_seq must be [{T}], got {tuple(first.shape)} and {tuple(second.shape)}")
        B = T
    else:
        _step_check(what, dev, block_table, first, second, ("seq_start", "seq_kv_len"))
        B = _sequences_check(what, first, second, block_table, T, max_new)
    if out is None:
        out = q.new_empty((T, H * hd))
    elif out.dtype is not q.dtype or out.shape != (T, H * hd) or out.get_device() != dev or not out.is_contiguous():
        raise KernelError(f"{what}: out must be a contiguous {q.dtype} [{T}, {H * hd}] tensor on {q.device}")
    if T == 0 or B == 0:
        return out
    # (no sequence brings more than all rows, none is longer than its row of the table)
    table, pages = block_table.data_ptr(), block_table.shape[1]
    held = pages * PAGE_TOKENS
    max_new = T if max_new > T else int(max_new)
    max_kv_len = held if max_kv_len > held else int(max_kv_len) if max_kv_len > 0 else 1
    keep_first = min(int(keep_first), held) if keep_first else 0
    window = max(-held, min(int(window), held)) if window else 0
    step = (first.data_ptr(), second.data_ptr(), None, None) if decode else (None, None, first.data_ptr(), second.data_ptr())
    cache = (k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), out.data_ptr())
    masks = (float(scale), window)
    rest = (_p(sink), keep_first, _p(slopes), _stream())
    rows = max_new * (H // G)
    seen = max_kv_len if window <= 0 else min(max_kv_len, window + keep_first + max_new + 2 * PAGE_TOKENS)
    need = (B * seen * 2 * G * hd + 2 * T * H * hd * q.element_size(), 4 * T * H * hd * seen) if TRACED else ()
    if not attention_kv8_mma_supported(q):
        ctas = B * G * (-(-rows // 32) if rows > 4 else 1)
        splits = n_splits or max(1, min(4 * SM_COUNT // ctas, seen // 64, 256, 65535 // G))
        ws = torch.empty((T * H * splits * (hd + 2),), dtype=torch.float32, device=q.device) if splits > 1 else None
        if CHECKED:
            _bounds("kv8", (), k_cache, block_table)
        code = _fn("kv8", "plm_kv8_attention_rows")(q.data_ptr(), dtype, *cache, _p(ws), *step, table, pages, T, B, max_new, H, G, hd, *masks, splits, *rest)
        _launched(code, lambda: f"{what} T={T} H={H} G={G} hd={hd} rows splits={splits}", 1 if ws is None else 2, *need)
    elif decode or (kv8_streams(B * G, rows, seen, hd) if n_splits is None else rows <= KV8_FEW_ROWS_MOST):
        lib, flags = _variant(hd, "attention_kv8")
        if CHECKED:
            _bounds(lib, flags, k_cache, block_table)
        tile, at_once, floats = kv8_few_plan(hd, rows)
        walks = B * G * -(-rows // tile)
        splits = kv8_cluster_splits(walks, at_once, -(-seen // PAGE_TOKENS), hd, tile) if n_splits is None else n_splits
        ws = None if splits else torch.empty((at_once * floats + 2 * walks,), dtype=torch.float32, device=q.device)
        code = _fn(lib, "plm_kv8_attention_few", flags)(q.data_ptr(), *cache, _p(ws), *step, table, pages, T, B, max_new, H, G, *masks, splits, at_once,
                                                        *rest)
        _launched(code, lambda: f"{what} T={T} H={H} G={G} hd={hd} few splits={splits}", 1 if splits else 2, *need)
    elif hd == 64 or hd == 128:
        lib, flags = _variant(hd, "attention_kv8_tc")
        if CHECKED:
            _bounds(lib, flags, k_cache, block_table)
        code = _fn(lib, "plm_kv8_attention_tc", flags)(q.data_ptr(), *cache, *step[2:], table, pages, B, max_new, H, G, *masks, status_word(q.device).data_ptr(),
                                                       *rest)
        _launched(code, lambda: f"{what} T={T} H={H} G={G} hd={hd} tc", 1, *need)
    else:
        lib, flags = _variant(hd, "attention_kv8")
        if CHECKED:
            _bounds(lib, flags, k_cache, block_table)
        code = _fn(lib, "plm_kv8_attention_tiles", flags)(q.data_ptr(), *cache, *step[2:], table, pages, B, max_new, H, G, *masks, *rest)
        _launched(code, lambda: f"{what} T={T} H={H} G={G} hd={hd} tiles", 1, *need)
    return out


def attention_kv8_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, tok_pos: torch.Tensor, tok_seq: torch.Tensor, block_table: torch.Tensor,
                         max_kv_len: int, num_kv_heads: int, scale: float, window: Optional[int] = None,
                         out: Optional[torch.Tensor] = None, sink: Optional[torch.Tensor] = None, keep_first: int = 0,
                         slopes: Optional[torch.Tensor] = None, n_splits: Optional[int] = None) -> torch.Tensor:
    """Attention of single query tokens (one per row of q [T, H, hd], at position tok_pos[t] of sequence tok_seq[t]) over the 8-bit
    cache; returns [T, H * hd].  `max_kv_len`: an upper bound of tok_pos + 1, for the choice of how many ranges the keys are cut
    into (`n_splits` sets it: 1 to 8 ranges, or 0, all keys of the step dealt out over one wave of CTAs).
    `window`, `sink`, `keep_first`, `slopes`: see `attention_rows`.  A row whose position is negative or beyond its sequence's row of the
    table is left as it is in `out`.  Tensors that begin off the boundary of the kernel's loads and stores (16 bytes; `out` of single tokens 4) are
    refused."""
    return _attend("attention_kv8_decode", q, k_cache, v_cache, k_scale, v_scale, block_table, tok_pos, tok_seq, True, 1, max_kv_len,
                   num_kv_heads, scale, window, out, sink, keep_first, slopes, n_splits)


def attention_kv8_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                          v_scale: torch.Tensor, seq_start: torch.Tensor, seq_kv_len: torch.Tensor, block_table: torch.Tensor,
                          max_new: int, max_kv_len: int, num_kv_heads: int, scale: float, window: Optional[int] = None,
                          out: Optional[torch.Tensor] = None, sink: Optional[torch.Tensor] = None, keep_first: int = 0,
                          slopes: Optional[torch.Tensor] = None, n_splits: Optional[int] = None) -> torch.Tensor:
    """Causal attention of every sequence's new tokens (rows seq_start[b] .. seq_start[b + 1] of q [T, H, hd], at most `max_new`) over
    its keys 0 .. seq_kv_len[b] - 1 (at most `max_kv_len`) in the 8-bit cache; returns [T, H * hd].  Rows of no sequence are left as they
    are in `out`.  `n_splits`: for at most KV8_FEW_ROWS_MOST rows a sequence and kv head (new tokens times the heads of a group), that
    keys are streamed, and in how many ranges.  The rest as in `attention_kv8_decode`."""
    return _attend("attention_kv8_prefill", q, k_cache, v_cache, k_scale, v_scale, block_table, seq_start, seq_kv_len, False, max_new, max_kv_len,
                   num_kv_heads, scale, window, out, sink, keep_first, slopes, n_splits)
