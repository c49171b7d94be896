// What the kernels of the 8-bit cache share.
//
// The format.  Keys and values are e4m3 numbers [pages, G, 64, hd] with one scale for each page and kv head, float32
// [pages, G], a power of two 2^e with KV8_E_MIN <= e <= KV8_E_MAX: the smallest with 448 * 2^e at or above the largest
// finite magnitude that the page holds (448 is e4m3's largest number).  What a place holds is number * scale; a value that is not finite
// is held as NaN, one beyond 448 * 2^KV8_E_MAX as that.  With scales that are powers of two a page whose scale has to grow
// keeps what it holds: its numbers' exponents shift, and only those that become subnormal (below 2^-6) are rounded again: off by
// 2^-10 of the scale as they come, by less than 2^-9 of it after any number of growths.
// The bounds of e keep 2^(e - e') of any two pages inside float32, and sums over numbers (below 2^9) times weights (below 2^12,
// see KV8_LIFT) in the unit of a page 2^80 below theirs for up to 2^27 keys; in a unit 2^100 below for 2^7 at the least.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

constexpr int KV8_E_MIN = -60, KV8_E_MAX = 40;

// Weights of bf16 attention are halves: exp2(score - reference) * 2^d.  The reference of a row lies 2^KV8_LIFT below its largest score so
// far, and follows once that is 2^KV8_RAISE further up; d, of a page whose values are in another unit than the sums, is at most
// KV8_SPAN, else the sums change their unit.  So a row's largest weight is at least 2^KV8_LIFT, no half passes 2^15, and a weight
// has a half's 11 bits down to 2^-20 of the largest and is off by at most 2^-31 of that below.  With the largest at 1 (LIFT 0,
// RAISE 8, SPAN 6) weights below 2^-25 of the largest were lost: where a first token draws the weight and holds next to
// nothing, all that 3,000 others give.  Single tokens take the same time; prompts (us, so / as now): 2,048 of 64 41.8 / 42.4, 1,000
// behind 15,000 of 128 274.4 / 275.6, 600 behind 3,000 69.7 / 70.5; with 7, 4, 4 42.9, 275.7, 71.1: sums are scaled more often.
constexpr int KV8_LIFT = 6, KV8_RAISE = 6, KV8_SPAN = 3;
static_assert(KV8_LIFT + KV8_RAISE + KV8_SPAN <= 15, "the largest half is below 2^16");

// Two e4m3 numbers, the low byte's first, as halves (exact; NaN stays NaN).
__device__ __forceinline__ uint32_t kv8_halves(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
// Four of them: the low two and the high two.
__device__ __forceinline__ void kv8_halves(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ float2 kv8_floats(uint32_t two) {
    const uint32_t h = kv8_halves(two);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Two floats as e4m3, to the nearest (ties to even), magnitudes above 448 held there; `a` in the low byte.
__device__ __forceinline__ uint32_t kv8_pack(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
    return r;
}
// Infinity and NaN as NaN.
__device__ __forceinline__ float kv8_finite_or_nan(float x) { return fabsf(x) < INFINITY ? x : __int_as_float(0x7fffffff); }
// |x|, and 0 for what is not finite
__device__ __forceinline__ float kv8_magnitude(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;
}
// The exponent of the scale for a largest magnitude: a = 1.f * 2^E <= 448 * 2^e = 1.75 * 2^(8 + e).
__device__ __forceinline__ int kv8_exponent(float a) {
    const uint32_t bits = __float_as_uint(a);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, KV8_E_MIN), KV8_E_MAX);
}
__device__ __forceinline__ float kv8_pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127
// A page's scale as a kernel reads it: the sums go by its exponent alone, so one that is no power of two, or out of bounds, would give
// other results in bfloat16 than in float32.  The checked build records it.
#ifdef PLM_CHECK
__device__ __forceinline__ float kv8_scale(float s) {
    const uint32_t bits = __float_as_uint(s);
    if (!(bits & 0x807fffffu) && bits >= (uint32_t)(KV8_E_MIN + 127) << 23 && bits <= (uint32_t)(KV8_E_MAX + 127) << 23) return s;
    if (plm_bounds.status) atomicCAS(plm_bounds.status, 0, 20);
    return 1.f;
}
#else
__device__ __forceinline__ float kv8_scale(float s) { return s; }
#endif
__device__ __forceinline__ int kv8_exponent_of_scale(float s) { return (int)(__float_as_uint(s) >> 23) - 127; }

// A step's sequence as attention sees it.  With tok_pos every row of q is a token of its own (`b` is its number), at
// position tok_pos[b] of the sequence whose pages are row tok_seq[b] of the table; otherwise `b` is a sequence of the step,
// its new tokens are rows seq_start[b] .. seq_start[b + 1] and its keys 0 .. seq_kv_len[b] - 1.  One whose positions its row of the table
// does not hold counts as one without rows: nothing is read or written for it.
struct Kv8Step {
    const int *tok_pos, *tok_seq, *seq_start, *seq_kv_len, *block_table;
    int max_pages;
};
struct Kv8Seq {
    int t0, n_new, pos0;                     // first row of q, rows, position of the first
    const int* pages;
};
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Step& s, int b) {
    Kv8Seq q;
    if (s.tok_pos) {
        q.t0 = b;
        q.n_new = 1;
        q.pos0 = PLM_POSITION(s.tok_pos[b]);
        q.pages = s.block_table + (size_t)PLM_SEQ_NO(s.tok_seq[b]) * s.max_pages;
    } else {
        q.t0 = s.seq_start[b];
        q.n_new = s.seq_start[b + 1] - q.t0;
        q.pos0 = q.n_new > 0 ? PLM_POSITION(s.seq_kv_len[b] - 1) + 1 - q.n_new : 0;
        q.pages = s.block_table + (size_t)b * s.max_pages;
    }
    if (q.n_new < 0 || q.pos0 < 0 || q.pos0 > s.max_pages * PLM_PAGE - q.n_new) q.n_new = 0;
    return q;
}

// The maximum that a partial result goes by where several are put together: ones with -inf have no weight, and a NaN among the scores,
// which is in l and not in the maximum, must have one.
__device__ __forceinline__ float kv8_top(float m, float l) { return l == l ? m : fmaxf(m, 0.f); }

// With a sink (one more term exp(sink) in the denominator) the factor that turns a row's sum_j exp2(s_j - m) v_j into its
// result: 1 / (l + exp2(sink log2e - m)), written so that a sink far above the scores does not overflow.  A row sees its own key at least: with
// m still -inf all its scores are -inf (a softmax of nothing, unless a sink is there) or NaN (then l is).
__device__ __forceinline__ float kv8_inverse(float m, float l, const float* sink) {
    if (m == -INFINITY) return sink && *sink > -INFINITY ? l : __int_as_float(0x7fffffff);
    if (!sink) return 1.f / l;
    const float sk = *sink * 1.4426950408889634f;
    if (sk <= m) return 1.f / (l + exp2f(sk - m));
    const float c = exp2f(m - sk);
    return c / fmaf(l, c, 1.f);
}
