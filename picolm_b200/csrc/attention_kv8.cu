// Attention of bfloat16 queries over the 8-bit cache (kv8.cuh) on the tensor cores (mma.sync m16n8k16, fp16 operands, fp32
// sums), compiled for one head size: -DPLM_HD=<head_dim>, a multiple of 16 up to 256.
//
// For a query at position p, head h, kv head g = h / (H / G), with the page of key t in page(t):
//   s_t = scale * ks[page(t), g] * (q . k8_t) [- slope (p - t)],   out = sum_t softmax(s)_t vs[page(t), g] v8_t
// over lo <= t <= p (or t < keep).  Every e4m3 number is a half; a query row becomes halves after a division by a power of two
// that puts its largest number into [2^13, 2^14) (then halves hold every bit of what was within 2^27 of it); the scales, being
// powers of two, stay outside the products: ks joins the factor on the scores, and the sum over values is kept in the unit
// 2^eo of some page's vs: a page in another unit either has its weights multiplied by the ratio or, where that is beyond 2^6,
// changes the unit (a factor on the sums, exact).
//
// Two kernels:
//   kv8_stream_kernel  few (token, head) rows a sequence and kv head, above all single tokens: bound by the cache's bytes.  A warp
//                      walks a range of the keys on its own, 16 or 32 at a time, from global memory straight into the fragments
//                      of its MMAs: no shared memory, no barrier on the way.  The keys are on the MMA's 16 rows and the
//                      (token, head) rows on its 8 columns, so that a group of four or eight heads does not leave half of the
//                      MMA empty: S^T = K Q^T, and out^T = V^T P^T, whose A operand takes pairs of keys a component; a
//                      byte permutation and a conversion make it of four rows of V.  The 8 columns of S^T become the
//                      B operand by movmatrix.  Four warps' partial results meet in shared memory, up to eight CTAs' in
//                      their cluster's, more through a workspace and a second kernel.
//   kv8_tile_kernel    prompts of head sizes that the tcgen05 kernel does not take: 64 rows a CTA, pages of 64 keys brought to
//                      shared memory as halves.
#include "kv8.cuh"

#ifndef PLM_HD
#define PLM_HD 128
#endif

namespace {

constexpr int HD = PLM_HD;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head_dim must be a multiple of 16 up to 256");
constexpr float LOG2E = 1.4426950408889634f;
constexpr int KS = HD / 16;                      // steps of the contraction over a head, and words of a key's row in a lane
constexpr int MT = HD / 16;                      // tiles of 16 components
constexpr int VW = (HD / 8 + 3) / 4;             // words of a value's row in a lane
constexpr int SB = HD <= 64 ? 2 : 1;             // blocks of 16 keys that a warp works on at a time
constexpr int KB = 16 * SB, UNITS = PLM_PAGE / KB;
constexpr int WARPS = 4, NT = 128;
constexpr float RAISE = 8.f;                     // a row's maximum may outgrow its reference by 2^RAISE before sums are scaled
constexpr int UNIT_SPAN = 6;                     // weights take a page's unit up to 2^6 from the sums'

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {      // an 8 x 8 matrix of halves in fragment order, transposed
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// bytes that are NaN (e4m3: 0x7f and 0xff): 0x80 in their places
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t without(uint32_t w, uint32_t marks) { return w & ~(marks | (marks - (marks >> 7))); }
__device__ __forceinline__ bool is_nan_byte(uint8_t b) { return (b & 0x7f) == 0x7f; }

// The power of two that a query row is divided by, from its largest finite magnitude.
__device__ __forceinline__ int row_exponent(float most) {
    return most > 0.f ? max((int)(__float_as_uint(most) >> 23) - 127, -100) - 13 : 0;
}

// A key's row in the four lanes (c = lane % 4) that share it: word w holds four components, the w-th step's of this lane.  Loads of 16,
// 8 and 4 bytes; which components a step contracts is free, as long as the queries' fragments say the same.
__device__ __forceinline__ int key_component(int w, int c) {
    constexpr int A = HD / 64, B = (HD / 32) & 1;
    if (w < 4 * A) return w / 4 * 64 + c * 16 + w % 4 * 4;
    if (B && w < 4 * A + 2) return 64 * A + c * 8 + (w - 4 * A) * 4;
    return 64 * A + 32 * B + c * 4;
}
__device__ __forceinline__ void load_key(uint32_t (&w)[KS], const uint8_t* row, int c) {
    constexpr int A = HD / 64, B = (HD / 32) & 1, C = (HD / 16) & 1;
#pragma unroll
    for (int i = 0; i < A; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + i * 64 + c * 16);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
    if (B) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + 64 * A + c * 8);
        w[4 * A] = v.x; w[4 * A + B] = v.y;
    }
    if (C) w[KS - 1] = *reinterpret_cast<const uint32_t*>(row + 64 * A + 32 * B + c * 4);
}
// A value's row in the eight lanes (n = lane / 4) that share it: bytes 2 m and 2 m + 1 of a lane are its components of the
// m-th tile: rows n and n + 8 of the MMA.
__device__ __forceinline__ int value_component(int m, int n) {
    constexpr int A = HD / 128, B = (HD / 64) & 1, C = (HD / 32) & 1;
    if (m < 8 * A) return m / 8 * 128 + n * 16 + m % 8 * 2;
    if (B && m < 8 * A + 4) return 128 * A + n * 8 + (m - 8 * A) * 2;
    if (C && m < 8 * A + 4 * B + 2) return 128 * A + 64 * B + n * 4 + (m - 8 * A - 4 * B) * 2;
    return 128 * A + 64 * B + 32 * C + n * 2;
}
__device__ __forceinline__ void load_value(uint32_t (&w)[VW], const uint8_t* row, int n) {
    constexpr int A = HD / 128, B = (HD / 64) & 1, C = (HD / 32) & 1, D = (HD / 16) & 1;
#pragma unroll
    for (int i = 0; i < A; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + i * 128 + n * 16);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
    if (B) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + 128 * A + n * 8);
        w[4 * A] = v.x; w[4 * A + B] = v.y;
    }
    if (C) w[4 * A + 2 * B] = *reinterpret_cast<const uint32_t*>(row + 128 * A + 64 * B + n * 4);
    if (D) w[VW - 1] = *reinterpret_cast<const uint16_t*>(row + 128 * A + 64 * B + 32 * C + n * 2);
}

struct Cache {
    const uint8_t *k, *v;
    const float *ks, *vs;
};

// What a CTA walks: the pages of kept first positions that lie before the window's, then the window's up to the last row's own.
struct Walk {
    int page_first, n_kept, n_pages;
    __device__ __forceinline__ Walk(int pos_first, int pos_last, int window, int keep) {
        const int lo = plm_first_key(pos_first, window);
        page_first = lo / PLM_PAGE;
        n_kept = plm_kept_pages(lo, keep);
        n_pages = n_kept + pos_last / PLM_PAGE - page_first + 1;
    }
    __device__ __forceinline__ int page_at(int i) const { return i < n_kept ? i : page_first + i - n_kept; }
};

// -------------------------------------------------------------------------------------------- few rows
constexpr int MAX_CLUSTER = 8;
constexpr size_t stream_smem(int ng) {           // queries' fragments; then the warps' results, what a CTA shows to its cluster
    return (size_t)ng * KS * 32 * 8 + (size_t)(WARPS + 1) * 8 * ng * (HD + 2) * 4;
}

// grid (ranges, G * tiles, sequences); NG groups of 8 (token, head) rows a CTA.  See Kv8Step for what a sequence is.
template <int NG, bool CLUSTER>
__global__ void __launch_bounds__(NT)
kv8_stream_kernel(const bf16* q, const Cache cache, bf16* __restrict__ out, float* __restrict__ ws, const Kv8Step step, int H, int G,
                  int tiles, float scale_log2, int window, const float* sink, int keep, const float* slopes) {
    constexpr int COLS = 8 * NG;
    extern __shared__ __align__(16) uint8_t sm_raw[];
    uint2* q_frag = reinterpret_cast<uint2*>(sm_raw);                              // [NG][KS][32]
    float* part = reinterpret_cast<float*>(sm_raw + (size_t)NG * KS * 32 * 8);     // [WARPS][COLS][HD + 2]
    float* mine = part + WARPS * COLS * (HD + 2);                                  // [COLS][HD + 2]
    __shared__ int row_exp[COLS];
    __shared__ int s_nan;                        // a value that not all rows see is NaN: looked at again at the end
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n8 = lane >> 2, c4 = lane & 3;
    const int g = blockIdx.y / tiles, tile = blockIdx.y - g * tiles, R = H / G;
    const int n_splits = gridDim.x, split = blockIdx.x;
    const Kv8Seq sq = kv8_seq(step, blockIdx.z);
    const int pair0 = tile * COLS, n_pairs = sq.n_new * R;
    if (pair0 >= n_pairs) return;                                                  // (with all CTAs of its cluster)
    const int n_cols = min(COLS, n_pairs - pair0);
    const int pos_first = sq.pos0 + pair0 / R, pos_last = sq.pos0 + (pair0 + n_cols - 1) / R;
    const int lo_first = plm_first_key(pos_first, window), lo_last = plm_first_key(pos_last, window);
    if (threadIdx.x == 0) s_nan = 0;

    // the queries as B operands: warp by warp a group of 8 rows, row n8's components key_component(w, c4) .. + 3
    for (int ng = warp; ng < NG; ng += WARPS) {
        const int pair = pair0 + ng * 8 + n8;
        const bool have = pair < n_pairs;
        const bf16* row = q + ((size_t)(sq.t0 + (have ? pair / R : 0)) * H + g * R + (have ? pair % R : 0)) * HD;
        uint2 w[KS];
        float most = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            w[s] = have ? *reinterpret_cast<const uint2*>(row + key_component(s, c4)) : make_uint2(0, 0);
            most = fmaxf(fmaxf(fmaxf(kv8_magnitude(__uint_as_float(w[s].x << 16)), kv8_magnitude(__uint_as_float(w[s].x & 0xffff0000u))),
                               fmaxf(kv8_magnitude(__uint_as_float(w[s].y << 16)), kv8_magnitude(__uint_as_float(w[s].y & 0xffff0000u)))), most);
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = row_exponent(most);
        const float down = kv8_pow2(-e);
#pragma unroll
        for (int s = 0; s < KS; ++s)
            q_frag[(ng * KS + s) * 32 + lane] =
                make_uint2(halves(__uint_as_float(w[s].x << 16) * down, __uint_as_float(w[s].x & 0xffff0000u) * down),
                           halves(__uint_as_float(w[s].y << 16) * down, __uint_as_float(w[s].y & 0xffff0000u) * down));
        if (c4 == 0) row_exp[ng * 8 + n8] = e;
    }

    // the warp's range of units of KB keys
    const Walk walk(pos_first, pos_last, window, keep);
    const int n_units = walk.n_pages * UNITS, per = (n_units + n_splits * WARPS - 1) / (n_splits * WARPS);
    const int u0 = (split * WARPS + warp) * per, u1 = min(n_units, u0 + per);
    auto number = [&](int u) { return PLM_PAGE_NO(sq.pages[walk.page_at(u / UNITS)]); };
    uint32_t kw[SB][2][KS], vw[SB][4][VW];
    float ks = 0.f, vs = 1.f;
    auto load_keys = [&](int u, int page) {
        const uint8_t* at = cache.k + (((size_t)page * G + g) * PLM_PAGE + u % UNITS * KB + n8) * HD;
#pragma unroll
        for (int b = 0; b < SB; ++b) {
            load_key(kw[b][0], at + b * 16 * HD, c4);
            load_key(kw[b][1], at + (b * 16 + 8) * HD, c4);
        }
    };
    auto load_values = [&](int u, int page) {                        // keys 2 c4, 2 c4 + 1, and those plus 8
        const uint8_t* at = cache.v + (((size_t)page * G + g) * PLM_PAGE + u % UNITS * KB + 2 * c4) * HD;
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) load_value(vw[b][i], at + (b * 16 + (i & 1) + (i >> 1) * 8) * HD, n8);
    };
    int page = 0, page_next = 0;
    if (u0 < u1) {
        page = number(u0);
        ks = cache.ks[(size_t)page * G + g];
        vs = cache.vs[(size_t)page * G + g];
        load_keys(u0, page);
        load_values(u0, page);
        page_next = number(min(u0 + 1, u1 - 1));
    }
    __syncthreads();                                                 // the queries' fragments are there

    // this lane's columns of S^T and out^T: rows 8 j + 2 c4 and + 1
    float m[NG][2], l[NG][2], cs[NG][2], slope[NG][2];
    int pos[NG][2], lo[NG][2];
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int pair = pair0 + j * 8 + c4 * 2 + e;
            const bool have = pair < n_pairs;
            m[j][e] = -INFINITY;
            l[j][e] = 0.f;
            cs[j][e] = have ? scale_log2 * kv8_pow2(max(-126, min(127, row_exp[j * 8 + c4 * 2 + e]))) : 0.f;
            slope[j][e] = slopes && have ? slopes[g * R + pair % R] * LOG2E : 0.f;
            pos[j][e] = have ? sq.pos0 + pair / R : -1;
            lo[j][e] = plm_first_key(pos[j][e], window);
        }
    float o[NG][MT][4];
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) o[j][t][0] = o[j][t][1] = o[j][t][2] = o[j][t][3] = 0.f;
    uint2 qr[NG == 1 ? KS : 1];
    if (NG == 1) {
#pragma unroll
        for (int s = 0; s < KS; ++s) qr[NG == 1 ? s : 0] = q_frag[s * 32 + lane];
    }
    int eo = kv8_exponent_of_scale(vs);

    for (int u = u0; u < u1; ++u) {
        const int key0 = walk.page_at(u / UNITS) * PLM_PAGE + u % UNITS * KB;
        const bool edge = key0 + KB - 1 > pos_first || key0 < lo_last;
        float s[SB][NG][4];
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
            for (int j = 0; j < NG; ++j) s[b][j][0] = s[b][j][1] = s[b][j][2] = s[b][j][3] = 0.f;
#pragma unroll
        for (int w = 0; w < KS; ++w) {
            uint32_t a[SB][4];
#pragma unroll
            for (int b = 0; b < SB; ++b) {
                a[b][0] = kv8_halves(kw[b][0][w] & 0xffffu);
                a[b][1] = kv8_halves(kw[b][1][w] & 0xffffu);
                a[b][2] = kv8_halves(kw[b][0][w] >> 16);
                a[b][3] = kv8_halves(kw[b][1][w] >> 16);
            }
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const uint2 f = NG == 1 ? qr[NG == 1 ? w : 0] : q_frag[(j * KS + w) * 32 + lane];
#pragma unroll
                for (int b = 0; b < SB; ++b) mma_f16(s[b][j], a[b], f.x, f.y);
            }
        }
        // the next unit's keys into the registers that are free now, its page's number having come with the last
        const float ks_now = ks, vs_now = vs;
        page = page_next;
        if (u + 1 < u1) {
            ks = cache.ks[(size_t)page * G + g];
            vs = cache.vs[(size_t)page * G + g];
            load_keys(u + 1, page);
            page_next = number(min(u + 2, u1 - 1));
        }
        float mx[NG][2];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float c = cs[j][e] * ks_now;
                mx[j][e] = -INFINITY;
#pragma unroll
                for (int b = 0; b < SB; ++b)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) s[b][j][2 * hi + e] *= c;
            }
            if (slopes) {
#pragma unroll
                for (int b = 0; b < SB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[b][j][i] = fmaf(slope[j][i & 1], (float)(key0 + b * 16 + n8 + (i >> 1) * 8 - pos[j][i & 1]), s[b][j][i]);
            }
            if (edge) {
#pragma unroll
                for (int b = 0; b < SB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + b * 16 + n8 + (i >> 1) * 8;
                        if (key > pos[j][i & 1] || (key < lo[j][i & 1] && key >= keep)) s[b][j][i] = -INFINITY;
                    }
            }
#pragma unroll
            for (int b = 0; b < SB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[j][i & 1] = fmaxf(mx[j][i & 1], s[b][j][i]);
        }
        bool raise = false;
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[j][e] = fmaxf(mx[j][e], __shfl_xor_sync(0xffffffffu, mx[j][e], 4));
                mx[j][e] = fmaxf(mx[j][e], __shfl_xor_sync(0xffffffffu, mx[j][e], 8));
                mx[j][e] = fmaxf(mx[j][e], __shfl_xor_sync(0xffffffffu, mx[j][e], 16));
                raise |= mx[j][e] > m[j][e] + RAISE || (m[j][e] == -INFINITY && mx[j][e] > -INFINITY);
            }
        const int ev = kv8_exponent_of_scale(vs_now);
        int d = ev - eo;
        if (__any_sync(0xffffffffu, raise) || d > UNIT_SPAN || d < -UNIT_SPAN) {
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                float down[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool up = mx[j][e] > m[j][e];
                    const float by = up ? m[j][e] - mx[j][e] : 0.f;                // -inf where nothing was seen before
                    down[e] = ex2(by - (float)d);
                    l[j][e] *= ex2(by);
                    if (up) m[j][e] = mx[j][e];
                }
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    o[j][t][0] *= down[0]; o[j][t][1] *= down[1];
                    o[j][t][2] *= down[0]; o[j][t][3] *= down[1];
                }
            }
            eo = ev;
            d = 0;
        }
        uint32_t pf[SB][NG][2];
        const float back = kv8_pow2(-d);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            float sum[2] = {0.f, 0.f};
            float off[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) off[e] = (float)d - (m[j][e] == -INFINITY ? 0.f : m[j][e]);
#pragma unroll
            for (int b = 0; b < SB; ++b) {
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[i] = ex2(s[b][j][i] + off[i & 1]);
                    sum[i & 1] += p[i];
                }
                pf[b][j][0] = turned(halves(p[0], p[1]));
                pf[b][j][1] = turned(halves(p[2], p[3]));
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) l[j][e] = fmaf(sum[e], back, l[j][e]);
        }
        if (edge) {
            // Places that no row sees hold whatever was left there: zeros.  A NaN that some rows see and others do not would
            // reach them all (0 * NaN): it is taken out, and put into the results of those that see it at the end.
            bool found = false;
#pragma unroll
            for (int b = 0; b < SB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + b * 16 + 2 * c4 + (i & 1) + (i >> 1) * 8;
                    const bool seen = key <= pos_last && (key >= lo_first || key < keep);
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        const uint32_t marks = nan_bytes(vw[b][i][w]);
                        found |= seen && marks;
                        vw[b][i][w] = seen ? without(vw[b][i][w], marks) : 0u;
                    }
                }
            if (found) s_nan = 1;
        }
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const uint32_t order = t & 1 ? 0x7362u : 0x5140u;
                const uint32_t x = __byte_perm(vw[b][0][t / 2], vw[b][1][t / 2], order);
                const uint32_t y = __byte_perm(vw[b][2][t / 2], vw[b][3][t / 2], order);
                const uint32_t a[4] = {kv8_halves(x & 0xffffu), kv8_halves(x >> 16), kv8_halves(y & 0xffffu), kv8_halves(y >> 16)};
#pragma unroll
                for (int j = 0; j < NG; ++j) mma_f16(o[j][t], a, pf[b][j][0], pf[b][j][1]);
            }
        if (u + 1 < u1) load_values(u + 1, page);
    }

    // the warps' results: part[warp][row] = sums in units of 1, [HD] = maximum, [HD + 1] = denominator
    {
        const float unit = kv8_pow2(max(-126, min(127, eo)));
        float* at = part + (size_t)warp * COLS * (HD + 2);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 4);
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 8);
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 16);
                float* row = at + (j * 8 + c4 * 2 + e) * (HD + 2);
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    *reinterpret_cast<float2*>(row + value_component(t, n8)) = make_float2(o[j][t][e] * unit, o[j][t][2 + e] * unit);
                if (n8 == 0) *reinterpret_cast<float2*>(row + HD) = make_float2(m[j][e], l[j][e]);
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_cols * HD; i += NT) {
        const int col = i / HD, d = i - col * HD;
        float mw[WARPS], mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            mw[w] = part[((size_t)w * COLS + col) * (HD + 2) + HD];
            mm = fmaxf(mm, mw[w]);
        }
        float acc = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float wgt = mw[w] == -INFINITY ? 0.f : exp2f(mw[w] - mm);
            acc = fmaf(wgt, part[((size_t)w * COLS + col) * (HD + 2) + d], acc);
            ll = fmaf(wgt, part[((size_t)w * COLS + col) * (HD + 2) + HD + 1], ll);
        }
        const int pair = pair0 + col;
        if (s_nan) {                                                 // the edge units of this CTA's range once more
            const int p = sq.pos0 + pair / R, lo_p = plm_first_key(p, window);
            const int end = min(n_units, (split + 1) * WARPS * per);
            for (int u = split * WARPS * per; u < end; ++u) {
                const int key0 = walk.page_at(u / UNITS) * PLM_PAGE + u % UNITS * KB;
                if (!(key0 + KB - 1 > pos_first || key0 < lo_last)) continue;
                const uint8_t* at = cache.v + (((size_t)number(u) * G + g) * PLM_PAGE + u % UNITS * KB) * HD + d;
                for (int k = 0; k < KB; ++k)
                    if (key0 + k <= p && (key0 + k >= lo_p || key0 + k < keep) && is_nan_byte(at[(size_t)k * HD])) acc = __int_as_float(0x7fffffff);
            }
        }
        const size_t row = (size_t)(sq.t0 + pair / R) * H + g * R + pair % R;
        if (CLUSTER) {
            mine[col * (HD + 2) + d] = acc;
            if (d == 0) { mine[col * (HD + 2) + HD] = mm; mine[col * (HD + 2) + HD + 1] = ll; }
        } else if (n_splits == 1) {
            out[row * HD + d] = __float2bfloat16_rn(acc * kv8_inverse(mm, ll, sink ? sink + g * R + pair % R : nullptr));
        } else {
            float* at = ws + (row * n_splits + split) * (HD + 2);
            at[d] = acc;
            if (d == 0) { at[HD] = mm; at[HD + 1] = ll; }
        }
    }
    if (CLUSTER) {
        cluster_sync_all();
        const int rank = (int)cluster_rank();                        // == split
        for (int i = rank * NT + threadIdx.x; i < n_cols * HD; i += n_splits * NT) {
            const int col = i / HD, d = i - col * HD, pair = pair0 + col;
            float ms[MAX_CLUSTER], ls[MAX_CLUSTER], as[MAX_CLUSTER], mm = -INFINITY;
#pragma unroll
            for (int s = 0; s < MAX_CLUSTER; ++s) {
                ms[s] = -INFINITY; ls[s] = 0.f; as[s] = 0.f;
                if (s < n_splits) {
                    const uint32_t at = cluster_map(mine + col * (HD + 2), (uint32_t)s);
                    ms[s] = cluster_ld_f32(at + HD * 4);
                    ls[s] = cluster_ld_f32(at + (HD + 1) * 4);
                    as[s] = cluster_ld_f32(at + d * 4);
                }
                mm = fmaxf(mm, ms[s]);
            }
            float acc = 0.f, ll = 0.f;
#pragma unroll
            for (int s = 0; s < MAX_CLUSTER; ++s) {
                if (ms[s] == -INFINITY) continue;
                const float wgt = exp2f(ms[s] - mm);
                acc = fmaf(wgt, as[s], acc);
                ll = fmaf(wgt, ls[s], ll);
            }
            out[((size_t)(sq.t0 + pair / R) * H + g * R + pair % R) * HD + d] =
                __float2bfloat16_rn(acc * kv8_inverse(mm, ll, sink ? sink + g * R + pair % R : nullptr));
        }
        cluster_sync_all();                                          // nobody reads this CTA's shared memory any more
    }
}

// out[row] = sum_s w_s acc_s / sum_s w_s l_s with w_s = exp2(m_s - max m), ranges in their order.  A block a row.
__global__ void __launch_bounds__(NT)
kv8_join_kernel(const float* ws, bf16* __restrict__ out, int n_splits, int H, const float* sink, const int* seq_start, int n_seqs) {
    extern __shared__ float weight[];                                // [n_splits]
    __shared__ float red[NT / 32], s_l;
    pdl_wait();
    pdl_launch_dependents();
    const size_t row = blockIdx.x;
    if (kv8_of_no_sequence((int)(row / H), seq_start, n_seqs)) return;
    const float* p = ws + row * n_splits * (HD + 2);
    float m = -INFINITY;
    for (int s = threadIdx.x; s < n_splits; s += NT) m = fmaxf(m, p[(size_t)s * (HD + 2) + HD]);
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    for (int s = threadIdx.x; s < n_splits; s += NT) {
        const float ms = p[(size_t)s * (HD + 2) + HD];
        weight[s] = ms == -INFINITY ? 0.f : exp2f(ms - m);
    }
    __syncthreads();
    if (threadIdx.x < 32) {                                          // ranges dealt out to 32 lanes, their sums in the tree's order
        float l = 0.f;
        for (int s = threadIdx.x; s < n_splits; s += 32)
            if (weight[s] != 0.f) l = fmaf(weight[s], p[(size_t)s * (HD + 2) + HD + 1], l);
        l = warp_sum(l);
        if (threadIdx.x == 0) s_l = l;
    }
    __syncthreads();
    const float inv = kv8_inverse(m, s_l, sink ? sink + row % H : nullptr);
    for (int d = threadIdx.x; d < HD; d += NT) {
        float acc = 0.f;
#pragma unroll 8
        for (int s = 0; s < n_splits; ++s)
            if (weight[s] != 0.f) acc = fmaf(weight[s], p[(size_t)s * (HD + 2) + d], acc);
        out[row * HD + d] = __float2bfloat16_rn(acc * inv);
    }
}

// -------------------------------------------------------------------------------------------- prompts
constexpr int LDS = HD + 8;                      // halves of a row in shared memory: ldmatrix without bank conflicts
constexpr size_t TILE_SMEM = (size_t)3 * 64 * LDS * 2;

// grid (tiles of 64 rows of the longest sequence, G, sequences): 16 rows a warp, keys and values a page at a time as halves in shared
// memory.  For head sizes up to 128 the next page's bytes are in registers meanwhile.
__global__ void __launch_bounds__(NT)
kv8_tile_kernel(const bf16* q, const Cache cache, bf16* __restrict__ out, const Kv8Step step, int H, int G, float scale_log2, int window,
                const float* sink, int keep, const float* slopes) {
    constexpr int CPR = HD / 16, CHUNKS = 64 * CPR / NT > 0 ? (64 * CPR + NT - 1) / NT : 1;       // 16-byte chunks of a page's rows
    constexpr bool AHEAD = HD <= 128;
    extern __shared__ __align__(16) uint8_t sm_raw[];
    __half* q_s = reinterpret_cast<__half*>(sm_raw);
    __half* k_s = q_s + 64 * LDS;
    __half* v_s = k_s + 64 * LDS;
    __shared__ int row_exp[64];
    __shared__ int s_nan;
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = blockIdx.y, R = H / G;
    const Kv8Seq sq = kv8_seq(step, blockIdx.z);
    const long n_rows = (long)sq.n_new * R;
    const int n_tiles = (int)((n_rows + 63) / 64);
    if ((int)blockIdx.x >= n_tiles) return;
    const long row0 = (long)(n_tiles - 1 - blockIdx.x) * 64;                       // the longest tiles first
    const int rows = (int)min(64L, n_rows - row0);
    const int pos_first = sq.pos0 + (int)(row0 / R), pos_last = sq.pos0 + (int)((row0 + rows - 1) / R);
    const int lo_first = plm_first_key(pos_first, window), lo_last = plm_first_key(pos_last, window);
    if (threadIdx.x == 0) s_nan = 0;

    for (int r = warp; r < 64; r += WARPS) {                                       // a row a warp: its largest number, then halves of it
        const long pair = row0 + r;
        const bf16* row = q + ((size_t)(sq.t0 + pair / R) * H + g * R + pair % R) * HD;
        float x[(HD + 63) / 64 * 2], most = 0.f;
#pragma unroll
        for (int i = 0; i < (HD + 63) / 64; ++i) {
            const int d = i * 64 + lane * 2;
            const uint32_t w = r < rows && d < HD ? *reinterpret_cast<const uint32_t*>(row + d) : 0u;
            x[2 * i] = __uint_as_float(w << 16);
            x[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
            most = fmaxf(most, fmaxf(kv8_magnitude(x[2 * i]), kv8_magnitude(x[2 * i + 1])));
        }
        const int e = row_exponent(warp_max(most));
        const float down = kv8_pow2(-e);
#pragma unroll
        for (int i = 0; i < (HD + 63) / 64; ++i) {
            const int d = i * 64 + lane * 2;
            if (d < HD) *reinterpret_cast<uint32_t*>(q_s + r * LDS + d) = halves(x[2 * i] * down, x[2 * i + 1] * down);
        }
        if (lane == 0) row_exp[r] = e;
    }

    const Walk walk(pos_first, pos_last, window, keep);
    uint4 kr[AHEAD ? CHUNKS : 1], vr[AHEAD ? CHUNKS : 1];
    float ks = 0.f, vs = 0.f;
    auto base_of = [&](int i) { return ((size_t)PLM_PAGE_NO(sq.pages[walk.page_at(i)]) * G + g); };
    auto ask = [&](int i) {
        const size_t at = base_of(i);
        ks = cache.ks[at];
        vs = cache.vs[at];
        if (AHEAD) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                const int x = c * NT + threadIdx.x;
                if (x < 64 * CPR) {
                    kr[AHEAD ? c : 0] = *reinterpret_cast<const uint4*>(cache.k + at * PLM_PAGE * HD + (size_t)x * 16);
                    vr[AHEAD ? c : 0] = *reinterpret_cast<const uint4*>(cache.v + at * PLM_PAGE * HD + (size_t)x * 16);
                }
            }
        }
    };
    auto widen = [&](__half* dst, uint4 w) {                                       // 16 numbers as halves
        const uint32_t in[4] = {w.x, w.y, w.z, w.w};
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) { h[2 * i] = kv8_halves(in[i] & 0xffffu); h[2 * i + 1] = kv8_halves(in[i] >> 16); }
        *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(dst + 8) = make_uint4(h[4], h[5], h[6], h[7]);
    };
    auto bring = [&](int i) {                                                      // page i of the walk into shared memory
        const size_t at = AHEAD ? 0 : base_of(i) * PLM_PAGE * HD;
        const int key0 = walk.page_at(i) * PLM_PAGE;
        const bool edge = key0 + PLM_PAGE - 1 > pos_first || key0 < lo_last;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int x = c * NT + threadIdx.x;
            if (x >= 64 * CPR) break;
            const int r = x / CPR, col = (x - r * CPR) * 16;
            const uint4 kv = AHEAD ? kr[AHEAD ? c : 0] : *reinterpret_cast<const uint4*>(cache.k + at + (size_t)x * 16);
            uint4 vv = AHEAD ? vr[AHEAD ? c : 0] : *reinterpret_cast<const uint4*>(cache.v + at + (size_t)x * 16);
            if (edge) {                                                            // see the kernel above
                const bool seen = key0 + r <= pos_last && (key0 + r >= lo_first || key0 + r < keep);
                const uint32_t mx = nan_bytes(vv.x), my = nan_bytes(vv.y), mz = nan_bytes(vv.z), mw = nan_bytes(vv.w);
                if (seen && (mx | my | mz | mw)) s_nan = 1;
                vv = seen ? make_uint4(without(vv.x, mx), without(vv.y, my), without(vv.z, mz), without(vv.w, mw)) : make_uint4(0, 0, 0, 0);
            }
            widen(k_s + r * LDS + col, kv);
            widen(v_s + r * LDS + col, vv);
        }
    };
    ask(0);
    __syncthreads();                                                               // the rows' exponents

    const int r_of[2] = {warp * 16 + (lane >> 2), warp * 16 + (lane >> 2) + 8};
    int pos[2], lo[2];
    float cs[2], slope[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
        const bool have = r_of[hi] < rows;
        pos[hi] = have ? sq.pos0 + (int)((row0 + r_of[hi]) / R) : -1;
        lo[hi] = plm_first_key(pos[hi], window);
        cs[hi] = scale_log2 * kv8_pow2(max(-126, min(127, row_exp[r_of[hi]])));
        slope[hi] = slopes && have ? slopes[g * R + (int)((row0 + r_of[hi]) % R)] * LOG2E : 0.f;
    }
    const int warp_pos_last = sq.pos0 + (int)((row0 + min(rows - 1, warp * 16 + 15)) / R);
    const bool warp_works = warp * 16 < rows;
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    int eo = kv8_exponent_of_scale(vs);

    for (int i = 0; i < walk.n_pages; ++i) {
        const float ks_now = ks;
        const int ev = kv8_exponent_of_scale(vs);
        bring(i);
        if (i + 1 < walk.n_pages) ask(i + 1);
        __syncthreads();
        const int key0 = walk.page_at(i) * PLM_PAGE;
        if (warp_works && key0 <= warp_pos_last) {
            float s[8][4];
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                uint32_t a[4];
                ldsm_x4(a, smem_u32(q_s + (warp * 16 + (lane & 15)) * LDS + k * 16 + (lane >> 4) * 8));
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    uint32_t b[4];
                    ldsm_x4(b, smem_u32(k_s + (j * 8 + (lane & 7) + (lane >> 4) * 8) * LDS + k * 16 + ((lane >> 3) & 1) * 8));
                    mma_f16(s[j], a, b[0], b[1]);
                    mma_f16(s[j + 1], a, b[2], b[3]);
                }
            }
            const float c[2] = {cs[0] * ks_now, cs[1] * ks_now};
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int hi = e >> 1, key = key0 + j * 8 + (lane & 3) * 2 + (e & 1);
                    const bool ok = key <= pos[hi] && (key >= lo[hi] || key < keep);
                    float x = s[j][e] * c[hi];
                    if (slopes) x = fmaf(slope[hi], (float)(key - pos[hi]), x);
                    s[j][e] = ok ? x : -INFINITY;
                    mx[hi] = fmaxf(mx[hi], s[j][e]);
                }
            float down[2], use[2];
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
                mx[hi] = fmaxf(mx[hi], __shfl_xor_sync(0xffffffffu, mx[hi], 1));
                mx[hi] = fmaxf(mx[hi], __shfl_xor_sync(0xffffffffu, mx[hi], 2));
                const float m_new = fmaxf(m[hi], mx[hi]);
                use[hi] = m_new == -INFINITY ? 0.f : m_new;
                l[hi] *= ex2(m[hi] - use[hi]);                                     // (-inf gives 0)
                down[hi] = ex2(m[hi] - use[hi] + (float)(eo - ev));
                m[hi] = m_new;
            }
            eo = ev;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[j][e] = ex2(s[j][e] - use[e >> 1]);
                    l[e >> 1] += s[j][e];                                          // (this lane's keys; the row's four lanes at the end)
                }
#pragma unroll
            for (int t = 0; t < HD / 8; ++t) {
                o[t][0] *= down[0]; o[t][1] *= down[0];
                o[t][2] *= down[1]; o[t][3] *= down[1];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t a[4] = {halves(s[2 * k][0], s[2 * k][1]), halves(s[2 * k][2], s[2 * k][3]),
                                       halves(s[2 * k + 1][0], s[2 * k + 1][1]), halves(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
                for (int t = 0; t < HD / 8; t += 2) {
                    uint32_t b[4];
                    ldsm_x4_t(b, smem_u32(v_s + (k * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * LDS + t * 8 + (lane >> 4) * 8));
                    mma_f16(o[t], a, b[0], b[1]);
                    mma_f16(o[t + 1], a, b[2], b[3]);
                }
            }
        }
        __syncthreads();                                                           // the page's place is free
    }
    const float unit = kv8_pow2(max(-126, min(127, eo)));
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
        l[hi] += __shfl_xor_sync(0xffffffffu, l[hi], 1);
        l[hi] += __shfl_xor_sync(0xffffffffu, l[hi], 2);
        if (r_of[hi] >= rows) continue;
        const long pair = row0 + r_of[hi];
        const int h = g * R + (int)(pair % R);
        const float inv = kv8_inverse(m[hi], l[hi], sink ? sink + h : nullptr) * unit;
        bf16* dst = out + ((size_t)(sq.t0 + pair / R) * H + h) * HD + (lane & 3) * 2;
#pragma unroll
        for (int t = 0; t < HD / 8; ++t) {
            float x = o[t][2 * hi] * inv, y = o[t][2 * hi + 1] * inv;
            if (s_nan) {
                for (int i = 0; i < walk.n_pages; ++i) {
                    const int key0 = walk.page_at(i) * PLM_PAGE;
                    if (!(key0 + PLM_PAGE - 1 > pos_first || key0 < lo_last)) continue;
                    const uint8_t* at = cache.v + base_of(i) * PLM_PAGE * HD + t * 8 + (lane & 3) * 2;
                    for (int k = 0; k < PLM_PAGE; ++k) {
                        if (key0 + k > pos[hi] || (key0 + k < lo[hi] && key0 + k >= keep)) continue;
                        if (is_nan_byte(at[(size_t)k * HD])) x = __int_as_float(0x7fffffff);
                        if (is_nan_byte(at[(size_t)k * HD + 1])) y = __int_as_float(0x7fffffff);
                    }
                }
            }
            *reinterpret_cast<__nv_bfloat162*>(dst + t * 8) = __floats2bfloat162_rn(x, y);
        }
    }
}

template <int NG>
int stream(const bf16* q, const Cache& cache, bf16* out, float* ws, const Kv8Step& step, int n_seqs, int max_new, int H, int G, float scale,
           int window, int n_splits, const float* sink, int keep, const float* slopes, cudaStream_t s) {
    static std::atomic<unsigned long long> d0{0}, d1{0};
    const size_t smem = stream_smem(NG);
    const bool cluster = n_splits > 1 && !ws;
    cudaError_t e = cluster ? plm_allow_smem(kv8_stream_kernel<NG, true>, smem, d0) : plm_allow_smem(kv8_stream_kernel<NG, false>, smem, d1);
    if (e != cudaSuccess) return (int)e;
    const long tiles = ((long)max_new * (H / G) + 8 * NG - 1) / (8 * NG);
    if (tiles * G > 65535) return PLM_ERR_SHAPE;
    const dim3 grid(n_splits, (unsigned)(tiles * G), n_seqs);
    if (cluster)
        return plm_status_of(launch_pdl_cluster(kv8_stream_kernel<NG, true>, grid, dim3(NT), dim3(n_splits, 1, 1), smem, s, q, cache, out, ws,
                                                step, H, G, (int)tiles, scale * LOG2E, window, sink, keep, slopes));
    return plm_status_of(launch_pdl(kv8_stream_kernel<NG, false>, grid, dim3(NT), smem, s, q, cache, out, ws, step, H, G, (int)tiles,
                                    scale * LOG2E, window, sink, keep, slopes));
}

bool bad_step(const int* tok_pos, const int* tok_seq, const int* seq_start, const int* seq_kv_len) {
    return !tok_pos != !tok_seq || !tok_pos == !seq_start || !seq_start != !seq_kv_len;
}

}  // namespace

// q [n_rows, H, HD] bf16, out [n_rows, H * HD] bf16.  Either tok_pos and tok_seq [n_seqs = n_rows] (single tokens, max_new 1) or
// seq_start [n_seqs + 1] and seq_kv_len [n_seqs].  Every sequence's keys are cut into n_splits ranges; up to eight meet in their
// cluster where ws is null, else ws holds n_rows * H * n_splits * (HD + 2) floats.
extern "C" int plm_kv8_attention_few(const void* q, const void* kc, const void* vc, const float* ks, const float* vs, void* out, float* ws,
                                     const int* tok_pos, const int* tok_seq, const int* seq_start, const int* seq_kv_len,
                                     const int* block_table, int max_pages, int n_rows, int n_seqs, int max_new, int H, int G,
                                     float scale, int window, int n_splits, const float* sink, int keep, const float* slopes,
                                     cudaStream_t s) {
    if (n_rows <= 0 || n_seqs <= 0 || max_new <= 0) return PLM_OK;
    if (H <= 0 || G <= 0 || H % G || n_seqs > 65535 || n_splits < 1 || (n_splits > 1 && !ws && n_splits > MAX_CLUSTER) || n_splits > 8192 ||
        keep < 0 || (long)n_rows * H > 0x7fffffffL)
        return PLM_ERR_SHAPE;
    if (bad_step(tok_pos, tok_seq, seq_start, seq_kv_len)) return PLM_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) & 15) return PLM_ERR_ALIGN;
    if (n_splits == 1) ws = nullptr;
    const Kv8Step step = {tok_pos, tok_seq, seq_start, seq_kv_len, block_table, max_pages};
    const Cache cache = {(const uint8_t*)kc, (const uint8_t*)vc, ks, vs};
    const long rows = (long)max_new * (H / G);
    int rc;
#define KV8_STREAM(NG_) rc = stream<NG_>((const bf16*)q, cache, (bf16*)out, ws, step, n_seqs, max_new, H, G, scale, window, n_splits, sink, keep, slopes, s)
    if (rows <= 8) KV8_STREAM(1);
    else if (rows <= 16 || HD > 128) KV8_STREAM(2);
    else KV8_STREAM((HD > 128 ? 2 : 4));
#undef KV8_STREAM
    if (rc != PLM_OK || !ws) return rc;
    return plm_status_of(launch_pdl(kv8_join_kernel, dim3((unsigned)((long)n_rows * H)), dim3(NT), n_splits * sizeof(float), s,
                                    (const float*)ws, (bf16*)out, n_splits, H, sink, seq_start, n_seqs));
}

// The same for prompts, rows of 64 at a time: seq_start [n_seqs + 1], seq_kv_len [n_seqs], at most max_new rows a sequence.
extern "C" int plm_kv8_attention_tiles(const void* q, const void* kc, const void* vc, const float* ks, const float* vs, void* out,
                                       const int* seq_start, const int* seq_kv_len, const int* block_table, int max_pages, int n_seqs,
                                       int max_new, int H, int G, float scale, int window, const float* sink, int keep,
                                       const float* slopes, cudaStream_t s) {
    if (n_seqs <= 0 || max_new <= 0) return PLM_OK;
    if (H <= 0 || G <= 0 || H % G || n_seqs > 65535 || G > 65535 || keep < 0) return PLM_ERR_SHAPE;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) & 15) return PLM_ERR_ALIGN;
    static std::atomic<unsigned long long> devices{0};
    cudaError_t e = plm_allow_smem(kv8_tile_kernel, TILE_SMEM, devices);
    if (e != cudaSuccess) return (int)e;
    const Kv8Step step = {nullptr, nullptr, seq_start, seq_kv_len, block_table, max_pages};
    const Cache cache = {(const uint8_t*)kc, (const uint8_t*)vc, ks, vs};
    const dim3 grid((unsigned)(((long)max_new * (H / G) + 63) / 64), G, n_seqs);
    return plm_status_of(launch_pdl(kv8_tile_kernel, grid, dim3(NT), TILE_SMEM, s, (const bf16*)q, cache, (bf16*)out, step, H, G,
                                    scale * LOG2E, window, sink, keep, slopes));
}
