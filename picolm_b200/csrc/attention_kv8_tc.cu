// Attention of prompts in bfloat16 over the 8-bit cache (kv8.cuh) on the fifth-generation tensor cores, compiled for one head
// size (-DPLM_HD = 64 or 128).  The mathematics is attention_kv8.cu's: e4m3 numbers as halves, a query row divided by a
// power of two as halves, the scales outside the products, the sums over values in the unit of some page's scale.
//
// A CTA takes 256 (token, head) rows of one sequence and kv head, two tiles of 128, and walks the sequence's pages of 64 keys; or
// 128 rows, which both tiles take against every other page each (SPLIT), and their results are put together at the end.
// Rows are (token, head in group) pairs, so all heads of a group meet a page in the CTA that has it, and a page's bytes
// become halves once for 256 rows.  Per page and tile:
//   S = Q K^T      tcgen05.mma, Q and K in shared memory (halves, 128-byte swizzle), S in tensor memory
//   softmax        a thread a row: its 64 scores out of tensor memory, running maximum and sum in fp32, probabilities as halves
//                  over the first half of the scores' place
//   O += P V       tcgen05.mma, P from tensor memory, V in shared memory (MN-major); O stays in tensor memory and is scaled only when
//                  a row's maximum outgrows its reference or a page's values have a scale beyond 2^KV8_SPAN from O's unit
// Warps 0..7 are the softmax threads of the two tiles (quarter = warp % 4), 8 and 9 make halves of keys' bytes, 10 and 11 of values',
// 12 and 14 issue the tiles' MMAs (12 owns the tensor memory), 13 asks for pages: a page's keys and values of a kv head are
// contiguous, so that each is one bulk copy of 4 or 8 KB into a ring of raw pages.  While one tile's threads work on page i, the
// tensor cores have P V of the other's; the scores of a tile have two places, so that Q K^T of the next page is there when
// its threads come for it.
//
// What bounds it.  Per page and 256 rows of heads of 128: shared memory's 128 bytes a cycle some 1,400 cycles (the products read Q and K 768
// and V 256, the conversion reads and writes 384), the 16,384 exponentials 1,024 of the special-function units, the products 1,024 of the
// tensor cores; a page takes some 2,100.  Heads of 64: 700, 1,024, 512 of some 1,600.  The rest is hand-overs: a wait on a barrier that is
// ready costs a warp 150 cycles here, a page is five of them in a row.  Measured, 32 heads over 8 of 128 (us): 1,000 tokens behind 15,000 keys
// 276 (920 TFLOP/s), 2,048 of 64 42 (415), 16 sequences of 9 tokens behind 3,000 37.  What made it so, at the first of those: keys and
// values converted by two teams that wait for nothing of each other, every load of a page asked for before any is used, one arrival a
// warp and not one a thread, waits that park (polling threads take the issue slots that the conversion needs): 292 -> 274.
// 128 rows a CTA, every other page a tile: where a wave holds all CTAs of 128 rows, or none has more (us, 256 rows / 128: 500 tokens
// behind 3,000 69 / 44, 16 times 9 behind 3,000 46 / 37, 600 behind 3,000, where it does not, 70 / 76).
//
// Every wait is bounded: one that runs out records where in `status`; the CTA stops issuing work, lets what is in flight land,
// frees its tensor memory and returns.
#include "tc_common.cuh"
#include "kv8.cuh"

#ifndef PLM_HD
#define PLM_HD 128
#endif

using namespace plm_tc;

namespace {

constexpr int HD = PLM_HD;
static_assert(HD == 64 || HD == 128, "built for head sizes 64 and 128");
constexpr float LOG2E = 1.4426950408889634f;
constexpr int CB = HD / 64;                       // blocks of 64 columns: a 128-byte line of halves each
constexpr int BQ = 128, TILES = 2, BKV = PLM_PAGE;
constexpr int RS = 4, KS = 3, VS = 3;             // raw pages, keys' and values' halves in their rings
constexpr int NT = 512;
constexpr uint32_t Q_BLOCK = BQ * 128, KV_BLOCK = BKV * 128;
constexpr uint32_t Q_BYTES = CB * Q_BLOCK, KV_BYTES = CB * KV_BLOCK, RAW_BYTES = BKV * HD;     // of one tensor's page
constexpr uint32_t TM_S = 0, TM_O = TILES * 128, TMEM_COLS = 512;
static_assert(TM_O + TILES * HD <= TMEM_COLS, "tensor memory");
constexpr size_t SMEM = 1024 + TILES * Q_BYTES + (KS + VS) * KV_BYTES + RS * 2 * RAW_BYTES + 320;
static_assert(SMEM + 1600 <= 227 * 1024, "shared memory, with what the kernel declares itself");
static_assert(8 * (2 * RS + 2 * KS + 2 * VS + 7 * TILES + TILES + 1) <= 320, "barriers");
// Registers a thread: launched with 128; the softmax's two warpgroups take 168 each, the other two keep 88: 2 * 168 + 2 * 88 = 4 * 128.
constexpr int SOFTMAX_REGS = 168, OTHER_REGS = 88;

#ifdef PLM_TEST_STALL
__device__ int plm_stall = 0;                     // a test build: the pages' barriers are told of more bytes than come
#endif
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) { tc_mma_bf16(d, a, b, idesc, accumulate); }
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// V [64 keys][64 columns] a block, columns contiguous: MN-major; 8-key groups 1,024 bytes apart, blocks KV_BLOCK.
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(KV_BLOCK >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D fp32, A and B fp16, M = 128, N = n; b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t instr_desc(int n, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
}
// bytes that are NaN (e4m3: 0x7f and 0xff): 0x80 in their places
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t without(uint32_t w, uint32_t marks) { return w & ~(marks | (marks - (marks >> 7))); }

struct Cache {
    const uint8_t *k, *v;
    const float *ks, *vs;
};

// grid (tiles of 256 rows, SPLIT: of 128, of the longest sequence, G, sequences).  EXTRA: instances for kept first positions and slopes; they walk from
// the tile's own pages to the oldest, along which slopes make the scores fall.
template <bool EXTRA, bool SPLIT>
__global__ void __launch_bounds__(NT, 1)
kv8_tc_kernel(const bf16* q, const Cache cache, bf16* __restrict__ out, const Kv8Step step, int H, int G, float scale_log2, int window,
              int* __restrict__ status, const float* sink, int keep, const float* slopes) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_smem = base, k_smem = q_smem + TILES * Q_BYTES, v_smem = k_smem + KS * KV_BYTES, raw = v_smem + VS * KV_BYTES;
    const uint32_t bars = raw + RS * 2 * RAW_BYTES;
    const uint32_t raw_full = bars, raw_empty = raw_full + 8 * RS, k_full = raw_empty + 8 * RS, k_empty = k_full + 8 * KS,
                   v_full = k_empty + 8 * KS, v_empty = v_full + 8 * VS, q_full = v_empty + 8 * VS, s_full = q_full + 8 * TILES,
                   p_ready = s_full + 16 * TILES, pv_full = p_ready + 16 * TILES, done = pv_full + 16 * TILES, other = done + 16;
    __shared__ uint32_t tmem_slot;
    __shared__ int s_abort, s_nan;
    __shared__ float other_m[BQ], other_l[BQ];                                     // split: what the second tile's rows came to
    __shared__ int other_eo[BQ];

    pdl_wait();
    // CTAs start in the order of their index: the longest tiles of all kv heads first, the short ones fill the end
    const unsigned lin = blockIdx.y * gridDim.x + blockIdx.x;
    const int g = lin % G, rank = lin / G, R = H / G;
    const Kv8Seq sq = kv8_seq(step, blockIdx.z);
    const long n_rows = (long)sq.n_new * R;
    constexpr int ROWS = SPLIT ? BQ : TILES * BQ;
    const int n_tiles = (int)((n_rows + ROWS - 1) / ROWS);
    if (rank >= n_tiles) return;
    const long row0 = (long)(n_tiles - 1 - rank) * ROWS;
    const int rows = (int)min((long)ROWS, n_rows - row0);
    const int used = rows > BQ ? 2 : 1;                                            // tiles that look at a page
    const int pos_first = sq.pos0 + (int)(row0 / R), pos_last = sq.pos0 + (int)((row0 + rows - 1) / R);
    const int lo_first = plm_first_key(pos_first, window), lo_last = plm_first_key(pos_last, window);
    const int page_first = lo_first / BKV, n_kept = EXTRA ? plm_kept_pages(lo_first, keep) : 0;
    const int n_pages = n_kept + pos_last / BKV - page_first + 1;
    auto page_at = [&](int i) {
        if (!EXTRA) return page_first + i;
        const int w = n_pages - 1 - i;
        return w < n_kept ? w : page_first + w - n_kept;
    };
    // pages that tile t works on: every other one, or the first of the walk (EXTRA: all of it)
    auto pages_of = [&](int t) {
        if (SPLIT) return (n_pages + 1 - t) >> 1;
        if (t >= used) return 0;
        if (EXTRA || t == used - 1) return n_pages;
        return (sq.pos0 + (int)((row0 + BQ - 1) / R)) / BKV - page_first + 1;
    };
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        s_abort = 0;
        s_nan = 0;
        for (int i = 0; i < RS; ++i) { mbar_init(raw_full + 8 * i, 1); mbar_init(raw_empty + 8 * i, 4); }
        for (int i = 0; i < KS; ++i) { mbar_init(k_full + 8 * i, 2); mbar_init(k_empty + 8 * i, used); }
        for (int i = 0; i < VS; ++i) { mbar_init(v_full + 8 * i, 2); mbar_init(v_empty + 8 * i, used); }
        for (int i = 0; i < TILES; ++i) mbar_init(q_full + 8 * i, 128);
        for (int i = 0; i < 2 * TILES; ++i) { mbar_init(s_full + 8 * i, 1); mbar_init(p_ready + 8 * i, 4); mbar_init(pv_full + 8 * i, 1); }
        mbar_init(done, 1);
        mbar_init(done + 8, 1);
        mbar_init(other, 128);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // The next kernel may begin once every CTA is here: one that wants tensor memory and then waits for this kernel must not
    // take what a CTA of this one still asks for.
    pdl_launch_dependents();

    if (warp < 8) {
        // ----------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
        const int t = warp >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane;                                         // the row within the tile
        const int t_row = SPLIT ? 0 : t * BQ, i_first = SPLIT ? t : 0;
        constexpr int i_step = SPLIT ? 2 : 1;
        const long pair = row0 + t_row + r;
        const bool have = t_row + r < rows;
        const int head = g * R + (have ? (int)(pair % R) : 0);
        const size_t q_row = (size_t)(sq.t0 + (have ? (int)(pair / R) : 0)) * H + head;
        const int pos = have ? sq.pos0 + (int)(pair / R) : -1, lo = plm_first_key(pos, window);
        const int tile_pos_first = sq.pos0 + (int)(min(row0 + t_row, n_rows - 1) / R);
        const int tile_pos_last = sq.pos0 + (int)(min(row0 + t_row + BQ - 1, n_rows - 1) / R);
        const int tile_lo_last = plm_first_key(tile_pos_last, window);
        const int my_pages = pages_of(t);
        float c_row;
        if (my_pages > 0) {                                                        // the row as halves, into shared memory
            uint4 w[HD / 8];
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) w[i] = have ? reinterpret_cast<const uint4*>(q + q_row * HD)[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    most = fmaxf(most, fmaxf(kv8_magnitude(__uint_as_float(x[k] << 16)), kv8_magnitude(__uint_as_float(x[k] & 0xffff0000u))));
            }
            // a power of two that puts the largest number into [2^13, 2^14)
            const int e = most > 0.f ? max((int)(__float_as_uint(most) >> 23) - 127, -100) - 13 : 0;
            const float down = kv8_pow2(-e);
            c_row = scale_log2 * kv8_pow2(max(-126, min(127, e)));
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                uint32_t h[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) h[k] = halves(__uint_as_float(x[k] << 16) * down, __uint_as_float(x[k] & 0xffff0000u) * down);
                if (!(SPLIT && t)) sts16(q_smem + t * Q_BYTES + (i >> 3) * Q_BLOCK + r * 128 + (((i & 7) ^ (r & 7)) << 4), h[0], h[1], h[2], h[3]);
            }
            fence_async();
            if (!(SPLIT && t)) mbar_arrive(q_full + 8 * t);
        }
        const float slope2 = EXTRA && slopes ? slopes[head] * LOG2E : 0.f;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t tm_o = tmem + lanes + TM_O + t * HD;
        float m_ref = -INFINITY, l = 0.f;
        int eo = 0;
        bool ok = true;
        float ks_next = 0.f, vs_next = 1.f;                                        // the page's scales, a page ahead,
        int page_next = 0;                                                         // and the number of the page after it
        if (my_pages > 0) {
            const size_t at = (size_t)PLM_PAGE_NO(sq.pages[page_at(i_first)]) * G + g;
            page_next = sq.pages[page_at(i_first + i_step * min(1, my_pages - 1))];
            ks_next = kv8_scale(cache.ks[at]);
            vs_next = kv8_scale(cache.vs[at]);
            eo = kv8_exponent_of_scale(vs_next);
        }
        for (int i = 0; i < my_pages && ok; ++i) {
            const float c = c_row * ks_next;
            const int ev = kv8_exponent_of_scale(vs_next);
            if (i + 1 < my_pages) {
                const size_t at = (size_t)PLM_PAGE_NO(page_next) * G + g;
                ks_next = kv8_scale(cache.ks[at]);
                vs_next = kv8_scale(cache.vs[at]);
                page_next = sq.pages[page_at(i_first + i_step * min(i + 2, my_pages - 1))];
            }
            const uint32_t s_tm = tmem + lanes + TM_S + t * 128 + (i & 1) * 64;
            if (!mbar_wait(s_full + 16 * t + 8 * (i & 1), (i >> 1) & 1, status, 72)) { ok = false; break; }
            tc_fence_after();
            const int key0 = page_at(i_first + i_step * i) * BKV;
            const bool need_mask = key0 + BKV - 1 > tile_pos_first || (key0 < tile_lo_last && (!EXTRA || key0 + BKV > keep));
            uint32_t s0[32], s1[32];
            tc_ld32(s_tm, s0);
            tc_ld32(s_tm + 32, s1);
            tc_wait_ld_into(s0);
            tc_wait_ld_into(s1);
            // scores in log2 units are s * c2 (with slopes they are made here, and c2 is 1)
            float c2 = c;
            if (EXTRA) {
                const uint64_t cc = pack2(c, c), sl = pack2(slope2, slope2);
                const float off = slope2 * (float)(key0 - pos), off_hi = slope2 * (float)(key0 + 32 - pos);
                const uint64_t o2 = pack2(off, off), o2h = pack2(off_hi, off_hi);
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const uint64_t jj = pack2((float)j, (float)(j + 1));
                    float x0, x1, y0, y1;
                    unpack2(fma2(pack2(__uint_as_float(s0[j]), __uint_as_float(s0[j + 1])), cc, fma2(jj, sl, o2)), x0, x1);
                    unpack2(fma2(pack2(__uint_as_float(s1[j]), __uint_as_float(s1[j + 1])), cc, fma2(jj, sl, o2h)), y0, y1);
                    s0[j] = __float_as_uint(x0); s0[j + 1] = __float_as_uint(x1);
                    s1[j] = __float_as_uint(y0); s1[j + 1] = __float_as_uint(y1);
                }
                c2 = 1.f;
            }
            if (need_mask) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const int ka = key0 + j, kb = key0 + 32 + j;
                    if (ka > pos || (ka < lo && (!EXTRA || ka >= keep))) s0[j] = 0xff800000u;
                    if (kb > pos || (kb < lo && (!EXTRA || kb >= keep))) s1[j] = 0xff800000u;
                }
            }
            float mx = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                mx = max3(mx, __uint_as_float(s0[j]), __uint_as_float(s1[j]));
                mx1 = max3(mx1, __uint_as_float(s0[j + 1]), __uint_as_float(s1[j + 1]));
                mx2 = max3(mx2, __uint_as_float(s0[j + 2]), __uint_as_float(s1[j + 2]));
                mx3 = max3(mx3, __uint_as_float(s0[j + 3]), __uint_as_float(s1[j + 3]));
            }
            mx = fmaxf(fmaxf(mx, mx1), fmaxf(mx2, mx3));
            const float m_cand = fmaxf(m_ref, mx * c2 - (float)KV8_LIFT);          // (c2 is positive)
            int d = ev - eo;
            const bool raise = m_cand > (m_ref == -INFINITY ? -INFINITY : m_ref + (float)KV8_RAISE);
            if (__any_sync(0xffffffffu, raise || d > KV8_SPAN || d < -KV8_SPAN)) {                // tcgen05.ld/st are warp-wide
                const float by = raise ? m_ref - m_cand : 0.f;                     // -inf where nothing was seen before
                if (i > 0) {
                    // O may only be touched once every P V issued so far has landed in it
                    if (!mbar_wait(pv_full + 16 * t + 8 * ((i - 1) & 1), ((i - 1) >> 1) & 1, status, 72)) { ok = false; break; }
                    tc_fence_after();
                    const float alpha = ex2(by - (float)d);
#pragma unroll
                    for (int x = 0; x < HD; x += 32) {
                        uint32_t ov[32];
                        tc_ld32(tm_o + x, ov);
                        tc_wait_ld_into(ov);
#pragma unroll
                        for (int j = 0; j < 32; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * alpha);
                        tc_st32(tm_o + x, ov);
                    }
                }
                if (raise) { l *= ex2(by); m_ref = m_cand; }
                eo = ev;
                d = 0;
            }
            const float off = (float)d - (m_ref == -INFINITY ? 0.f : m_ref);
            const uint64_t cc = pack2(c2, c2), oo = pack2(off, off);
            uint32_t p[32];
            uint64_t sum2 = 0;                                                     // two partial sums, (0.f, 0.f)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                float a0, a1, b0, b1;
                unpack2(fma2(pack2(__uint_as_float(s0[2 * j]), __uint_as_float(s0[2 * j + 1])), cc, oo), a0, a1);
                unpack2(fma2(pack2(__uint_as_float(s1[2 * j]), __uint_as_float(s1[2 * j + 1])), cc, oo), b0, b1);
                a0 = ex2(a0); a1 = ex2(a1); b0 = ex2(b0); b1 = ex2(b1);
                sum2 = add2(sum2, add2(pack2(a0, a1), pack2(b0, b1)));
                p[j] = halves(a0, a1);
                p[16 + j] = halves(b0, b1);
            }
            float sum_lo, sum_hi;
            unpack2(sum2, sum_lo, sum_hi);
            l = fmaf(sum_lo + sum_hi, kv8_pow2(-d), l);
            tc_st32(s_tm, p);                                                      // over the scores, which this thread has read
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready + 16 * t + 8 * (i & 1));
        }
        if (ok && my_pages > 0 && !mbar_wait(pv_full + 16 * t + 8 * ((my_pages - 1) & 1), ((my_pages - 1) >> 1) & 1, status, 72)) ok = false;
        tc_fence_after();
        // Split: the second tile's sums lie in the same lanes of tensor memory, so the first tile's threads take them from there.
        const bool joins = SPLIT && n_pages > 1;
        if (joins && t == 1 && ok) {
            other_m[r] = kv8_top(m_ref, l);
            other_l[r] = l;
            other_eo[r] = eo;
            mbar_arrive(other);
        }
        float inv = 0.f, inv_other = 0.f;
        if (ok && t < used) {
            const float unit = kv8_pow2(max(-126, min(127, eo)));
            if (joins && (!mbar_wait(other, 0, status, 72) || !mbar_wait(pv_full + 16 + 8 * ((pages_of(1) - 1) & 1), ((pages_of(1) - 1) >> 1) & 1, status, 72))) ok = false;
            if (joins && ok) {
                tc_fence_after();
                const float m0 = kv8_top(m_ref, l), m1 = other_m[r], m = fmaxf(m0, m1);
                const float w0 = m0 == -INFINITY ? 0.f : ex2(m0 - m), w1 = m1 == -INFINITY ? 0.f : ex2(m1 - m);
                const float both = kv8_inverse(m, fmaf(w0, l, w1 * other_l[r]), sink ? sink + head : nullptr);
                inv = both * w0 * unit;
                inv_other = both * w1 * kv8_pow2(max(-126, min(127, other_eo[r])));
            } else {
                inv = kv8_inverse(m_ref, l, sink ? sink + head : nullptr) * unit;
            }
        }
        if (!ok) s_abort = 1;
        if (ok && t < used) {
            bf16* dst = out + q_row * HD;
            const bool nan = *(volatile int*)&s_nan != 0;                          // (set before the P V that has landed was asked for)
#pragma unroll 1
            for (int x = 0; x < HD; x += 32) {
                uint32_t ov[32];
                tc_ld32(tm_o + x, ov);                                             // warp-wide, also for rows that are not written
                tc_wait_ld_into(ov);
#pragma unroll
                for (int j = 0; j < 32; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * inv);
                if (joins) {
                    uint32_t more[32];
                    tc_ld32(tm_o + HD + x, more);
                    tc_wait_ld_into(more);
#pragma unroll
                    for (int j = 0; j < 32; ++j) ov[j] = __float_as_uint(fmaf(__uint_as_float(more[j]), inv_other, __uint_as_float(ov[j])));
                }
                if (nan) {                                                         // the edge pages once more, see the conversion
                    for (int i = 0; i < n_pages; ++i) {
                        const int key0 = page_at(i) * BKV;
                        if (!(key0 + BKV - 1 > pos_first || key0 < lo_last)) continue;
                        const uint8_t* v = cache.v + ((size_t)PLM_PAGE_NO(sq.pages[page_at(i)]) * G + g) * RAW_BYTES + x;
                        for (int k = 0; k < BKV; ++k) {
                            if (key0 + k > pos || (key0 + k < lo && key0 + k >= keep)) continue;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if ((v[k * HD + j] & 0x7f) == 0x7f) ov[j] = 0x7fffffffu;
                        }
                    }
                }
                if (have) {
#pragma unroll
                    for (int y = 0; y < 32; y += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const __nv_bfloat162 v2 = __floats2bfloat162_rn(__uint_as_float(ov[y + 2 * j]), __uint_as_float(ov[y + 2 * j + 1]));
                            w[j] = *reinterpret_cast<const uint32_t*>(&v2);
                        }
                        *reinterpret_cast<uint4*>(dst + x + y) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
    } else if (warp < 12) {
        // -------------------------------------------------------------- bytes to halves
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        // Two teams of two warps, one for keys and one for values, which take their own time.
        const int tid = (threadIdx.x - 256) & 63;
        const bool values = warp >= 10;
        bool ok = true;
        // 16 numbers at a time: chunk j of a row becomes 16-byte chunks 2 (j % 4) and + 1 of its line in block j / 4, each at
        // its place of the 128-byte swizzle.  Of heads of 128 eight lanes have one row: those of the second block write their second
        // chunk first, so that the eight meet 32 banks.
        constexpr int CPR = HD / 16, CHUNKS = BKV * CPR / 64;
        const bool swap = HD == 128 && (tid & 4);
        auto widen = [&](uint32_t dst, int r, int j, uint4 w) {
            uint32_t h[8];
            kv8_halves(swap ? w.z : w.x, h[0], h[1]);
            kv8_halves(swap ? w.w : w.y, h[2], h[3]);
            kv8_halves(swap ? w.x : w.z, h[4], h[5]);
            kv8_halves(swap ? w.y : w.w, h[6], h[7]);
            const uint32_t line = dst + (j >> 2) * KV_BLOCK + r * 128;
            const int c = (j & 3) * 2 + (swap ? 1 : 0);
            sts16(line + ((c ^ (r & 7)) << 4), h[0], h[1], h[2], h[3]);
            sts16(line + (((c ^ 1) ^ (r & 7)) << 4), h[4], h[5], h[6], h[7]);
        };
        static_assert(KS == VS, "one place for both");
        const uint32_t full = values ? v_full : k_full, empty = values ? v_empty : k_empty, to = values ? v_smem : k_smem;
        int rs = 0, rp = 0, hs = 0, hp = 0;                                        // places in the rings and their parities
        for (int i = 0; i < n_pages && ok; ++i) {
            ok = mbar_wait(raw_full + 8 * rs, rp, status, 71);
            if (!ok) break;
            const uint32_t src = raw + rs * 2 * RAW_BYTES + (values ? RAW_BYTES : 0) + tid * 16;
            uint4 w[CHUNKS];                                                       // (all asked for before any is waited for)
#pragma unroll
            for (int x = 0; x < CHUNKS; ++x) w[x] = lds16(src + x * 1024);
            __syncwarp();
            if (lane == 0) mbar_arrive(raw_empty + 8 * rs);
            ok = mbar_wait(empty + 8 * hs, hp ^ 1, status, 71);
            if (!ok) break;
            const int key0 = page_at(i) * BKV;
            if (values && (key0 + BKV - 1 > pos_first || key0 < lo_last)) {
                // Places that no row sees hold whatever was left there: zeros.  A NaN that some rows see and others do not would
                // reach them all (0 * NaN): it is taken out, and put into the results of those that see it at the end.
#pragma unroll
                for (int x = 0; x < CHUNKS; ++x) {
                    const int key = key0 + (x * 64 + tid) / CPR;
                    const bool seen = key <= pos_last && (key >= lo_first || key < keep);
                    const uint32_t mx = nan_bytes(w[x].x), my = nan_bytes(w[x].y), mz = nan_bytes(w[x].z), mw = nan_bytes(w[x].w);
                    if (seen && (mx | my | mz | mw)) *(volatile int*)&s_nan = 1;
                    w[x] = seen ? make_uint4(without(w[x].x, mx), without(w[x].y, my), without(w[x].z, mz), without(w[x].w, mw)) : make_uint4(0, 0, 0, 0);
                }
            }
#pragma unroll
            for (int x = 0; x < CHUNKS; ++x) widen(to + hs * KV_BYTES, (x * 64 + tid) / CPR, (x * 64 + tid) % CPR, w[x]);
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * hs);
            if (++rs == RS) { rs = 0; rp ^= 1; }
            if (++hs == KS) { hs = 0; hp ^= 1; }
        }
        if (!ok) s_abort = 1;
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp == 12 || warp == 14) {
            // ---------------------------------------------------------- MMA issuers, one a tile (the whole warp walks, one elected lane
            // issues).  One for both was what the tiles waited for: a page's waits, fences and issues are a chain of some 800 cycles.
            // A tile's j-th page is the walk's page i_first + i_step * j; where both walk all pages, those behind its own are passed by.
            const int t = (warp - 12) >> 1, mine = pages_of(t), all = SPLIT ? mine : n_pages, q_tile = SPLIT ? 0 : t;
            const int i_first = SPLIT ? t : 0;
            constexpr int i_step = SPLIT ? 2 : 1;
            const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0), q_at = q_smem + q_tile * Q_BYTES;
            constexpr uint32_t idesc_s = instr_desc(BKV, false), idesc_o = instr_desc(HD, true);
            auto scores = [&](int j) {                                             // S[j % 2] = Q K(i)^T, and K(i)'s place is free
                const int i = i_first + i_step * j;
                const uint32_t k_at = k_smem + (i % KS) * KV_BYTES;
                if (elect_one()) {
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_ss(tmem_u + TM_S + t * 128 + (j & 1) * 64, smem_desc_sw128(q_at + cb * Q_BLOCK) + (uint64_t)(k * 2),
                                   smem_desc_sw128(k_at + cb * KV_BLOCK) + (uint64_t)(k * 2), idesc_s, (cb > 0 || k > 0) ? 1u : 0u);
                    tc_commit(s_full + 16 * t + 8 * (j & 1));
                    tc_commit(k_empty + 8 * (i % KS));
                }
                __syncwarp();
            };
            auto keys = [&](int j) {
                const int i = i_first + i_step * j;
                return mbar_wait_warp(k_full + 8 * (i % KS), (i / KS) & 1, status, 70);
            };
            auto pass = [&](uint32_t bar) { if (lane == 0) mbar_arrive(bar); };    // a page that this tile does not look at
            bool ok = mine > 0;
            if (ok) {
                ok = mbar_wait_warp(q_full + 8 * q_tile, 0, status, 70);
                for (int j = 0; j < 2 && j < all && ok; ++j) {                     // the scores' places
                    ok = keys(j);
                    if (!ok) break;
                    tc_fence_after();
                    if (j < mine) scores(j);
                    else pass(k_empty + 8 * (j % KS));
                }
                for (int j = 0; j < all && ok; ++j) {
                    const int nxt = j + 2, i = i_first + i_step * j;
                    // (the ring holds three pages: the keys of a split tile's page after the next come when this one's values are done with)
                    ok = !*(volatile int*)&s_abort && mbar_wait_warp(v_full + 8 * (i % VS), (i / VS) & 1, status, 70) &&
                         (SPLIT || nxt >= all || keys(nxt));
                    if (!ok) break;
                    if (j < mine) {
                        ok = __all_sync(0xffffffffu, mbar_wait(p_ready + 16 * t + 8 * (j & 1), (j >> 1) & 1, status, 70));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t v_at = v_smem + (i % VS) * KV_BYTES, p_tm = tmem_u + TM_S + t * 128 + (j & 1) * 64;
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < BKV / 16; ++k)                     // 16 keys a step
                                mma_ts(tmem_u + TM_O + t * HD, p_tm + k * 8, smem_desc_sw128_mn(v_at + k * 2048), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
                            tc_commit(pv_full + 16 * t + 8 * (j & 1));
                            tc_commit(v_empty + 8 * (i % VS));
                        }
                        __syncwarp();
                    } else {
                        pass(v_empty + 8 * (i % VS));
                    }
                    if (SPLIT && nxt < all) {
                        ok = keys(nxt);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    // P(j) lies in the place of S(j + 2): the MMAs of one thread run in their order
                    if (nxt < mine) scores(nxt);
                    else if (nxt < all) pass(k_empty + 8 * (nxt % KS));
                }
                if (!ok) {                                                         // what was issued lands before the memory is given back
                    s_abort = 1;
                    if (elect_one()) tc_commit(done + 8 * t);
                    __syncwarp();
                    mbar_wait_warp(done + 8 * t, 0, nullptr, 0);
                }
            }
        } else if (warp == 13 && lane == 0) {
            // ---------------------------------------------------------- pages, as they are
            int issued = 0;
            for (int i = 0; i < n_pages; ++i) {
                const int rs = i % RS;
                const size_t at = ((size_t)PLM_PAGE_NO(sq.pages[page_at(i)]) * G + g) * RAW_BYTES;
                if (*(volatile int*)&s_abort) break;
                if (!mbar_wait(raw_empty + 8 * rs, ((i / RS) & 1) ^ 1, status, 73)) { s_abort = 1; break; }
#ifdef PLM_TEST_STALL
                mbar_expect_tx(raw_full + 8 * rs, 2 * RAW_BYTES + (plm_stall ? 64 : 0));
#else
                mbar_expect_tx(raw_full + 8 * rs, 2 * RAW_BYTES);
#endif
                bulk_load(raw + rs * 2 * RAW_BYTES, cache.k + at, RAW_BYTES, raw_full + 8 * rs);
                bulk_load(raw + rs * 2 * RAW_BYTES + RAW_BYTES, cache.v + at, RAW_BYTES, raw_full + 8 * rs);
                issued = i + 1;
            }
            for (int i = max(0, issued - RS); i < issued; ++i) mbar_wait(raw_full + 8 * (i % RS), (i / RS) & 1, nullptr, 0);      // all have landed
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

}  // namespace

// q [T, H, HD] bf16, caches [pages, G, 64, HD] e4m3 with scales [pages, G], out [T, H * HD] bf16.  seq_start [n_seqs + 1]: offsets of each
// sequence's new tokens, at most max_new; seq_kv_len [n_seqs]: its length after the step.  `status`: a device int that stays 0 unless a
// bounded wait ran out.
extern "C" int plm_kv8_attention_tc(const void* q, const void* kc, const void* vc, const float* ks, const float* vs, void* out,
                                    const int* seq_start, const int* seq_kv_len, const int* block_table, int max_pages, int n_seqs,
                                    int max_new, int H, int G, float scale, int window, int* status, const float* sink, int keep,
                                    const float* slopes, cudaStream_t stream) {
    if (n_seqs <= 0 || max_new <= 0) return PLM_OK;
    if (H <= 0 || G <= 0 || H % G || n_seqs > 65535 || G > 65535 || keep < 0 || !status) return PLM_ERR_SHAPE;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)out) & 15) return PLM_ERR_ALIGN;
    const bool more = keep > 0 || slopes;
    const Kv8Step step = {nullptr, nullptr, seq_start, seq_kv_len, block_table, max_pages};
    const Cache cache = {(const uint8_t*)kc, (const uint8_t*)vc, ks, vs};
    const long rows = (long)max_new * (H / G), halves_of = (rows + BQ - 1) / BQ;
    const bool split = rows <= BQ || halves_of * G * n_seqs <= PLM_SM_COUNT;      // (see the kernel)
    const dim3 grid((unsigned)(split ? halves_of : (halves_of + 1) / 2), G, n_seqs);
    auto launch = [&](auto kernel, std::atomic<unsigned long long>& devices) {
        cudaError_t e = plm_allow_smem(kernel, SMEM, devices);
        if (e != cudaSuccess) return (int)e;
        return plm_status_of(launch_pdl(kernel, grid, dim3(NT), SMEM, stream, (const bf16*)q, cache, (bf16*)out, step, H, G, scale * LOG2E, window, status,
                                        sink, keep, slopes));
    };
    static std::atomic<unsigned long long> devices[4];
    if (more) return split ? launch(kv8_tc_kernel<true, true>, devices[0]) : launch(kv8_tc_kernel<true, false>, devices[1]);
    return split ? launch(kv8_tc_kernel<false, true>, devices[2]) : launch(kv8_tc_kernel<false, false>, devices[3]);
}

#ifdef PLM_TEST_STALL
extern "C" int plm_test_stall(int on, cudaStream_t stream) {
    return (int)cudaMemcpyToSymbolAsync(plm_stall, &on, sizeof(on), 0, cudaMemcpyHostToDevice, stream);
}
#endif
