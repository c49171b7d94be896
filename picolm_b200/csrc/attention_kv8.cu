// Attention of bfloat16 queries over the 8-bit cache (kv8.cuh) on the tensor cores (mma.sync m16n8k16, fp16 operands, fp32
// sums), compiled for one head size: -DPLM_HD=<head_dim>, a multiple of 16 up to 256.
//
// For a query at position p, head h, kv head g = h / (H / G), with the page of key t in page(t):
//   s_t = scale * ks[page(t), g] * (q . k8_t) [- slope (p - t)],   out = sum_t softmax(s)_t vs[page(t), g] v8_t
// over lo <= t <= p (or t < keep).  Every e4m3 number is a half; a query row becomes halves after a division by a power of two
// that puts its largest number into [2^13, 2^14) (then halves hold every bit of what was within 2^27 of it); the scales, being
// powers of two, stay outside the products: ks joins the factor on the scores, and the sum over values is kept in the unit
// 2^eo of some page's vs: a page in another unit either has its weights multiplied by the ratio or, where that is beyond 2^KV8_SPAN,
// changes the unit (a factor on the sums, exact).
//
// Two kernels:
//   kv8_stream_kernel  few (token, head) rows a sequence and kv head, above all single tokens: bound by the cache's bytes.  A warp
//                      walks keys on its own, 16 or 32 at a time, through a ring of its own in shared memory (cp.async; no
//                      barrier but the warp's).  The keys are on the MMA's 16 rows and the
//                      (token, head) rows on its 8 columns, so that a group of four or eight heads does not leave half of the
//                      MMA empty: S^T = K Q^T, and out^T = V^T P^T, whose A operand takes pairs of keys a component; a
//                      byte permutation and a conversion make it of four rows of V.  The 8 columns of S^T become the
//                      B operand by movmatrix.  Four warps' partial results meet in shared memory; CTAs' in their cluster's,
//                      or (few walks of long contexts) through a workspace and a second kernel, all keys of a step being
//                      dealt out evenly over one wave of CTAs.
//                      Measured, 32 heads over 8 (us, of the copy rate): 8 tokens behind 32,768 keys of 128 72, 0.79; 64 behind
//                      4,096 of 64 37, 0.69; one behind 2,001 of 64 6.0 (a launch that reads almost nothing takes 4.5).
//                      The cache in 16 bits takes 126, 60 and 6.  What a step waits for beside its bytes: in clusters the
//                      CTAs' starts and meetings, some 1 us of an SM each, dealt out the second kernel, some 6 us with its
//                      start.  16 keys cost a warp 228 instructions.
//   kv8_tile_kernel    longer prompts of head sizes that the tcgen05 kernel does not take: 64 rows a CTA, pages of 64 keys brought to
//                      shared memory as halves.  Measured, 32 heads over 8 (us): a prompt of 1,000 of 80 66 (0.05 of the bf16 rate), of
//                      96 83, of 112 88, of 256 159; 500 behind 7,500 374, 342, 364, 893.  The legacy MMAs, and a page that every
//                      CTA widens for its 64 rows, are what takes it.
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
constexpr int WARPS = 4, NT = 128;
constexpr float LIFT = KV8_LIFT, RAISE = KV8_RAISE;

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
// A value's row in the eight lanes (n = lane / 4) that share it: bytes 2 m and 2 m + 1 of a lane are its components of the
// m-th tile: rows n and n + 8 of the MMA.
__device__ __forceinline__ int value_component(int m, int n) {
    constexpr int A = HD / 128, B = (HD / 64) & 1, C = (HD / 32) & 1;
    if (m < 8 * A) return m / 8 * 128 + n * 16 + m % 8 * 2;
    if (B && m < 8 * A + 4) return 128 * A + n * 8 + (m - 8 * A) * 2;
    if (C && m < 8 * A + 4 * B + 2) return 128 * A + 64 * B + n * 4 + (m - 8 * A - 4 * B) * 2;
    return 128 * A + 64 * B + 32 * C + n * 2;
}
// Rows as they lie in shared memory: 16-byte chunk j of row r.  For heads of 64 and of multiples of 128 the chunks of a 128-byte line
// change places by the row, so that the lanes of the loads below (rows n for keys, 2 c for values) find 32 banks.
__device__ __forceinline__ uint32_t key_chunk(int r, int j) {
    if constexpr (HD == 64) return (r >> 1) * 128 + ((((r & 1) * 4 + j) ^ (((r >> 1) & 3) * 2)) << 4);
    else if constexpr (HD % 128 == 0) return r * HD + (j >> 3) * 128 + (((j & 7) ^ ((r & 1) * 4)) << 4);
    else return r * HD + j * 16;
}
__device__ __forceinline__ uint32_t value_chunk(int r, int j) {
    if constexpr (HD == 64) return key_chunk(r, j);
    else if constexpr (HD % 128 == 0) return r * HD + (j >> 3) * 128 + (((j & 7) ^ (((r >> 1) & 3) * 2)) << 4);
    else return r * HD + j * 16;
}
// The same as a lane's place and constants: chunk 32 x + lane of a tile lies at key_place / value_place of `at` = the chunk
// function of chunk `lane`.  (Eight rows further on the places are the same, and 32 chunks are 8, 4 or 2 rows.)
__device__ __forceinline__ uint32_t key_place(uint32_t at, int x) { return at + x * 512; }
__device__ __forceinline__ uint32_t value_place(uint32_t at, int x) {
    return (HD == 128 ? at ^ ((x & 1) * 64) : HD == 256 ? at ^ ((x & 3) * 32) : at) + x * 512;
}
template <typename T> __device__ __forceinline__ T lds(uint32_t at) {
    T v;
    if constexpr (sizeof(T) == 16)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    else if constexpr (sizeof(T) == 8)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
// Row n of eight at shared-memory address `rows`; at = key_chunk(n, c).  (The places of row n + 8 i are 8 HD i further on.)
__device__ __forceinline__ void load_key(uint32_t (&w)[KS], uint32_t rows, uint32_t at, int n, int c) {
    constexpr int A = HD / 64, B = (HD / 32) & 1, C = (HD / 16) & 1;
#pragma unroll
    for (int i = 0; i < A; ++i) {
        const uint4 v = lds<uint4>(rows + (HD % 128 == 0 ? (at ^ ((i & 1) * 64)) + (i >> 1) * 128 : at + i * 64));
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
    if (B) {
        const uint2 v = lds<uint2>(rows + n * HD + 64 * A + c * 8);
        w[4 * A] = v.x; w[4 * A + B] = v.y;
    }
    if (C) w[KS - 1] = lds<uint32_t>(rows + n * HD + 64 * A + 32 * B + c * 4);
}
// Row 2 c + e of eight; at = where row 2 c's first bytes of this lane lie.
__device__ __forceinline__ uint32_t value_at(int n, int c) {
    if constexpr (HD == 64) return value_chunk(2 * c, n >> 1) + (n & 1) * 8;
    else if constexpr (HD >= 128) return value_chunk(2 * c, n);
    else return 2 * c * HD + (HD >= 64 ? n * 8 : 0);
}
__device__ __forceinline__ void load_value(uint32_t (&w)[VW], uint32_t rows, uint32_t at, int n, int c, int e) {
    constexpr int A = HD / 128, B = (HD / 64) & 1, C = (HD / 32) & 1, D = (HD / 16) & 1;
#pragma unroll
    for (int i = 0; i < A; ++i) {
        const uint4 v = lds<uint4>(rows + at + e * HD + i * 128);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
    const uint32_t row = rows + (2 * c + e) * HD + 128 * A;
    if (B) {
        const uint2 v = lds<uint2>(HD == 64 ? rows + (at ^ (e * 64)) : HD < 128 ? rows + at + e * HD : row + n * 8);
        w[4 * A] = v.x; w[4 * A + B] = v.y;
    }
    if (C) w[4 * A + 2 * B] = lds<uint32_t>(row + 64 * B + n * 4);
    if (D) {                                         // two bytes; the load takes the four that they lie in
        const uint32_t v = lds<uint32_t>(row + 64 * B + 32 * C + (n & ~1) * 2);
        w[VW - 1] = n & 1 ? v >> 16 : v & 0xffffu;
    }
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
constexpr int MAX_CTAS = 6 * PLM_SM_COUNT;       // (a float a warp fits the second kernel's shared memory)
constexpr int ROW = HD + 2;                      // floats of a partial result's row: sums, maximum, denominator
constexpr int SM_SMEM = 228 * 1024;              // shared memory of an SM
// (CTAS, an SM: what registers allow, and shared memory by one unit less in the ring where it must, in both forms of the kernel: heads of
// 112 with three CTAs of two units / two of three 57 / 64 us for 64 sequences of 4,096; two rows' groups of 32 of heads of 128 and of 16 of 240
// share an SM since a CTA's sums lie over its first warp's: 8 sequences of 8,192 keys with 32 rows 39 -> 31, with 16 of 240 46 -> 38.)
template <int NG> struct Few {
    enum : int {
        SB = HD * NG <= 256 && HD <= 128 ? 2 : 1,                    // blocks of 16 keys at a time
        KB = 16 * SB,
        TILE = KB * HD,                                              // bytes of KB keys
        CTAS = NG == 1 ? (HD <= 64 ? 4 : HD <= 128 ? 3 : 2) : NG == 2 && HD <= 64 ? 3 : 2,      // an SM
        Q_BYTES = NG > 1 ? WARPS * NG * KS * 32 * 8 : 0,             // the queries' fragments (of one group: in registers)
        AFTER = (WARPS * ROW + 2) * 8 * NG * 4,                      // the warps' results; what a CTA shows to its cluster: in the first's place
        SLACK = 1024 + 128,                                          // a CTA's beside: the system's, what the kernel declares itself
        MOST = SM_SMEM / CTAS - SLACK - Q_BYTES,                     // of a CTA for its ring
        WANTED = TILE >= 4096 ? 2 : TILE >= 2048 ? 3 : 4,
        STAGES = WARPS * WANTED * 2 * TILE <= MOST ? WANTED : WANTED - 1,                       // units a warp has in its ring
        RING = WARPS * STAGES * 2 * TILE,
        SMEM = Q_BYTES + (RING > AFTER ? (int)RING : (int)AFTER),
    };
    static_assert(STAGES >= 2 && CTAS * (SMEM + SLACK) <= SM_SMEM, "as many CTAs an SM as the work is dealt out to");
};

// The rows of one sequence and kv head, COLS at a time, against its keys: how the work is dealt out.  A sequence's walk is one of
// units of KB keys, the same for all its tiles of rows and kv heads; all walks of the step in a row (sequence by sequence, and
// there (kv head, tile) by (kv head, tile)) are cut into one equal range for each warp.  So a ragged batch keeps all SMs busy to the
// end; a warp meets at most two walks that are not wholly its own, and leaves partial results for those.
constexpr int MIN_UNITS = 4;                     // of a warp's range, so that its start and a partial result are worth it
template <int COLS, int KB> struct Deal {
    const Kv8Step& step;
    int n_seqs, G, R, window, keep, most;         // (most: tiles of a sequence that the launch knows of)
    __device__ __forceinline__ void of(int b, int& units, int& tiles) const {
        const Kv8Seq q = kv8_seq(step, b);
        units = tiles = 0;
        if (q.n_new <= 0) return;
        const int last = q.pos0 + q.n_new - 1;
        const Walk w(q.pos0, last, window, keep);
        units = w.n_pages * (PLM_PAGE / KB) - (PLM_PAGE - 1 - last % PLM_PAGE) / KB;
        tiles = min(most, (q.n_new * R + COLS - 1) / COLS);
    }
    __device__ __forceinline__ unsigned long long all(int b) const {
        int u, t;
        of(b, u, t);
        return (unsigned long long)u * t * G;
    }
    // A whole warp, number `w` of n_warps: its units of all, and the sequence that the first belongs to with the units before that.
    __device__ __forceinline__ bool range(int w, int n_warps, unsigned long long& per, unsigned long long& at, unsigned long long& end, int& b,
                                          unsigned long long& before) const {
        constexpr int HOLD = 4;                                      // 128 sequences are asked for once
        const int lane = threadIdx.x & 31;
        unsigned long long held[HOLD], total = 0;
#pragma unroll
        for (int i = 0; i < HOLD; ++i) total += held[i] = i * 32 + lane < n_seqs ? all(i * 32 + lane) : 0;
        for (int i = HOLD * 32 + lane; i < n_seqs; i += 32) total += all(i);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        per = (total + n_warps - 1) / n_warps;
        per = per < MIN_UNITS ? MIN_UNITS : per;
        at = per * w;
        end = at + per < total ? at + per : total;
        if (at >= end) return false;
        before = 0;
        for (int i0 = 0; i0 < n_seqs; i0 += 32) {
            const unsigned long long mine = i0 == 0 ? held[0] : i0 == 32 ? held[1] : i0 == 64 ? held[2] : i0 == 96 ? held[3]
                                                                                                          : i0 + lane < n_seqs ? all(i0 + lane) : 0;
            unsigned long long sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            const unsigned here = __ballot_sync(0xffffffffu, before + sum > at);
            if (here) {
                const int f = __ffs(here) - 1;
                before += __shfl_sync(0xffffffffu, sum - mine, f);
                b = i0 + f;
                return true;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        return false;
    }
};

// NG groups of 8 (token, head) rows a warp.  CLUSTER: grid (ranges, G * tiles, sequences), the ranges of a walk are the CTAs of a
// cluster.  Else: any number of warps, see Deal; `ws` holds two partial results a warp: [0] of a walk that an earlier warp began,
// [1] of one that a later warp ends, each [COLS][ROW], and `pieces` [n_seqs * G * tiles] which warp began each walk and how many
// have a piece of it.
template <int NG, bool CLUSTER>
__global__ void __launch_bounds__(NT, Few<NG>::CTAS)
kv8_stream_kernel(const bf16* q, const Cache cache, bf16* __restrict__ out, float* __restrict__ ws, int2* __restrict__ pieces, const Kv8Step step,
                  int n_seqs, int H, int G, int tiles, float scale_log2, int window, const float* sink, int keep, const float* slopes) {
    constexpr int COLS = 8 * NG, SB = Few<NG>::SB, KB = Few<NG>::KB, TILE = Few<NG>::TILE, STAGES = Few<NG>::STAGES;
    constexpr unsigned UNITS = PLM_PAGE / KB;
    extern __shared__ __align__(128) uint8_t sm_raw[];                             // [WARPS][NG][KS][32] queries, [WARPS][STAGES][keys, values]
    __shared__ float scales[WARPS][STAGES][2];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n8 = lane >> 2, c4 = lane & 3;
    const int R = H / G;
    uint2* q_frag = reinterpret_cast<uint2*>(sm_raw) + (NG > 1 ? warp * NG * KS * 32 : 0);
    const uint32_t ring = smem_u32(sm_raw + Few<NG>::Q_BYTES) + warp * STAGES * 2 * TILE, scales_s = smem_u32(&scales[warp][0][0]);
    const uint32_t key_to = key_chunk(lane / (HD / 16), lane % (HD / 16)), value_to = value_chunk(lane / (HD / 16), lane % (HD / 16));
    const uint32_t key_from = key_chunk(n8, c4), value_from = value_at(n8, c4);

    // A warp's piece: units u0, u0 + stride, .. below u1 of the walk of rows pair0 .. of sequence sq and kv head g.  finish(o, m, l): the sums
    // out^T in units of 1, maximum and denominator of this lane's rows 8 j + 2 c4 and + 1.
    auto piece = [&](const Kv8Seq& sq, int g, int tile, int u0, int u1, int stride, auto&& finish) {
        const int pair0 = tile * COLS, n_pairs = sq.n_new * R;
        const int n_cols = min(COLS, n_pairs - pair0);
        const int pos_first = sq.pos0 + pair0 / R, pos_last = sq.pos0 + (pair0 + n_cols - 1) / R;
        const int lo_first = plm_first_key(pos_first, window), lo_last = plm_first_key(pos_last, window);
        const Walk walk(sq.pos0, sq.pos0 + sq.n_new - 1, window, keep);

        // The ring's first units are asked for before the queries are looked at.  A unit's keys and values are groups of their own, each
        // asked for as soon as its place is free.
        auto number = [&](unsigned u) { return PLM_PAGE_NO(sq.pages[walk.page_at((int)(u / UNITS))]); };
        auto offset = [&](unsigned u, unsigned block) { return (size_t)block * (PLM_PAGE * HD) + u % UNITS * TILE; };
        constexpr int CHUNKS = TILE / 16;
        auto ask_keys = [&](unsigned u, unsigned block, int stage) {
            const uint8_t* from = cache.k + offset(u, block) + lane * 16;
            const uint32_t to = ring + stage * (2 * TILE);
#pragma unroll
            for (int x = 0; x < CHUNKS; x += 32)
                if (CHUNKS % 32 == 0 || x + lane < CHUNKS) cp_async16(to + key_place(key_to, x / 32), from + x * 16);
            if (lane < 2) cp_async4(scales_s + (stage * 2 + lane) * 4, (lane ? cache.vs : cache.ks) + block);
        };
        auto ask_values = [&](unsigned u, unsigned block, int stage) {
            const uint8_t* from = cache.v + offset(u, block) + lane * 16;
            const uint32_t to = ring + stage * (2 * TILE) + TILE;
#pragma unroll
            for (int x = 0; x < CHUNKS; x += 32)
                if (CHUNKS % 32 == 0 || x + lane < CHUNKS) cp_async16(to + value_place(value_to, x / 32), from + x * 16);
        };
        unsigned block = 0;                                          // page and kv head of the unit asked for last
        int page_next = 0;                                           // page of the one after it
#pragma unroll
        for (int i = 0; i < STAGES; ++i) {
            if (u0 + i * stride < u1) {
                block = (unsigned)number(u0 + i * stride) * G + g;
                ask_keys(u0 + i * stride, block, i);
                cp_commit();
                ask_values(u0 + i * stride, block, i);
                cp_commit();
            } else {
                cp_commit();
                cp_commit();
            }
        }
        if (u0 + STAGES * stride < u1) page_next = number(u0 + STAGES * stride);

        // The queries as B operands, a group of 8 rows at a time: this lane has row n8's components key_component(w, c4) .. + 3.
        float m[NG][2], l[NG][2], cs[NG][2];
        uint2 qr[NG == 1 ? KS : 1];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const int pair = pair0 + j * 8 + n8;
            const bool have = pair < n_pairs;
            const bf16* row = q + ((size_t)(sq.t0 + (have ? pair / R : 0)) * H + g * R + (have ? pair % R : 0)) * HD;
            uint2 w[KS];
            float most = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s) w[s] = have ? *reinterpret_cast<const uint2*>(row + key_component(s, c4)) : make_uint2(0, 0);
#pragma unroll
            for (int s = 0; s < KS; ++s)
                most = fmaxf(fmaxf(fmaxf(kv8_magnitude(__uint_as_float(w[s].x << 16)), kv8_magnitude(__uint_as_float(w[s].x & 0xffff0000u))),
                                   fmaxf(kv8_magnitude(__uint_as_float(w[s].y << 16)), kv8_magnitude(__uint_as_float(w[s].y & 0xffff0000u)))), most);
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int e = row_exponent(most);
            const float down = kv8_pow2(-e);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint2 f = make_uint2(halves(__uint_as_float(w[s].x << 16) * down, __uint_as_float(w[s].x & 0xffff0000u) * down),
                                           halves(__uint_as_float(w[s].y << 16) * down, __uint_as_float(w[s].y & 0xffff0000u) * down));
                if (NG == 1) qr[NG == 1 ? s : 0] = f;
                else q_frag[(j * KS + s) * 32 + lane] = f;           // (its reader is this lane)
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                m[j][k] = -INFINITY;
                l[j][k] = 0.f;
                cs[j][k] = scale_log2 * kv8_pow2(max(-126, min(127, __shfl_sync(0xffffffffu, e, (c4 * 2 + k) * 4))));
            }
        }
        float o[NG][MT][4];
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) o[j][t][0] = o[j][t][1] = o[j][t][2] = o[j][t][3] = 0.f;
        int eo = 0, stage = 0;
        bool nan_found = false;
        for (int u = u0; u < u1; u += stride) {
            const uint32_t tile = ring + stage * (2 * TILE);
            const int key0 = walk.page_at((int)((unsigned)u / UNITS)) * PLM_PAGE + (int)((unsigned)u % UNITS) * KB;
            const bool edge = key0 + KB - 1 > pos_first || key0 < lo_last;
            float s[SB][NG][4];
#pragma unroll
            for (int b = 0; b < SB; ++b)
#pragma unroll
                for (int j = 0; j < NG; ++j) s[b][j][0] = s[b][j][1] = s[b][j][2] = s[b][j][3] = 0.f;
            cp_wait<2 * STAGES - 1>();                               // this unit's keys are there
            __syncwarp();
            const float ks_now = kv8_scale(scales[warp][stage][0]);
            const int ev = kv8_exponent_of_scale(kv8_scale(scales[warp][stage][1]));
            uint32_t kw[SB][2][KS];
#pragma unroll
            for (int b = 0; b < SB; ++b) {
                load_key(kw[b][0], tile + b * 16 * HD, key_from, n8, c4);
                load_key(kw[b][1], tile + (b * 16 + 8) * HD, key_from, n8, c4);
            }
#pragma unroll
            for (int w = 0; w < KS; ++w) {
                uint32_t a[SB][4];
#pragma unroll
                for (int b = 0; b < SB; ++b) {
                    kv8_halves(kw[b][0][w], a[b][0], a[b][2]);
                    kv8_halves(kw[b][1][w], a[b][1], a[b][3]);
                }
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const uint2 f = NG == 1 ? qr[NG == 1 ? w : 0] : q_frag[(j * KS + w) * 32 + lane];
#pragma unroll
                    for (int b = 0; b < SB; ++b) mma_f16(s[b][j], a[b], f.x, f.y);
                }
            }
            __syncwarp();                                            // its place is free
            const bool more = u + STAGES * stride < u1;
            if (more) {
                block = (unsigned)page_next * G + g;
                ask_keys(u + STAGES * stride, block, stage);
                page_next = number(min(u + (STAGES + 1) * stride, u1 - 1));
            }
            cp_commit();
            // scores in log2 units are s * c (with slopes and masks they are made here, and c is 1)
            float c[NG][2], mx[NG][2];
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) c[j][e] = cs[j][e] * ks_now;
            if (edge || slopes) {
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int pair = pair0 + j * 8 + c4 * 2 + e;
                        const int pos = pair < n_pairs ? sq.pos0 + pair / R : -1, lo = plm_first_key(pos, window);
                        const float slope = slopes && pair < n_pairs ? slopes[g * R + pair % R] * LOG2E : 0.f;
#pragma unroll
                        for (int b = 0; b < SB; ++b)
#pragma unroll
                            for (int hi = 0; hi < 2; ++hi) {
                                const int key = key0 + b * 16 + n8 + hi * 8;
                                const float x = fmaf(slope, (float)(key - pos), s[b][j][2 * hi + e] * c[j][e]);
                                s[b][j][2 * hi + e] = key > pos || (key < lo && key >= keep) ? -INFINITY : x;
                            }
                        c[j][e] = 1.f;
                    }
            }
            bool raise = false;
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = fmaxf(s[0][j][e], s[0][j][2 + e]);
                    if (SB == 2) x = fmaxf(x, fmaxf(s[SB - 1][j][e], s[SB - 1][j][2 + e]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    mx[j][e] = x * c[j][e] - LIFT;                   // (c is positive)
                    raise |= mx[j][e] > (m[j][e] == -INFINITY ? -INFINITY : m[j][e] + RAISE);
                }
            int d = ev - eo;
            if (__any_sync(0xffffffffu, raise || d > KV8_SPAN || d < -KV8_SPAN)) {
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float down[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool up = mx[j][e] > m[j][e];
                        const float by = up ? m[j][e] - mx[j][e] : 0.f;            // -inf where nothing was seen before
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
                float sum[2] = {0.f, 0.f}, off[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) off[e] = (float)d - (m[j][e] == -INFINITY ? 0.f : m[j][e]);
#pragma unroll
                for (int b = 0; b < SB; ++b) {
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[i] = ex2(fmaf(s[b][j][i], c[j][i & 1], off[i & 1]));
                        sum[i & 1] += p[i];
                    }
                    pf[b][j][0] = turned(halves(p[0], p[1]));
                    pf[b][j][1] = turned(halves(p[2], p[3]));
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) l[j][e] = fmaf(sum[e], back, l[j][e]);
            }
            cp_wait<2 * STAGES - 1>();                               // its values are there
            __syncwarp();
            uint32_t vw[SB][4][VW];
#pragma unroll
            for (int b = 0; b < SB; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) load_value(vw[b][k], tile + TILE + (b * 16 + (k >> 1) * 8) * HD, value_from, n8, c4, k & 1);
            if (edge) {
                // Places that no row sees hold whatever was left there: zeros.  A NaN that some rows see and others do not would
                // reach them all (0 * NaN): it is taken out, and put into the results of those that see it at the end.
#pragma unroll
                for (int b = 0; b < SB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + b * 16 + 2 * c4 + (i & 1) + (i >> 1) * 8;
                        const bool seen = key <= pos_last && (key >= lo_first || key < keep);
#pragma unroll
                        for (int w = 0; w < VW; ++w) {
                            const uint32_t marks = nan_bytes(vw[b][i][w]);
                            nan_found |= seen && marks;
                            vw[b][i][w] = seen ? without(vw[b][i][w], marks) : 0u;
                        }
                    }
            }
#pragma unroll
            for (int b = 0; b < SB; ++b)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const uint32_t order = t & 1 ? 0x7362u : 0x5140u;
                    const uint32_t x = __byte_perm(vw[b][0][t / 2], vw[b][1][t / 2], order);
                    const uint32_t y = __byte_perm(vw[b][2][t / 2], vw[b][3][t / 2], order);
                    uint32_t a[4];
                    kv8_halves(x, a[0], a[1]);
                    kv8_halves(y, a[2], a[3]);
#pragma unroll
                    for (int j = 0; j < NG; ++j) mma_f16(o[j][t], a, pf[b][j][0], pf[b][j][1]);
                }
            __syncwarp();
            if (more) ask_values(u + STAGES * stride, block, stage);
            cp_commit();
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        const float unit = kv8_pow2(max(-126, min(127, eo)));
#pragma unroll
        for (int j = 0; j < NG; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 4);
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 8);
                l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 16);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][t][e] *= unit;
        }
        if (__any_sync(0xffffffffu, nan_found)) {                    // the piece's edge units once more
            for (int u = u0; u < u1; u += stride) {
                const int key0 = walk.page_at((int)((unsigned)u / UNITS)) * PLM_PAGE + (int)((unsigned)u % UNITS) * KB;
                if (!(key0 + KB - 1 > pos_first || key0 < lo_last)) continue;
                const uint8_t* at = cache.v + offset(u, (unsigned)number(u) * G + g);
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        const uint8_t* v = at + (size_t)k * HD + value_component(t, n8);
                        const bool n0 = is_nan_byte(v[0]), n1 = is_nan_byte(v[1]);
                        if (!(n0 || n1)) continue;
#pragma unroll
                        for (int j = 0; j < NG; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int pair = pair0 + j * 8 + c4 * 2 + e, p = sq.pos0 + pair / R, lo = plm_first_key(p, window);
                                if (pair >= n_pairs || key0 + k > p || (key0 + k < lo && key0 + k >= keep)) continue;
                                if (n0) o[j][t][e] = __int_as_float(0x7fffffff);
                                if (n1) o[j][t][2 + e] = __int_as_float(0x7fffffff);
                            }
                    }
            }
        }
        finish(o, m, l);
    };
    // a lane's part of a row [ROW]: sums, maximum, denominator
    auto put = [&](float* row, const float (&o)[MT][4], int e, float m, float l) {
#pragma unroll
        for (int t = 0; t < MT; ++t) *reinterpret_cast<float2*>(row + value_component(t, n8)) = make_float2(o[t][e], o[t][2 + e]);
        if (n8 == 0) *reinterpret_cast<float2*>(row + HD) = make_float2(kv8_top(m, l), l);
    };

    const Deal<COLS, KB> deal = {step, n_seqs, G, R, window, keep, tiles};
    if constexpr (CLUSTER) {
        float* part = reinterpret_cast<float*>(sm_raw + Few<NG>::Q_BYTES);         // after the walk, in the rings' place: [WARPS][COLS][ROW]
        float* mine = part;                                                        // [COLS][ROW], each number where the one thread that needs it
        float* tops = part + WARPS * COLS * ROW;                                   // had the first warp's; [COLS][2] maximum and denominator
        const int g = blockIdx.y / tiles, tile = blockIdx.y - g * tiles, n_splits = gridDim.x, rank = blockIdx.x;
        const Kv8Seq sq = kv8_seq(step, blockIdx.z);
        int units, n_tiles;
        deal.of(blockIdx.z, units, n_tiles);
        if (tile >= n_tiles) return;                                               // (with all CTAs of its cluster)
        const int per = (units + n_splits - 1) / n_splits;
        const int pair0 = tile * COLS, n_cols = min(COLS, sq.n_new * R - pair0);
        piece(sq, g, tile, min(units, rank * per) + warp, min(units, (rank + 1) * per), WARPS, [&](auto& o, auto& m, auto& l) {
            __syncthreads();                                                       // all rings are free
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (j * 8 + c4 * 2 + e < n_cols) put(part + (size_t)(warp * COLS + j * 8 + c4 * 2 + e) * ROW, o[j], e, m[j][e], l[j][e]);
        });
        __syncthreads();
        for (int i = threadIdx.x; i < n_cols * HD; i += NT) {
            const int col = i / HD, d = i - col * HD;
            float mw[WARPS], mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                mw[w] = part[((size_t)w * COLS + col) * ROW + HD];
                mm = fmaxf(mm, mw[w]);
            }
            float acc = 0.f, ll = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float wgt = mw[w] == -INFINITY ? 0.f : exp2f(mw[w] - mm);
                acc = fmaf(wgt, part[((size_t)w * COLS + col) * ROW + d], acc);
                ll = fmaf(wgt, part[((size_t)w * COLS + col) * ROW + HD + 1], ll);
            }
            if (n_splits == 1) {                                                   // nobody to meet
                const int pair = pair0 + col, h = g * R + pair % R;
                out[((size_t)(sq.t0 + pair / R) * H + h) * HD + d] = __float2bfloat16_rn(acc * kv8_inverse(mm, ll, sink ? sink + h : nullptr));
                continue;
            }
            mine[col * ROW + d] = acc;
            if (d == 0) { tops[col * 2] = mm; tops[col * 2 + 1] = ll; }
        }
        if (n_splits == 1) return;
        cluster_sync_all();
        for (int i = rank * NT + threadIdx.x; i < n_cols * HD; i += n_splits * NT) {
            const int col = i / HD, d = i - col * HD, pair = pair0 + col;
            float ms[MAX_CLUSTER], ls[MAX_CLUSTER], as[MAX_CLUSTER], mm = -INFINITY;
#pragma unroll
            for (int s = 0; s < MAX_CLUSTER; ++s) {
                ms[s] = -INFINITY; ls[s] = 0.f; as[s] = 0.f;
                if (s < n_splits) {
                    const uint32_t top = cluster_map(tops + col * 2, (uint32_t)s);
                    ms[s] = cluster_ld_f32(top);
                    ls[s] = cluster_ld_f32(top + 4);
                    as[s] = cluster_ld_f32(cluster_map(mine + col * ROW + d, (uint32_t)s));
                }
                mm = fmaxf(mm, ms[s]);
            }
            float acc = 0.f, ll = 0.f;
#pragma unroll
            for (int s = 0; s < MAX_CLUSTER; ++s) {
                const float wgt = ms[s] == -INFINITY ? 0.f : exp2f(ms[s] - mm);    // (its sum is zero, or NaN where a value is)
                acc = fmaf(wgt, as[s], acc);
                ll = fmaf(wgt, ls[s], ll);
            }
            const int h = g * R + pair % R;
            out[((size_t)(sq.t0 + pair / R) * H + h) * HD + d] = __float2bfloat16_rn(acc * kv8_inverse(mm, ll, sink ? sink + h : nullptr));
        }
        cluster_sync_all();                                          // nobody reads this CTA's shared memory any more
    } else {
        const int w = blockIdx.x * WARPS + warp;
        unsigned long long per, at, end, before;
        int b, units, n_tiles;
        if (!deal.range(w, gridDim.x * WARPS, per, at, end, b, before)) return;
        deal.of(b, units, n_tiles);
        unsigned rest = (unsigned)((at - before) / units);           // (kv head, tile) within the sequence
        int u0 = (int)(at - before - (unsigned long long)rest * units);
        while (true) {
            const int u1 = (int)min((unsigned long long)units, u0 + (end - at));
            const int g = (int)rest / n_tiles, tile = (int)rest - g * n_tiles, pair0 = tile * COLS;
            const Kv8Seq sq = kv8_seq(step, b);
            const int n_cols = min(COLS, sq.n_new * R - pair0);
            const bool whole = u0 == 0 && u1 == units;
            float* where = ws + ((size_t)w * 2 + (u0 == 0 ? 1 : 0)) * COLS * ROW;
            if (u0 == 0 && lane == 0)                                // this warp, and those whose range begins within the walk
                pieces[((size_t)b * G + g) * tiles + tile] = make_int2(w, 1 + (int)((at + units - 1) / per - w));
            piece(sq, g, tile, u0, u1, 1, [&](auto& o, auto& m, auto& l) {
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int col = j * 8 + c4 * 2 + e, pair = pair0 + col;
                        if (col >= n_cols) continue;
                        if (whole) {
                            const int h = g * R + pair % R;
                            const float inv = kv8_inverse(m[j][e], l[j][e], sink ? sink + h : nullptr);
                            bf16* row = out + ((size_t)(sq.t0 + pair / R) * H + h) * HD;
#pragma unroll
                            for (int t = 0; t < MT; ++t)
                                *reinterpret_cast<__nv_bfloat162*>(row + value_component(t, n8)) = __floats2bfloat162_rn(o[j][t][e] * inv, o[j][t][2 + e] * inv);
                        } else {
                            put(where + col * ROW, o[j], e, m[j][e], l[j][e]);
                        }
                    }
            });
            at += u1 - u0;
            if (at >= end) break;
            __syncwarp();                                            // the ring and the queries' place are free
            u0 = 0;
            if (++rest == (unsigned)(n_tiles * G)) {
                rest = 0;
                do { deal.of(++b, units, n_tiles); } while (units == 0);
            }
        }
    }
}

// The partial results of walks that several warps shared: out[row] = sum_w f_w acc_w / sum_w f_w l_w with f_w = exp2(m_w - max m), warps in
// their order.  A thread takes a component of a row, eight warps' results at a time, all asked for at once: two trips to memory for
// most walks of a large step.  grid (G * tiles, 256ths of a tile's rows, sequences).
constexpr int JOIN = 256, AT_ONCE = 8;
template <int NG>
__global__ void __launch_bounds__(JOIN)
kv8_join_kernel(const float* ws, const int2* pieces, bf16* __restrict__ out, const Kv8Step step, int H, int G, int tiles, const float* sink) {
    constexpr int COLS = 8 * NG;
    pdl_wait();
    pdl_launch_dependents();
    const int R = H / G, b = blockIdx.z, at = blockIdx.y * JOIN + threadIdx.x, row = at / HD, d = at - row * HD;
    const int g = blockIdx.x / tiles, tile = blockIdx.x - g * tiles, pair = tile * COLS + row;
    const Kv8Seq sq = kv8_seq(step, b);
    if (tile * COLS >= sq.n_new * R) return;                         // (no walk)
    const int2 who = pieces[((size_t)b * G + g) * tiles + tile];
    if (who.y == 1 || row >= COLS || pair >= sq.n_new * R) return;      // one warp had it all, or no such row
    auto place = [&](int i) { return ws + ((size_t)((who.x + i) * 2 + (i == 0 ? 1 : 0)) * COLS + row) * ROW; };
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int i0 = 0; i0 < who.y; i0 += AT_ONCE) {
        float ms[AT_ONCE], ls[AT_ONCE], as[AT_ONCE], top = m;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const bool have = i0 + i < who.y;
            const float* p = place(have ? i0 + i : i0);
            ms[i] = p[HD]; ls[i] = p[HD + 1]; as[i] = p[d];
            if (!have) { ms[i] = -INFINITY; as[i] = 0.f; }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) top = fmaxf(top, ms[i]);
        const float f = m == -INFINITY ? 0.f : exp2f(m - top);
        l *= f;
        acc *= f;
        m = top;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const float w = ms[i] == -INFINITY ? 0.f : exp2f(ms[i] - top);         // (its sum is zero, or NaN where a value is)
            l = fmaf(w, ls[i], l);
            acc = fmaf(w, as[i], acc);
        }
    }
    const int h = g * R + pair % R;
    out[((size_t)(sq.t0 + pair / R) * H + h) * HD + d] = __float2bfloat16_rn(acc * kv8_inverse(m, l, sink ? sink + h : nullptr));
}

// The same for walks that many warps shared (few sequences): a block a row, in strands of every (512 / LANES)-th warp, the strands in
// their order.  grid (G * tiles, rows of a tile, sequences).
constexpr int LANES = HD <= 64 ? 64 : HD <= 128 ? 128 : 256;         // threads, one a component
template <int NG>
__global__ void __launch_bounds__(512)
kv8_join_many_kernel(const float* ws, const int2* pieces, bf16* __restrict__ out, const Kv8Step step, int H, int G, int tiles, const float* sink) {
    constexpr int COLS = 8 * NG, THREADS = 512, STRANDS = THREADS / LANES;
    extern __shared__ float factor[];                                // one a warp of the walk
    __shared__ float red[THREADS / 32], sums[THREADS];
    pdl_wait();
    pdl_launch_dependents();
    const int R = H / G, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = blockIdx.x / tiles, tile = blockIdx.x - g * tiles, pair = tile * COLS + blockIdx.y;
    const Kv8Seq sq = kv8_seq(step, b);
    if (pair >= sq.n_new * R) return;
    const int2 who = pieces[((size_t)b * G + g) * tiles + tile];
    const int n = who.y;
    if (n == 1) return;                                              // one warp had it all
    auto place = [&](int i) { return ws + ((size_t)((who.x + i) * 2 + (i == 0 ? 1 : 0)) * COLS + blockIdx.y) * ROW; };
    // everything that a thread reads of the first pieces is asked for before anything is waited for
    const int strand = threadIdx.x / LANES, d = threadIdx.x % LANES;
    float ahead[AT_ONCE], m = -INFINITY, l_first = 0.f;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
        const int i = strand + k * STRANDS;
        ahead[k] = d < HD && i < n ? place(i)[d] : 0.f;
    }
    if ((int)threadIdx.x < n) l_first = place(threadIdx.x)[HD + 1];
    for (int i = threadIdx.x; i < n; i += THREADS) m = fmaxf(m, factor[i] = place(i)[HD]);
    m = warp_max(m);
    if (lane == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < THREADS / 32; ++k) m = fmaxf(m, red[k]);
    float l = 0.f;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const float f = factor[i] == -INFINITY ? 0.f : exp2f(factor[i] - m);
        factor[i] = f;
        l = fmaf(f, i == (int)threadIdx.x ? l_first : place(i)[HD + 1], l);
    }
    l = warp_sum(l);
    __syncthreads();
    if (lane == 0) red[warp] = l;
    float acc = 0.f;
    if (d < HD) {
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
            if (strand + k * STRANDS < n) acc = fmaf(factor[strand + k * STRANDS], ahead[k], acc);
#pragma unroll 8
        for (int i = strand + AT_ONCE * STRANDS; i < n; i += STRANDS) acc = fmaf(factor[i], place(i)[d], acc);
    }
    sums[threadIdx.x] = acc;
    __syncthreads();
    if (strand == 0 && d < HD) {
        l = 0.f;
#pragma unroll
        for (int k = 0; k < THREADS / 32; ++k) l += red[k];
#pragma unroll
        for (int k = 1; k < STRANDS; ++k) acc += sums[k * LANES + d];
        const int h = g * R + pair % R;
        out[((size_t)(sq.t0 + pair / R) * H + h) * HD + d] = __float2bfloat16_rn(acc * kv8_inverse(m, l, sink ? sink + h : nullptr));
    }
}

// -------------------------------------------------------------------------------------------- prompts
#if PLM_HD != 64 && PLM_HD != 128                // (those on tcgen05: attention_kv8_tc.cu)
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
constexpr int LDS = HD + 8;                      // halves of a row in shared memory: ldmatrix without bank conflicts
constexpr size_t TILE_SMEM = (size_t)3 * 64 * LDS * 2;

// grid (tiles of 64 rows of the longest sequence, G, sequences): 16 rows a warp, keys and values a page at a time as halves in shared
// memory.  For head sizes up to 128 the next page's bytes are in registers meanwhile.
__global__ void __launch_bounds__(NT)
kv8_tile_kernel(const bf16* q, const Cache cache, bf16* __restrict__ out, const Kv8Step step, int H, int G, float scale_log2, int window,
                const float* sink, int keep, const float* slopes) {
    constexpr int CPR = HD / 16, CHUNKS = 64 * CPR / NT > 0 ? (64 * CPR + NT - 1) / NT : 1;       // 16-byte chunks of a page's rows
    constexpr bool AHEAD = HD <= 128;
    extern __shared__ __align__(128) uint8_t sm_raw[];
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
        ks = kv8_scale(cache.ks[at]);
        vs = kv8_scale(cache.vs[at]);
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
        for (int i = 0; i < 4; ++i) kv8_halves(in[i], h[2 * i], h[2 * i + 1]);
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
                const float m_new = fmaxf(m[hi], mx[hi] - LIFT);
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

#endif

template <int NG>
int stream(const bf16* q, const Cache& cache, bf16* out, void* ws, const Kv8Step& step, int n_seqs, int max_new, int H, int G, float scale,
           int window, int n_splits, int n_ctas, const float* sink, int keep, const float* slopes, cudaStream_t s) {
    static std::atomic<unsigned long long> d0{0}, d1{0};
    const size_t smem = Few<NG>::SMEM;
    cudaError_t e = ws ? plm_allow_smem(kv8_stream_kernel<NG, false>, smem, d1) : plm_allow_smem(kv8_stream_kernel<NG, true>, smem, d0);
    if (e != cudaSuccess) return (int)e;
    const long rows = (long)max_new * (H / G), tiles = (rows + 8 * NG - 1) / (8 * NG);
    if (tiles * G > 65535) return PLM_ERR_SHAPE;
    float* none = nullptr;
    int2* pieces = nullptr;
    if (!ws)
        return plm_status_of(launch_pdl_cluster(kv8_stream_kernel<NG, true>, dim3(n_splits, (unsigned)(tiles * G), n_seqs), dim3(NT), dim3(n_splits, 1, 1),
                                                smem, s, q, cache, out, none, pieces, step, n_seqs, H, G, (int)tiles, scale * LOG2E, window, sink, keep, slopes));
    // (no more CTAs than the step can have work for)
    const long most = (tiles * G * n_seqs * ((long)step.max_pages * (PLM_PAGE / Few<NG>::KB)) + WARPS * MIN_UNITS - 1) / (WARPS * MIN_UNITS);
    if (n_ctas > most) n_ctas = (int)most;
    float* part = reinterpret_cast<float*>(ws);
    pieces = reinterpret_cast<int2*>(part + (size_t)n_ctas * WARPS * 2 * 8 * NG * ROW);
    int rc = plm_status_of(launch_pdl(kv8_stream_kernel<NG, false>, dim3(n_ctas), dim3(NT), smem, s, q, cache, out, part, pieces, step, n_seqs, H, G,
                                      (int)tiles, scale * LOG2E, window, sink, keep, slopes));
    if (rc != PLM_OK) return rc;
    const unsigned n_walks = (unsigned)(tiles * G), n_rows = (unsigned)(rows < 8 * NG ? rows : 8 * NG);
    if ((long)n_ctas * WARPS > 10L * n_walks * n_seqs)
        return plm_status_of(launch_pdl(kv8_join_many_kernel<NG>, dim3(n_walks, n_rows, n_seqs), dim3(512), (size_t)n_ctas * WARPS * sizeof(float), s,
                                        (const float*)part, (const int2*)pieces, out, step, H, G, (int)tiles, sink));
    return plm_status_of(launch_pdl(kv8_join_kernel<NG>, dim3(n_walks, (n_rows * HD + JOIN - 1) / JOIN, n_seqs), dim3(JOIN), 0, s, (const float*)part,
                                    (const int2*)pieces, out, step, H, G, (int)tiles, sink));
}

// (token, head) rows that a CTA of the streaming kernel takes at a time, for at most `rows` of a sequence and kv head.
int groups_of(long rows) { return rows <= 8 ? 1 : rows <= 16 || HD > 128 ? 2 : 4; }

bool bad_step(const int* tok_pos, const int* tok_seq, const int* seq_start, const int* seq_kv_len) {
    return !tok_pos != !tok_seq || !tok_pos == !seq_start || !seq_start != !seq_kv_len;
}

}  // namespace

// CTAs that run at once, and floats of workspace for a CTA, for at most `rows` (token, head) rows of a sequence and kv head; two more
// for every sequence, kv head and tile of that many rows.
extern "C" int plm_kv8_few_ctas(int rows) {
    const int ng = groups_of(rows);
#if PLM_HD <= 128
    if (ng == 4) return PLM_SM_COUNT * (int)Few<4>::CTAS;
#endif
    return PLM_SM_COUNT * (ng == 1 ? (int)Few<1>::CTAS : (int)Few<2>::CTAS);
}
extern "C" int plm_kv8_few_floats(int rows) { return WARPS * 2 * 8 * groups_of(rows) * ROW; }
extern "C" int plm_kv8_few_tile(int rows) { return 8 * groups_of(rows); }

// q [n_rows, H, HD] bf16, out [n_rows, H * HD] bf16.  Either tok_pos and tok_seq [n_seqs = n_rows] (single tokens, max_new 1) or
// seq_start [n_seqs + 1] and seq_kv_len [n_seqs].  With ws null every sequence's keys are cut into n_splits ranges (at most eight), which
// meet in a cluster; else all keys of the step are dealt out to n_ctas CTAs (see the functions above for the
// size of ws).
extern "C" int plm_kv8_attention_few(const void* q, const void* kc, const void* vc, const float* ks, const float* vs, void* out, void* ws,
                                     const int* tok_pos, const int* tok_seq, const int* seq_start, const int* seq_kv_len,
                                     const int* block_table, int max_pages, int n_rows, int n_seqs, int max_new, int H, int G,
                                     float scale, int window, int n_splits, int n_ctas, const float* sink, int keep, const float* slopes,
                                     cudaStream_t s) {
    if (n_rows <= 0 || n_seqs <= 0 || max_new <= 0) return PLM_OK;
    if (H <= 0 || G <= 0 || H % G || n_seqs > 65535 || (ws ? n_ctas < 1 || n_ctas > MAX_CTAS : n_splits < 1 || n_splits > MAX_CLUSTER) || keep < 0) return PLM_ERR_SHAPE;
    if (bad_step(tok_pos, tok_seq, seq_start, seq_kv_len)) return PLM_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) & 15 || (uintptr_t)out & 3) return PLM_ERR_ALIGN;      // (out: pairs of bf16)
    const Kv8Step step = {tok_pos, tok_seq, seq_start, seq_kv_len, block_table, max_pages};
    const Cache cache = {(const uint8_t*)kc, (const uint8_t*)vc, ks, vs};
    const int groups = groups_of((long)max_new * (H / G));
    if (groups == 1) return stream<1>((const bf16*)q, cache, (bf16*)out, ws, step, n_seqs, max_new, H, G, scale, window, n_splits, n_ctas, sink, keep, slopes, s);
    if (groups == 2) return stream<2>((const bf16*)q, cache, (bf16*)out, ws, step, n_seqs, max_new, H, G, scale, window, n_splits, n_ctas, sink, keep, slopes, s);
#if PLM_HD <= 128
    if (groups == 4)
        return stream<4>((const bf16*)q, cache, (bf16*)out, ws, step, n_seqs, max_new, H, G, scale, window, n_splits, n_ctas, sink, keep, slopes, s);
#endif
    return PLM_ERR_UNSUPPORTED;
}

#if PLM_HD != 64 && PLM_HD != 128
// The same for prompts, rows of 64 at a time: seq_start [n_seqs + 1], seq_kv_len [n_seqs], at most max_new rows a sequence.
extern "C" int plm_kv8_attention_tiles(const void* q, const void* kc, const void* vc, const float* ks, const float* vs, void* out,
                                       const int* seq_start, const int* seq_kv_len, const int* block_table, int max_pages, int n_seqs,
                                       int max_new, int H, int G, float scale, int window, const float* sink, int keep,
                                       const float* slopes, cudaStream_t s) {
    if (n_seqs <= 0 || max_new <= 0) return PLM_OK;
    if (H <= 0 || G <= 0 || H % G || n_seqs > 65535 || G > 65535 || keep < 0) return PLM_ERR_SHAPE;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) & 15 || (uintptr_t)out & 3) return PLM_ERR_ALIGN;
    static std::atomic<unsigned long long> devices{0};
    cudaError_t e = plm_allow_smem(kv8_tile_kernel, TILE_SMEM, devices);
    if (e != cudaSuccess) return (int)e;
    const Kv8Step step = {nullptr, nullptr, seq_start, seq_kv_len, block_table, max_pages};
    const Cache cache = {(const uint8_t*)kc, (const uint8_t*)vc, ks, vs};
    const dim3 grid((unsigned)(((long)max_new * (H / G) + 63) / 64), G, n_seqs);
    return plm_status_of(launch_pdl(kv8_tile_kernel, grid, dim3(NT), TILE_SMEM, s, (const bf16*)q, cache, (bf16*)out, step, H, G,
                                    scale * LOG2E, window, sink, keep, slopes));
}
#endif
