// The 8-bit cache (kv8.cuh says what it holds): a step's keys and values into it, with the rotary encoding on the way, and
// attention over it in fp32 on the CUDA cores (the float32 run, and head sizes that the tensor-core kernels refuse).
#include "kv8.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// ------------------------------------------------------------------------------------------------ append
// q_in [T, H heads], k_in and v_in [T, G heads] of hd numbers, rows ldq / ldk / ldv apart (the three parts of one
// projection's rows, or rows of their own).  q' = R(pos) q goes to q_out [T, H, hd]; k' = R(pos) k and v to the cache.  The step's
// sequence b brings rows seq_start[b] .. seq_start[b + 1], its last position is seq_kv_len[b] - 1.  Tables cos / sin
// [n_table, rot / 2], null: no rotation; pairing 0: (x[i], x[i + rot / 2]), 1: (x[2i], x[2i + 1]).  Page 0 is nobody's: it is not written.
struct Append {
    const void *q_in, *k_in, *v_in;
    void* q_out;
    uint8_t *kc, *vc;
    float *ks, *vs;
    const float *cos_t, *sin_t;
    const int *seq_start, *seq_kv_len, *block_table;
    long ldq, ldk, ldv;
    int max_pages, n_table, H, G, hd, rot, pairing;
};

template <typename T, int N> struct Pack;
template <> struct Pack<float, 4> { typedef float4 type; };
template <> struct Pack<bf16, 8> { typedef uint4 type; };
template <> struct Pack<bf16, 4> { typedef uint2 type; };
template <> struct Pack<float, 1> { typedef float type; };
template <> struct Pack<bf16, 1> { typedef uint16_t type; };

template <typename T, int N> __device__ __forceinline__ void load_group(const T* p, float* x) {
    typedef typename Pack<T, N>::type P;
    const P w = *reinterpret_cast<const P*>(p);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32<T>(e[i]);
}
template <typename T, int N> __device__ __forceinline__ void store_group(T* p, const float* x) {
    typedef typename Pack<T, N>::type P;
    P w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = from_f32<T>(x[i]);
    *reinterpret_cast<P*>(p) = w;
}

// A unit is 2 * N numbers of one row: N pairs of the rotation, or 2 * N numbers in a row that are not rotated.  N numbers lie together and
// are one load: 16 bytes where the rotated part of a head and the head are multiples of 2 N, 8 bytes or one number where not.
template <int N> struct Unit {
    int ia, ib;                                  // where its first and its second N numbers lie in the head
    int angle;                                   // its first pair's column of the tables, -1: not rotated
    __device__ __forceinline__ Unit(int u, int rot, int pairing, bool rotate) {
        const bool turned = rotate && 2 * N * u < rot;
        if (turned && pairing == 0) { ia = N * u; ib = ia + rot / 2; }
        else { ia = 2 * N * u; ib = ia + N; }
        angle = turned ? N * u : -1;
    }
};
template <int N> struct Angles {
    float c[N], s[N];
    __device__ __forceinline__ void load(const Append& a, const Unit<N>& u, int pos) {
        if (u.angle < 0) return;
        const size_t at = (size_t)min(pos, a.n_table - 1) * (a.rot / 2) + u.angle;
        constexpr int M = N < 4 ? N : 4;
#pragma unroll
        for (int i = 0; i < N; i += M) {
            load_group<float, M>(a.cos_t + at + i, c + i);
            load_group<float, M>(a.sin_t + at + i, s + i);
        }
    }
    __device__ __forceinline__ void turn(float* x, const Append& a, const Unit<N>& u) const {
        if (u.angle < 0) return;
        if (a.pairing == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float p = x[i], q = x[N + i];
                x[i] = rope_first(p, q, c[i], s[i]);
                x[N + i] = rope_second(p, q, c[i], s[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = rope_first(p, q, c[i], s[i]);
                x[2 * i + 1] = rope_second(p, q, c[i], s[i]);
            }
        }
    }
};

// An item is the rows of the step that lie on one page, of one key or value head (they decide with what the page already holds about its
// scale and go in) or of Q_HEADS query heads (which share the angles: a table's row is as long as a head's).  W warps an item: 4 or 8 for
// prompts (an item is up to 64 rows, a CTA; what a thread loads stays in its registers until the scale is known), 1 for a few
// tokens a sequence (four items a CTA).  EVEN: a row's units divide the item's threads, so that a thread has one place in a row
// and every so many rows (no division on the way).
// One read of the projection, one write of what it becomes: bound by memory for prompts, by the launch for single tokens.  Measured (us,
// what it reads within the L2): a prompt of 2,048, 32 heads over 8 of 64 6.3 to 7.4 (9.9 from memory: 2.4 TB/s), 7 sequences of 1,011 in
// float32, 15 heads over 5 of 80 with 40 rotated 19.3 (3.2 TB/s), 64 single tokens 3.2, one 2.6; where every open page's scale grows, and
// what it holds is rounded again, 6.3 and 3.5.  A page's warps read, meet for its scale and write, with one wave
// of items an SM and half.  16 bytes a load and four query heads an item: a prompt of 8,192 39 -> 30.
constexpr int Q_HEADS = 4;
template <int N> struct Held { enum : int { UNITS = N == 8 ? 2 : 4 }; };      // units that a thread keeps between the two passes; more are read again
template <typename T, int N, int W, bool EVEN>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W)
kv8_append_kernel(const Append a) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int ITEMS = W == 1 ? 4 : 1, S = 32 * W, KEEP = W == 1 ? 1 : (int)Held<N>::UNITS;
    const int q_items = (a.H + Q_HEADS - 1) / Q_HEADS;
    const int item = blockIdx.y * ITEMS + (W == 1 ? threadIdx.x >> 5 : 0);
    const int tid = W == 1 ? threadIdx.x & 31 : threadIdx.x;
    const int b = blockIdx.z;
    if (item >= q_items + 2 * a.G) return;
    const int t0 = a.seq_start[b], n_new = a.seq_start[b + 1] - t0;
    if (n_new <= 0) return;
    const int pos0 = PLM_POSITION(a.seq_kv_len[b] - 1) + 1 - n_new;
    if (pos0 < 0) return;                                        // more tokens than the sequence is long
    const int page_no = pos0 / PLM_PAGE + blockIdx.x;
    const int first = max(pos0, page_no * PLM_PAGE), rows = min(pos0 + n_new, (page_no + 1) * PLM_PAGE) - first;
    if (rows <= 0) return;
    const int units = a.hd / (2 * N), total = rows * units;
    const int t_first = t0 + first - pos0;                       // the token of the item's first row
    const int u0 = EVEN ? tid % units : 0, r0 = EVEN ? tid / units : 0, r_step = EVEN ? S / units : 0;
    // the thread's j-th unit: its row and its place in the row
    auto row_of = [&](int j) { return EVEN ? r0 + j * r_step : (tid + j * S) / units; };
    auto place_of = [&](int j) { return EVEN ? u0 : (tid + j * S) % units; };
    const int mine = tid < total ? (total - tid + S - 1) / S : 0;

    if (item < q_items) {
        const int h0 = item * Q_HEADS, heads = min(Q_HEADS, a.H - h0);
        const T* src = reinterpret_cast<const T*>(a.q_in) + (size_t)h0 * a.hd;
        T* dst = reinterpret_cast<T*>(a.q_out) + (size_t)h0 * a.hd;
        for (int j = 0; j < mine; ++j) {
            const int r = row_of(j);
            const Unit<N> u(place_of(j), a.rot, a.pairing, a.cos_t != nullptr);
            const T* from = src + (size_t)(t_first + r) * a.ldq;
            T* to = dst + (size_t)(t_first + r) * a.H * a.hd;
            float x[Q_HEADS][2 * N];
            Angles<N> t;
#pragma unroll
            for (int h = 0; h < Q_HEADS; ++h) {
                if (h >= heads) break;
                load_group<T, N>(from + h * a.hd + u.ia, x[h]);
                load_group<T, N>(from + h * a.hd + u.ib, x[h] + N);
            }
            t.load(a, u, first + r);
#pragma unroll
            for (int h = 0; h < Q_HEADS; ++h) {
                if (h >= heads) break;
                t.turn(x[h], a, u);
                store_group<T, N>(to + h * a.hd + u.ia, x[h]);
                store_group<T, N>(to + h * a.hd + u.ib, x[h] + N);
            }
        }
        return;
    }
    const bool key = item < q_items + a.G;
    const int g = item - q_items - (key ? 0 : a.G);
    if (page_no >= a.max_pages) return;
    const int page = PLM_PAGE_NO(a.block_table[(size_t)b * a.max_pages + page_no]);
    if (page <= 0) return;
    const T* src = reinterpret_cast<const T*>(key ? a.k_in : a.v_in) + (size_t)g * a.hd;
    const long ld = key ? a.ldk : a.ldv;
    uint8_t* held = (key ? a.kc : a.vc) + ((size_t)page * a.G + g) * PLM_PAGE * a.hd;
    float* scale_at = (key ? a.ks : a.vs) + (size_t)page * a.G + g;
    const bool rotate = key && a.cos_t != nullptr;
    const int place = first % PLM_PAGE;                          // rows before it are there already
    const int e_old = place ? kv8_exponent_of_scale(kv8_scale(*scale_at)) : KV8_E_MIN;

    auto read = [&](int j, float* x) {
        const int r = row_of(j);
        const Unit<N> u(place_of(j), a.rot, a.pairing, rotate);
        const T* p = src + (size_t)(t_first + r) * ld;
        load_group<T, N>(p + u.ia, x);
        load_group<T, N>(p + u.ib, x + N);
        Angles<N> t;
        t.load(a, u, first + r);
        t.turn(x, a, u);
    };
    float x[KEEP][2 * N], most = 0.f;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        if (j >= mine) break;
        read(j, x[j]);
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) most = fmaxf(most, kv8_magnitude(x[j][i]));
    }
    for (int j = KEEP; j < mine; ++j) {
        float y[2 * N];
        read(j, y);
#pragma unroll
        for (int k = 0; k < 2 * N; ++k) most = fmaxf(most, kv8_magnitude(y[k]));
    }
    most = warp_max(most);
    if (W > 1) {
        __shared__ float red[W];
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) most = fmaxf(most, red[w]);
    }
    const int e = max(e_old, kv8_exponent(most));
    if (place && e != e_old) {                                   // rows that are there, held against the larger scale
        const float down = kv8_pow2(max(e_old - e, -126));
        for (int i = tid; i < place * a.hd / 8; i += S) {
            uint2 w = reinterpret_cast<const uint2*>(held)[i];
            uint32_t* words = &w.x;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 lo = kv8_floats(words[k] & 0xffffu), hi = kv8_floats(words[k] >> 16);
                words[k] = kv8_pack(lo.x * down, lo.y * down) | kv8_pack(hi.x * down, hi.y * down) << 16;
            }
            reinterpret_cast<uint2*>(held)[i] = w;
        }
    }
    const float up = kv8_pow2(-e);
    auto put = [&](int j, const float* y) {
        const int r = row_of(j);
        const Unit<N> u(place_of(j), a.rot, a.pairing, rotate);
        uint8_t* p = held + (size_t)(place + r) * a.hd;
        if constexpr (N >= 4) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t w[N / 4];
#pragma unroll
                for (int i = 0; i < N / 4; ++i) {
                    const float* z = y + half * N + 4 * i;
                    w[i] = kv8_pack(kv8_finite_or_nan(z[0]) * up, kv8_finite_or_nan(z[1]) * up) |
                           kv8_pack(kv8_finite_or_nan(z[2]) * up, kv8_finite_or_nan(z[3]) * up) << 16;
                }
                uint8_t* to = p + (half ? u.ib : u.ia);
                if constexpr (N == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[N / 4 - 1]);
                else *reinterpret_cast<uint32_t*>(to) = w[0];
            }
        } else {
            const uint32_t two = kv8_pack(kv8_finite_or_nan(y[0]) * up, kv8_finite_or_nan(y[1]) * up);
            p[u.ia] = (uint8_t)two;
            p[u.ib] = (uint8_t)(two >> 8);
        }
    };
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        if (j >= mine) break;
        put(j, x[j]);
    }
    for (int j = KEEP; j < mine; ++j) {
        float y[2 * N];
        read(j, y);
        put(j, y);
    }
    if (W == 1) __syncwarp();                                    // (all have read the scale; more warps met at the maximum)
    if (tid == 0) *scale_at = kv8_pow2(e);
}

template <typename T, int N, bool EVEN>
int append(const Append& a, int n_seqs, int max_new, cudaStream_t stream) {
    const int pages = 1 + (max_new + 62) / PLM_PAGE, items = (a.H + Q_HEADS - 1) / Q_HEADS + 2 * a.G;
    // a warp takes an item of few rows as fast as more do, and four times as many items are in flight on an SM
    if (max_new <= 4)
        return plm_status_of(launch_pdl(kv8_append_kernel<T, N, 1, EVEN>, dim3(pages, (items + 3) / 4, n_seqs), dim3(128), 0, stream, a));
    // four warps where a thread then keeps all it reads
    if (PLM_PAGE * a.hd / (2 * N) <= 128 * (int)Held<N>::UNITS)
        return plm_status_of(launch_pdl(kv8_append_kernel<T, N, 4, EVEN>, dim3(pages, items, n_seqs), dim3(128), 0, stream, a));
    return plm_status_of(launch_pdl(kv8_append_kernel<T, N, 8, EVEN>, dim3(pages, items, n_seqs), dim3(256), 0, stream, a));
}
template <typename T, int N>
int append(const Append& a, int n_seqs, int max_new, cudaStream_t stream) {
    const int units = a.hd / (2 * N);
    return (units & (units - 1)) == 0 && units <= 32 ? append<T, N, true>(a, n_seqs, max_new, stream) : append<T, N, false>(a, n_seqs, max_new, stream);
}

// ------------------------------------------------------------------------------------------------ attention, fp32
// A CTA of four warps takes WARPS * RPW (token, query head) rows of one sequence and kv head, RPW a warp, and a range of the
// keys that any of them sees, a group of 32 or (eight rows a warp) 64 at a time: keys and values as floats in shared memory (number * scale is
// exact there), a lane one or two keys for the scores, a lane VEC components for the sums; running maximum a row, its sum in each lane's part.  The ranges' partial results
// (sum, maximum, denominator) meet in kv8_merge_kernel.  For eight rows and two keys 64 products a lane take ten 16-byte reads (with one
// key nine for 32: 59 us where 52 are now).  Measured: two prompts of 301 tokens, 32 heads over 8 of 64 52 us (10.6 TFLOP/s); no pipe is full
// (FFMA 30 %, shared memory 31 %, 1.9 instructions a cycle): 12 warps an SM, which meet twice a group, with nothing asked for ahead.  The same
// takes single tokens' time: one behind 2,001 keys 19 us, eight behind 4,096 52, eight behind 8,192 of 128 225 (their bytes: 0.3, 3.5, 14).
constexpr int WARPS = 4;

template <bool V> struct Const { static constexpr bool value = V; };
__host__ __device__ constexpr int keys_a_lane(int rows_a_warp) { return rows_a_warp > 1 ? 2 : 1; }

template <typename T, int RPW, int VEC>
__global__ void __launch_bounds__(WARPS * 32)
kv8_rows_kernel(const T* q, const uint8_t* kc, const uint8_t* vc, const float* ksc, const float* vsc, T* __restrict__ out,
                float* __restrict__ ws, const Kv8Step step, int H, int G, int hd, float scale_log2, int window, int n_splits,
                const float* sink, int keep, const float* slopes) {
    constexpr int ROWS = WARPS * RPW, WIDE = 32 * VEC, KPL = keys_a_lane(RPW), KG = 32 * KPL;
    extern __shared__ __align__(16) float sm[];
    float* ks = sm;                                  // [KG][hd + 4]
    float* vs = ks + KG * (hd + 4);                  // [KG][WIDE], zero from hd on
    float* qs = vs + KG * WIDE;                      // [ROWS][hd]
    float* ps = qs + ROWS * hd;                      // [ROWS][KG]
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = H / G;
    // CTAs start in the order of their index: the tiles that see most keys first, of all kv heads
    const unsigned lin = blockIdx.y * gridDim.x + blockIdx.x;
    const int which = lin % gridDim.y, g = which / n_splits, split = which - g * n_splits;
    const Kv8Seq sq = kv8_seq(step, blockIdx.z);
    const long n_pairs = (long)sq.n_new * R, pair0 = ((n_pairs + ROWS - 1) / ROWS - 1 - (long)(lin / gridDim.y)) * ROWS;
    if (pair0 < 0) return;
    const int pos_first = sq.pos0 + (int)(pair0 / R), pos_last = sq.pos0 + (int)(min(pair0 + ROWS, n_pairs) - 1) / R;
    // the walk: kept first positions that lie before the window's first group, then the window's
    const int lo0 = plm_first_key(pos_first, window), g_lo = lo0 / KG;
    const int n_kept = min((keep + KG - 1) / KG, g_lo), n_groups = n_kept + pos_last / KG - g_lo + 1;
    const int per = (n_groups + n_splits - 1) / n_splits, w0 = split * per, w1 = min(n_groups, w0 + per);

    const int quads = hd / 4;
    for (int i = threadIdx.x; i < ROWS * quads; i += WARPS * 32) {
        const long pair = pair0 + i / quads;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (pair < n_pairs) load_group<T, 4>(q + ((sq.t0 + pair / R) * H + g * R + pair % R) * hd + i % quads * 4, x);
        *reinterpret_cast<float4*>(qs + i * 4) = make_float4(x[0], x[1], x[2], x[3]);
    }
    for (int i = threadIdx.x; i < KG * (WIDE - hd); i += WARPS * 32) vs[i / (WIDE - hd) * WIDE + hd + i % (WIDE - hd)] = 0.f;

    float acc[RPW][VEC], m[RPW], l[RPW], slope[RPW];
    int pos[RPW], lo[RPW];
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
        const long pair = pair0 + r * WARPS + warp;
        pos[r] = pair < n_pairs ? sq.pos0 + (int)(pair / R) : -1;
        lo[r] = plm_first_key(pos[r], window);
        slope[r] = slopes && pair < n_pairs ? slopes[g * R + pair % R] * LOG2E : 0.f;
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[r][i] = 0.f;
    }
    for (int w = w0; w < w1; ++w) {
        const int key0 = (w < n_kept ? w : g_lo + w - n_kept) * KG;
        const int page = PLM_PAGE_NO(sq.pages[key0 / PLM_PAGE]);
        const size_t base = (((size_t)page * G + g) * PLM_PAGE + key0 % PLM_PAGE) * hd;
        const float sk = kv8_scale(ksc[(size_t)page * G + g]), sv = kv8_scale(vsc[(size_t)page * G + g]);
        __syncthreads();                                             // what was there has been read (and q is there)
        bool nan = false;
        for (int i = threadIdx.x; i < KG * quads; i += WARPS * 32) {
            const int j = i / quads, c = i % quads * 4;
            float4 kv = make_float4(0.f, 0.f, 0.f, 0.f), vv = kv;
            if (key0 + j <= pos_last) {                              // (places behind hold whatever an earlier owner left)
                const uint32_t kw = *reinterpret_cast<const uint32_t*>(kc + base + (size_t)j * hd + c);
                const uint32_t vw = *reinterpret_cast<const uint32_t*>(vc + base + (size_t)j * hd + c);
                const float2 k0 = kv8_floats(kw & 0xffffu), k1 = kv8_floats(kw >> 16);
                const float2 v0 = kv8_floats(vw & 0xffffu), v1 = kv8_floats(vw >> 16);
                kv = make_float4(k0.x * sk, k0.y * sk, k1.x * sk, k1.y * sk);
                vv = make_float4(v0.x * sv, v0.y * sv, v1.x * sv, v1.y * sv);
                nan |= !(v0.x == v0.x && v0.y == v0.y && v1.x == v1.x && v1.y == v1.y);
            }
            *reinterpret_cast<float4*>(ks + j * (hd + 4) + c) = kv;
            *reinterpret_cast<float4*>(vs + j * WIDE + c) = vv;
        }
        nan = __syncthreads_or(nan);
        float dot[KPL][RPW];
#pragma unroll
        for (int n = 0; n < KPL; ++n)
#pragma unroll
            for (int r = 0; r < RPW; ++r) dot[n][r] = 0.f;
        const float* kr = ks + lane * (hd + 4);
#pragma unroll 4
        for (int c = 0; c < hd; c += 4) {
            float4 k4[KPL];
#pragma unroll
            for (int n = 0; n < KPL; ++n) k4[n] = *reinterpret_cast<const float4*>(kr + n * 32 * (hd + 4) + c);
#pragma unroll
            for (int r = 0; r < RPW; ++r) {
                const float4 q4 = *reinterpret_cast<const float4*>(qs + (r * WARPS + warp) * hd + c);
#pragma unroll
                for (int n = 0; n < KPL; ++n)
                    dot[n][r] = fmaf(q4.x, k4[n].x, fmaf(q4.y, k4[n].y, fmaf(q4.z, k4[n].z, fmaf(q4.w, k4[n].w, dot[n][r]))));
            }
        }
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            float most = -INFINITY;
#pragma unroll
            for (int n = 0; n < KPL; ++n) {
                const int key = key0 + n * 32 + lane;
                const bool ok = key <= pos[r] && (key >= lo[r] || key < keep);
                dot[n][r] = ok ? fmaf(slope[r], (float)(key - pos[r]), dot[n][r] * scale_log2) : -INFINITY;
                most = fmaxf(most, dot[n][r]);
            }
            const float m_new = fmaxf(m[r], warp_max(most)), m_use = m_new == -INFINITY ? 0.f : m_new;
            const float down = exp2f(m[r] - m_use);
            l[r] *= down;
            m[r] = m_new;
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[r][i] *= down;
#pragma unroll
            for (int n = 0; n < KPL; ++n) {
                const float p = exp2f(dot[n][r] - m_use);
                l[r] += p;
                ps[(r * WARPS + warp) * KG + n * 32 + lane] = p;
            }
        }
        __syncwarp();
        // NaN among the values: it counts for the rows that see its place, whatever their weight, and for no others (0 * NaN)
        auto add = [&](auto skips) {
#pragma unroll 2
            for (int j0 = 0; j0 < KG; j0 += 4) {
                float4 p4[RPW];
#pragma unroll
                for (int r = 0; r < RPW; ++r) p4[r] = *reinterpret_cast<const float4*>(ps + (r * WARPS + warp) * KG + j0);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i += VEC < 4 ? 2 : 4) {
                        if constexpr (VEC < 4) *reinterpret_cast<float2*>(v + i) = *reinterpret_cast<const float2*>(vs + (j0 + k) * WIDE + lane * VEC + i);
                        else *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(vs + (j0 + k) * WIDE + lane * VEC + i);
                    }
#pragma unroll
                    for (int r = 0; r < RPW; ++r) {
                        const float p = k == 0 ? p4[r].x : k == 1 ? p4[r].y : k == 2 ? p4[r].z : p4[r].w;
                        const int key = key0 + j0 + k;
                        const bool skip = decltype(skips)::value && !(key <= pos[r] && (key >= lo[r] || key < keep));
#pragma unroll
                        for (int i = 0; i < VEC; ++i) acc[r][i] = fmaf(p, skip ? 0.f : v[i], acc[r][i]);
                    }
                }
            }
        };
        if (nan) add(Const<true>());
        else add(Const<false>());
    }
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
        const long pair = pair0 + r * WARPS + warp;
        if (pair >= n_pairs) continue;                               // (the whole warp)
        l[r] = warp_sum(l[r]);
        const size_t row = (sq.t0 + pair / R) * H + g * R + pair % R;
        const float inv = n_splits > 1 ? 1.f : kv8_inverse(m[r], l[r], sink ? sink + g * R + pair % R : nullptr);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int d = lane * VEC + i;
            if (d >= hd) continue;
            if (n_splits > 1) ws[(row * n_splits + split) * (hd + 2) + d] = acc[r][i];
            else out[row * hd + d] = from_f32<T>(acc[r][i] * inv);
        }
        if (n_splits > 1 && lane == 0) {
            ws[(row * n_splits + split) * (hd + 2) + hd] = kv8_top(m[r], l[r]);
            ws[(row * n_splits + split) * (hd + 2) + hd + 1] = l[r];
        }
    }
}

// out[row] = sum_s w_s acc_s / sum_s w_s l_s with w_s = exp2(m_s - max m), ranges in their order; ws [rows, n_splits, hd + 2]:
// acc, m, l.  A block a row, a thread a component (or several); grid (tokens of a sequence * H, sequences).
template <typename T>
__global__ void __launch_bounds__(128)
kv8_merge_kernel(const float* ws, T* __restrict__ out, const Kv8Step step, int n_splits, int hd, int H, const float* sink) {
    pdl_wait();
    pdl_launch_dependents();
    const Kv8Seq sq = kv8_seq(step, blockIdx.y);
    if ((int)(blockIdx.x / H) >= sq.n_new) return;
    const size_t row = (size_t)sq.t0 * H + blockIdx.x;
    const float* p = ws + row * n_splits * (hd + 2);
    float m = -INFINITY, l = 0.f;
    for (int s = 0; s < n_splits; ++s) m = fmaxf(m, p[(size_t)s * (hd + 2) + hd]);
    for (int s = 0; s < n_splits; ++s) {
        const float ms = p[(size_t)s * (hd + 2) + hd];
        if (ms != -INFINITY) l = fmaf(exp2f(ms - m), p[(size_t)s * (hd + 2) + hd + 1], l);
    }
    const float inv = kv8_inverse(m, l, sink ? sink + row % H : nullptr);
    for (int d = threadIdx.x; d < hd; d += 128) {
        float acc = 0.f;
        for (int s = 0; s < n_splits; ++s) {
            const float ms = p[(size_t)s * (hd + 2) + hd];
            acc = fmaf(ms == -INFINITY ? 0.f : exp2f(ms - m), p[(size_t)s * (hd + 2) + d], acc);       // (its sum is zero, or NaN where a value is)
        }
        out[row * hd + d] = from_f32<T>(acc * inv);
    }
}

size_t rows_smem(int rows, int wide, int hd) {
    const int group = 32 * keys_a_lane(rows / WARPS);
    return (size_t)(group * (hd + 4) + group * wide + rows * hd + rows * group) * sizeof(float);
}

template <typename T, int RPW, int VEC>
int rows_launch(dim3 grid, const void* q, const void* kc, const void* vc, const float* ks, const float* vs, void* out, float* ws,
                const Kv8Step& step, int H, int G, int hd, float scale, int window, int n_splits, const float* sink, int keep,
                const float* slopes, cudaStream_t stream) {
    static std::atomic<unsigned long long> devices{0};
    const size_t smem = rows_smem(WARPS * RPW, 32 * VEC, hd);
    cudaError_t e = plm_allow_smem(kv8_rows_kernel<T, RPW, VEC>, rows_smem(WARPS * RPW, 32 * VEC, 32 * VEC), devices);
    if (e != cudaSuccess) return (int)e;
    return plm_status_of(launch_pdl(kv8_rows_kernel<T, RPW, VEC>, grid, dim3(WARPS * 32), smem, stream, (const T*)q,
                                    (const uint8_t*)kc, (const uint8_t*)vc, ks, vs, (T*)out, ws, step, H, G, hd, scale * LOG2E,
                                    window, n_splits, sink, keep, slopes));
}

template <typename T>
int rows_any(const void* q, const void* kc, const void* vc, const float* ks, const float* vs, void* out, float* ws,
             const Kv8Step& step, int n_seqs, int max_new, int H, int G, int hd, float scale, int window, int n_splits,
             const float* sink, int keep, const float* slopes, cudaStream_t stream) {
    const int R = H / G;
    const long pairs = (long)max_new * R;
    // few rows: one a warp, so that the CTAs are many; else eight, so that what is brought to shared memory is used often
    const bool few = pairs <= WARPS;
    const long tiles = few ? 1 : (pairs + 8 * WARPS - 1) / (8 * WARPS);
    if (tiles > 0x7fffffffL || (long)max_new * H > 0x7fffffffL || (long)G * n_splits > 65535 || n_seqs > 65535) return PLM_ERR_SHAPE;
    const dim3 grid((unsigned)tiles, G * n_splits, n_seqs);
    int rc;
#define KV8_ROWS(RPW_, VEC_) rc = rows_launch<T, RPW_, VEC_>(grid, q, kc, vc, ks, vs, out, ws, step, H, G, hd, scale, window, n_splits, sink, keep, slopes, stream)
    if (hd <= 64) { if (few) KV8_ROWS(1, 2); else KV8_ROWS(8, 2); }
    else if (hd <= 128) { if (few) KV8_ROWS(1, 4); else KV8_ROWS(8, 4); }
    else { if (few) KV8_ROWS(1, 8); else KV8_ROWS(8, 8); }
#undef KV8_ROWS
    if (rc != PLM_OK || n_splits == 1) return rc;
    return plm_status_of(launch_pdl(kv8_merge_kernel<T>, dim3((unsigned)((long)max_new * H), n_seqs), dim3(128), 0, stream, (const float*)ws,
                                    (T*)out, step, n_splits, hd, H, sink));
}

}  // namespace

// See `Append`.  dtype is that of the rows; q_in and q_out may be null with H = 0 (keys and values alone).
extern "C" int plm_kv8_append(const void* q_in, const void* k_in, const void* v_in, int dtype, long ldq, long ldk, long ldv,
                              void* q_out, void* kc, void* vc, float* ks, float* vs, const float* cos_t, const float* sin_t,
                              int n_table, const int* seq_start, const int* seq_kv_len, const int* block_table, int max_pages,
                              int n_seqs, int max_new, int H, int G, int hd, int rot, int pairing, cudaStream_t stream) {
    if (n_seqs <= 0 || max_new <= 0) return PLM_OK;
    if (H < 0 || G <= 0 || hd <= 0 || hd % 8 || hd > 256 || rot < 0 || rot > hd || rot % 2 || n_seqs > 65535 || max_pages <= 0 ||
        H + 2L * G > 65535 || (cos_t && (n_table <= 0 || rot == 0)) || (H > 0 && (!q_in || !q_out)))
        return PLM_ERR_SHAPE;
    if (pairing != 0 && pairing != 1) return PLM_ERR_UNSUPPORTED;
    if (((uintptr_t)kc | (uintptr_t)vc) & 15) return PLM_ERR_ALIGN;
    const Append a = {q_in, k_in, v_in, q_out, (uint8_t*)kc, (uint8_t*)vc, ks, vs, cos_t, sin_t, seq_start, seq_kv_len, block_table,
                      ldq, ldk, ldv, max_pages, n_table, H, G, hd, rot, pairing};
    // N numbers at a time where all of them lie on a boundary of their own size, in the rows, the tables and the cache
    const uintptr_t rows = (uintptr_t)q_in | (uintptr_t)k_in | (uintptr_t)v_in | (uintptr_t)q_out, tables = (uintptr_t)cos_t | (uintptr_t)sin_t;
    const int item = dtype == PLM_F32 ? 4 : 2;
    auto fits = [&](int n) {
        return hd % (2 * n) == 0 && (!cos_t || (rot % (2 * n) == 0 && !(tables & 15))) && !(rows & (n * item - 1)) && !((ldq | ldk | ldv) & (n - 1));
    };
    if (dtype == PLM_F32) return fits(4) ? append<float, 4>(a, n_seqs, max_new, stream) : append<float, 1>(a, n_seqs, max_new, stream);
    if (dtype == PLM_BF16)
        return fits(8) ? append<bf16, 8>(a, n_seqs, max_new, stream)
                       : fits(4) ? append<bf16, 4>(a, n_seqs, max_new, stream) : append<bf16, 1>(a, n_seqs, max_new, stream);
    return PLM_ERR_DTYPE;
}

// Attention on the CUDA cores.  q [n_rows, H, hd], out [n_rows, H * hd]; either tok_pos and tok_seq [n_seqs = n_rows] (single
// tokens) or seq_start [n_seqs + 1] and seq_kv_len [n_seqs].  ws: n_rows * H * n_splits * (hd + 2) floats where n_splits > 1.
extern "C" int plm_kv8_attention_rows(const void* q, int dtype, const void* kc, const void* vc, const float* ks, const float* vs,
                                      void* out, float* ws, const int* tok_pos, const int* tok_seq, const int* seq_start,
                                      const int* seq_kv_len, const int* block_table, int max_pages, int n_rows, int n_seqs,
                                      int max_new, int H, int G, int hd, float scale, int window, int n_splits, const float* sink,
                                      int keep, const float* slopes, cudaStream_t stream) {
    if (n_rows <= 0 || n_seqs <= 0 || max_new <= 0) return PLM_OK;
    if (H <= 0 || G <= 0 || H % G || hd <= 0 || hd % 8 || hd > 256 || n_splits < 1 || (n_splits > 1 && !ws) || keep < 0) return PLM_ERR_SHAPE;
    if (!tok_pos != !tok_seq || !tok_pos == !seq_start || !seq_start != !seq_kv_len) return PLM_ERR_UNSUPPORTED;
    if ((uintptr_t)q & 15 || ((uintptr_t)kc | (uintptr_t)vc) & 3) return PLM_ERR_ALIGN;      // (the caches: four bytes at a time)
    const Kv8Step step = {tok_pos, tok_seq, seq_start, seq_kv_len, block_table, max_pages};
    if (dtype == PLM_F32)
        return rows_any<float>(q, kc, vc, ks, vs, out, ws, step, n_seqs, max_new, H, G, hd, scale, window, n_splits, sink, keep, slopes, stream);
    if (dtype == PLM_BF16)
        return rows_any<bf16>(q, kc, vc, ks, vs, out, ws, step, n_seqs, max_new, H, G, hd, scale, window, n_splits, sink, keep, slopes, stream);
    return PLM_ERR_DTYPE;
}
