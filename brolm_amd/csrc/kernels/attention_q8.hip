// Attention of a batched step over the paged 8-bit KV cache (layout and entry
// points in kv_pages.hip and brolm_hip.h): decode rows and prompt chunks of
// several requests in one call.
//
// A request's rows and the query heads of one KV head make columns, column c =
// (row c / G, head c % G); a workgroup takes 16 columns of one KV head and walks
// their keys in tiles of 64, one tile per wavefront at a time:
//   S^T = K Q^T on v_mfma_i32_16x16x64_i8, the codes of K as they are stored: q is
//         written in three 8-bit parts times a power of two, whose products are exact,
//         so S has q to 2^-23 of its largest element (components above 2^-11 of it
//         exactly; with two parts, 2^-15, a channel 300 times the others cost 4e-3 of
//         the output; the third takes 0.5 % of the time of a long decode step);
//   softmax in FP32 (base 2, running maximum and sum per column); a tile's scales
//         enter as one factor per 16 keys, which lie in one page;
//   O^T += V^T P^T on v_mfma_f32_16x16x32_f16: V codes as FP16 integers, P times
//         its page's scale of V.  The running maximum is that of score + log2(scale),
//         so P stays inside FP16 (below 2^15) and what contributes 2^-21 of a column's
//         largest part still has 11 bits.  A second product adds what P's rounding left:
//         the output's error is then that of its own rounding (2.1e-4 relative; 3.1e-4
//         with one), for 1 % of the time, which goes with the bytes (48 requests of 8,000
//         to 16,000 keys 211 us, 208 with one).
//         Prompt chunks, which the arithmetic bounds, leave it out.
// The 16 keys that a lane holds of S^T are consecutive (fragment t takes the rows
// 16 i + 4 t + j): P is an operand as it stands, and its V^T counterpart is one
// 16-byte load of 16 tokens of a head dim, as the cache stores them.  K and V go
// from memory to the matrix operands without LDS.
//
// A column tile's keys are split over workgroups where there are few tiles; each
// leaves a record (O, m, l), the last one to arrive adds them in split order.
//
// Single tokens are bound by their bytes: 48 requests of 8,000 to 16,000 keys, 8 KV heads of
// 128, 212 us, 5.6 TB/s of codes (8 heads of 64: 107 us, 5.4; 4 of 256: 260 us, 4.4, one
// wavefront a SIMD); one of 700 keys by latency (9.8 us: lengths, table, rows, the merge).
#include <algorithm>

#include "gemm_job.h"
#include "kv_pages.h"

namespace bx {
namespace {

typedef _Float16 qa_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 qa_h2 __attribute__((ext_vector_type(2)));
typedef float qa_f4 __attribute__((ext_vector_type(4)));
typedef int qa_i4 __attribute__((ext_vector_type(4)));
typedef u4v __attribute__((aligned(2))) qa_any16;
typedef u2v __attribute__((aligned(2))) qa_any8;

constexpr int kQaThreads = 256;
constexpr int kQaMaxGroup = 16;
constexpr int kQaLazy = 8;      // the running maximum moves when exceeded by 2^8
constexpr int kQaReserve = 7;   // P is 2^7 at that maximum; 2^(8 + 7) < 65504
// V scales as P carries them: weights divided by one add up inside FP32.  127 times the least
// is 0 in FP16, the most is infinite.
constexpr float kQaLeastScale = 0x1p-64f, kQaMostScale = 0x1p64f;
constexpr int kQaMaxSplits = 256;   // their weights (16 columns) fit the LDS of the wavefronts' shares
constexpr int64_t kQaRecBytes = 128 << 20;   // records of either kind of tile, at most
constexpr int kQaNarrowReq = 256;    // requests whose narrow tiles a wavefront counts in four steps
constexpr int kQaNarrowCols = 64;    // columns a request up to which narrow tiles serve any batch
constexpr int64_t kQaNarrowWork = (int64_t)1 << 27;   // bytes of K that they read, for more columns
constexpr int kQaWords = 32768;   // arrival counters of either kind of tile

struct QaArgs {
    const uint16_t* q;
    int64_t q_stride;
    int rows;
    const int32_t *starts, *lens;
    int n_req;
    const int32_t* table;
    int max_blocks, pshift, n_pages;
    const int8_t *Kc, *Vc;
    const float *ks, *vs;
    int n_kv, G, window;
    uint16_t* out;
    int64_t out_stride;
    int narrow, S;
    uint64_t* cnt;
    unsigned char* recs;
    uint32_t tag;
};

// The first key that the row at position p sees (p below 0 where there are more rows than
// keys; the window may be anything up to 2^31 - 1).
__device__ __forceinline__ int first_key(int p, int window) { return window > 0 && p >= window ? p - window + 1 : 0; }

// Four int8 codes as FP16 integers: 1024 + (c + 128) by byte placement, less 1152.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = w ^ 0x80808080u;
    const qa_h2 off{(_Float16)-1152.0f, (_Float16)-1152.0f};
    const qa_h2 a = __builtin_bit_cast(qa_h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
    const qa_h2 b = __builtin_bit_cast(qa_h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
    lo = __builtin_bit_cast(uint32_t, a);
    hi = __builtin_bit_cast(uint32_t, b);
}

__device__ __forceinline__ float exp2_int(int e) {   // 2^e, 0 below the normal range
    return e < -126 ? 0.f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23);
}

// op over lanes l, l ^ 16, l ^ 32, l ^ 48, in each of them: the two halves of the rows (of
// the wavefront) that a lane swap hands out, without a trip through the LDS.
template <class F>
__device__ __forceinline__ uint32_t quad_of(uint32_t v, F&& op) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op((uint32_t)a[0], (uint32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return op((uint32_t)b[0], (uint32_t)b[1]);
}
__device__ __forceinline__ float quad_max(float v) {
    return __uint_as_float(quad_of(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ float quad_sum(float v) {
    return __uint_as_float(quad_of(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
__device__ __forceinline__ uint32_t quad_max_u(uint32_t v) {
    return quad_of(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}

// The V scale that P carries for the lane's 16 keys.  A page of which the wavefront sees no key
// (seen) may have been given back and hold anything; one with a NaN or an infinity that is seen
// (weird: some lane has one) is multiplied apart.
struct QaScale {
    float sv, r;   // as it is; in P
    bool weird;

    __device__ __forceinline__ void next(float scale, bool seen) {
        sv = seen ? scale : 1.f;
        const bool fin = sv < INFINITY;
        weird = __any(!fin);
        r = fin ? fminf(fmaxf(sv, kQaLeastScale), kQaMostScale) : 1.f;
    }
};

// One step of the softmax for 64 keys of NF columns a lane: s[n][t][e] are the products of
// q and the codes of key 4 t + e of the lane's 16, f their factor in base-2 units; hide(n,
// t, e) is asked where `masked`.  m is the running maximum of score + log2(V scale), of each
// column by itself: P, the weight times the V scale, is then near 2^kQaReserve where a column's
// largest contributions are, whatever the scales of other pages or of those that only other
// columns see, and as an FP16 operand loses bits only for what is 2^-21 of them.  It moves only
// when exceeded by 2^kQaLazy (rescale(al) then gets the factors of O).  l is the sum of P / V scale.
// SPLIT: pb[n][2 .. 3] gets what the rounding of pb[n][0 .. 1] left.
template <int NF, bool SPLIT, class H, class F>
__device__ __forceinline__ void qa_softmax(float (&s)[NF][4][4], float f0, const float (&cf)[NF], bool masked, H&& hide,
                                           const QaScale& sc, float (&m)[NF], float (&l)[NF], qa_h8 (&pb)[NF][SPLIT ? 4 : 2],
                                           F&& rescale) {
    // the exponents against the maximum so far: most tiles exceed it nowhere, and one that
    // does moves them.  (The largest exponent costs half the instructions that the largest
    // product does, which the compiler makes canonical first.)
    float f[NF], nm[NF], nr[NF], mx[NF];
    const float lr = __builtin_amdgcn_logf(sc.r) + (float)kQaReserve;   // base 2
    bool over = false;
#pragma unroll
    for (int n = 0; n < NF; ++n) {
        f[n] = cf[n] * f0;
        nm[n] = m[n] == -INFINITY ? 0.f : -m[n];
        nr[n] = nm[n] + lr;
    }
    if (masked) {
#pragma unroll
        for (int n = 0; n < NF; ++n) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][t][e] = hide(n, t, e) ? -INFINITY : s[n][t][e] * f[n];
            f[n] = 1.f;
        }
    }
#pragma unroll
    for (int n = 0; n < NF; ++n) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][t][e] = __builtin_fmaf(s[n][t][e], f[n], nr[n]);
                mx[n] = t + e == 0 ? s[n][t][e] : fmaxf(mx[n], s[n][t][e]);
            }
        over |= mx[n] > (m[n] == -INFINITY ? -INFINITY : (float)(kQaReserve + kQaLazy));
    }
    if (__any(over)) {
        float al[NF];
#pragma unroll
        for (int n = 0; n < NF; ++n) {
            const float mn = fmaxf(m[n], quad_max(mx[n] - nm[n] - (float)kQaReserve));
            const float d = mn == m[n] ? 0.f : -mn - nm[n];
            al[n] = mn == m[n] ? 1.f : __builtin_amdgcn_exp2f(m[n] - mn);
            l[n] *= al[n];
            m[n] = mn;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][t][e] += d;
        }
        rescale(al);
    }
    const float ir = __builtin_amdgcn_rcpf(sc.r);
    if (!sc.weird) {
#pragma unroll
        for (int n = 0; n < NF; ++n) {
            float ls[4];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(s[n][t][e]);
                    ls[e] = t == 0 ? p : ls[e] + p;
                    const _Float16 h = (_Float16)p;
                    pb[n][t / 2][4 * (t % 2) + e] = h;
                    if constexpr (SPLIT) pb[n][2 + t / 2][4 * (t % 2) + e] = (_Float16)(p - (float)h);
                }
            l[n] = __builtin_fmaf((ls[0] + ls[1]) + (ls[2] + ls[3]), ir, l[n]);
        }
    } else {   // a hidden key weighs nothing whatever its page's scale
#pragma unroll
        for (int n = 0; n < NF; ++n)
#pragma unroll 1
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = 0.f;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (q == t) x = s[n][q][e];
                    const float p = __builtin_amdgcn_exp2f(x);
                    l[n] = __builtin_fmaf(p, ir, l[n]);
                    const float pr = sc.sv < INFINITY ? p : x == -INFINITY ? 0.f : p * sc.sv;
                    const _Float16 h = (_Float16)pr;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (q == t) {
                            pb[n][q / 2][4 * (q % 2) + e] = h;
                            if constexpr (SPLIT) pb[n][2 + q / 2][4 * (q % 2) + e] = (_Float16)(pr - (float)h);
                        }
                }
    }
}

// The query columns of a wavefront as B operands of the integer products: lane l
// holds column l % 16, head dims 64 c + 16 (l / 16) .. of part c.
template <int HD>
struct QaQuery {
    qa_i4 hi[HD / 64], mid[HD / 64], lo[HD / 64];
    float scale;   // q = (65536 hi + 256 mid + lo) scale; NaN where q holds one or an infinity
    u4v w[HD / 64][2];

    // the loads apart from the arithmetic: the first tile is requested between them
    __device__ __forceinline__ void load(const uint16_t* col) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                w[c][i] = *reinterpret_cast<const qa_any16*>(col + 64 * c + 16 * (lane >> 4) + 8 * i);
    }
    __device__ __forceinline__ void split(bool real) {
        uint32_t m = 0u;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!real) w[c][i] = u4v{0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t a = w[c][i][e] & 0x7fff7fffu;
                    m = max(m, max(a & 0xffffu, a >> 16));
                }
            }
        m = quad_max_u(m);
        const float amax = h2f((uint16_t)m);
        const bool fin = m < 0x7c00u;
        // the power of two that brings amax below 127 * 65536 + 127 * 256 + 127, a whole number
        int k = 22 - ((int)(__float_as_uint(amax) >> 23) - 127);
        if (amax * exp2_int(k) > 8355711.f) --k;
        const float mul = fin && m > 0u ? exp2_int(k) : 0.f;
        scale = fin ? (m > 0u ? exp2_int(-k) : 0.f) : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint32_t h4 = 0u, m4 = 0u, l4 = 0u;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int e = 4 * d + b;
                    const uint16_t x = (uint16_t)(w[c][e / 8][(e % 8) / 2] >> (16 * (e & 1)));
                    const int q = fin ? (int)rintf(h2f(x) * mul) : 0;
                    const int m = (q + 128) >> 8, h = (m + 128) >> 8;   // parts in [-128, 127]
                    h4 |= (uint32_t)(h & 0xff) << (8 * b);
                    m4 |= (uint32_t)(m & 0xff) << (8 * b);
                    l4 |= (uint32_t)(q & 0xff) << (8 * b);
                }
                hi[c][d] = (int)h4;
                mid[c][d] = (int)m4;
                lo[c][d] = (int)l4;
            }
    }
};

// A tile of 64 keys on its way: K as the A operands of the integer products
// (fragment t, part c: lane l holds key 16 (l % 16 / 4) + 4 t + l % 4), V^T as the
// sources of the A operands of P V (part j: lane l holds head dim 16 j + l % 16 of
// the keys 16 (l / 16) ..), the scales of the lane's 16 keys.
template <int HD>
struct QaTile {
    qa_i4 k[4][HD / 64];
    u4v v[HD / 16];
    float sk, sv;
    bool ok;
};

// NT: rows by streaming loads (below, at the launch).
template <int HD, bool NT>
__device__ __forceinline__ void qa_tile(const QaArgs& a, unsigned block, unsigned char* smem) {
    constexpr int NC = HD / 64, NJ = HD / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lc = lane & 15, lg = lane >> 4, G = a.G, page = 1 << a.pshift;

    // ---- block -> (tile of 16 columns, split, KV head)
    const int g = (int)(block % (unsigned)a.n_kv);
    const unsigned rest = block / (unsigned)a.n_kv;
    const int s = (int)(rest % (unsigned)a.S), tile = (int)(rest / (unsigned)a.S);
    int r = tile, c0 = 0;
    if (a.narrow) {
        // the tiles that have columns, numbered through: no empty block stands between two
        // that work, or they would share their CUs and leave others idle
        constexpr int N = kQaNarrowReq / 64;
        int cnt[N], base = 0;
        r = -1;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = min(64 * n + lane, a.n_req - 1), n_i = a.starts[i + 1] - a.starts[i];
            cnt[n] = 64 * n + lane < a.n_req ? (int)(((int64_t)max(0, min(n_i, a.rows)) * G + 15) / 16) : 0;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int end = base + (int)wave_prefix((uint32_t)cnt[n]);
            const uint64_t in = __ballot(end > tile && end - cnt[n] <= tile);
            if (in) {
                const int at = __builtin_ctzll(in);
                r = 64 * n + at;
                c0 = 16 * (tile - (__builtin_amdgcn_readlane(end, at) - __builtin_amdgcn_readlane(cnt[n], at)));
            }
            base = __builtin_amdgcn_readlane(end, 63);
        }
        if (r < 0) return;
    }
    const int row0 = a.starts[r], n_new = a.starts[r + 1] - row0;
    if (row0 < 0 || n_new <= 0 || row0 > a.rows - n_new) return;
    const int64_t ncol = (int64_t)n_new * G;
    if (!a.narrow && ncol > 16) return;
    const int cols = (int)min((int64_t)16, ncol - c0);
    const int len = (int)min((int64_t)max(0, a.lens[r]), (int64_t)a.max_blocks << a.pshift);
    // positions of the tile's first and last row, and of this lane's column
    const int p0 = len - n_new;
    const int t_first = c0 / G, t_last = (c0 + cols - 1) / G;
    const bool real = lc < cols;
    const int col = c0 + (real ? lc : 0), tok = col / G, head = g * G + col % G;
    auto low = [&](int p) { return first_key(p, a.window); };
    const int plast = real ? p0 + tok : -1, plow = low(p0 + tok);
    const int kend = max(0, p0 + t_last + 1), k64 = low(p0 + t_first) / 64;
    const int n64 = max(0, (kend + 63) / 64 - k64);
    // Tiles to a workgroup: the S-th part at least.  A round of its four wavefronts takes 1.8 us
    // and a record 0.33 us to join (heads of 128; the rounds of 256 twice that), so where that
    // leaves few, the square root of all (one request of 8,000 keys 18.6 -> 14.9 us, 16,000 20.7
    // -> 17.6); and up to 512 keys stay in one piece (300 keys 9.7 -> 8.5, 500 9.9 -> 8.7; 700
    // 10.0 in three, 10.1 in one).
    const int root = 4 * max(1, (int)((HD > 128 ? 0.18f : 0.25f) * __builtin_amdgcn_sqrtf((float)n64) + 0.5f));
    const int ku = n64 <= 8 ? 8 : max(root, (n64 + a.S - 1) / a.S), T = max(1, (n64 + ku - 1) / ku);
    if (s >= T) return;
    const int tb = s * ku, te = min(n64, tb + ku);

    // ---- tiles: page ids two steps ahead, keys and values one
    const int32_t* const trow = a.table + (int64_t)r * a.max_blocks;
    const int last_block = max(0, (kend - 1) >> a.pshift);
    auto entry = [&](int i, int grp) {   // page of 16 keys of tile i
        return *gptr<int32_t>(trow + min(((k64 + i) * 64 + 16 * grp) >> a.pshift, last_block));
    };
    auto load16 = [&]<class T>(const int8_t* p) {
        if constexpr (NT) return (T)__builtin_nontemporal_load(gptr<T>(p));
        else return (T)*gptr<T>(p);
    };
    // Rows of tile i, whose pages are pk (K lanes) and pv (V lanes).  Behind the last tile
    // every lane reads the pool's first bytes instead: the same loads in every turn of the
    // loop, so that a wait counts exactly those of its own tile, and no traffic.
    auto fetch = [&](QaTile<HD>& x, int i, int pk, int pv) {
        const int key = (k64 + i) * 64;
        const bool live = i < te;
        x.ok = pv >= 0 && pv < a.n_pages;
        const int64_t hk = (int64_t)(pk >= 0 && pk < a.n_pages ? pk : 0) * a.n_kv + g;
        const int64_t hv = (int64_t)(x.ok ? pv : 0) * a.n_kv + g;
        const int64_t ko = (hk * page + ((key + 16 * (lc >> 2) + (lc & 3)) & (page - 1))) * HD + 16 * lg;
        const int64_t vo = (hv * HD + lc) * page + ((key + 16 * lg) & (page - 1));
        const int8_t* const kp = a.Kc + (live ? ko : 0);
        const int8_t* const vp = a.Vc + (live ? vo : 0);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c) x.k[t][c] = load16.template operator()<qa_i4>(kp + 4 * t * HD + 64 * c);
#pragma unroll
        for (int j = 0; j < NJ; ++j) x.v[j] = load16.template operator()<u4v>(vp + 16 * j * page);
        x.sk = *gptr<float>(a.ks + (live ? hv : 0));
        x.sv = *gptr<float>(a.vs + (live ? hv : 0));
    };

    QaQuery<HD> qy;
    QaTile<HD> x0, x1;
    const int i0 = tb + wave;
    int pk = entry(i0, lc >> 2), pv = entry(i0, lg);
    qy.load(a.q + (int64_t)(row0 + tok) * a.q_stride + (int64_t)head * HD);
    const int k2 = pk, v2 = pv;
    pk = entry(i0 + 4, lc >> 2);
    pv = entry(i0 + 4, lg);
    fetch(x0, i0, k2, v2);
    __builtin_amdgcn_sched_barrier(0);
    qy.split(real);
    const float cf = qy.scale * (1.4426950408889634f / sqrtf((float)HD));
    qa_f4 o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = qa_f4{0.f, 0.f, 0.f, 0.f};
    float mm[1] = {-INFINITY}, ll[1] = {0.f};
    const float cfs[1] = {cf};
    QaScale sc;
    auto rescale = [&](float al) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j] *= al;
    };

    auto compute = [&](const QaTile<HD>& x, int i) {
        const int key = (k64 + i) * 64, kk = key + 16 * lg;
        // S: lane l, element e of y[t] holds key 16 (l / 16) + 4 t + e of column l % 16
        float y[1][4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            qa_i4 h{0, 0, 0, 0}, m{0, 0, 0, 0}, w{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                h = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.k[t][c], qy.hi[c], h, 0, 0, 0);
                m = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.k[t][c], qy.mid[c], m, 0, 0, 0);
                w = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.k[t][c], qy.lo[c], w, 0, 0, 0);
            }
            // 256 h + m below 2^31 (256 * 256 * 128 * 129), the rest below 2^22
#pragma unroll
            for (int e = 0; e < 4; ++e) y[0][t][e] = __builtin_fmaf((float)(h[e] * 256 + m[e]), 256.f, (float)w[e]);
            if (t == 1) __builtin_amdgcn_sched_barrier(0);   // two fragments' integer sums at a time
        }
        const bool whole = key + 63 <= p0 + t_first && key >= low(p0 + t_last) && __all(x.ok);
        sc.next(x.sv, x.ok && kk <= p0 + t_last && kk + 15 >= low(p0 + t_first));
        qa_h8 pb[1][4];
        qa_softmax<1, true>(
            y, x.sk, cfs, !whole,
            [&](int, int t, int e) { return !x.ok || kk + 4 * t + e > plast || kk + 4 * t + e < plow; }, sc, mm, ll, pb,
            [&](const float (&al)[1]) { rescale(al[0]); });
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t e0, e1, e2, e3;
                codes_f16(x.v[j][2 * u], e0, e1);
                codes_f16(x.v[j][2 * u + 1], e2, e3);
                const u4v w{e0, e1, e2, e3};
                const qa_h8 vf = __builtin_bit_cast(qa_h8, w);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pb[0][u], o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pb[0][2 + u], o[j], 0, 0, 0);
            }
    };
    // the page ids of the tile after next are requested before the next tile's rows: loads
    // complete in order, so ids behind the rows would hold up the fetch that needs them
    // until the rows have come
    auto ahead = [&](QaTile<HD>& x, int i) {
        const int k1 = pk, v1 = pv;
        pk = entry(i + 4, lc >> 2);
        pv = entry(i + 4, lg);
        fetch(x, i, k1, v1);
    };
    if constexpr (HD <= 128) {
        for (int i = i0; i < te; i += 8) {
            ahead(x1, i + 4);
            compute(x0, i);
            if (i + 4 >= te) break;
            ahead(x0, i + 8);
            compute(x1, i + 4);
        }
    } else {   // one tile's registers
        for (int i = i0; i < te; i += 4) {
            compute(x0, i);
            ahead(x0, i + 4);
        }
    }
    const float m = mm[0], l = quad_sum(ll[0]);

    // ---- the four wavefronts' shares -> head dims j = wave, wave + 4, .. of each
    qa_f4* const so = reinterpret_cast<qa_f4*>(smem);            // [wave][j][lane]
    float* const sml = reinterpret_cast<float*>(so + 4 * NJ * 64);   // [wave][m, l][column]
#pragma unroll
    for (int j = 0; j < NJ; ++j) so[(wave * NJ + j) * 64 + lane] = o[j];
    if (lane < 16) {
        sml[wave * 32 + lane] = m;
        sml[wave * 32 + 16 + lane] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.f, wt[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sml[w * 32 + lc]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float mw = sml[w * 32 + lc];
        wt[w] = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
        L += wt[w] * sml[w * 32 + 16 + lc];
    }
    qa_f4 acc[NJ / 4];
#pragma unroll
    for (int jj = 0; jj < NJ / 4; ++jj) {
        acc[jj] = qa_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) acc[jj] += so[(w * NJ + wave + 4 * jj) * 64 + lane] * wt[w];
    }
    auto store = [&](float sum) {
        if (!real) return;
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        uint16_t* const orow = a.out + (int64_t)(row0 + tok) * a.out_stride + (int64_t)head * HD + 4 * lg;
#pragma unroll
        for (int jj = 0; jj < NJ / 4; ++jj) {
            u2v w;
            w.x = (uint32_t)f2h(acc[jj][0] * inv) | ((uint32_t)f2h(acc[jj][1] * inv) << 16);
            w.y = (uint32_t)f2h(acc[jj][2] * inv) | ((uint32_t)f2h(acc[jj][3] * inv) << 16);
            *reinterpret_cast<qa_any8*>(orow + 16 * (wave + 4 * jj)) = w;
        }
    };
    if (T == 1) {
        store(L);
        return;
    }

    // ---- this split's record, then the sum of all by the last to arrive
    constexpr int kRec = NJ * 1024 + 128;   // O as the lanes hold it, m and l per column
    unsigned char* const grp = a.recs + ((int64_t)tile * a.n_kv + g) * a.S * kRec;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(grp, 0, 0x7fffffff, 0x00020000);
    if (real) {
#pragma unroll
        for (int jj = 0; jj < NJ / 4; ++jj)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4v, acc[jj]), rs,
                                                   s * kRec + (wave + 4 * jj) * 1024 + lane * 16, 0, kSc1);
        if (wave == 0 && lane < 16) {
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(M), rs, s * kRec + NJ * 1024 + 8 * lane, 0, kSc1);
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(L), rs, s * kRec + NJ * 1024 + 8 * lane + 4, 0, kSc1);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint64_t* const word = a.cnt + tile * a.n_kv + g;
    uint32_t* const last = reinterpret_cast<uint32_t*>(smem);
    if (threadIdx.x == 0) {
        *last = tagged_arrive(word, a.tag) == (uint32_t)T ? 1u : 0u;
        if (*last) __hip_atomic_store(word, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last) return;
    // every record's weight exp2(m - M) into LDS: lanes of group lg take the records lg, lg +
    // 4, .. of their column; then O, sixteen records on their way at a time
    float* const sw = reinterpret_cast<float*>(smem) + 16;   // [record][column]
    const int mine = 8 * (real ? lc : 0);
    M = -INFINITY;
    for (int t = lg; t < T; t += 4)
        M = fmaxf(M, __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, t * kRec + NJ * 1024 + mine, 0, kSc1)));
    M = quad_max(M);
    L = 0.f;
    for (int t = lg; t < T; t += 4) {
        const u2v ml = __builtin_bit_cast(u2v, __builtin_amdgcn_raw_buffer_load_b64(rs, t * kRec + NJ * 1024 + mine, 0, kSc1));
        const float mt = __uint_as_float(ml.x), w = mt == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mt - M);
        L += w * __uint_as_float(ml.y);
        if (wave == 0) sw[t * 16 + lc] = w;
    }
    L = quad_sum(L);
    __syncthreads();
#pragma unroll
    for (int jj = 0; jj < NJ / 4; ++jj) acc[jj] = qa_f4{0.f, 0.f, 0.f, 0.f};
    constexpr int B = 32 / (NJ / 4) > 16 ? 16 : 32 / (NJ / 4);   // records at a time
    for (int t0 = 0; t0 < T; t0 += B) {
        u4v ov[B][NJ / 4];
#pragma unroll
        for (int u = 0; u < B; ++u)
#pragma unroll
            for (int jj = 0; jj < NJ / 4; ++jj)
                ov[u][jj] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(
                                                        rs, min(t0 + u, T - 1) * kRec + (wave + 4 * jj) * 1024 + 256 * lg + 2 * mine,
                                                        0, kSc1));
#pragma unroll
        for (int u = 0; u < B; ++u) {
            const float w = t0 + u < T ? sw[(t0 + u) * 16 + lc] : 0.f;
            if (t0 + u < T) {
#pragma unroll
                for (int jj = 0; jj < NJ / 4; ++jj) acc[jj] += __builtin_bit_cast(qa_f4, ov[u][jj]) * w;
            }
        }
    }
    store(L);
}

// Prompt chunks: requests with more than 16 columns, where narrow tiles would cost more (the
// plan below).  A workgroup takes 128 columns of one KV head, a wavefront 32 of them, and all
// four share each tile of 64 keys in LDS as FP16 integers: a thread loads 16 codes at a time
// two tiles ahead, converts them once for the 128 columns and stores them double-buffered
// (one barrier a tile; 16-byte chunks XOR-swizzled).  S^T = K Q^T is then one FP16 product with
// q as it is.
// Prompts of 2,047 and 2,010 rows, 32 / 8 heads of 128: 101 us, 667 TFLOP/s (heads of 64: 72 us;
// 16 / 4 heads of 256: 166); 1,500 rows at 12,000 keys 800.  What bounds it: two wavefronts a
// SIMD (245 registers, 64 KB of LDS a workgroup), whose VALU work (exponents, exponentials,
// sums and the conversion of codes, about 360 instructions for every 64 matrix instructions)
// fills 59 % of the time, the matrix cores a quarter, and 28 % of whose cycles wait, for
// counters or at the tile's barrier.  Eight wavefronts that share a tile convert half as much
// for 5 % and leave a batch half as many workgroups; holding the next tile's conversion over
// the softmax spills (194 us).  Heads of 256 spill as it is (30 registers), at one wavefront a SIMD.
template <int HD>
struct QrShape {
    static constexpr int CH = HD / 8;             // 16-byte chunks of a K row
    static constexpr int kK = 64 * HD * 2;        // bytes of a K tile, as many of V
    static constexpr int kBuf = 2 * kK;
    static constexpr int NI = HD / 64;            // pieces of 16 codes a thread and matrix
    static constexpr int kShare = HD / 16 * 2 * 1024;   // O of a wavefront in a record
    static constexpr int kRec = 4 * kShare + 128 * 8;   // a split's record: O, then m and l per column
    // chunk c of key k sits at c ^ kswz(k), of head dim d at c ^ vswz(d): the 16 lanes that
    // the LDS serves at once, 16 keys of a fragment or 16 head dims, then cover its 64
    // banks, and so do the stores but those of K at 256
    static __device__ __forceinline__ int kswz(int k) {
        return CH == 8 ? ((k >> 4) & 3) << 1 | ((k >> 1) & 1) : ((k >> 4) & 3) << 2 | (k & 3);
    }
    static __device__ __forceinline__ int vswz(int d) { return (d >> 1) & 7; }
};

template <int HD>
__device__ __forceinline__ void qa_rows_tile(const QaArgs& a, unsigned block, unsigned blocks, unsigned char* smem) {
    using S = QrShape<HD>;
    constexpr int NS = HD / 32, NJ = HD / 16, NI = S::NI, KB = HD > 128 ? 1 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lc = lane & 15, lg = lane >> 4, G = a.G, page = 1 << a.pshift;

    // ---- block -> (column tile, split, KV head): the last tiles first, they see the
    // most keys
    const unsigned b = blocks - 1 - block, rest = b / (unsigned)a.n_kv;
    const int g = (int)(b % (unsigned)a.n_kv), s = (int)(rest % (unsigned)a.S);
    const int64_t tile = rest / (unsigned)a.S;
    int r = 0;
    {
        int hi = a.n_req;
        while (hi - r > 1) {
            const int mid = (r + hi) >> 1;
            if ((int64_t)a.starts[mid] * G / 128 + mid <= tile) r = mid;
            else hi = mid;
        }
    }
    const int row0 = a.starts[r], n_new = a.starts[r + 1] - row0;
    const int ti = (int)(tile - ((int64_t)row0 * G / 128 + r));
    if (row0 < 0 || n_new <= 0 || row0 > a.rows - n_new || ti < 0) return;
    const int64_t ncol = (int64_t)n_new * G, c0 = 128 * (int64_t)ti;
    if (c0 >= ncol || ncol <= 16) return;   // up to 16 columns are qa_kernel's
    const int len = (int)min((int64_t)max(0, a.lens[r]), (int64_t)a.max_blocks << a.pshift);
    const int p0 = len - n_new;
    auto low = [&](int p) { return first_key(p, a.window); };
    const int t_first = (int)(c0 / G), t_last = (int)((min(c0 + 128, ncol) - 1) / G);
    const int kend = max(0, p0 + t_last + 1), k64 = low(p0 + t_first) / 64;
    const int n64 = max(0, (kend + 63) / 64 - k64);
    const int ku = max(4, (n64 + a.S - 1) / a.S), T = max(1, (n64 + ku - 1) / ku);
    if (s >= T) return;
    const int tb = s * ku, te = min(n64, tb + ku);

    // ---- this wavefront's columns: fragment f, lane l: column 16 f + l % 16 of its 32
    const int64_t w0 = c0 + 32 * wave;
    const bool works = w0 < ncol;
    bool real[2];
    int tok[2], head[2], plast[2], plow[2];
    qa_h8 qf[2][NS];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        const int64_t c = w0 + 16 * f + lc;
        real[f] = c < ncol;
        const int64_t cc = real[f] ? c : c0;
        tok[f] = (int)(cc / G);
        head[f] = g * G + (int)(cc % G);
        plast[f] = real[f] ? p0 + tok[f] : -1;
        plow[f] = low(p0 + tok[f]);
        const uint16_t* const q = a.q + (int64_t)(row0 + tok[f]) * a.q_stride + (int64_t)head[f] * HD + 8 * lg;
#pragma unroll
        for (int d = 0; d < NS; ++d)
            qf[f][d] = __builtin_bit_cast(qa_h8, (u4v)*reinterpret_cast<const qa_any16*>(q + 32 * d));
    }
    const int w_first = p0 + (int)(min(w0, ncol - 1) / G), w_last = p0 + (int)((min(w0 + 32, ncol) - 1) / G);

    // ---- tiles through registers: piece i of a thread is 16 codes of key 16 grp + .. (K)
    // and of head dim .. (V) of the 16 keys grp = thread / HD + i (256 / HD)
    const int32_t* const trow = a.table + (int64_t)r * a.max_blocks;
    const int last_block = max(0, (kend - 1) >> a.pshift);
    const int in = threadIdx.x % HD, grp0 = __builtin_amdgcn_readfirstlane(threadIdx.x / HD);
    const int kkey = in / (HD / 16), kunit = in % (HD / 16);   // K: key of the 16, piece of the row
    u4v kx[NI], vx[NI];
    // page ids a turn before the rows that they lead to, and those of the lane's 16 keys
    int ids[NI], ps;
    auto page_at = [&](int i, int grp) {
        return *gptr<int32_t>(trow + min(((k64 + i) * 64 + 16 * grp) >> a.pshift, last_block));
    };
    auto look = [&](int i) {
#pragma unroll
        for (int n = 0; n < NI; ++n) ids[n] = page_at(i, grp0 + n * (256 / HD));
        ps = page_at(i, lg);
    };
    auto issue = [&](int i) {
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int key = (k64 + i) * 64 + 16 * (grp0 + n * (256 / HD));
            const int pg = ids[n] < 0 || ids[n] >= a.n_pages ? 0 : ids[n];
            const int64_t hp = (int64_t)pg * a.n_kv + g;
            kx[n] = *gptr<u4v>(a.Kc + (hp * page + (key & (page - 1)) + kkey) * HD + 16 * kunit);
            vx[n] = *gptr<u4v>(a.Vc + (hp * HD + in) * page + (key & (page - 1)));
        }
    };
    auto land = [&](int buf) {
        unsigned char* const kt = smem + buf * S::kBuf;
        unsigned char* const vt = kt + S::kK;
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int grp = grp0 + n * (256 / HD), key = 16 * grp + kkey;
            u4v* const krow = reinterpret_cast<u4v*>(kt + key * HD * 2);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t x0, x1, x2, x3;
                codes_f16(kx[n][2 * e], x0, x1);
                codes_f16(kx[n][2 * e + 1], x2, x3);
                krow[(2 * kunit + e) ^ S::kswz(key)] = u4v{x0, x1, x2, x3};
            }
            u4v* const vrow = reinterpret_cast<u4v*>(vt + in * 128);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t x0, x1, x2, x3;
                codes_f16(vx[n][2 * e], x0, x1);
                codes_f16(vx[n][2 * e + 1], x2, x3);
                vrow[(2 * grp + e) ^ S::vswz(in)] = u4v{x0, x1, x2, x3};
            }
        }
    };
    // the scales of the lane's 16 keys and whether their page is one
    float sk, sv, sk2, sv2;
    bool ok, ok2;
    auto scales = [&] {
        ok2 = ps >= 0 && ps < a.n_pages;
        const int64_t hp = (int64_t)(ok2 ? ps : 0) * a.n_kv + g;
        sk2 = *gptr<float>(a.ks + hp);
        sv2 = *gptr<float>(a.vs + hp);
    };

    qa_f4 o[2][NJ];
    float m[2], l[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        m[f] = -INFINITY;
        l[f] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[f][j] = qa_f4{0.f, 0.f, 0.f, 0.f};
    }
    const float sl2 = 1.4426950408889634f / sqrtf((float)HD), cfs[2] = {sl2, sl2};
    QaScale sc;
    if (tb < te) {
        look(tb);
        issue(tb);
        scales();
        look(tb + 1);
        land(0);
        issue(tb + 1);
    }
    __syncthreads();
    for (int i = tb; i < te; ++i) {
        const int cur = (i - tb) & 1, key = (k64 + i) * 64;
        const unsigned char* const kt = smem + cur * S::kBuf;
        const unsigned char* const vt = kt + S::kK;
        sk = sk2;
        sv = sv2;
        ok = ok2;
        scales();   // of the next tile
        look(i + 2);
        if (works && key <= w_last && key + 63 >= low(w_first)) {
            // fragments from LDS a step ahead of the products that take them (heads of 256
            // have no registers for K's)
            float y[2][4][4];
            qa_h8 kf[KB][NS];
            auto k_read = [&](int t) {
                const int kr = 16 * (lc >> 2) + 4 * t + (lc & 3);
#pragma unroll
                for (int d = 0; d < NS; ++d)
                    kf[t % KB][d] = *reinterpret_cast<const qa_h8*>(kt + kr * HD * 2 + (((4 * d + lg) ^ S::kswz(kr)) << 4));
            };
            if (KB > 1) k_read(0);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (t + KB - 1 < 4) k_read(t + KB - 1);
                if constexpr (KB > 1) __builtin_amdgcn_sched_barrier(0);
                qa_f4 acc[2] = {qa_f4{0.f, 0.f, 0.f, 0.f}, qa_f4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int d = 0; d < NS; ++d)
#pragma unroll
                    for (int f = 0; f < 2; ++f)
                        acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t % KB][d], qf[f][d], acc[f], 0, 0, 0);
#pragma unroll
                for (int f = 0; f < 2; ++f)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[f][t][e] = acc[f][e];
            }
            const bool whole = key + 63 <= w_first && key >= low(w_last) && __all(ok);
            const int kk = key + 16 * lg;
            sc.next(sv, ok && kk <= w_last && kk + 15 >= low(w_first));
            qa_h8 pb[2][2];
            qa_softmax<2, false>(
                y, sk, cfs, !whole,
                [&](int f, int t, int e) { return !ok || kk + 4 * t + e > plast[f] || kk + 4 * t + e < plow[f]; }, sc, m, l, pb,
                [&](const float (&al)[2]) {
#pragma unroll
                    for (int f = 0; f < 2; ++f)
#pragma unroll
                        for (int j = 0; j < NJ; ++j) o[f][j] *= al[f];
                });
            qa_h8 vf[2][2];
            auto v_read = [&](int j) {
                const int d = 16 * j + lc;
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    vf[j % 2][u] = *reinterpret_cast<const qa_h8*>(vt + d * 128 + (((2 * lg + u) ^ S::vswz(d)) << 4));
            };
            v_read(0);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                if (j + 1 < NJ) v_read(j + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int f = 0; f < 2; ++f)
                        o[f][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[j % 2][u], pb[f][u], o[f][j], 0, 0, 0);
            }
        }
        if (i + 1 < te) {
            land(cur ^ 1);
            if (i + 2 < te) issue(i + 2);   // (a tile past the last has the last block's page)
        }
        __syncthreads();
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) l[f] = quad_sum(l[f]);
    auto store = [&](int f, float sum) {
        if (!real[f]) return;
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        uint16_t* const orow = a.out + (int64_t)(row0 + tok[f]) * a.out_stride + (int64_t)head[f] * HD + 4 * lg;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            u2v w;
            w.x = (uint32_t)f2h(o[f][j][0] * inv) | ((uint32_t)f2h(o[f][j][1] * inv) << 16);
            w.y = (uint32_t)f2h(o[f][j][2] * inv) | ((uint32_t)f2h(o[f][j][3] * inv) << 16);
            *reinterpret_cast<qa_any8*>(orow + 16 * j) = w;
        }
    };
    if (T == 1) {
        if (works) {
            store(0, l[0]);
            store(1, l[1]);
        }
        return;
    }

    // ---- this split's record; the last workgroup adds them in split order, each
    // wavefront its own columns
    unsigned char* const grp = a.recs + (tile * a.n_kv + g) * (int64_t)a.S * S::kRec;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(grp, 0, 0x7fffffff, 0x00020000);
    auto o_at = [&](int t, int f, int j) { return t * S::kRec + wave * S::kShare + (f * NJ + j) * 1024 + lane * 16; };
    auto ml_at = [&](int t, int f) { return t * S::kRec + 4 * S::kShare + (32 * wave + 16 * f + lc) * 8; };
    if (works) {
#pragma unroll
        for (int f = 0; f < 2; ++f) {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4v, o[f][j]), rs, o_at(s, f, j), 0, kSc1);
            if (lane < 16)
                __builtin_amdgcn_raw_buffer_store_b64(u2v{__float_as_uint(m[f]), __float_as_uint(l[f])}, rs, ml_at(s, f), 0, kSc1);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint64_t* const word = a.cnt + tile * a.n_kv + g;
    uint32_t* const last = reinterpret_cast<uint32_t*>(smem);   // (the tiles are done with)
    if (threadIdx.x == 0) {
        *last = tagged_arrive(word, a.tag) == (uint32_t)T ? 1u : 0u;
        if (*last) __hip_atomic_store(word, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last || !works) return;
    float M[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f};
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int f = 0; f < 2; ++f)
            M[f] = fmaxf(M[f], __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, ml_at(t, f), 0, kSc1)));
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[f][j] = qa_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int t = 0; t < T; ++t) {
        u2v ml[2];
        u4v ov[2][NJ];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            ml[f] = __builtin_bit_cast(u2v, __builtin_amdgcn_raw_buffer_load_b64(rs, ml_at(t, f), 0, kSc1));
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                ov[f][j] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(rs, o_at(t, f, j), 0, kSc1));
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const u2v x = ml[f];
            const float mt = __uint_as_float(x.x), w = mt == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mt - M[f]);
            L[f] += w * __uint_as_float(x.y);
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[f][j] += __builtin_bit_cast(qa_f4, ov[f][j]) * w;
        }
    }
    store(0, L[0]);
    store(1, L[1]);
}

template <int HD, bool NT>
__global__ __launch_bounds__(kQaThreads, HD > 128 ? 1 : 2) void qa_kernel(QaArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    qa_tile<HD, NT>(a, blockIdx.x, smem);
}

// Both kinds of tiles in one launch, the long ones first: decode rows fill the CUs that
// the chunks leave, or leave last.
template <int HD>
__global__ __launch_bounds__(kQaThreads, HD > 128 ? 1 : 2) void qa_both_kernel(QaArgs rows, QaArgs a, unsigned row_blocks) {
    extern __shared__ __align__(16) unsigned char smem[];
    if (blockIdx.x < row_blocks) qa_rows_tile<HD>(rows, blockIdx.x, row_blocks, smem);
    else qa_tile<HD, false>(a, blockIdx.x - row_blocks, smem);
}

// How a call is laid out.  Requests of up to 16 columns: a tile each in qa_kernel, their
// keys over S workgroups; where longer ones are allowed for (max_new), those as several
// such tiles (narrow), or in qa_rows_tile, `tiles` of 128 columns at most, their keys over
// Sr workgroups.
struct QaPlan {
    bool rows_too, narrow;
    int S, Sr;
    int64_t tiles16, tiles;
    size_t rec_bytes, rrec_bytes;
    // the counters have a place of their own whatever the call's shape, so that a workspace
    // that serves different shapes keeps them at zero
    static constexpr size_t kCounters = (size_t)2 * kQaWords * 8;
    size_t bytes() const { return kCounters + rec_bytes + rrec_bytes; }
};

QaPlan qa_plan(int rows, int n_req, int n_q, int n_kv, int hd, int max_new, int max_len) {
    QaPlan p{};
    const int64_t G = n_q / n_kv, cus = num_cus();
    auto up = [](int64_t x) { return ((size_t)x + 255) / 256 * 256; };
    // `tiles` of 16 columns at most, `likely` of them with any
    auto small = [&](int64_t tiles, int64_t likely) {
        // about a workgroup a CU, and no more than 4096 keys to one (ragged batches: a long
        // conversation among short ones); 256 keys, a tile for each wavefront, at least.
        // 16 requests of 750 to 1,500 keys, 16 / 8 heads of 128: 1 a CU 14.4 us, 2 a CU 16.5;
        // one of 16,000, 32 / 8 heads: 17.6 and 24.7; 48 of 8,000 to 16,000: 4096 keys to one
        // 209 us, 2048 223, 8192 226.
        const int64_t rec = hd * 64 + 128;
        const int64_t S = std::min<int64_t>({std::max<int64_t>({1, cus / (likely * n_kv), ((int64_t)max_len + 4095) / 4096}),
                                             ((int64_t)max_len + 255) / 256, kQaMaxSplits, kQaRecBytes / (tiles * n_kv * rec)});
        p.tiles16 = tiles;
        p.S = tiles * n_kv > kQaWords ? 1 : (int)std::max<int64_t>(1, S);
        p.rec_bytes = p.S > 1 ? up(tiles * n_kv * p.S * rec) : 0;
    };
    small(n_req, n_req);
    p.rows_too = (int64_t)max_new * G > 16;
    // what the batch is taken to be: requests with one row and, as many as the rest needs,
    // with max_new
    const int64_t more = std::max<int64_t>(0, (int64_t)rows - n_req), most = std::max(2, max_new);
    const int64_t longer = std::min<int64_t>(n_req, (more + most - 2) / (most - 1));
    if (p.rows_too && n_req <= kQaNarrowReq) {
        // Narrow tiles for all rows: 31 us for a million keys of a tile of 16 columns where the
        // chip is full, against 14 with all of a tile of 128, which is paid for whole; and
        // where it is not full, more workgroups with less to do.  32 / 8 heads of 128, narrow
        // against 128: 48 requests of 8,000 to 16,000 keys, 8 rows each 313 and 471 us, 12 411
        // and 578; 16 of 750 to 1,500, 8 rows 17.0 and 29.4, 16 rows 25.3 and 35.8, 32 rows
        // 42.2 and 41.7; one of 8,000, 64 rows 33.6 and 41.4; one prompt of 300, 16 / 8
        // heads 10.8 and 16.8, of 1,000 27.2 and 26.8.  (Above kQaNarrowReq requests a few rows each
        // go to tiles of 128: 256 requests of 750 to 1,500 keys, 8 rows each, 183 us, 257 of them 244.)
        const int64_t likely = n_req - longer + ((more + longer) * G + 15) / 16;
        if ((int64_t)max_new * G <= kQaNarrowCols || likely * n_kv * max_len <= kQaNarrowWork / hd) {
            small(n_req + (int64_t)rows * G / 16, likely);
            p.narrow = true;
            p.rows_too = false;
        }
    }
    if (p.rows_too) {
        // `tiles` at most.  As many workgroups as have room at once, two a CU (one with heads
        // of 256), less one for every second CU where single tokens need some; a few more
        // would run alone at the end.  32 / 8 heads of 128: 400 rows beside 7 single tokens at
        // 6,000 keys 77 us in four parts, 97 in five (520 workgroups), 90 in three; 500 beside
        // 39 at 4,000 89 in three, 104 in four; three of 126 to 200 rows and one token at 3,000
        // 53 in three, 64 in four (544).  16 / 4 heads of 256, 500 rows at 4,000 90 in four,
        // 122 in eight.
        p.tiles = (int64_t)rows * G / 128 + n_req;
        const int64_t tb = p.tiles * n_kv, rec = (int64_t)hd * 512 + 1024, slots = hd > 128 ? cus : 2 * cus;
        const int64_t singles = hd > 128 ? 0 : std::min(cus / 2, (n_req - longer) * n_kv * p.S);
        const int64_t likely = std::max<int64_t>(1, ((more + longer) * G + 127) / 128 + longer - 1) * n_kv;
        const int64_t cap = std::max<int64_t>(1, std::min(((int64_t)max_len + 511) / 512, kQaRecBytes / (tb * rec)));
        int64_t Sr = std::max<int64_t>(1, std::min({(slots - singles + likely / 2) / likely, slots / likely, cap}));
        // More than one round where that is shorter by 15 %: a part takes its share of the
        // keys and about four tiles' time to begin and to join (32 / 8 heads of 128, 1,500 rows
        // at 8,000 keys: one round of 376 workgroups 281 us, 254 in parts; 1,100 beside 29
        // single tokens at 12,000 447 and 358; 16 / 4 heads of 256, three chunks of 326 to 400
        // rows at 2,000: 148 workgroups 142, 444 127).
        auto time = [&](int64_t n) { return ((likely * n + slots - 1) / slots) * (max_len / 64.0 / n + 4.0); };
        const double once = time(Sr);
        double least = 0.85 * once;
        for (int64_t n = slots / likely + 1; n <= std::min<int64_t>(8, cap); ++n)
            if (time(n) < least) {
                least = time(n);
                Sr = n;
            }
        p.Sr = tb > kQaWords ? 1 : (int)Sr;
        p.rrec_bytes = p.Sr > 1 ? up(tb * p.Sr * rec) : 0;
    }
    return p;
}

}  // namespace
}  // namespace bx

using namespace bx;

extern "C" {

size_t bx_attention_paged_q8_workspace_bytes(int rows, int n_req, int n_q, int n_kv, int hd, int max_new, int max_len) {
    if (rows <= 0 || n_req <= 0 || n_kv <= 0 || n_q <= 0 || n_q % n_kv || hd <= 0 || max_new <= 0 || max_len <= 0) return 0;
    return qa_plan(rows, n_req, n_q, n_kv, hd, max_new, max_len).bytes();
}

int bx_attention_paged_q8_f16(const uint16_t* q, int64_t q_stride, int rows, const int32_t* starts, const int32_t* lens,
                              int n_req, int max_new, int max_len, const int32_t* table, int max_blocks, int page,
                              int n_pages, const int8_t* Kc, const int8_t* Vc, const float* k_scale,
                              const float* v_scale, int n_q, int n_kv, int hd, int window, uint16_t* out,
                              int64_t out_stride, void* ws, size_t ws_bytes, void* stream) {
    if (!q || !starts || !lens || !table || !out || !ws) return fail(BX_EINVAL, "attention_paged_q8: null pointer");
    if (int rc = kv_cache_check("attention_paged_q8", n_kv, hd, page, n_pages, Kc, Vc, k_scale, v_scale)) return rc;
    if (rows <= 0 || n_req <= 0 || max_new <= 0 || max_len <= 0 || max_blocks <= 0 || n_q <= 0 || n_q % n_kv || window < 0)
        return fail(BX_EINVAL, "attention_paged_q8: bad shape");
    if (n_q / n_kv > kQaMaxGroup) return fail(BX_EUNSUPPORTED, "attention_paged_q8: GQA group larger than 16");
    if (q_stride < (int64_t)n_q * hd || out_stride < (int64_t)n_q * hd)
        return fail(BX_EINVAL, "attention_paged_q8: row stride below n_q * head_dim");
    if ((int64_t)max_blocks * page > 0x7fffffff - 4095)   // the tiles asked for ahead lie below 2^31 too
        return fail(BX_EUNSUPPORTED, "attention_paged_q8: more than 2^31 - 4096 tokens a request");
    const QaPlan p = qa_plan(rows, n_req, n_q, n_kv, hd, max_new, max_len);
    if (ws_bytes < p.bytes() || (reinterpret_cast<uintptr_t>(ws) & 15))
        return fail(BX_EINVAL, "attention_paged_q8: workspace too small or not 16-byte aligned");
    const int64_t blocks = p.tiles16 * n_kv * p.S, rblocks = p.tiles * n_kv * p.Sr;
    if (blocks + rblocks > 0x7fffffff)
        return fail(BX_EUNSUPPORTED, "attention_paged_q8: too many rows and heads");
    QaArgs a{};
    a.q = q; a.q_stride = q_stride; a.rows = rows; a.starts = starts; a.lens = lens; a.n_req = n_req;
    a.table = table; a.max_blocks = max_blocks; a.pshift = __builtin_ctz((unsigned)page); a.n_pages = n_pages;
    a.Kc = Kc; a.Vc = Vc; a.ks = k_scale; a.vs = v_scale;
    a.n_kv = n_kv; a.G = n_q / n_kv; a.window = window; a.out = out; a.out_stride = out_stride;
    unsigned char* const w = static_cast<unsigned char*>(ws);
    QaArgs ar = a;
    a.narrow = p.narrow;
    a.S = p.S;
    a.cnt = reinterpret_cast<uint64_t*>(w);
    a.recs = w + QaPlan::kCounters;
    a.tag = next_launch_tag();
    ar.S = p.Sr;
    ar.cnt = a.cnt + kQaWords;
    ar.recs = a.recs + p.rec_bytes;
    ar.tag = next_launch_tag();
    hipStream_t st = as_stream(stream);
    auto run = [&](auto hdc) -> int {
        constexpr int HD = decltype(hdc)::value, lds = HD / 16 * 4096 + 512, rlds = 2 * QrShape<HD>::kBuf;
        auto allow = [&](std::atomic<uint64_t>& done, auto kernel, int bytes) {
            return bytes <= 64 * 1024 ? BX_OK : allow_lds(done, reinterpret_cast<const void*>(kernel), bytes,
                                                          "attention_paged_q8: LDS attribute");
        };
        if (p.rows_too) {
            static std::atomic<uint64_t> allowed{0};
            if (int rc = allow(allowed, &qa_both_kernel<HD>, std::max(lds, rlds))) return rc;
            qa_both_kernel<HD><<<(unsigned)(blocks + rblocks), kQaThreads, std::max(lds, rlds), st>>>(ar, a, (unsigned)rblocks);
        } else {
            // streaming loads where the keys may be more than the 256 MB cache holds (48
            // requests of 8,000 to 16,000 keys, 1.2 GB: 226 -> 209 us); smaller sets may
            // still be there (16 of 750 to 1,500, 37 MB: 14.4 us, streaming 16.6), and heads of
            // 256, one wavefront a SIMD, wait longer for them (234 us, streaming 243); the narrow
            // tiles of a request share its keys (48 of 8,000 to 16,000, 8 rows each: 313 us,
            // streaming 406)
            const bool nt = HD <= 128 && !p.narrow && (int64_t)n_req * max_len * n_kv * hd * 2 > (int64_t)256 << 20;
            const auto kernel = nt ? qa_kernel<HD, HD <= 128> : qa_kernel<HD, false>;
            static std::atomic<uint64_t> allowed[2];
            if (int rc = allow(allowed[nt], kernel, lds)) return rc;
            kernel<<<(unsigned)blocks, kQaThreads, lds, st>>>(a);
        }
        return launch_check("attention_paged_q8");
    };
    if (hd == 64) return run(std::integral_constant<int, 64>{});
    if (hd == 128) return run(std::integral_constant<int, 128>{});
    return run(std::integral_constant<int, 256>{});
}

}  // extern "C"
