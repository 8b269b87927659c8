// Attention of a batched step over the paged 8-bit KV cache (layout and entry
// points in kv_pages.hip and brolm_hip.h): decode rows and prompt chunks of
// several requests in one call.
//
// A request's rows and the query heads of one KV head make columns, column c =
// (row c / G, head c % G); a workgroup takes 16 columns of one KV head and walks
// their keys in tiles of 64, one tile per wavefront at a time:
//   S^T = K Q^T on v_mfma_i32_16x16x64_i8, the codes of K as they are stored: q is
//         written as 256 hi + lo in two 8-bit parts times a power of two, both
//         products are exact, and S = 256 S_hi + S_lo has q to 2^-15 of its largest
//         element (components above 2^-5 of it exactly);
//   softmax in FP32 (base 2, running maximum and sum per column); a tile's scales
//         enter as one factor per 16 keys, which lie in one page;
//   O^T += V^T P^T on v_mfma_f32_16x16x32_f16: V codes as FP16 integers, P times
//         its page's scale of V.  That factor is taken relative to the largest
//         scale so far, as a power of two with 2^7 in reserve, so P stays inside
//         FP16 (below 2^15) and a page 2^20 times smaller than the largest still has
//         11 bits.
// The 16 keys that a lane holds of S^T are consecutive (fragment t takes the rows
// 16 i + 4 t + j): P is an operand as it stands, and its V^T counterpart is one
// 16-byte load of 16 tokens of a head dim, as the cache stores them.  K and V go
// from memory to the matrix operands without LDS.
//
// A column tile's keys are split over workgroups where there are few tiles; each
// leaves a record (O, m, l), the last one to arrive adds them in split order.
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
constexpr int kQaReserve = 7;   // 2^(8 + 7) < 65504
constexpr int kQaMinExp = 6;    // least exponent field of the reference scale

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
    int direct, S;
    uint64_t* cnt;
    unsigned char* recs;
    uint32_t tag;
};

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

__device__ __forceinline__ float quad_max(float v) {   // over lanes l, l ^ 16, l ^ 32, l ^ 48
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// The query columns of a wavefront as B operands of the integer products: lane l
// holds column l % 16, head dims 64 c + 16 (l / 16) .. of part c.
template <int HD>
struct QaQuery {
    qa_i4 hi[HD / 64], lo[HD / 64];
    float scale;   // q = (256 hi + lo) scale; NaN where q holds one or an infinity

    __device__ __forceinline__ void load(const uint16_t* col, bool real) {
        const int lane = threadIdx.x & 63;
        u4v w[HD / 64][2];
        uint32_t m = 0u;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                w[c][i] = *reinterpret_cast<const qa_any16*>(col + 64 * c + 16 * (lane >> 4) + 8 * i);
                if (!real) w[c][i] = u4v{0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t a = w[c][i][e] & 0x7fff7fffu;
                    m = max(m, max(a & 0xffffu, a >> 16));
                }
            }
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        const float amax = h2f((uint16_t)m);
        const bool fin = m < 0x7c00u;
        // the power of two that brings amax just below 32640 = 127 * 256 + 128
        int k = 14 - ((int)(__float_as_uint(amax) >> 23) - 127);
        if (amax * exp2_int(k) >= 32639.5f) --k;
        const float mul = fin && m > 0u ? exp2_int(k) : 0.f;
        scale = fin ? (m > 0u ? exp2_int(-k) : 0.f) : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint32_t h4 = 0u, l4 = 0u;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int e = 4 * d + b;
                    const uint16_t x = (uint16_t)(w[c][e / 8][(e % 8) / 2] >> (16 * (e & 1)));
                    const int q = fin ? (int)rintf(h2f(x) * mul) : 0;
                    const int h = (q + 128) >> 8;
                    h4 |= (uint32_t)(h & 0xff) << (8 * b);
                    l4 |= (uint32_t)((q - 256 * h) & 0xff) << (8 * b);
                }
                hi[c][d] = (int)h4;
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

template <int HD>
__global__ __launch_bounds__(kQaThreads, HD > 128 ? 1 : 2) void qa_kernel(QaArgs a) {
    constexpr int NC = HD / 64, NJ = HD / 16;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lc = lane & 15, lg = lane >> 4, G = a.G, page = 1 << a.pshift;

    // ---- block -> (column tile, split, KV head), the KV head fastest: with 8 of
    // them an XCD keeps to one, and the tiles of a request share its L2
    const int g = (int)(blockIdx.x % (unsigned)a.n_kv);
    const int64_t rest = blockIdx.x / (unsigned)a.n_kv;
    const int s = (int)(rest % a.S);
    const int64_t tile = rest / a.S;
    int r = (int)tile, ti = 0;
    if (!a.direct) {
        // request r owns the tiles from starts[r] G / 16 + r on (at least as many as
        // its columns fill)
        int lo = 0, hi = a.n_req;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((int64_t)a.starts[mid] * G / 16 + mid <= tile) lo = mid;
            else hi = mid;
        }
        r = lo;
        ti = (int)(tile - ((int64_t)a.starts[r] * G / 16 + r));
    }
    const int row0 = a.starts[r], n_new = a.starts[r + 1] - row0;
    if (row0 < 0 || n_new <= 0 || row0 > a.rows - n_new || ti < 0) return;
    const int64_t ncol = (int64_t)n_new * G, c0 = 16 * (int64_t)ti;
    if (c0 >= ncol) return;
    const int cols = (int)min((int64_t)16, ncol - c0);
    const int len = (int)min((int64_t)a.lens[r], (int64_t)a.max_blocks << a.pshift);
    // positions of the tile's first and last row, and of this lane's column
    const int p0 = len - n_new;
    const int t_first = (int)(c0 / G), t_last = (int)((c0 + cols - 1) / G);
    const bool real = lc < cols;
    const int64_t col = c0 + (real ? lc : 0);
    const int tok = (int)(col / G), head = g * G + (int)(col % G);
    auto low = [&](int p) { return a.window > 0 ? max(0, p - a.window + 1) : 0; };
    const int plast = real ? p0 + tok : -1, plow = low(p0 + tok);
    const int kend = max(0, p0 + t_last + 1), k64 = low(p0 + t_first) / 64;
    const int n64 = max(0, (kend + 63) / 64 - k64);
    const int ku = max(4, (n64 + a.S - 1) / a.S), T = max(1, (n64 + ku - 1) / ku);
    if (s >= T) return;
    const int tb = s * ku, te = min(n64, tb + ku);

    // ---- tiles: page ids two steps ahead, keys and values one
    const int32_t* const trow = a.table + (int64_t)r * a.max_blocks;
    const int last_block = max(0, (kend - 1) >> a.pshift);
    auto entry = [&](int i, int grp) {   // page of 16 keys of tile i
        return trow[min(((k64 + i) * 64 + 16 * grp) >> a.pshift, last_block)];
    };
    auto fetch = [&](QaTile<HD>& x, int i, int pk, int pv) {
        const int key = (k64 + i) * 64;
        x.ok = pv >= 0 && pv < a.n_pages;
        const int64_t hk = (int64_t)(pk >= 0 && pk < a.n_pages ? pk : 0) * a.n_kv + g;
        const int64_t hv = (int64_t)(x.ok ? pv : 0) * a.n_kv + g;
        const int8_t* const kp =
            a.Kc + (hk * page + ((key + 16 * (lc >> 2) + (lc & 3)) & (page - 1))) * HD + 16 * lg;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c) x.k[t][c] = *gptr<qa_i4>(kp + 4 * t * HD + 64 * c);
        const int8_t* const vp = a.Vc + (hv * HD + lc) * page + ((key + 16 * lg) & (page - 1));
#pragma unroll
        for (int j = 0; j < NJ; ++j) x.v[j] = *gptr<u4v>(vp + (int64_t)16 * j * page);
        x.sk = a.ks[hv];
        x.sv = a.vs[hv];
    };

    QaQuery<HD> qy;
    QaTile<HD> x0, x1;
    int i0 = tb + wave;
    int pk = 0, pv = 0;
    if (i0 < te) {
        pk = entry(i0, lc >> 2);
        pv = entry(i0, lg);
    }
    qy.load(a.q + (int64_t)(row0 + tok) * a.q_stride + (int64_t)head * HD, real);
    if (i0 < te) fetch(x0, i0, pk, pv);
    if (i0 + 4 < te) {
        pk = entry(i0 + 4, lc >> 2);
        pv = entry(i0 + 4, lg);
    }
    const float cf = qy.scale * (1.4426950408889634f / sqrtf((float)HD));
    qa_f4 o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = qa_f4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    int eref = kQaMinExp;

    auto compute = [&](const QaTile<HD>& x, int i) {
        const int key = (k64 + i) * 64;
        // S: lane l, element r of y[t] holds key 16 (l / 16) + 4 t + r of column l % 16
        float y[4][4];
        const float f = cf * x.sk;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            qa_i4 h{0, 0, 0, 0}, w{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                h = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.k[t][c], qy.hi[c], h, 0, 0, 0);
                w = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.k[t][c], qy.lo[c], w, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) y[t][e] = (float)(h[e] * 256 + w[e]) * f;
        }
        const bool whole = key + 63 <= p0 + t_first && key >= low(p0 + t_last) && __all(x.ok);
        const int kk = key + 16 * lg;
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!x.ok || kk + 4 * t + e > plast || kk + 4 * t + e < plow) y[t][e] = -INFINITY;
        }
        float mx = y[0][0];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, y[t][e]);
        mx = quad_max(mx);
        if (__any(mx > m + (float)kQaLazy)) {
            const float mn = fmaxf(m, mx), al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[j] *= al;
            m = mn;
        }
        // the scale of V: a NaN or an infinity takes no part in the reference
        const bool fin = x.sv < INFINITY;
        int ev = fin ? (int)(__float_as_uint(x.sv) >> 23) : 0;
        ev = max(ev, __shfl_xor(ev, 16));
        ev = __builtin_amdgcn_readfirstlane(max(ev, __shfl_xor(ev, 32)));
        if (ev > eref) {
            const float al = exp2_int(eref - ev);
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[j] *= al;
            eref = ev;
        }
        const float rv = x.sv * exp2_int(126 + kQaReserve - eref);
        const float nm = m == -INFINITY ? 0.f : -m;
        qa_h8 pb[2];
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(y[t][e] + nm);
                ls[e] += p;
                pb[t / 2][4 * (t % 2) + e] = (_Float16)(p * rv);
            }
        if (__any(!fin)) {   // a hidden key weighs nothing whatever its page's scale
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (y[t][e] == -INFINITY) pb[t / 2][4 * (t % 2) + e] = (_Float16)0.f;
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                u4v w;
                uint32_t e0, e1, e2, e3;
                codes_f16(x.v[j][2 * u], e0, e1);
                codes_f16(x.v[j][2 * u + 1], e2, e3);
                w = u4v{e0, e1, e2, e3};
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(qa_h8, w), pb[u], o[j], 0, 0, 0);
            }
    };
    auto next_ids = [&](int i) {
        if (i < te) {
            pk = entry(i, lc >> 2);
            pv = entry(i, lg);
        }
    };
    if constexpr (HD <= 128) {
        for (int i = i0; i < te;) {
            if (i + 4 < te) fetch(x1, i + 4, pk, pv);
            next_ids(i + 8);
            compute(x0, i);
            i += 4;
            if (i >= te) break;
            if (i + 4 < te) fetch(x0, i + 4, pk, pv);
            next_ids(i + 8);
            compute(x1, i);
            i += 4;
        }
    } else {   // one tile's registers
        for (int i = i0; i < te; i += 4) {
            compute(x0, i);
            if (i + 4 < te) fetch(x0, i + 4, pk, pv);
            next_ids(i + 8);
        }
    }
    l = quad_sum(l);
    const float unit = exp2_int(eref - 126 - kQaReserve);

    // ---- the four wavefronts' shares -> head dims j = wave, wave + 4, .. of each
    qa_f4* const so = reinterpret_cast<qa_f4*>(smem);            // [wave][j][lane]
    float* const sml = reinterpret_cast<float*>(so + 4 * NJ * 64);   // [wave][m, l][column]
#pragma unroll
    for (int j = 0; j < NJ; ++j) so[(wave * NJ + j) * 64 + lane] = o[j] * unit;
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
    unsigned char* const grp = a.recs + (tile * a.n_kv + g) * (int64_t)a.S * kRec;
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
    M = -INFINITY;
    for (int t = 0; t < T; ++t)
        M = fmaxf(M, __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, t * kRec + NJ * 1024 + 8 * (real ? lc : 0), 0, kSc1)));
    L = 0.f;
#pragma unroll
    for (int jj = 0; jj < NJ / 4; ++jj) acc[jj] = qa_f4{0.f, 0.f, 0.f, 0.f};
    for (int t0 = 0; t0 < T; t0 += 4) {
        u2v ml[4];
        u4v ov[4][NJ / 4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = min(t0 + u, T - 1);
            ml[u] = __builtin_bit_cast(u2v, __builtin_amdgcn_raw_buffer_load_b64(rs, t * kRec + NJ * 1024 + 8 * (real ? lc : 0), 0, kSc1));
#pragma unroll
            for (int jj = 0; jj < NJ / 4; ++jj)
                ov[u][jj] = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(
                                                        rs, t * kRec + (wave + 4 * jj) * 1024 + (16 * lg + (real ? lc : 0)) * 16, 0, kSc1));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (t0 + u >= T) break;
            const float mt = __uint_as_float(ml[u].x), w = mt == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mt - M);
            L += w * __uint_as_float(ml[u].y);
#pragma unroll
            for (int jj = 0; jj < NJ / 4; ++jj) acc[jj] += __builtin_bit_cast(qa_f4, ov[u][jj]) * w;
        }
    }
    store(L);
}

// How a call is laid out: 16 columns at most per request (direct: a tile is a
// request) or tiles over all columns; splits of a tile's keys.
struct QaPlan {
    int direct, S;
    int64_t tiles;
    size_t cnt_bytes, rec_bytes;
};

QaPlan qa_plan(int rows, int n_req, int n_q, int n_kv, int hd, int max_new, int max_len) {
    QaPlan p{};
    const int G = n_q / n_kv, cus = num_cus();
    p.direct = (int64_t)max_new * G <= 16;
    p.tiles = p.direct ? n_req : (int64_t)rows * G / 16 + n_req;
    // two workgroups a CU, and no more than 2048 keys to one where a tile is a
    // request (ragged batches: one long conversation among short ones); at least
    // 256 keys, a tile for each wavefront
    const int64_t blocks = p.tiles * n_kv;
    int64_t S = std::max<int64_t>(1, 2 * cus / blocks);
    if (p.direct) S = std::max<int64_t>(S, (max_len + 2047) / 2048);
    p.S = (int)std::min<int64_t>({S, (max_len + 255) / 256, 1024});
    p.cnt_bytes = ((size_t)blocks * 8 + 255) / 256 * 256;
    p.rec_bytes = p.S > 1 ? (size_t)blocks * p.S * (hd * 64 + 128) : 0;
    return p;
}

}  // namespace
}  // namespace bx

using namespace bx;

extern "C" {

size_t bx_attention_paged_q8_workspace_bytes(int rows, int n_req, int n_q, int n_kv, int hd, int max_new, int max_len) {
    if (rows <= 0 || n_req <= 0 || n_kv <= 0 || n_q <= 0 || n_q % n_kv || hd <= 0 || max_new <= 0 || max_len <= 0) return 0;
    const QaPlan p = qa_plan(rows, n_req, n_q, n_kv, hd, max_new, max_len);
    return p.cnt_bytes + p.rec_bytes;
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
    if ((int64_t)max_blocks * page > 0x7fffffff - 128)
        return fail(BX_EUNSUPPORTED, "attention_paged_q8: more than 2^31 - 129 tokens a request");
    const QaPlan p = qa_plan(rows, n_req, n_q, n_kv, hd, max_new, max_len);
    if (ws_bytes < p.cnt_bytes + p.rec_bytes || (reinterpret_cast<uintptr_t>(ws) & 15))
        return fail(BX_EINVAL, "attention_paged_q8: workspace too small or not 16-byte aligned");
    if (p.tiles * n_kv * p.S > 0x7fffffff) return fail(BX_EUNSUPPORTED, "attention_paged_q8: too many rows and heads");
    QaArgs a{};
    a.q = q; a.q_stride = q_stride; a.rows = rows; a.starts = starts; a.lens = lens; a.n_req = n_req;
    a.table = table; a.max_blocks = max_blocks; a.pshift = __builtin_ctz((unsigned)page); a.n_pages = n_pages;
    a.Kc = Kc; a.Vc = Vc; a.ks = k_scale; a.vs = v_scale;
    a.n_kv = n_kv; a.G = n_q / n_kv; a.window = window; a.out = out; a.out_stride = out_stride;
    a.direct = p.direct; a.S = p.S;
    a.cnt = static_cast<uint64_t*>(ws);
    a.recs = static_cast<unsigned char*>(ws) + p.cnt_bytes;
    a.tag = next_launch_tag();
    const dim3 grid((unsigned)(p.tiles * n_kv * p.S));
    const int lds = hd / 16 * 4096 + 512;
    hipStream_t st = as_stream(stream);
    if (hd == 64) {
        qa_kernel<64><<<grid, kQaThreads, lds, st>>>(a);
    } else if (hd == 128) {
        qa_kernel<128><<<grid, kQaThreads, lds, st>>>(a);
    } else {
        static std::atomic<uint64_t> allowed{0};
        if (int rc = allow_lds(allowed, reinterpret_cast<const void*>(&qa_kernel<256>), lds, "attention_paged_q8: LDS attribute"))
            return rc;
        qa_kernel<256><<<grid, kQaThreads, lds, st>>>(a);
    }
    return launch_check("attention_paged_q8");
}

}  // extern "C"
