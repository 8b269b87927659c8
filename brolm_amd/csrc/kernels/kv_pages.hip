// The paged 8-bit KV cache of a batched step: which page a token goes to
// (bx_kv_plan), its K / V rows into the pages (bx_kv_append_q8_f16) and rows
// back out (bx_kv_read_q8_f16).  The attention over it is attention_q8.hip.
//
// A page holds P tokens of every KV head: K codes [page][head][token][hd] and V
// codes [page][head][hd][token], so that the attention's matrix operands (16
// bytes along hd for Q K^T, 16 bytes along the tokens for P V) are plain 16-byte
// loads.  One FP32 scale per page, head and matrix: value = code * scale, codes
// in [-127, 127].
#include <type_traits>

#include "kv_pages.h"

namespace bx {
namespace {

// ------------------------------------------------------------------ the plan
//
// Request r grows by delta[r] tokens (or gives -delta[r] back).  Every workgroup
// forms the same prefix sums over the requests in LDS (rows of the step, pages
// taken, pages given back), then fills its own share of the rows and of the moved
// pages: a row finds its request by binary search.  The state that a caller may
// hand over in place (lens over past, the ring's ends) is written by the workgroup
// that arrives last, when all have read it.
// Latency bounds it: 16 requests with a token each 3.9 us, 384 requests with 36,000 rows 8.3
// (0.6 MB; the prefix, the search and the last workgroup's turn one after the other).

constexpr int kPlanThreads = 256;
constexpr int kPlanRows = 512;    // rows per workgroup

struct PlanArgs {
    const int32_t *past, *delta;
    int n_req, pshift, n_pages, max_blocks, max_rows;
    int32_t *table, *ring;
    const int64_t* ends_in;
    int64_t* ends_out;
    int32_t *lens, *starts, *pos, *status;
    int64_t* slots;
    uint64_t* word;
    uint32_t tag;
};

// Exclusive prefixes of three values over the workgroup in thread order, and their sums.
__device__ __forceinline__ void plan_scan(int64_t (&v)[3], int64_t (&total)[3], int64_t (*red)[kPlanThreads / 64]) {
    const int w = threadIdx.x >> 6;
    int64_t inc[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        inc[i] = wave_prefix(v[i]);
        if ((threadIdx.x & 63) == 63) red[i][w] = inc[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        int64_t before = 0, sum = 0;
#pragma unroll
        for (int k = 0; k < kPlanThreads / 64; ++k) {
            if (k < w) before += red[i][k];
            sum += red[i][k];
        }
        total[i] = sum;
        v[i] = before + inc[i] - v[i];
    }
}

// The last i in [0, n) with p[i] <= x (p ascending, p[0] = 0 <= x).
__device__ __forceinline__ int plan_find(const int32_t* p, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs a) {
    // per request: first row, pages taken and pages given before it
    __shared__ int32_t s_row[kPlanMaxReq], s_take[kPlanMaxReq], s_give[kPlanMaxReq];
    __shared__ int64_t red[3][kPlanThreads / 64];
    __shared__ int s_bad;
    __shared__ uint32_t s_last;
    const int t = threadIdx.x, n = a.n_req, page = 1 << a.pshift;
    const int64_t head = a.ends_in[0], tail = a.ends_in[1], room = (int64_t)a.max_blocks << a.pshift;
    if (t == 0) s_bad = 0;
    __syncthreads();

    // ---- prefix sums, `per` consecutive requests a thread
    const int per = (n + kPlanThreads - 1) / kPlanThreads, r0 = min(n, t * per), r1 = min(n, r0 + per);
    int64_t rows = 0, take = 0, give = 0;
    int bad = 0;
    for (int r = r0; r < r1; ++r) {
        const int64_t old = a.past[r], d = a.delta[r], len = old + d;
        if (old < 0 || len < 0 || old > room) bad |= BX_KV_PLAN_BAD_LENGTH;
        else if (len > room) bad |= BX_KV_PLAN_TABLE_FULL;
        else {
            const int ob = (int)((old + page - 1) >> a.pshift), nb = (int)((len + page - 1) >> a.pshift);
            rows += d > 0 ? d : 0;
            take += nb > ob ? nb - ob : 0;
            give += ob > nb ? ob - nb : 0;
        }
    }
    int64_t pre[3] = {rows, take, give}, sum[3];
    plan_scan(pre, sum, red);
    rows = pre[0], take = pre[1], give = pre[2];
    const int64_t n_rows = sum[0], n_take = sum[1], n_give = sum[2];
    if (head < 0 || tail < head || tail - head > a.n_pages || tail - head + n_give > a.n_pages) bad |= BX_KV_PLAN_BAD_RING;
    else if (n_take > tail - head) bad |= BX_KV_PLAN_NO_PAGES;
    if (n_rows > a.max_rows) bad |= BX_KV_PLAN_ROWS_FULL;
    if (bad) atomicOr(&s_bad, bad);
    __syncthreads();
    bad = s_bad;
    if (!bad)
        for (int r = r0; r < r1; ++r) {
            const int old = a.past[r], d = a.delta[r];
            const int ob = (int)(((int64_t)old + page - 1) >> a.pshift), nb = (int)(((int64_t)old + d + page - 1) >> a.pshift);
            s_row[r] = (int)rows;
            s_take[r] = (int)take;
            s_give[r] = (int)give;
            rows += d > 0 ? d : 0;
            take += nb > ob ? nb - ob : 0;
            give += ob > nb ? ob - nb : 0;
        }
    __syncthreads();

    // ---- the rows: position and slot; -1 behind the last one
    const int live = bad ? 0 : (int)n_rows;
    const int hm = bad ? 0 : (int)(head % a.n_pages), tm = bad ? 0 : (int)(tail % a.n_pages);
    auto ring_at = [&](int base, int i) { return base < a.n_pages - i ? base + i : base - (a.n_pages - i); };
    auto blocks_of = [&](int len) { return (int)(((int64_t)len + page - 1) >> a.pshift); };
    const int first = (int)blockIdx.x * kPlanRows, n_own = min(a.max_rows - first, kPlanRows);   // (up to 2^31 - 1 rows)
    for (int o = t; o < n_own; o += kPlanThreads) {
        const int i = first + o;
        int p = -1;
        int64_t slot = -1;
        if (i < live) {
            const int r = plan_find(s_row, n, i), old = a.past[r];
            p = old + i - s_row[r];
            const int b = p >> a.pshift, ob = blocks_of(old);
            const int pg = b < ob ? a.table[(int64_t)r * a.max_blocks + b] : a.ring[ring_at(hm, s_take[r] + b - ob)];
            if (pg >= 0 && pg < a.n_pages) slot = ((int64_t)pg << a.pshift) + (p & (page - 1));
        }
        a.pos[i] = p;
        a.slots[i] = slot;
    }
    // ---- the pages: taken ones from the ring's head to the table, given ones from
    // the table to its tail (the ring's used part and the entries read are not
    // written: a page is in the ring or in the table)
    if (!bad) {
        for (int i = (int)blockIdx.x * kPlanThreads + t; i < (int)n_take; i += (int)gridDim.x * kPlanThreads) {
            const int r = plan_find(s_take, n, i);
            a.table[(int64_t)r * a.max_blocks + blocks_of(a.past[r]) + i - s_take[r]] = a.ring[ring_at(hm, i)];
        }
        for (int i = (int)blockIdx.x * kPlanThreads + t; i < (int)n_give; i += (int)gridDim.x * kPlanThreads) {
            const int r = plan_find(s_give, n, i);
            const int kept = blocks_of(a.past[r] + a.delta[r]);
            a.ring[ring_at(tm, i)] = a.table[(int64_t)r * a.max_blocks + kept + i - s_give[r]];
        }
    }
    // ---- the requests' state, by the last workgroup to come here
    __syncthreads();
    if (gridDim.x > 1) {
        if (t == 0) {
            s_last = tagged_arrive(a.word, a.tag) == gridDim.x ? 1u : 0u;
            if (s_last) __hip_atomic_store(a.word, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!s_last) return;
    }
    for (int r = t; r < n; r += kPlanThreads) {
        a.lens[r] = a.past[r] + (bad ? 0 : a.delta[r]);
        a.starts[r] = bad ? 0 : s_row[r];
    }
    if (t == 0) {
        a.starts[n] = live;
        a.ends_out[0] = head + (bad ? 0 : n_take);
        a.ends_out[1] = tail + (bad ? 0 : n_give);
        a.status[0] = bad;
    }
}

// ---------------------------------------------------------------- the append
//
// A run is a row whose predecessor in the call is not the token before it in the
// same page, with the rows after it that are: the tokens that one page receives.
// Per run, head and matrix:
//   amax over the run, s = max(s_old, amax / 127) (s_old = 0 for a page that was
//   empty); where s grew, the page's earlier codes c become rint(c s_old / s); the
//   new codes are rint(x / s).
// Both roundings are exact to the last border: a new code's remainder x - q s is
// exact in FP32 (x and q s are multiples of s's last place, and the remainder is
// below s), the earlier codes' quotient is formed in FP64, where c s_old is exact.
// |x| is compared as the FP16 bit pattern, which orders NaN last: a page with a
// NaN or an infinity gets such a scale, and every value of it becomes NaN or infinite.
//
// A wavefront's unit is 16 tokens of one head, in registers from the one load to
// the store: of K a lane holds 8 head dims of hd / 32 tokens, of V 4 head dims of hd /
// 16 consecutive tokens, which are consecutive bytes of the token-minor page.  Every
// byte is read, requantized and written by one lane.  A run inside one unit (a decode
// step's rows) is one wavefront's; for a longer one the four wavefronts of a workgroup are
// the units of the page (and of 4 / (units) heads where a page has fewer) and share its
// amax through LDS.
// 16 rows of 8 heads of 128: 4.4 us, slots, scale and rows, stores in series.  Three prompts of
// 7,389 rows: 15.6 us for 46 MB, 2.9 TB/s: a workgroup's runs come one after the other, slots,
// rows, the maximum's barrier, codes, and the rounding is a third of the time (19.7 us with the
// exact form for every value).  Heads of 256 in pages of 128 spill 13 registers.

typedef u4v __attribute__((aligned(2))) any16;
typedef u2v __attribute__((aligned(2))) any8;

struct AppendArgs {
    const uint16_t* x[2];   // K rows, V rows
    int64_t stride[2];
    int rows, n_kv, pshift, window;
    int64_t n_slots;
    const int64_t* slots;
    int8_t* codes[2];
    float* scale[2];
};

// rint(x / s), ties to even; inv is about 1 / s, s > 0 and finite.
__device__ __forceinline__ int q8_code(float x, float s, float inv) {
    const float q = rintf(x * inv);
    const float r = __builtin_fmaf(-q, s, x), a = fabsf(r), h = 0.5f * s;
    // one step off at most: the remainder says whether and which way (equal: the even one)
    const bool off = (a > h) | ((a == h) & (((int)q & 1) != 0));
    return (int)q + (off ? (r > 0.f ? 1 : -1) : 0);
}

__device__ __forceinline__ uint32_t pk_max_abs(uint32_t m, uint32_t x) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    const us2 a = __builtin_bit_cast(us2, m), b = __builtin_bit_cast(us2, x & 0x7fff7fffu);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
}

__device__ __forceinline__ int byte_of(uint32_t w, int i) { return (int8_t)(w >> (8 * i)); }
__device__ __forceinline__ uint32_t put_byte(uint32_t w, int i, int c) {
    return (w & ~(0xffu << (8 * i))) | ((uint32_t)(c & 0xff) << (8 * i));
}

// WHICH 0: K, 1: V; NCH units of 16 tokens a page.  SOLO: the run lies inside one unit, head
// hs of the workgroup's; else hs is not read.
template <int HD, int WHICH, int NCH, bool SOLO>
__device__ __forceinline__ void append_run(const AppendArgs& a, int row, int n, int64_t slot, int hs, uint32_t* red) {
    constexpr int HPW = NCH < 4 ? 4 / NCH : 1;           // heads a workgroup takes
    constexpr int U = NCH > 4 && !SOLO ? NCH / 4 : 1;    // units a wavefront takes
    constexpr int page = 16 * NCH;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (!SOLO) hs = NCH < 4 ? wave / NCH : 0;
    const int head = (int)blockIdx.y * HPW + hs;
    const bool there = head < a.n_kv;
    const int off = (int)(slot & (page - 1));
    auto unit = [&](int u) { return SOLO ? off >> 4 : (NCH < 4 ? wave % NCH : wave) + 4 * u; };
    const int64_t hp = (slot >> a.pshift) * a.n_kv + (there ? head : 0);
    const int64_t st = a.stride[WHICH];
    // row of token tk of the page: x + tk st
    const uint16_t* const x = a.x[WHICH] + ((int64_t)row - off) * st + (int64_t)head * HD;
    float* const sp = a.scale[WHICH] + hp;
    int8_t* const codes = a.codes[WHICH] + hp * page * HD;
    const uint32_t old_bits = off > 0 && there ? __float_as_uint(*sp) : 0u;
    // K: piece j of a lane is token kt + j KR, head dims kd ..; V: row j of a lane is
    // token vt + j, head dims vd .. vd + 3
    constexpr int KL = HD / 32, KR = 512 / HD, VT = HD / 16;
    const int kt = lane / (HD / 8), kd = 8 * (lane % (HD / 8));
    const int vt = lane / (HD / 4) * VT, vd = 4 * (lane % (HD / 4));
    u4v kx[U][KL];
    u2v vx[U][VT];
    uint32_t old[U][4][VT / 4];   // V: the lane's bytes of 4 head dims
    uint32_t m2 = 0u;
    auto fresh = [&](int tk) { return tk >= off && tk < off + n; };
    auto v_piece = [&](int c, int d) { return codes + (int64_t)(vd + d) * page + 16 * c + vt; };
    auto load_old = [&](int u, int c) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const uint32_t* const p = reinterpret_cast<const uint32_t*>(v_piece(c, d));
#pragma unroll
            for (int i = 0; i < VT / 4; ++i) old[u][d][i] = p[i];
        }
    };
    bool has_new[U], part[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = unit(u), t0 = 16 * c;
        has_new[u] = there && t0 < off + n && t0 + 16 > off;
        part[u] = has_new[u] && WHICH == 1 && !(t0 + vt >= off && t0 + vt + VT <= off + n);
        // tokens outside the run read its nearest row and count as zero: loads without
        // branches between them
        auto near = [&](int tk) { return x + (int64_t)min(max(tk, off), off + n - 1) * st; };
        if constexpr (WHICH == 0) {
            if (has_new[u]) {
#pragma unroll
                for (int j = 0; j < KL; ++j) kx[u][j] = *reinterpret_cast<const any16*>(near(t0 + kt + j * KR) + kd);
#pragma unroll
                for (int j = 0; j < KL; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        m2 = pk_max_abs(m2, kx[u][j][i] & (fresh(t0 + kt + j * KR) ? 0xffffffffu : 0u));
            }
        } else if (has_new[u]) {
            if (part[u]) load_old(u, c);
#pragma unroll
            for (int j = 0; j < VT; ++j) vx[u][j] = *reinterpret_cast<const any8*>(near(t0 + vt + j) + vd);
#pragma unroll
            for (int j = 0; j < VT; ++j) {
                const uint32_t in = fresh(t0 + vt + j) ? 0xffffffffu : 0u;
                m2 = pk_max_abs(pk_max_abs(m2, vx[u][j].x & in), vx[u][j].y & in);
            }
        }
    }
    uint32_t m = max(m2 & 0xffffu, m2 >> 16);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    if constexpr (NCH > 1 && !SOLO) {
        if (lane == 0) red[wave] = m;
        __syncthreads();
        m = 0u;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (NCH >= 4 || w / NCH == hs) m = max(m, red[w]);
    }
    if (!there) return;
    const uint32_t new_bits = max(old_bits, __float_as_uint(h2f((uint16_t)m) / 127.0f));
    const float s_old = __uint_as_float(old_bits), s = __uint_as_float(new_bits);
    const bool live = s > 0.f && s < INFINITY;   // else every code is 0
    const float div = live ? s : INFINITY, inv = live ? 1.0f / s : 0.f;
    const bool grew = off > 0 && new_bits != old_bits;
    if ((SOLO || unit(0) == 0) && lane == 0) *sp = s;
    const uint32_t mask = live ? 0xffffffffu : 0u;
    // the codes of four values, half h of each of four dwords: x inv + 1.5 2^23 has the rounded
    // integer in its low byte.  x inv is x / s to 127 2^-24: right unless it lies within 2e-5
    // of a half, which some lane's does one time in a hundred
    auto code4 = [&](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, int h0, int h1, int h2, int h3) -> uint32_t {
        auto val = [&](uint32_t w, int h) { return h2f((uint16_t)((w & mask) >> (16 * h))); };
        const float x4[4] = {val(w0, h0), val(w1, h1), val(w2, h2), val(w3, h3)};
        uint32_t u[4];
        float far = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y = __builtin_fmaf(x4[i], inv, 12582912.f);
            far = fmaxf(far, fabsf(__builtin_fmaf(x4[i], inv, -(y - 12582912.f))));
            u[i] = __float_as_uint(y);
        }
        if (__any(far > 0.49998f)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = (uint32_t)q8_code(x4[i], div, inv);
        }
        const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
        return lo | hi;
    };
    // the earlier codes of one dword, the first of them token tk's and the others
    // `step` tokens apart, requantized in place
    auto move4 = [&](uint32_t* p, int tk, int step) {
        uint32_t y = *p;
#pragma unroll 1
        for (int b = 0; b < 4; ++b)
            if (tk + b * step < off)
                y = put_byte(y, b, live ? (int)rint((double)byte_of(y, b) * (double)s_old / (double)s) : 0);
        *p = y;
    };
    if (grew) {
        auto move = [&](int c) {
            const int t0 = 16 * c;
            if constexpr (WHICH == 0) {
#pragma unroll 1
                for (int j = 0; j < 2 * KL; ++j) {
                    const int tk = t0 + kt + j / 2 * KR;
                    if (tk < off) move4(reinterpret_cast<uint32_t*>(codes + tk * HD + kd) + (j & 1), tk, 0);
                }
            } else {
#pragma unroll 1
                for (int d = 0; d < 4; ++d)
#pragma unroll 1
                    for (int i = 0; i < VT / 4; ++i)
                        if (t0 + vt + 4 * i < off) move4(reinterpret_cast<uint32_t*>(v_piece(c, d)) + i, t0 + vt + 4 * i, 1);
            }
        };
        if constexpr (SOLO) {
#pragma unroll 1
            for (int c = 0; 16 * c < off; ++c) move(c);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (16 * unit(u) < off) move(unit(u));
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (part[u]) load_old(u, unit(u));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = unit(u), t0 = 16 * c;
        if (!has_new[u]) continue;
        if constexpr (WHICH == 0) {
#pragma unroll
            for (int j = 0; j < KL; ++j) {
                const int tk = t0 + kt + j * KR;
                if (fresh(tk)) {
                    const u4v w = kx[u][j];
                    *reinterpret_cast<u2v*>(codes + tk * HD + kd) =
                        u2v{code4(w.x, w.x, w.y, w.y, 0, 1, 0, 1), code4(w.z, w.z, w.w, w.w, 0, 1, 0, 1)};
                }
            }
        } else if (t0 + vt < off + n && t0 + vt + VT > off) {   // new tokens among the lane's
#pragma unroll
            for (int i = 0; i < VT / 4; ++i) {
                // bytes of the run's tokens
                const int tk = t0 + vt + 4 * i, lo = min(4, max(0, off - tk)), hi = min(4, max(0, off + n - tk));
                const uint32_t keep = ~(hi > lo ? (0xffffffffu >> (8 * (4 - hi + lo))) << (8 * lo) : 0u);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t y = code4(vx[u][4 * i][d / 2], vx[u][4 * i + 1][d / 2], vx[u][4 * i + 2][d / 2],
                                             vx[u][4 * i + 3][d / 2], d & 1, d & 1, d & 1, d & 1);
                    old[u][d][i] = part[u] ? (old[u][d][i] & keep) | (y & ~keep) : y;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < VT / 4; ++i) reinterpret_cast<uint32_t*>(v_piece(c, d))[i] = old[u][d][i];
        }
    }
}

// Workgroup (window of rows, heads, K or V): the runs that start in its window.
template <int HD, int NCH>
__global__ __launch_bounds__(256, HD > 128 ? 3 : 4) void kv_append_kernel(AppendArgs a) {
    __shared__ uint32_t red[2][4];
    const int64_t row0 = (int64_t)blockIdx.x * a.window;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int page = 16 * NCH, HPW = NCH < 4 ? 4 / NCH : 1;
    auto slot_at = [&](int64_t r) { return r >= 0 && r < a.rows ? a.slots[r] : -1; };
    // lane l: row row0 + l; what starts a run in the window, and what continues none
    const int64_t r = row0 + lane, own = slot_at(r), prev = slot_at(r - 1);
    const bool valid = own >= 0 && own < a.n_slots, next = valid && (own & (page - 1)) != 0 && own == prev + 1;
    const uint64_t starts = __ballot(lane < a.window && valid && !next), stops = __ballot(!next);
    // runs inside one unit: a wavefront each
    uint64_t longer = 0;
    int turn = 0;
    for (uint64_t todo = starts; todo; todo &= todo - 1) {
        const int i = __builtin_ctzll(todo);
        const uint64_t behind = i < 63 ? stops >> (i + 1) : 0;
        const int64_t slot = __shfl(own, i);
        const int n = behind ? __builtin_ctzll(behind) + 1 : 64;
        if (n > 16 - (int)(slot & 15)) {
            longer |= 1ull << i;
            continue;
        }
        // wavefront w: head w % HPW of the workgroup's, every (4 / HPW)th run
        if (turn++ % (4 / HPW) != wave / HPW) continue;
        if (blockIdx.z == 0) append_run<HD, 0, NCH, true>(a, (int)(row0 + i), n, slot, wave % HPW, nullptr);
        else append_run<HD, 1, NCH, true>(a, (int)(row0 + i), n, slot, wave % HPW, nullptr);
    }
    if constexpr (NCH == 1) return;   // a page is one unit
    // longer ones: all four, one after the other (red alternates: one barrier a run)
    for (int k = 0; longer; k ^= 1) {
        const int i = __builtin_ctzll(longer);
        longer &= longer - 1;
        const int row = (int)(row0 + i);
        const int64_t slot = __shfl(own, i);
        const int left = page - (int)(slot & (page - 1));   // tokens to the page's end
        const uint64_t behind = i < 63 ? stops >> (i + 1) : 0;
        int n = behind ? __builtin_ctzll(behind) + 1 : 64 - i;
        if (!behind)
            for (int q = n; q < left; q += 64) {
                const uint64_t same = __ballot(q + lane < left && slot_at((int64_t)row + q + lane) == slot + q + lane);
                const int c = ~same ? __builtin_ctzll(~same) : 64;
                n += c;
                if (c < 64) break;
            }
        if (blockIdx.z == 0) append_run<HD, 0, NCH, false>(a, row, n, slot, 0, red[k]);
        else append_run<HD, 1, NCH, false>(a, row, n, slot, 0, red[k]);
    }
}

// ------------------------------------------------------------------ the read
//
// A wavefront takes 16 rows of one head.  Of K a lane reads 16 codes of a row.  Of V
// it takes the pieces of 16 tokens of a page that begin among its rows (a row that
// is not the next token of the row before it, or the first of a piece): a lane holds
// 4 head dims of hd / 16 tokens.
// 203 rows of 8 heads of 128: 4.4 us, slots, then codes and scales.  30,011 rows of 8 heads of
// 64, 92 MB: 26 us from memory, 3.5 TB/s (a copy has 5.2), 20 us where the 256 MB cache still
// has the codes.
struct ReadArgs {
    const int64_t* slots;
    int rows, n_kv, pshift;
    int64_t n_slots;
    const int8_t* codes[2];
    const float* scale[2];
    uint16_t* y[2];
    int64_t stride[2];
};

__device__ __forceinline__ uint32_t q8_pair(int c0, int c1, float s) {
    return (uint32_t)f2h(f32_fence((float)c0 * s)) | ((uint32_t)f2h(f32_fence((float)c1 * s)) << 16);
}

template <int HD>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int which = (int)(item & 1), head = (int)((item >> 1) % a.n_kv);
    const int64_t row0 = (item >> 1) / a.n_kv * 16;
    const int lane = threadIdx.x & 63, page = 1 << a.pshift;
    if (row0 >= a.rows) return;
    auto slot_at = [&](int64_t r) { return r >= 0 && r < a.rows ? a.slots[r] : -1; };
    if (which == 0) {
        constexpr int LR = HD / 16, RP = 64 / LR;   // lanes a row, rows at once
        int64_t slot[16 / RP];
        u4v w[16 / RP];
        float s[16 / RP];
#pragma unroll
        for (int j = 0; j < 16 / RP; ++j) {
            slot[j] = slot_at(row0 + j * RP + lane / LR);
            if (slot[j] >= a.n_slots) slot[j] = -1;
        }
#pragma unroll
        for (int j = 0; j < 16 / RP; ++j) {
            const int64_t at = slot[j] < 0 ? 0 : slot[j], hp = (at >> a.pshift) * a.n_kv + head;
            w[j] = *gptr<u4v>(a.codes[0] + (hp * page + (at & (page - 1))) * HD + 16 * (lane % LR));
            s[j] = a.scale[0][hp];
        }
#pragma unroll
        for (int j = 0; j < 16 / RP; ++j) {
            if (slot[j] < 0) continue;
            any16* const y = reinterpret_cast<any16*>(a.y[0] + (row0 + j * RP + lane / LR) * a.stride[0] +
                                                      (int64_t)head * HD + 16 * (lane % LR));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u4v z;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t b = w[j][2 * h + i / 2];
                    z[i] = q8_pair(byte_of(b, 2 * (i & 1)), byte_of(b, 2 * (i & 1) + 1), s[j]);
                }
                y[h] = z;
            }
        }
        return;
    }
    const int64_t own = slot_at(row0 + lane), prev = slot_at(row0 + lane - 1);
    const bool first = lane < 16 && own >= 0 && own < a.n_slots && ((own & 15) == 0 || own != prev + 1);
    uint64_t todo = __ballot(first);
    constexpr int VT = HD / 16;
    const int vt = lane / (HD / 4) * VT, vd = 4 * (lane % (HD / 4));
    while (todo) {
        const int i = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int64_t slot = __shfl(own, i);
        const int o = (int)(slot & 15);   // its place in the piece
        const uint64_t same = __ballot(lane < 16 - o && slot_at(row0 + i + lane) == slot + lane);
        const int n = __builtin_ctzll(~same);
        const int64_t hp = (slot >> a.pshift) * a.n_kv + head;
        const int8_t* const p = a.codes[1] + (hp * HD + vd) * page + ((slot & (page - 1)) - o) + vt;
        const float s = a.scale[1][hp];
        uint32_t w[4][VT / 4];
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int q = 0; q < VT / 4; ++q) w[d][q] = reinterpret_cast<const uint32_t*>(p + d * page)[q];
#pragma unroll
        for (int j = 0; j < VT; ++j) {
            const int tk = vt + j;
            if (tk < o || tk >= o + n) continue;
            u2v z;
            z.x = q8_pair(byte_of(w[0][j / 4], j % 4), byte_of(w[1][j / 4], j % 4), s);
            z.y = q8_pair(byte_of(w[2][j / 4], j % 4), byte_of(w[3][j / 4], j % 4), s);
            *reinterpret_cast<any8*>(a.y[1] + (row0 + i + tk - o) * a.stride[1] + (int64_t)head * HD + vd) = z;
        }
    }
}

}  // namespace

int kv_cache_check(const char* what, int n_kv, int hd, int page, int n_pages, const int8_t* Kc, const int8_t* Vc,
                const float* ks, const float* vs) {
    if (!Kc || !Vc || !ks || !vs) return fail(BX_EINVAL, std::string(what) + ": null cache pointer");
    if (n_kv <= 0 || n_pages <= 0) return fail(BX_EINVAL, std::string(what) + ": bad cache shape");
    if (!kv_page_ok(page)) return fail(BX_EUNSUPPORTED, std::string(what) + ": pages hold 16, 32, 64 or 128 tokens");
    if (hd != 64 && hd != 128 && hd != 256)
        return fail(BX_EUNSUPPORTED, std::string(what) + ": head_dim must be 64, 128 or 256");
    if ((reinterpret_cast<uintptr_t>(Kc) | reinterpret_cast<uintptr_t>(Vc)) & 15)
        return fail(BX_EINVAL, std::string(what) + ": codes not 16-byte aligned");
    return BX_OK;
}

}  // namespace bx

using namespace bx;

extern "C" {

size_t bx_kv_plan_workspace_bytes(void) { return 256; }

int bx_kv_plan(const int32_t* past, const int32_t* delta, int n_req, int page, int n_pages, int32_t* table,
               int max_blocks, int32_t* ring, const int64_t* ends_in, int64_t* ends_out, int32_t* lens, int32_t* starts,
               int64_t* slots, int32_t* pos, int max_rows, int32_t* status, void* ws, size_t ws_bytes, void* stream) {
    if (!past || !delta || !table || !ring || !ends_in || !ends_out || !lens || !starts || !slots || !pos || !status || !ws)
        return fail(BX_EINVAL, "kv_plan: null pointer");
    if (n_req <= 0 || n_pages <= 0 || max_blocks <= 0 || max_rows <= 0) return fail(BX_EINVAL, "kv_plan: bad shape");
    if (n_req > kPlanMaxReq) return fail(BX_EUNSUPPORTED, "kv_plan: more than 4096 requests");
    if (!kv_page_ok(page)) return fail(BX_EUNSUPPORTED, "kv_plan: pages hold 16, 32, 64 or 128 tokens");
    if ((int64_t)max_blocks * page > 0x7fffffff) return fail(BX_EUNSUPPORTED, "kv_plan: more than 2^31 - 1 tokens a request");
    if (ws_bytes < bx_kv_plan_workspace_bytes() || (reinterpret_cast<uintptr_t>(ws) & 7))
        return fail(BX_EINVAL, "kv_plan: workspace too small or not 8-byte aligned");
    if (delta == lens || starts == past || starts == delta || starts == lens)
        return fail(BX_EINVAL, "kv_plan: only lens may lie over past, and ends_out over ends_in");
    PlanArgs a{};
    a.past = past; a.delta = delta; a.n_req = n_req; a.pshift = __builtin_ctz((unsigned)page); a.n_pages = n_pages;
    a.max_blocks = max_blocks; a.max_rows = max_rows; a.table = table; a.ring = ring; a.ends_in = ends_in;
    a.ends_out = ends_out; a.lens = lens; a.starts = starts; a.pos = pos; a.status = status; a.slots = slots;
    a.word = static_cast<uint64_t*>(ws);
    a.tag = next_launch_tag();
    const unsigned grid = ((unsigned)max_rows + kPlanRows - 1) / kPlanRows;
    kv_plan_kernel<<<grid, kPlanThreads, 0, as_stream(stream)>>>(a);
    return launch_check("kv_plan");
}

int bx_kv_append_q8_f16(const uint16_t* k, int64_t k_stride, const uint16_t* v, int64_t v_stride, int rows, int n_kv,
                        int hd, const int64_t* slots, int page, int n_pages, int8_t* Kc, int8_t* Vc, float* k_scale,
                        float* v_scale, void* stream) {
    if (!k || !v || !slots) return fail(BX_EINVAL, "kv_append_q8: null pointer");
    if (int rc = kv_cache_check("kv_append_q8", n_kv, hd, page, n_pages, Kc, Vc, k_scale, v_scale)) return rc;
    const int64_t width = (int64_t)n_kv * hd;
    if (rows <= 0 || k_stride < width || v_stride < width) return fail(BX_EINVAL, "kv_append_q8: bad shape");
    AppendArgs a{};
    a.x[0] = k; a.x[1] = v; a.stride[0] = k_stride; a.stride[1] = v_stride;
    a.rows = rows; a.n_kv = n_kv; a.pshift = __builtin_ctz((unsigned)page);
    a.n_slots = (int64_t)n_pages * page;
    a.slots = slots; a.codes[0] = Kc; a.codes[1] = Vc; a.scale[0] = k_scale; a.scale[1] = v_scale;
    // a row to a workgroup for few rows, as many as it has wavefronts for their heads where
    // rows are many (decode rows are a wavefront each), 32 for prompts: three of 7,389 rows
    // together, 8 heads of 128, pages of 64, 15.6 us (16 rows a workgroup 24.0; 64 the same, but
    // 18.4 for 16.6 with pages of 128), 1,000 decode rows 29.2 us (a row a workgroup 34.9)
    const int per = page < 64 ? 64 / page : 1;   // heads a workgroup takes
    a.window = rows <= 256 ? 1 : rows <= 2048 ? 4 / per : 32;
    const unsigned windows = ((unsigned)rows + a.window - 1) / a.window;
    if ((n_kv + per - 1) / per > 65535) return fail(BX_EUNSUPPORTED, "kv_append_q8: too many heads");
    const dim3 grid(windows, (unsigned)((n_kv + per - 1) / per), 2);
    hipStream_t st = as_stream(stream);
    auto run = [&](auto hdc) {
        constexpr int HD = decltype(hdc)::value;
        if (page == 16) kv_append_kernel<HD, 1><<<grid, 256, 0, st>>>(a);
        else if (page == 32) kv_append_kernel<HD, 2><<<grid, 256, 0, st>>>(a);
        else if (page == 64) kv_append_kernel<HD, 4><<<grid, 256, 0, st>>>(a);
        else kv_append_kernel<HD, 8><<<grid, 256, 0, st>>>(a);
    };
    if (hd == 64) run(std::integral_constant<int, 64>{});
    else if (hd == 128) run(std::integral_constant<int, 128>{});
    else run(std::integral_constant<int, 256>{});
    return launch_check("kv_append_q8");
}

int bx_kv_read_q8_f16(const int64_t* slots, int rows, int n_kv, int hd, int page, int n_pages, const int8_t* Kc,
                      const int8_t* Vc, const float* k_scale, const float* v_scale, uint16_t* k, int64_t k_stride,
                      uint16_t* v, int64_t v_stride, void* stream) {
    if (!k || !v || !slots) return fail(BX_EINVAL, "kv_read_q8: null pointer");
    if (int rc = kv_cache_check("kv_read_q8", n_kv, hd, page, n_pages, Kc, Vc, k_scale, v_scale)) return rc;
    const int64_t width = (int64_t)n_kv * hd;
    if (rows <= 0 || k_stride < width || v_stride < width) return fail(BX_EINVAL, "kv_read_q8: bad shape");
    ReadArgs a{};
    a.slots = slots; a.rows = rows; a.n_kv = n_kv; a.pshift = __builtin_ctz((unsigned)page);
    a.n_slots = (int64_t)n_pages * page;
    a.codes[0] = Kc; a.codes[1] = Vc; a.scale[0] = k_scale; a.scale[1] = v_scale;
    a.y[0] = k; a.y[1] = v; a.stride[0] = k_stride; a.stride[1] = v_stride;
    const int64_t items = ((int64_t)rows + 15) / 16 * n_kv * 2, blocks = (items + 3) / 4;
    if (blocks > 0x7fffffff) return fail(BX_EUNSUPPORTED, "kv_read_q8: too many rows and heads");
    const dim3 grid((unsigned)blocks);
    hipStream_t st = as_stream(stream);
    if (hd == 64) kv_read_kernel<64><<<grid, 256, 0, st>>>(a);
    else if (hd == 128) kv_read_kernel<128><<<grid, 256, 0, st>>>(a);
    else kv_read_kernel<256><<<grid, 256, 0, st>>>(a);
    return launch_check("kv_read_q8");
}

}  // extern "C"
