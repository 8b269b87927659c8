// The paged 8-bit KV cache of a batched step: which page a token goes to
// (bx_kv_plan), its K / V rows into the pages (bx_kv_append_q8_f16) and rows
// back out (bx_kv_read_q8_f16).  The attention over it is attention_q8.hip.
//
// A page holds P tokens of every KV head: K codes [page][head][token][hd] and V
// codes [page][head][hd][token], so that the attention's matrix operands (16
// bytes along hd for Q K^T, 16 bytes along the tokens for P V) are plain 16-byte
// loads.  One FP32 scale per page, head and matrix: value = code * scale, codes
// in [-127, 127].
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

constexpr int kPlanThreads = 256;
constexpr int kPlanRows = 1024;   // rows per workgroup

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

// Exclusive prefix over the workgroup in thread order; *total gets the sum.
__device__ __forceinline__ int64_t plan_scan(int64_t v, int64_t* red, int64_t* total) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(inc, o);
        if (l >= o) inc += y;
    }
    __syncthreads();
    if (l == 63) red[w] = inc;
    __syncthreads();
    int64_t before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 64; ++i) {
        if (i < w) before += red[i];
        sum += red[i];
    }
    *total = sum;
    return before + inc - v;
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
    __shared__ int64_t red[kPlanThreads / 64];
    __shared__ int s_bad;
    __shared__ uint32_t s_last;
    const int t = threadIdx.x, n = a.n_req, page = 1 << a.pshift;
    const int64_t head = a.ends_in[0], tail = a.ends_in[1], room = (int64_t)a.max_blocks << a.pshift;
    if (t == 0) s_bad = 0;
    __syncthreads();

    // ---- prefix sums, kPlanPer consecutive requests a thread
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
    int64_t n_rows, n_take, n_give;
    rows = plan_scan(rows, red, &n_rows);
    take = plan_scan(take, red, &n_take);
    give = plan_scan(give, red, &n_give);
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
    auto ring_at = [&](int base, int i) { return base + i < a.n_pages ? base + i : base + i - a.n_pages; };
    auto blocks_of = [&](int len) { return (int)(((int64_t)len + page - 1) >> a.pshift); };
    const int end = min(a.max_rows, ((int)blockIdx.x + 1) * kPlanRows);
    for (int i = (int)blockIdx.x * kPlanRows + t; i < end; i += kPlanThreads) {
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
// One wavefront writes a run of one head, of K or of V:
//   amax over the run, s = max(s_old, amax / 127) (s_old = 0 for a page that was
//   empty); where s grew, the page's earlier codes c become rint(c s_old / s); the
//   new codes are rint(x / s).
// Both roundings are exact to the last border: a new code's remainder x - q s is
// exact in FP32 (x and q s are multiples of s's last place, and the remainder is
// below s), the earlier codes' quotient is formed in FP64, where c s_old is exact.
// |x| is compared as the FP16 bit pattern, which orders NaN last: a page with a
// NaN or an infinity gets such a scale, and every value of it becomes NaN.

typedef u4v __attribute__((aligned(2))) any16;

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
    float q = rintf(x * inv);
    const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s;
    // one step off at most: the remainder says which way (equal: the even one)
    const bool odd = ((int)q & 1) != 0;
    if (r > h || (r == h && odd)) q += 1.f;
    else if (r < -h || (r == -h && odd)) q -= 1.f;
    return (int)q;
}

__device__ __forceinline__ uint32_t pk_max_abs(uint32_t m, uint32_t x) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    const us2 a = __builtin_bit_cast(us2, m), b = __builtin_bit_cast(us2, x & 0x7fff7fffu);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
}

// The earlier codes of four bytes, requantized: those of tokens below `keep` (byte i
// holds token t0 + i); others as they are.
__device__ __forceinline__ int requant(int c, float s_old, float s_new) {
    return (int)rint((double)c * (double)s_old / (double)s_new);
}

template <int HD>
__device__ void append_run(const AppendArgs& a, int row, int n, int head, int which) {
    constexpr int CH = HD / 8;        // 16-byte pieces of a row
    constexpr int RP = 64 / CH > 0 ? 64 / CH : 1;   // rows a wavefront reads at once
    const int lane = threadIdx.x & 63, page = 1 << a.pshift;
    const int64_t slot = a.slots[row], pg = slot >> a.pshift;
    const int off = (int)(slot & (page - 1));
    const int64_t hp = pg * a.n_kv + head;
    const uint16_t* const x = a.x[which] + (int64_t)row * a.stride[which] + (int64_t)head * HD;
    const int64_t st = a.stride[which];
    float* const sp = a.scale[which] + hp;
    int8_t* const codes = a.codes[which] + hp * page * HD;
    const uint32_t old_bits = off > 0 ? __float_as_uint(*sp) : 0u;
    uint32_t m2 = 0u;
    for (int i = lane / CH; i < n; i += RP) {
        const u4v w = *reinterpret_cast<const any16*>(x + (int64_t)i * st + 8 * (lane % CH));
        m2 = pk_max_abs(pk_max_abs(pk_max_abs(pk_max_abs(m2, w.x), w.y), w.z), w.w);
    }
    uint32_t m = max(m2 & 0xffffu, m2 >> 16);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    const uint32_t new_bits = max(old_bits, __float_as_uint(h2f((uint16_t)m) / 127.0f));
    const float s_old = __uint_as_float(old_bits), s = __uint_as_float(new_bits);
    const bool live = s > 0.f && s < INFINITY;   // else every code is 0
    const float inv = live ? 1.0f / s : 0.f;
    if (lane == 0) *sp = s;
    auto code = [&](uint16_t h) { return live ? q8_code(h2f(h), s, inv) : 0; };
    const bool grew = off > 0 && new_bits != old_bits;
    auto moved = [&](int c) { return live ? requant(c, s_old, s) : 0; };
    if (which == 0) {
        if (grew) {
            u4v* const p = reinterpret_cast<u4v*>(codes);
            for (int i = lane; i < off * HD / 16; i += 64) {
                u4v w = p[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t y = 0u;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        y |= (uint32_t)(moved((int8_t)(w[j] >> (8 * b))) & 0xff) << (8 * b);
                    w[j] = y;
                }
                p[i] = w;
            }
        }
        for (int i = lane / CH; i < n; i += RP) {
            const u4v w = *reinterpret_cast<const any16*>(x + (int64_t)i * st + 8 * (lane % CH));
            u2v y{0u, 0u};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                y[j / 4] |= (uint32_t)(code((uint16_t)(w[j / 2] >> (16 * (j & 1)))) & 0xff) << (8 * (j & 3));
            *reinterpret_cast<u2v*>(codes + (int64_t)(off + i) * HD + 8 * (lane % CH)) = y;
        }
        return;
    }
    // V: pieces of 16 tokens of one head dim; a piece that also holds earlier tokens
    // (or ones behind the run) keeps their bytes
    for (int c0 = grew ? 0 : off & ~15; c0 < off + n; c0 += 16) {
        const bool whole = c0 >= off && c0 + 16 <= off + n;
        for (int d = lane; d < HD; d += 64) {
            u4v* const p = reinterpret_cast<u4v*>(codes + (int64_t)d * page + c0);
            u4v w{0u, 0u, 0u, 0u};
            if (!whole) w = *p;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int tk = c0 + j, sh = 8 * (j & 3);
                int y = (int8_t)(w[j / 4] >> sh);
                if (tk >= off && tk < off + n) y = code(x[(int64_t)(tk - off) * st + d]);
                else if (grew && tk < off) y = moved(y);
                w[j / 4] = (w[j / 4] & ~(0xffu << sh)) | ((uint32_t)(y & 0xff) << sh);
            }
            *p = w;
        }
    }
}

template <int HD>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    // wavefront -> (window of rows, head, K or V); the runs that start in its window
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int which = (int)(item & 1), head = (int)((item >> 1) % a.n_kv);
    const int64_t row0 = (item >> 1) / a.n_kv * a.window;
    const int lane = threadIdx.x & 63, page = 1 << a.pshift;
    if (row0 >= a.rows) return;
    auto slot_at = [&](int64_t r) { return r >= 0 && r < a.rows ? a.slots[r] : -1; };
    const int64_t r = row0 + lane;
    const int64_t own = slot_at(r), prev = slot_at(r - 1);
    const bool first = lane < a.window && own >= 0 && own < a.n_slots && ((own & (page - 1)) == 0 || own != prev + 1);
    uint64_t todo = __ballot(first);
    while (todo) {
        const int i = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int row = (int)(row0 + i);
        const int64_t slot = a.slots[row];
        const int left = page - (int)(slot & (page - 1));   // tokens to the page's end
        int n = 0;
        for (int k = 0; k < left; k += 64) {
            const uint64_t same = __ballot(k + lane < left && slot_at((int64_t)row + k + lane) == slot + k + lane);
            const int c = ~same ? __builtin_ctzll(~same) : 64;
            n += c;
            if (c < 64) break;
        }
        append_run<HD>(a, row, n, head, which);
    }
}

// ------------------------------------------------------------------ the read
//
// A wavefront takes 16 rows of one head, of K or of V.  K rows are 16-byte loads;
// V, token-minor, is read in 16-byte pieces of 16 tokens of a head dim where the
// rows are consecutive tokens of one page, else byte by byte.
struct ReadArgs {
    const int64_t* slots;
    int rows, n_kv, pshift;
    int64_t n_slots;
    const int8_t* codes[2];
    const float* scale[2];
    uint16_t* y[2];
    int64_t stride[2];
};

__device__ __forceinline__ uint16_t q8_value(int c, float s) { return f2h(f32_fence((float)c * s)); }

template <int HD>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int which = (int)(item & 1), head = (int)((item >> 1) % a.n_kv);
    const int64_t row0 = (item >> 1) / a.n_kv * 16;
    const int lane = threadIdx.x & 63, page = 1 << a.pshift;
    if (row0 >= a.rows) return;
    const int n = (int)min((int64_t)16, a.rows - row0);
    for (int i = 0; i < n; ++i) {
        const int64_t slot = a.slots[row0 + i];
        if (slot < 0 || slot >= a.n_slots) continue;
        const int64_t hp = (slot >> a.pshift) * a.n_kv + head;
        const int off = (int)(slot & (page - 1));
        const float s = a.scale[which][hp];
        const int8_t* const c = a.codes[which] + hp * page * HD;
        uint16_t* const y = a.y[which] + (row0 + i) * a.stride[which] + (int64_t)head * HD;
        for (int d = lane; d < HD; d += 64) y[d] = q8_value(which ? c[(int64_t)d * page + off] : c[off * HD + d], s);
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
    a.window = rows <= 512 ? 1 : 16;
    const int64_t items = ((int64_t)rows + a.window - 1) / a.window * n_kv * 2, blocks = (items + 3) / 4;
    if (blocks > 0x7fffffff) return fail(BX_EUNSUPPORTED, "kv_append_q8: too many rows and heads");
    const dim3 grid((unsigned)blocks);
    hipStream_t st = as_stream(stream);
    if (hd == 64) kv_append_kernel<64><<<grid, 256, 0, st>>>(a);
    else if (hd == 128) kv_append_kernel<128><<<grid, 256, 0, st>>>(a);
    else kv_append_kernel<256><<<grid, 256, 0, st>>>(a);
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
