// The draw of a batched step: one id per row of FP16 logits, each row with its own
// temperature, top-k, top-p, min-p and random number (the rules of reference
// src/detail/generate.cpp:68-142, with min-p, for many rows at once).
//
// One workgroup a row, nothing sorted.  An FP16 logit has at most 65,536 values,
// and its bits, with the negative ones flipped, order like the values: the row
// becomes a histogram over that key, 16-bit counts in 128 KB of LDS.  Counts are
// integers (any order of the additions gives the same), and a level's mass is its count
// times exp((l - max) / T) in FP64, so every cut and the draw are decided in FP64
// whatever the number of ids: equal logits are one level, ids within it stand in
// ascending order.  Blocks of 64 keys get their count and mass, a prefix over the
// 1024 blocks (largest keys first) places each cut in a block and one wavefront
// finishes it there.  The kept ids are the first n in that order:
//   n = min(top_k, ids with e >= min_p, the first place where the running mass
//       reaches top_p of the whole), at least 1;
// the draw is the first place among them where the running mass exceeds u times
// the mass of the n.  A last look at the row finds that place's id among those of
// its level.
//
// A 16-bit count wraps for more than 65,535 equal logits; the counts then add up
// to less than the vocabulary, and the row is done again in pieces that cannot.
#include <cmath>

#include "common.h"

namespace bx {
namespace {

constexpr int kSrThreads = 1024;
constexpr int kSrWaves = kSrThreads / 64;
constexpr int kSrBlocks = 1024;              // blocks of 64 keys
constexpr int kSrHist = 65536 * 2;           // bytes
constexpr int kSrPiece = 65528;              // ids whose counts fit 16 bits, a multiple of 8
constexpr int kSrMaxVocab = 4194304;

typedef u4v __attribute__((aligned(2))) sr_any16;

struct SrArgs {
    const uint16_t* logits;
    int64_t stride;
    int V;
    const float* temp;
    const int32_t* top_k;
    const float *top_p, *min_p;
    const double* u;
    int32_t* out;
};

// Keys of two logits: -0 as +0, NaN as -infinity, then ordered bits.
__device__ __forceinline__ uint32_t key_pair(uint32_t x) {
    typedef short s2 __attribute__((ext_vector_type(2)));
    const h2 ninf{(_Float16)-INFINITY, (_Float16)-INFINITY}, zero{(_Float16)0.f, (_Float16)0.f};
    const uint32_t y = as_u32(__builtin_elementwise_max(as_h2(x), ninf) + zero);
    const s2 sg = __builtin_bit_cast(s2, y) >> 15;
    return y ^ (__builtin_bit_cast(uint32_t, sg) | 0x80008000u);
}
__device__ __forceinline__ double key_value(int key) {
    return (double)h2f((uint16_t)(key & 0x8000 ? key ^ 0x8000 : ~key));
}

// f(first id, key pairs of 8 ids) over ids [lo, hi) of the row, `lanes` lanes of
// which this is number `me`; lo a multiple of 8.  Ids at hi and behind: `pad`.
template <class F>
__device__ __forceinline__ void for_keys(const uint16_t* row, int lo, int hi, int me, int lanes, F&& f) {
    for (int i = lo + 8 * me; i < hi; i += 8 * lanes) {
        u4v w;
        if (i + 8 <= hi) {
            w = *reinterpret_cast<const sr_any16*>(row + i);
        } else {
            w = u4v{0u, 0u, 0u, 0u};
            for (int j = 0; j < hi - i; ++j) w[j / 2] |= (uint32_t)row[i + j] << (16 * (j & 1));
        }
        f(i, u4v{key_pair(w.x), key_pair(w.y), key_pair(w.z), key_pair(w.w)});
    }
}
__device__ __forceinline__ int key_of(const u4v& k, int j) { return (int)((k[j / 2] >> (16 * (j & 1))) & 0xffffu); }

// Ids [lo, hi) into the histogram; returns the largest key this thread saw.
__device__ int sr_count(const uint16_t* row, int lo, int hi, uint32_t* hist) {
    int top = 0;
    for_keys(row, lo, hi, threadIdx.x, kSrThreads, [&](int i, const u4v& k) {
        const int n = min(8, hi - i);
        // masked vocabularies: whole stretches of one value are added once
        const uint32_t one = (uint32_t)__builtin_amdgcn_readfirstlane((int)k.x), pair = (one & 0xffffu) * 0x10001u;
        const bool same = n == 8 && k.x == pair && k.y == pair && k.z == pair && k.w == pair;
        const uint64_t all = __ballot(same);
        if (same) {
            const int key = (int)(pair & 0xffffu);
            top = max(top, key);
            if ((threadIdx.x & 63) == __builtin_ctzll(all))
                atomicAdd(&hist[key >> 1], (uint32_t)(8 * __popcll(all)) << (16 * (key & 1)));
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j >= n) break;
            const int key = key_of(k, j);
            top = max(top, key);
            atomicAdd(&hist[key >> 1], 1u << (16 * (key & 1)));
        }
    });
    return top;
}

__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
    return v;
}

struct SrShared {
    uint32_t cnt[kSrBlocks];   // ids of block b (largest keys first), then of blocks 0 .. b
    double mass[kSrBlocks];
    uint32_t red_n[kSrWaves];
    double red_m[kSrWaves];
    uint32_t level[64];        // counts of one block's keys
    int red_i[kSrWaves];
    int found[4];
    int key, nth;
};

// One block's levels, largest key first: count, e, and what stands before each.
struct SrLevels {
    uint32_t c, before_n;
    double e, before_m;
    int key;
};

__global__ __launch_bounds__(kSrThreads) void sample_rows_kernel(SrArgs a) {
    extern __shared__ __align__(16) uint32_t hist[];
    __shared__ SrShared s;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, V = a.V;
    const uint16_t* const row = a.logits + (int64_t)blockIdx.x * a.stride;
    const float temp = a.temp[blockIdx.x];
    auto all_max = [&](int v) {
        v = wave_max_i(v);
        __syncthreads();
        if (lane == 0) s.red_i[wave] = v;
        __syncthreads();
        int r = s.red_i[0];
        for (int i = 1; i < kSrWaves; ++i) r = max(r, s.red_i[i]);
        return r;
    };
    int key, nth;
    if (!(temp > 0.f)) {
        int top = 0;
        for_keys(row, 0, V, t, kSrThreads, [&](int i, const u4v& k) {
            for (int j = 0; j < min(8, V - i); ++j) top = max(top, key_of(k, j));
        });
        key = all_max(top);
        nth = 0;
    } else {
        auto clear = [&] {
            for (int i = t; i < kSrHist / 16; i += kSrThreads) reinterpret_cast<u4v*>(hist)[i] = u4v{0u, 0u, 0u, 0u};
            __syncthreads();
        };
        s.cnt[t] = 0u;
        s.mass[t] = 0.0;
        clear();
        const int top = all_max(sr_count(row, 0, V, hist));   // barriers: the histogram is whole
        const double vmax = key_value(top), inv_t = 1.0 / (double)temp;
        auto weight = [&](int k) {   // exp((l - max) / T)
            if (k == top) return 1.0;
            const double e = exp((key_value(k) - vmax) * inv_t);
            return e >= 0.0 ? e : 0.0;
        };
        auto count_at = [&](int k) { return (hist[k >> 1] >> (16 * (k & 1))) & 0xffffu; };
        // a wavefront a block, lane i its i-th largest key
        auto block_sums = [&] {
            for (int b = wave; b < kSrBlocks; b += kSrWaves) {
                const int k = ((kSrBlocks - 1 - b) << 6) + 63 - lane;
                const uint32_t c = count_at(k);
                if (!__any(c != 0u)) continue;
                double m = c != 0u && k <= top ? (double)c * weight(k) : 0.0;
                uint32_t n = c;
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) {
                    n += (uint32_t)__shfl_xor((int)n, o);
                    m += __shfl_xor(m, o);
                }
                if (lane == 0) {
                    s.cnt[b] += n;
                    s.mass[b] += m;
                }
            }
            __syncthreads();
        };
        block_sums();
        // inclusive prefix over the blocks, thread t block t
        uint32_t n_in;
        double m_in;
        auto prefix = [&] {
            n_in = s.cnt[t];
            m_in = s.mass[t];
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t n = (uint32_t)__shfl_up((int)n_in, o);
                const double m = __shfl_up(m_in, o);
                if (lane >= o) {
                    n_in += n;
                    m_in += m;
                }
            }
            if (lane == 63) {
                s.red_n[wave] = n_in;
                s.red_m[wave] = m_in;
            }
            __syncthreads();
            for (int w = 0; w < wave; ++w) {
                n_in += s.red_n[w];
                m_in += s.red_m[w];
            }
        };
        prefix();
        uint32_t total = 0;
        for (int w = 0; w < kSrWaves; ++w) total += s.red_n[w];
        __syncthreads();
        bool whole = true;   // the histogram holds the row
        if (total != (uint32_t)V) {
            whole = false;
            s.cnt[t] = 0u;
            s.mass[t] = 0.0;
            for (int lo = 0; lo < V; lo += kSrPiece) {
                clear();
                sr_count(row, lo, min(V, lo + kSrPiece), hist);
                __syncthreads();
                block_sums();
            }
            prefix();
            __syncthreads();
        }
        s.cnt[t] = n_in;
        s.mass[t] = m_in;
        if (t < 4) s.found[t] = kSrBlocks - 1;
        __syncthreads();

        // the levels of block b in every wavefront
        auto levels = [&](int b) {
            SrLevels x;
            x.key = ((kSrBlocks - 1 - b) << 6) + 63 - lane;
            if (whole) {
                x.c = count_at(x.key);
            } else {
                __syncthreads();
                if (t < 64) s.level[t] = 0u;
                __syncthreads();
                for_keys(row, 0, V, t, kSrThreads, [&](int i, const u4v& k) {
                    for (int j = 0; j < min(8, V - i); ++j)
                        if (key_of(k, j) >> 6 == kSrBlocks - 1 - b) atomicAdd(&s.level[63 - (key_of(k, j) & 63)], 1u);
                });
                __syncthreads();
                x.c = s.level[lane];
            }
            x.e = x.c != 0u ? weight(x.key) : 0.0;
            uint32_t n = x.c;
            double m = (double)x.c * x.e;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = (uint32_t)__shfl_up((int)n, o);
                const double z = __shfl_up(m, o);
                if (lane >= o) {
                    n += y;
                    m += z;
                }
            }
            // what stands before a level: the inclusive sums of the lane above
            uint32_t pn = (uint32_t)__shfl_up((int)n, 1);
            double pm = __shfl_up(m, 1);
            if (lane == 0) pn = 0u, pm = 0.0;
            x.before_n = (b > 0 ? s.cnt[b - 1] : 0u) + pn;
            x.before_m = (b > 0 ? s.mass[b - 1] : 0.0) + pm;
            return x;
        };
        auto last_lane = [](uint64_t mask) { return 63 - __builtin_clzll(mask); };

        // ---- how many ids are kept
        uint32_t n = (uint32_t)V;
        const int k = a.top_k ? a.top_k[blockIdx.x] : 0;
        if (k > 0) n = min(n, (uint32_t)k);
        const double mp = a.min_p ? (double)a.min_p[blockIdx.x] : 0.0;
        const double tp = a.top_p ? (double)a.top_p[blockIdx.x] : 1.0;
        const double goal = tp * s.mass[kSrBlocks - 1];
        const bool cut_m = !(mp <= 0.0), cut_p = tp < 1.0;
        // the blocks where they end: the first whose smallest key is below min_p, the
        // first whose running mass reaches the goal
        if (cut_m && !(weight((kSrBlocks - 1 - t) << 6) >= mp) && ((kSrBlocks - 1 - t) << 6) <= top) atomicMin(&s.found[0], t);
        if (cut_p && n_in > 0u && m_in >= goal) atomicMin(&s.found[1], t);
        __syncthreads();
        if (cut_m) {
            const SrLevels x = levels(s.found[0]);
            const uint64_t in = __ballot(x.c != 0u && x.e >= mp);
            uint32_t kept = __shfl((int)x.before_n, 0);
            if (in) kept = (uint32_t)__shfl((int)(x.before_n + x.c), last_lane(in));
            n = min(n, max(1u, kept));
        }
        if (cut_p) {
            const SrLevels x = levels(s.found[1]);
            const uint64_t any = __ballot(x.c != 0u), in = __ballot(x.c != 0u && x.before_m + (double)x.c * x.e >= goal);
            const double need = ceil((goal - x.before_m) / (x.e > 0.0 ? x.e : 1.0));
            const uint32_t part = (uint32_t)fmin(fmax(need, 1.0), (double)max(1u, x.c));
            uint32_t kept = n;
            if (in) kept = (uint32_t)__shfl((int)(x.before_n + part), __builtin_ctzll(in));
            else if (any) kept = (uint32_t)__shfl((int)(x.before_n + x.c), last_lane(any));
            n = min(n, kept);
        }
        // ---- their mass, and the place of the draw
        if (n_in >= n) atomicMin(&s.found[2], t);
        __syncthreads();
        const int bk = s.found[2];
        SrLevels x = levels(bk);
        const uint64_t end = __ballot(x.c != 0u && x.before_n < n && n <= x.before_n + x.c);
        const double upto = x.before_m + (double)(n - x.before_n) * x.e;
        const double goal_u = a.u[blockIdx.x] * __shfl(upto, end ? __builtin_ctzll(end) : 0);
        if (m_in > goal_u) atomicMin(&s.found[3], t);
        __syncthreads();
        const int bd = min(bk, s.found[3]);
        if (bd != bk) x = levels(bd);
        const uint32_t c = x.before_n < n ? min(x.c, n - x.before_n) : 0u;   // kept ids of the level
        const uint64_t any = __ballot(c != 0u), hit = __ballot(c != 0u && x.before_m + (double)c * x.e > goal_u);
        const double place = x.e > 0.0 ? floor((goal_u - x.before_m) / x.e) : 0.0;
        const int at = hit ? __builtin_ctzll(hit) : any ? last_lane(any) : 0;
        const int own = hit ? (int)fmin(fmax(place, 0.0), (double)max(1u, c) - 1.0) : (int)max(1u, c) - 1;
        key = __shfl(x.key, at);
        nth = __shfl(own, at);
    }

    // ---- the nth id (ascending) whose key this is: a stretch of ids a wavefront
    const int seg = ((V + kSrWaves - 1) / kSrWaves + 511) & ~511, lo = min(V, wave * seg), hi = min(V, lo + seg);
    int mine = 0;
    for_keys(row, lo, hi, lane, 64, [&](int i, const u4v& k) {
        for (int j = 0; j < min(8, hi - i); ++j) mine += key_of(k, j) == key ? 1 : 0;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o);
    __syncthreads();
    if (lane == 0) s.red_i[wave] = mine;
    __syncthreads();
    for (int w = 0; w < wave; ++w) nth -= s.red_i[w];
    if (nth < 0 || nth >= mine) return;   // another wavefront's
    for (int base = lo; base < hi; base += 512) {
        int c = 0;
        u4v kk{0u, 0u, 0u, 0u};
        const int i0 = base + 8 * lane, n = max(0, min(8, hi - i0));
        for_keys(row, base, min(hi, base + 512), lane, 64, [&](int, const u4v& k) { kk = k; });
        for (int j = 0; j < n; ++j) c += key_of(kk, j) == key ? 1 : 0;
        int inc = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(inc, o);
            if (lane >= o) inc += y;
        }
        const int before = inc - c;
        if (nth >= before && nth < inc) {
            int seen = before;
            for (int j = 0; j < n; ++j)
                if (key_of(kk, j) == key && seen++ == nth) a.out[blockIdx.x] = i0 + j;
        }
        nth -= __shfl(inc, 63);
        if (nth < 0) return;
    }
}

}  // namespace
}  // namespace bx

using namespace bx;

extern "C" int bx_sample_rows_f16(const uint16_t* logits, int64_t stride, int rows, int vocab, const float* temperature,
                                  const int32_t* top_k, const float* top_p, const float* min_p, const double* u,
                                  int32_t* out, void* stream) {
    if (!logits || !temperature || !u || !out) return fail(BX_EINVAL, "sample_rows: null pointer");
    if (rows <= 0 || vocab <= 0 || stride < vocab) return fail(BX_EINVAL, "sample_rows: bad shape");
    if (vocab > kSrMaxVocab) return fail(BX_EUNSUPPORTED, "sample_rows: vocabulary above 4194304 ids");
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_lds(allowed, reinterpret_cast<const void*>(&sample_rows_kernel), kSrHist, "sample_rows: LDS attribute"))
        return rc;
    SrArgs a{logits, stride, vocab, temperature, top_k, top_p, min_p, u, out};
    sample_rows_kernel<<<(unsigned)rows, kSrThreads, kSrHist, as_stream(stream)>>>(a);
    return launch_check("sample_rows");
}
