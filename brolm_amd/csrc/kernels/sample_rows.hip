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
// Up to 155,648 ids the row is read once and stays in registers as keys (76 of the
// 128 that a thread has); a longer one is read again for the last look.  The
// exponentials are 2^(n / 64) from a table times a polynomial of degree 5 in the
// rest (a table-driven reduction, relative error below 2^-50): 16 instructions
// where the library's exp has about 80.
//
// A 16-bit count wraps for more than 65,535 equal logits; the counts then add up
// to less than the vocabulary, and the row is done again in pieces that cannot.
#include <cmath>
#include <type_traits>

#include "common.h"

namespace bx {
namespace {

constexpr int kSrThreads = 1024;
constexpr int kSrWaves = kSrThreads / 64;
constexpr int kSrBlocks = 1024;              // blocks of 64 keys
constexpr int kSrHist = 65536 * 2;           // bytes
constexpr int kSrPiece = 7 * 8192;           // ids whose counts fit 16 bits, a multiple of kSrStep
constexpr int kSrMaxVocab = 4194304;
constexpr int kSrStep = 8 * kSrThreads;      // ids of one load of the workgroup
constexpr int kSrKeep = 19;                  // loads of a row that stays in registers

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

__device__ __forceinline__ int key_of(const u4v& k, int j) { return (int)((k[j / 2] >> (16 * (j & 1))) & 0xffffu); }

// Keys of ids i .. i + 7 of the row (8 at most; 0, which no logit has, behind the last).
__device__ __forceinline__ u4v load_keys(const uint16_t* row, int i, int hi) {
    u4v w{0u, 0u, 0u, 0u};
    if (i + 8 <= hi) {
        w = *reinterpret_cast<const sr_any16*>(row + i);
        return u4v{key_pair(w.x), key_pair(w.y), key_pair(w.z), key_pair(w.w)};
    }
    for (int j = 0; j < hi - i; ++j) w[j / 2] |= (key_pair(row[i + j]) & 0xffffu) << (16 * (j & 1));
    return w;
}

// A row's keys, eight ids a thread and step: in registers, or read again each time.
template <bool KEEP>
struct SrRow {
    const uint16_t* row;
    int V;
    u4v k[KEEP ? kSrKeep : 1];

    __device__ __forceinline__ void init(const uint16_t* r, int v) {
        row = r;
        V = v;
        if constexpr (KEEP) {
#pragma unroll
            for (int q = 0; q < kSrKeep; ++q) {
                const int i = q * kSrStep + 8 * (int)threadIdx.x;
                k[q] = u4v{0u, 0u, 0u, 0u};
                if (q * kSrStep < V && i + 8 <= V) k[q] = *reinterpret_cast<const sr_any16*>(row + i);
            }
#pragma unroll
            for (int q = 0; q < kSrKeep; ++q) {
                const int i = q * kSrStep + 8 * (int)threadIdx.x;
                if (q * kSrStep < V) {
                    if (i + 8 <= V) k[q] = u4v{key_pair(k[q].x), key_pair(k[q].y), key_pair(k[q].z), key_pair(k[q].w)};
                    else k[q] = load_keys(row, i, V);
                }
            }
        }
    }
    // f(first id, its 8 keys, all of them ids) for ids [lo, hi); lo and hi multiples of
    // kSrStep, or hi the vocabulary
    template <class F>
    __device__ __forceinline__ void each(int lo, int hi, F&& f) const {
        if constexpr (KEEP) {
#pragma unroll
            for (int q = 0; q < kSrKeep; ++q) {
                const int i = q * kSrStep + 8 * (int)threadIdx.x;
                if (q * kSrStep >= lo && q * kSrStep < hi) f(i, k[q], (q + 1) * kSrStep <= V);
                __builtin_amdgcn_sched_barrier(0);   // one step's temporaries at a time
            }
        } else {
            again(lo, hi, f);
        }
    }
    // the same from memory
    template <class F>
    __device__ __forceinline__ void again(int lo, int hi, F&& f) const {
#pragma unroll 1
        for (int b = lo; b < hi; b += kSrStep) {
            const int i = b + 8 * (int)threadIdx.x;
            f(i, load_keys(row, i, V), b + kSrStep <= V);
        }
    }
};

// The larger key of each half of a dword.  (The elements are copied first: a bit cast of
// a vector's element in place reads the vector's first one.)
__device__ __forceinline__ uint32_t max_pairs(uint32_t top, const u4v& k) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    us2 m = __builtin_bit_cast(us2, top);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = k[i];
        m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, w));
    }
    return __builtin_bit_cast(uint32_t, m);
}

// The keys of one step into the histogram; the largest key this thread has seen in top.
__device__ __forceinline__ void sr_count(const u4v& k, bool all, uint32_t* hist, uint32_t& top) {
    top = max_pairs(top, k);
    // masked vocabularies: whole stretches of one value are added once
    const uint32_t one = (uint32_t)__builtin_amdgcn_readfirstlane((int)k.x), pair = (one & 0xffffu) * 0x10001u;
    const bool same = pair != 0u && k.x == pair && k.y == pair && k.z == pair && k.w == pair;
    const uint64_t many = __ballot(same);
    if (many) {
        const int key = (int)(pair & 0xffffu);
        if ((threadIdx.x & 63) == __builtin_ctzll(many))
            atomicAdd(&hist[key >> 1], (uint32_t)(8 * __popcll(many)) << (16 * (key & 1)));
    }
    if (same) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int key = key_of(k, j);
        if (all || key != 0) atomicAdd(&hist[key >> 1], 1u << (16 * (key & 1)));
    }
}

// Sums over the 16 lanes of a row, in every lane of it (quads, mirrored halves).
__device__ __forceinline__ double row16_sum(double v) {
    auto move = [](double x, auto ctrl) {
        constexpr int C = decltype(ctrl)::value;
        const u2v w = __builtin_bit_cast(u2v, x);
        const u2v y{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, C, 0xf, 0xf, false),
                    (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, C, 0xf, 0xf, false)};
        return __builtin_bit_cast(double, y);
    };
    v += move(v, std::integral_constant<int, 0xB1>{});
    v += move(v, std::integral_constant<int, 0x4E>{});
    v += move(v, std::integral_constant<int, 0x141>{});
    v += move(v, std::integral_constant<int, 0x140>{});
    return v;
}
__device__ __forceinline__ uint32_t row16_sum(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false);
    return v;
}

__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
    return v;
}

struct SrShared {
    uint32_t cnt[kSrBlocks];   // ids of block b (largest keys first), then of blocks 0 .. b
    double mass[kSrBlocks];
    double pow2[64];           // 2^(i / 64)
    uint32_t red_n[kSrWaves];
    double red_m[kSrWaves];
    uint32_t level[64];        // counts of one block's keys
    int red_i[kSrWaves];
    int found[4];
    int hits[kSrKeep * kSrWaves];   // of a step and wavefront
    int pick[2];
};

// One block's levels, largest key first: count, e, and what stands before each.
struct SrLevels {
    uint32_t c, before_n;
    double e, before_m;
    int key;
};

template <bool KEEP>
__global__ __launch_bounds__(kSrThreads) void sample_rows_kernel(SrArgs a) {
    extern __shared__ __align__(16) uint32_t hist[];
    __shared__ SrShared s;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, V = a.V;
    const float temp = a.temp[blockIdx.x];
    SrRow<KEEP> row;
    row.init(a.logits + (int64_t)blockIdx.x * a.stride, V);
    auto all_max = [&](uint32_t pair) {
        const int v = wave_max_i((int)max(pair & 0xffffu, pair >> 16));
        __syncthreads();
        if (lane == 0) s.red_i[wave] = v;
        __syncthreads();
        int r = s.red_i[0];
        for (int i = 1; i < kSrWaves; ++i) r = max(r, s.red_i[i]);
        return r;
    };
    int key, nth;
    if (!(temp > 0.f)) {
        uint32_t top = 0u;
        row.each(0, V, [&](int, const u4v& k, bool) { top = max_pairs(top, k); });
        key = all_max(top);
        nth = 0;
    } else {
        auto clear = [&] {
            for (int i = t; i < kSrHist / 16; i += kSrThreads) reinterpret_cast<u4v*>(hist)[i] = u4v{0u, 0u, 0u, 0u};
            __syncthreads();
        };
        if (t < 64) s.pow2[t] = exp2((double)t * 0.015625);
        clear();
        uint32_t seen = 0u;
        row.each(0, V, [&](int, const u4v& k, bool all) { sr_count(k, all, hist, seen); });
        const int top = all_max(seen);   // barriers: the histogram is whole
        // exp((l - max) / T): 2^(y / 64) with y = 64 log2(e) (l - max) / T = n + f
        const double vmax = key_value(top), step = 92.332482616893656877 / (double)temp;
        auto weight = [&](int k) {
            const double y = fmax((key_value(k) - vmax) * step, -80000.0);
            const double n = rint(y), z = (y - n) * 0.010830424696249145094;   // ln(2) / 64
            const int q = (int)n;
            double p = fma(z, 1.0 / 120.0, 1.0 / 24.0);
            p = fma(p, z, 1.0 / 6.0);
            p = fma(p, z, 0.5);
            p = fma(p, z, 1.0);
            p = fma(p, z, 1.0);
            const double e = ldexp(s.pow2[q & 63] * p, q >> 6);
            return k == top ? 1.0 : y >= -79999.0 ? e : 0.0;
        };
        auto count_at = [&](int k) { return (hist[k >> 1] >> (16 * (k & 1))) & 0xffffu; };
        // a wavefront takes four blocks at a time, a lane four keys of them (its 16
        // lanes are a block); added to what an earlier piece of the row left there
        auto block_sums = [&](bool add) {
            for (int b = 4 * wave; b < kSrBlocks; b += 4 * kSrWaves) {
                const int k0 = ((kSrBlocks - 1 - b) << 6) + 60 - 4 * lane;
                const u2v w = *reinterpret_cast<const u2v*>(hist + (k0 >> 1));
                uint32_t n = (w.x & 0xffffu) + (w.x >> 16) + (w.y & 0xffffu) + (w.y >> 16);
                double m = 0.0;
                if (__any(n != 0u)) {
                    if (n != 0u) {
                        m = (double)(w.x & 0xffffu) * weight(k0) + (double)(w.x >> 16) * weight(k0 + 1) +
                            (double)(w.y & 0xffffu) * weight(k0 + 2) + (double)(w.y >> 16) * weight(k0 + 3);
                    }
                    n = row16_sum(n);
                    m = row16_sum(m);
                }
                if ((lane & 15) == 0) {
                    const int at = b + (lane >> 4);
                    s.cnt[at] = add ? s.cnt[at] + n : n;
                    s.mass[at] = add ? s.mass[at] + m : m;
                }
            }
            __syncthreads();
        };
        block_sums(false);
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
            for (int lo = 0; lo < V; lo += kSrPiece) {
                clear();
                row.again(lo, min(V, lo + kSrPiece), [&](int, const u4v& k, bool all) { sr_count(k, all, hist, seen); });
                __syncthreads();
                block_sums(lo > 0);
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
                row.again(0, V, [&](int, const u4v& k, bool) {
                    for (int j = 0; j < 8; ++j)
                        if (key_of(k, j) >> 6 == kSrBlocks - 1 - b && key_of(k, j) != 0)
                            atomicAdd(&s.level[63 - (key_of(k, j) & 63)], 1u);
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

    // ---- the nth id (ascending) whose key this is
    const uint32_t pair = (uint32_t)key * 0x10001u;
    auto matches = [&](const u4v& k) {   // of the lane's 8 ids
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 off{0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = k[i] ^ pair;
            off += __builtin_elementwise_min(__builtin_bit_cast(us2, w), us2{1, 1});
        }
        return 8 - (int)off[0] - (int)off[1];
    };
    auto wave_inclusive = [&](int v) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(v, o);
            if (lane >= o) v += y;
        }
        return v;
    };
    // the id in the wavefront's 512 keys of one step, which hold the n-th
    auto finish = [&](int i, const u4v& k, int n) {
        const int c = matches(k);
        int before = wave_inclusive(c) - c;
        if (n < before || n >= before + c) return;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (key_of(k, j) == key && before++ == n) a.out[blockIdx.x] = i + j;
    };
    auto wave_total = [&](const u4v& k) {
        const int c = matches(k);
        return __any(c > 0) ? __shfl(wave_inclusive(c), 63) : 0;
    };
    // steps in groups of kSrKeep: hits of each (step, wavefront), in order of the ids
    for (int lo = 0; lo < V; lo += kSrKeep * kSrStep) {
        const int hi = min(V, lo + kSrKeep * kSrStep), steps = (hi - lo + kSrStep - 1) / kSrStep;
        row.each(lo, hi, [&](int i, const u4v& k, bool) {
            const int c = wave_total(k);
            if (lane == 0) s.hits[(i - lo) / kSrStep * kSrWaves + wave] = c;
        });
        if (t == 0) s.pick[0] = -1;
        __syncthreads();
        if (wave == 0) {
            constexpr int kPer = (kSrKeep * kSrWaves + 63) / 64;
            int c[kPer], sum = 0;
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                const int e = kPer * lane + q;
                c[q] = e < steps * kSrWaves ? s.hits[e] : 0;
                sum += c[q];
            }
            int before = wave_inclusive(sum) - sum;
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                if (nth >= before && nth < before + c[q]) {
                    s.pick[0] = kPer * lane + q;
                    s.pick[1] = nth - before;
                }
                before += c[q];
            }
            if (lane == 63) s.red_i[0] = before;
        }
        __syncthreads();
        const int pick = s.pick[0], n = s.pick[1];
        if (pick >= 0) {
            if (wave == pick % kSrWaves) {
                const int i = lo + pick / kSrWaves * kSrStep + 8 * t;
                finish(i, load_keys(row.row, i, V), n);
            }
            return;
        }
        nth -= s.red_i[0];
        __syncthreads();
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
    static std::atomic<uint64_t> allowed[2];
    const bool keep = vocab <= kSrKeep * kSrStep;
    const auto kernel = keep ? sample_rows_kernel<true> : sample_rows_kernel<false>;
    if (int rc = allow_lds(allowed[keep], reinterpret_cast<const void*>(kernel), kSrHist, "sample_rows: LDS attribute"))
        return rc;
    SrArgs a{logits, stride, vocab, temperature, top_k, top_p, min_p, u, out};
    kernel<<<(unsigned)rows, kSrThreads, kSrHist, as_stream(stream)>>>(a);
    return launch_check("sample_rows");
}
