// The draw of a batched step: one id per row of FP16 logits, each row with its own
// temperature, top-k, top-p, min-p and random number (the rules of reference
// src/detail/generate.cpp:68-142, with min-p, for many rows at once).
//
// One workgroup a row, nothing sorted.  An FP16 logit has at most 65,536 values: the
// row becomes a histogram over its bit patterns, 16-bit counts in 128 KB of LDS.
// Counts are integers (any order of the additions gives the same), and a level's mass
// is its count times exp((l - max) / T) in FP64, so every cut and the draw are
// decided in FP64 whatever the number of ids: equal logits are one level, ids within it
// stand in ascending order.  A level's key is its pattern with the negative ones flipped, which
// orders like the value.  Blocks of 64 keys get their count and mass, a prefix over
// the 1024 blocks (largest keys first) places each cut in a block and one wavefront
// finishes it there.  The kept ids are the first n in that order:
//   n = min(top_k, ids with e >= min_p, the first place where the running mass
//       reaches top_p of the whole), at least 1;
// the draw is the first place among them where the running mass exceeds u times
// the mass of the n.  A last look at the row finds that place's id among those of
// its level.
//
// The exponentials are 2^(n / 64) from a table times a polynomial of degree 5 in the
// rest (a table-driven reduction, relative error below 2^-50, to which the rounding of the
// argument adds (max - l) / T 2^-52), and of four neighbouring keys one only: keys of one
// exponent are evenly spaced, so each weighs a constant times the next.
//
// 16 rows of 151,936 ids: 31 us, 200 rows: 39.  What bounds it: one CU a row, whose LDS makes
// 64 additions in about 16 cycles (15 us a row), the levels' exponentials (6 us), and the two
// looks at the row.
//
// A 16-bit count wraps for more than 65,535 equal logits; the counts then add up
// to less than the vocabulary, and the row is done again in pieces that cannot, and read once
// more for each cut: 16 rows of 151,936 ids, 100,000 of them at -infinity, 256 us.  (45,000 of
// them 58 us: their additions meet in one place of the histogram.)
#include <cmath>

#include "common.h"

namespace bx {
namespace {

constexpr int kSrThreads = 1024;
constexpr int kSrWaves = kSrThreads / 64;
constexpr int kSrBlocks = 1024;              // blocks of 64 keys
constexpr int kSrHist = 32768 * 4;           // bytes: positive patterns in the low halves, negative in the high
constexpr int kSrStep = 8 * kSrThreads;      // ids of one load of the workgroup
constexpr int kSrPiece = 7 * kSrStep;        // ids whose counts fit 16 bits
constexpr int kSrPart = 16;                  // steps looked through at once for the chosen id
constexpr int kSrMaxVocab = 4194304;
constexpr uint32_t kSrNegInf = 0xfc00u;
constexpr int kSrLowest = 0x3ff;             // key of -infinity, the smallest (NaN count as it)

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

// The key of a logit: -0 as +0, NaN as -infinity, then ordered bits.
__device__ __forceinline__ int key_of(uint32_t b) {
    if ((b & 0x7fffu) > 0x7c00u) b = kSrNegInf;
    if (b == 0x8000u) b = 0u;
    return (int)(b ^ (b & 0x8000u ? 0xffffu : 0x8000u));
}
__device__ __forceinline__ uint32_t key_bits(int key) { return (uint32_t)(key & 0x8000 ? key ^ 0x8000 : ~key & 0xffff); }
__device__ __forceinline__ double key_value(int key) { return (double)h2f((uint16_t)key_bits(key)); }
__device__ __forceinline__ uint32_t half_of(const u4v& w, int j) { return (w[j / 2] >> (16 * (j & 1))) & 0xffffu; }

// Ids i .. i + 7 of the row (8 at most), -infinity behind the last.
__device__ __forceinline__ u4v load_tail(const uint16_t* row, int i, int V) {
    u4v w{0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (i + j < V) w[j / 2] ^= ((uint32_t)row[i + j] ^ kSrNegInf) << (16 * (j & 1));
    return w;
}

// f(first id, its 8 logits, whether all are ids) for ids [lo, hi) of the row, eight a
// thread and step; lo a multiple of kSrStep, hi too or the vocabulary V.  Four steps
// are requested while the four before them are worked on.  (The row kept in 76
// registers a thread, every pass unrolled over it, was 100 KB of code and slower.)
template <class F>
__device__ __forceinline__ void each_step(const uint16_t* row, int V, int lo, int hi, F&& f) {
    const int me = 8 * (int)threadIdx.x;
    u4v w[4];
    auto fetch = [&](u4v (&x)[4], int b) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = b + q * kSrStep + me;
            x[q] = u4v{0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};
            if (i + 8 <= V) x[q] = *reinterpret_cast<const sr_any16*>(row + i);
        }
    };
    fetch(w, lo);
#pragma unroll 1
    for (int b = lo; b < hi; b += 4 * kSrStep) {
        u4v next[4];
        fetch(next, b + 4 * kSrStep);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int s = b + q * kSrStep;
            if (s >= hi) break;
            const bool all = s + kSrStep <= V;
            if (!all && s + me + 8 > V && s + me < V) w[q] = load_tail(row, s + me, V);
            f(s + me, w[q], all);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = next[q];
    }
}

// The larger value of each half of a dword, NaN left out.  (The elements are copied first: a
// bit cast of a vector's element in place reads the vector's first one.)
__device__ __forceinline__ uint32_t max_halves(uint32_t top, const u4v& x) {
    h2 m = as_h2(top);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = x[i];
        m = __builtin_elementwise_max(m, as_h2(w));
    }
    return as_u32(m);
}

// The logits of one step into the histogram; the largest this thread has seen in top.
__device__ __forceinline__ void sr_count(int i, const u4v& x, bool all, int V, uint32_t* hist, uint32_t& top) {
    top = max_halves(top, x);
    // masked vocabularies: whole stretches of one value are added once
    const uint32_t one = (uint32_t)__builtin_amdgcn_readfirstlane((int)x.x), pair = (one & 0xffffu) * 0x10001u;
    const bool same = ((x.x ^ pair) | (x.y ^ pair) | (x.z ^ pair) | (x.w ^ pair)) == 0u && (all || i + 8 <= V);
    const uint64_t many = __ballot(same);
    if (many) {
        if ((threadIdx.x & 63) == __builtin_ctzll(many))
            atomicAdd(&hist[pair & 0x7fffu], (uint32_t)(8 * __popcll(many)) << ((pair >> 11) & 16u));
    }
    if (same) return;
    char* const h = reinterpret_cast<char*>(hist);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (!all && i + j >= V) break;
        const uint32_t w = x[j / 2];
        // 1 into the low half, 65536 for a set sign
        if (j & 1) atomicAdd(reinterpret_cast<uint32_t*>(h + ((w >> 14) & 0x1fffcu)), __builtin_amdgcn_ubfe(w, 31, 1) * 65535u + 1u);
        else atomicAdd(reinterpret_cast<uint32_t*>(h + ((w << 2) & 0x1fffcu)), __builtin_amdgcn_ubfe(w, 15, 1) * 65535u + 1u);
    }
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
    double ratio[64];          // weight of a key to that of the key above it, by key >> 10
    uint32_t red_n[kSrWaves];
    double red_m[kSrWaves];
    uint32_t level[64];        // counts of one block's keys
    int red_i[kSrWaves];
    int hits[kSrPart * kSrWaves];   // of a step and wavefront
    int pick[3];
    uint32_t nan, wrap;
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
    const float temp = a.temp[blockIdx.x];
    const uint16_t* const row = a.logits + (int64_t)blockIdx.x * a.stride;
    auto all_max = [&](uint32_t pair) {   // the largest key of the row
        const int v = wave_max_i(max(key_of(pair & 0xffffu), key_of(pair >> 16)));
        __syncthreads();
        if (lane == 0) s.red_i[wave] = v;
        __syncthreads();
        int r = s.red_i[0];
        for (int i = 1; i < kSrWaves; ++i) r = max(r, s.red_i[i]);
        return r;
    };
    int key, nth;
    int ties = 0;   // ids of that key
    uint32_t seen = 0xfc00fc00u;
    if (!(temp > 0.f)) {
        each_step(row, V, 0, V, [&](int, const u4v& x, bool) { seen = max_halves(seen, x); });
        key = all_max(seen);
        nth = 0;
    } else {
        auto clear = [&] {
            for (int i = t; i < kSrHist / 16; i += kSrThreads) reinterpret_cast<u4v*>(hist)[i] = u4v{0u, 0u, 0u, 0u};
            if (t == 0) s.nan = s.wrap = 0u;
            __syncthreads();
        };
        // after a barrier behind the counting: -0 joins +0, NaN join -infinity; a count
        // that wraps here is reported
        auto fold = [&] {
            if (t < 0x3ff) {
                const uint32_t c = hist[0x7c01 + t];
                if (c != 0u) {
                    atomicAdd(&s.nan, (c & 0xffffu) + (c >> 16));
                    hist[0x7c01 + t] = 0u;
                }
            }
            __syncthreads();
            if (t == 0) {
                const uint32_t z = (hist[0] & 0xffffu) + (hist[0] >> 16), n = (hist[0x7c00] >> 16) + s.nan;
                hist[0] = z & 0xffffu;
                hist[0x7c00] = (hist[0x7c00] & 0xffffu) | (n << 16);
                s.wrap = (z | n) >> 16;
            }
            __syncthreads();
        };
        if (t < 64) s.pow2[t] = exp2((double)t * 0.015625);
        clear();
        each_step(row, V, 0, V, [&](int i, const u4v& x, bool all) { sr_count(i, x, all, V, hist, seen); });
        const int top = all_max(seen);   // barriers: the histogram is whole
        fold();
        // exp((l - max) / T): 2^(y / 64) with y = 64 log2(e) (l - max) / T = n + f
        const double vmax = key_value(top), step = 92.332482616893656877 / (double)temp;
        auto power = [&](double y) {   // y <= 0
            y = fmax(y, -80000.0);
            const double n = rint(y), z = (y - n) * 0.010830424696249145094;   // ln(2) / 64
            const int q = (int)n;
            double p = fma(z, 1.0 / 120.0, 1.0 / 24.0);
            p = fma(p, z, 1.0 / 6.0);
            p = fma(p, z, 0.5);
            p = fma(p, z, 1.0);
            p = fma(p, z, 1.0);
            const double e = ldexp(s.pow2[q & 63] * p, q >> 6);
            return y > -80000.0 ? e : 0.0;
        };
        auto weight = [&](int k) { return k == top ? 1.0 : power((key_value(k) - vmax) * step); };
        auto count_at = [&](int k) {
            const uint32_t b = key_bits(k);
            return (hist[b & 0x7fffu] >> ((b >> 11) & 16u)) & 0xffffu;
        };
        // 1,024 keys share their spacing, so a key's weight is that of the key above it
        // times one factor
        if (t < 64) s.ratio[t] = power((key_value((t << 10) + 512) - key_value((t << 10) + 513)) * step);
        __syncthreads();
        // a wavefront takes four blocks of positive keys and the four of the same patterns
        // with a sign; a lane four keys of each (its 16 lanes are a block); added to what an
        // earlier piece of the row left there
        auto block_sums = [&](bool add) {
            for (int b = 4 * wave; b < kSrBlocks / 2; b += 4 * kSrWaves) {
                const int p0 = 64 * b + 4 * lane;
                const u4v w = *reinterpret_cast<const u4v*>(hist + p0);
#pragma unroll
                for (int neg = 0; neg < 2; ++neg) {
                    // counts by descending key
                    uint32_t c[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[j] = neg ? w[j] >> 16 : w[3 - j] & 0xffffu;
                    const int k = neg ? 0x7fff - p0 : 0x8000 + p0 + 3;   // the first one's key
                    uint32_t n = (c[0] + c[1]) + (c[2] + c[3]);
                    double m = 0.0;
                    if (__any(n != 0u)) {
                        if (k < top && k - 3 > kSrLowest) {
                            const double r = s.ratio[k >> 10];
                            m = weight(k) * fma(fma(fma((double)c[3], r, (double)c[2]), r, (double)c[1]), r, (double)c[0]);
                        } else if (n != 0u) {   // the largest key, -infinity
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (c[j] != 0u) m += (double)c[j] * weight(k - j);
                        }
                        n = row16_sum(n);
                        m = row16_sum(m);
                    }
                    if ((lane & 15) == 0) {
                        const int at = kSrBlocks - 1 - (k >> 6);
                        s.cnt[at] = add ? s.cnt[at] + n : n;
                        s.mass[at] = add ? s.mass[at] + m : m;
                    }
                }
            }
            __syncthreads();
        };
        block_sums(false);
        // inclusive prefix over the blocks, thread t block t.  The sums form a tree, so a block
        // without ids could differ from the block before it by a rounding; it takes that one's
        // mass instead (a wavefront's lanes from the last with ids, and the wavefronts before it
        // are added in one order), and a search for the first block past a goal ends in one
        // that has ids.
        uint32_t n_in;
        double m_in;
        auto prefix = [&] {
            const uint32_t own = s.cnt[t];
            n_in = wave_prefix(own);
            m_in = wave_prefix(s.mass[t]);
            const uint64_t some = __ballot(own != 0u) & (~0ull >> (63 - lane));
            const double last = __shfl(m_in, some ? 63 - __builtin_clzll(some) : 0);
            m_in = some ? last : 0.0;
            if (lane == 63) {
                s.red_n[wave] = n_in;
                s.red_m[wave] = m_in;
            }
            __syncthreads();
            double before = 0.0;
            for (int w = 0; w < wave; ++w) {
                n_in += s.red_n[w];
                before += s.red_m[w];
            }
            m_in += before;
        };
        prefix();
        uint32_t total = 0;
        for (int w = 0; w < kSrWaves; ++w) total += s.red_n[w];
        __syncthreads();
        bool whole = true;   // the histogram holds the row
        if (total != (uint32_t)V || s.wrap != 0u) {
            whole = false;
            for (int lo = 0; lo < V; lo += kSrPiece) {
                clear();
                each_step(row, V, lo, min(V, lo + kSrPiece), [&](int i, const u4v& x, bool all) { sr_count(i, x, all, V, hist, seen); });
                __syncthreads();
                fold();
                block_sums(lo > 0);
            }
            prefix();
            __syncthreads();
        }
        s.cnt[t] = n_in;
        s.mass[t] = m_in;
        __syncthreads();

        // the levels of block b
        auto levels = [&](int b) {
            SrLevels x;
            x.key = ((kSrBlocks - 1 - b) << 6) + 63 - lane;
            if (whole) {
                x.c = count_at(x.key);
            } else {
                __syncthreads();
                if (t < 64) s.level[t] = 0u;
                __syncthreads();
                each_step(row, V, 0, V, [&](int i, const u4v& x8, bool) {
                    for (int j = 0; j < 8; ++j) {
                        const int kj = key_of(half_of(x8, j));
                        if (i + j < V && kj >> 6 == kSrBlocks - 1 - b) atomicAdd(&s.level[63 - (kj & 63)], 1u);
                    }
                });
                __syncthreads();
                x.c = s.level[lane];
            }
            x.e = x.c != 0u ? weight(x.key) : 0.0;
            const uint32_t n = wave_prefix(x.c);
            const double m = wave_prefix((double)x.c * x.e);
            // what stands before a level: the inclusive sums of the lane above
            uint32_t pn = (uint32_t)__shfl_up((int)n, 1);
            double pm = __shfl_up(m, 1);
            if (lane == 0) pn = 0u, pm = 0.0;
            x.before_n = (b > 0 ? s.cnt[b - 1] : 0u) + pn;
            x.before_m = (b > 0 ? s.mass[b - 1] : 0.0) + pm;
            return x;
        };
        auto last_lane = [](uint64_t mask) { return 63 - __builtin_clzll(mask); };
        // the first block that passes (blocks behind it pass too, but for a rounding), else the
        // last one
        auto first_block = [&](auto&& pass) {
            const uint64_t far = __ballot(pass(16 * lane + 15));
            if (!far) return kSrBlocks - 1;
            const int b = 16 * __builtin_ctzll(far);
            return b + (int)__builtin_ctzll(__ballot(pass(b + (lane & 15))));
        };

        // ---- the cuts and the draw: one wavefront (where the histogram holds the row)
        if (wave == 0 || !whole) {
            // how many ids are kept
            uint32_t n = (uint32_t)V;
            const int k = a.top_k ? a.top_k[blockIdx.x] : 0;
            if (k > 0) n = min(n, (uint32_t)k);
            const double mp = a.min_p ? (double)a.min_p[blockIdx.x] : 0.0;
            const double tp = a.top_p ? (double)a.top_p[blockIdx.x] : 1.0;
            if (!(mp <= 0.0)) {
                // the first block whose smallest key is below min_p
                const SrLevels x = levels(first_block([&](int b) {
                    const int low = (kSrBlocks - 1 - b) << 6;
                    return low <= top && !(weight(low) >= mp);
                }));
                const uint64_t in = __ballot(x.c != 0u && x.e >= mp);
                uint32_t kept = (uint32_t)__shfl((int)x.before_n, 0);
                if (in) kept = (uint32_t)__shfl((int)(x.before_n + x.c), last_lane(in));
                n = min(n, max(1u, kept));
            }
            if (tp < 1.0) {
                // the first place where the running mass reaches the goal
                const double goal = tp * s.mass[kSrBlocks - 1];
                const SrLevels x = levels(first_block([&](int b) { return s.cnt[b] > 0u && s.mass[b] >= goal; }));
                const uint64_t any = __ballot(x.c != 0u);
                const uint64_t in = __ballot(x.c != 0u && x.before_m + (double)x.c * x.e >= goal);
                const double need = ceil((goal - x.before_m) / (x.e > 0.0 ? x.e : 1.0));
                const uint32_t part = (uint32_t)fmin(fmax(need, 1.0), (double)max(1u, x.c));
                uint32_t kept = n;
                if (in) kept = (uint32_t)__shfl((int)(x.before_n + part), __builtin_ctzll(in));
                else if (any) kept = (uint32_t)__shfl((int)(x.before_n + x.c), last_lane(any));
                n = min(n, kept);
            }
            // their mass, and the place of the draw
            const int bk = first_block([&](int b) { return s.cnt[b] >= n; });
            SrLevels x = levels(bk);
            const uint64_t end = __ballot(x.c != 0u && x.before_n < n && n <= x.before_n + x.c);
            const double upto = x.before_m + (double)(n - x.before_n) * x.e;
            // (not below 0: the blocks before the first with ids have a mass of 0)
            const double goal = fmax(a.u[blockIdx.x] * __shfl(upto, end ? __builtin_ctzll(end) : 0), 0.0);
            const int bd = min(bk, first_block([&](int b) { return s.mass[b] > goal; }));
            if (bd != bk) x = levels(bd);
            const uint32_t c = x.before_n < n ? min(x.c, n - x.before_n) : 0u;   // kept ids of the level
            const uint64_t any = __ballot(c != 0u), hit = __ballot(c != 0u && x.before_m + (double)c * x.e > goal);
            const double place = x.e > 0.0 ? floor((goal - x.before_m) / x.e) : 0.0;
            const int at = hit ? __builtin_ctzll(hit) : any ? last_lane(any) : 0;
            const int own = hit ? (int)fmin(fmax(place, 0.0), (double)max(1u, c) - 1.0) : (int)max(1u, c) - 1;
            if (t == at) {
                s.pick[0] = x.key;
                s.pick[1] = own;
                s.pick[2] = (int)x.c;
            }
        }
        __syncthreads();
        key = s.pick[0];
        nth = s.pick[1];
        ties = s.pick[2];
        __syncthreads();
    }

    // ---- the nth id (ascending) whose key this is: patterns compared as they are, zero
    // without its sign; NaN beside -infinity are looked at one by one
    const bool low = key == kSrLowest;
    const uint32_t care = key == 0x8000 ? 0x7fff7fffu : 0xffffffffu, pair = key_bits(key) * 0x10001u;
    auto match = [&](int i, const u4v& x, int j) {
        return i + j < V && (low ? key_of(half_of(x, j)) == key : ((half_of(x, j) ^ pair) & care & 0xffffu) == 0u);
    };
    auto some = [&](const u4v& x) {   // does one of the 8 match (or lie behind the row)
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 m{0xffff, 0xffff};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = (x[i] ^ pair) & care;
            m = __builtin_elementwise_min(m, __builtin_bit_cast(us2, w));
        }
        return low || m[0] == 0 || m[1] == 0;
    };
    auto matches = [&](int i, const u4v& x) {
        int c = 0;
        if (some(x)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) c += match(i, x, j) ? 1 : 0;
        }
        return c;
    };
    if (nth == 0) {   // the first: each thread's, then the least of them
        int mine = 0x7fffffff;
        each_step(row, V, 0, V, [&](int i, const u4v& x, bool) {
            if (mine != 0x7fffffff || !some(x)) return;
#pragma unroll
            for (int j = 7; j >= 0; --j)
                if (match(i, x, j)) mine = i + j;
        });
        mine = 0x7fffffff - wave_max_i(0x7fffffff - mine);
        if (lane == 0) s.red_i[wave] = mine;
        __syncthreads();
        if (t == 0) {
            for (int w = 0; w < kSrWaves; ++w) mine = min(mine, s.red_i[w]);
            a.out[blockIdx.x] = mine;
        }
        return;
    }
    if (ties <= kSrThreads) {   // all of them into a list; a thread ranks one
        int* const list = reinterpret_cast<int*>(hist);
        if (t == 0) s.pick[0] = 0;
        __syncthreads();
        each_step(row, V, 0, V, [&](int i, const u4v& x, bool) {
            if (!some(x)) return;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (match(i, x, j)) list[min(atomicAdd(&s.pick[0], 1), kSrThreads - 1)] = i + j;
        });
        __syncthreads();
        if (t < ties) {
            const int mine = list[t];
            int before = 0;
            for (int i = 0; i < ties; ++i) before += list[i] < mine ? 1 : 0;
            if (before == nth) a.out[blockIdx.x] = mine;
        }
        return;
    }
    auto wave_inclusive = [&](int v) { return (int)wave_prefix((uint32_t)v); };
    // the id in the wavefront's 512 keys of one step, which hold the n-th
    auto finish = [&](int i, const u4v& x, int n) {
        const int c = matches(i, x);
        int before = wave_inclusive(c) - c;
        if (n < before || n >= before + c) return;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (match(i, x, j) && before++ == n) a.out[blockIdx.x] = i + j;
    };
    auto wave_total = [&](int i, const u4v& x) {
        const int c = matches(i, x);
        return __any(c > 0) ? __shfl(wave_inclusive(c), 63) : 0;
    };
    // steps in groups of kSrPart: hits of each (step, wavefront), in order of the ids
    for (int lo = 0; lo < V; lo += kSrPart * kSrStep) {
        const int hi = min(V, lo + kSrPart * kSrStep), steps = (hi - lo + kSrStep - 1) / kSrStep;
        each_step(row, V, lo, hi, [&](int i, const u4v& x, bool) {
            const int c = wave_total(i, x);
            if (lane == 0) s.hits[(i - lo) / kSrStep * kSrWaves + wave] = c;
        });
        if (t == 0) s.pick[0] = -1;
        __syncthreads();
        if (wave == 0) {
            constexpr int kPer = (kSrPart * kSrWaves + 63) / 64;
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
                finish(i, load_tail(row, i, V), n);
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
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_lds(allowed, reinterpret_cast<const void*>(&sample_rows_kernel), kSrHist, "sample_rows: LDS attribute"))
        return rc;
    SrArgs a{logits, stride, vocab, temperature, top_k, top_p, min_p, u, out};
    sample_rows_kernel<<<(unsigned)rows, kSrThreads, kSrHist, as_stream(stream)>>>(a);
    return launch_check("sample_rows");
}
