// Shared prefixes of a paged serving step (bx_prefix_plan): request r's rows come
// behind the first keys of another request, which are computed once for all that
// share them (bx_attention_prefix_q8_f16, attention_q8.hip).
//
// Keys shared by request r: min(shared_lens[r], lens[parent[r]]).  The rows that
// share any are listed parent by parent, in the order of rows within one: the
// requests' numbers (parent, request) are sorted, and a prefix sum of their row
// counts in that order is where each request's rows begin in the list.  Every
// workgroup sorts for itself, then fills its own share of the rows.
// The sort is bitonic; a wavefront holds 64 E consecutive numbers in registers, so that all
// but the few exchanges between wavefronts go without LDS and barriers.
// Latency bounds it (loads in series, the sort's steps, the rows): 17 requests 4.0 us; 740 with
// 25,000 rows 10.0 (17.9 with the numbers in LDS and a barrier a step); 4,040 requests 28.
#include <type_traits>

#include "kv_pages.h"

namespace bx {
namespace {

constexpr int kPrefixThreads = 512;
constexpr int kPrefixRows = 512;   // rows a workgroup

struct PrefixArgs {
    const int32_t *parent, *shared_lens, *starts, *lens, *pos_in;
    int n_req, max_rows, slots;     // slots: a power of two, n_req or more, at most 512 E
    int32_t *pos, *shared, *order, *groups, *group_starts;
};

// The value of lane l ^ J: without a trip through the LDS but for 4.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    const int lane = threadIdx.x & 63;
    if constexpr (J == 1) return dpp_of<0xB1>(v);
    else if constexpr (J == 2) return dpp_of<0x4E>(v);
    else if constexpr (J == 8) return dpp_of<0x128>(v);   // the row of 16, half way round
    else if constexpr (J == 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (uint32_t)((lane & 16) ? s[0] : s[1]);
    } else if constexpr (J == 32) {
        const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (uint32_t)((lane & 32) ? s[0] : s[1]);
    } else return (uint32_t)__shfl_xor((int)v, J);
}

template <int E>
__global__ __launch_bounds__(kPrefixThreads) void prefix_plan_kernel(PrefixArgs a) {
    // the sorted numbers (parent << 12 | request; none: all ones), later the requests' shared keys
    constexpr int N = kPrefixThreads * E;
    static_assert(N <= kPlanMaxReq);
    __shared__ uint32_t s_key[N];
    __shared__ int32_t s_start[N + 1], s_at[N];
    __shared__ uint32_t red[2][kPrefixThreads / 64];
    const int t = threadIdx.x, n = a.n_req, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // rows of request r; starts that do not ascend within the step's rows give none
    auto count = [&](int r) {
        const int b = s_start[r], e = s_start[r + 1];
        return b >= 0 && e > b && e <= a.max_rows ? e - b : 0;
    };
    for (int r = t; r <= n; r += kPrefixThreads) s_start[r] = a.starts[r];
    __syncthreads();
    // number e of this thread: request 64 E wave + 64 i + lane
    uint32_t key[E];
    int share[E];
    auto number = [&](int i) { return 64 * (E * wave + i) + lane; };
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int r = number(i), p = r < n ? a.parent[r] : -1;
        share[i] = p >= 0 && p < n && p != r ? max(0, min(a.shared_lens[r], a.lens[p])) : 0;
        key[i] = share[i] > 0 && count(r) > 0 ? (uint32_t)p << 12 | (uint32_t)r : 0xffffffffu;
    }

    // ---- bitonic sort, ascending
    for (int k = 2; k <= a.slots; k <<= 1) {
        uint32_t other[E];
        auto keep = [&](int j) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int e = number(i);
                key[i] = ((e & k) == 0) == ((e & j) == 0) ? min(key[i], other[i]) : max(key[i], other[i]);
            }
        };
        for (int j = k >> 1; j >= 64; j >>= 1) {
            if (j >= 64 * E) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < E; ++i) s_key[number(i)] = key[i];
                __syncthreads();
#pragma unroll
                for (int i = 0; i < E; ++i) other[i] = s_key[number(i) ^ j];
            } else {
#pragma unroll
                for (int d = 1; d < E; d *= 2)
                    if (j == 64 * d)
#pragma unroll
                        for (int i = 0; i < E; ++i) other[i] = key[i ^ d];
            }
            keep(j);
        }
        auto lanes = [&]<int J>(std::integral_constant<int, J>) {
            if (J >= k) return;
#pragma unroll
            for (int i = 0; i < E; ++i) other[i] = lane_xor<J>(key[i]);
            keep(J);
        };
        lanes(std::integral_constant<int, 32>{});
        lanes(std::integral_constant<int, 16>{});
        lanes(std::integral_constant<int, 8>{});
        lanes(std::integral_constant<int, 4>{});
        lanes(std::integral_constant<int, 2>{});
        lanes(std::integral_constant<int, 1>{});
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; ++i) s_key[number(i)] = key[i];
    __syncthreads();

    // ---- rows and groups before each of them, `per` consecutive ones a thread
    const int per = (a.slots + kPrefixThreads - 1) / kPrefixThreads, i0 = min(a.slots, t * per), i1 = min(a.slots, i0 + per);
    auto first = [&](int i) { return i == 0 || (s_key[i - 1] >> 12) != (s_key[i] >> 12); };
    uint32_t rows = 0, groups = 0;   // (a step's rows are below 2^31)
    for (int i = i0; i < i1; ++i)
        if (s_key[i] != 0xffffffffu) {
            rows += (uint32_t)count((int)(s_key[i] & 0xfff));
            groups += first(i) ? 1u : 0u;
        }
    uint32_t before[2], total[2];
    {
        const uint32_t own[2] = {rows, groups};
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            before[v] = wave_prefix(own[v]);
            if (lane == 63) red[v][wave] = before[v];
            before[v] -= own[v];
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            total[v] = 0u;
#pragma unroll
            for (int w = 0; w < kPrefixThreads / 64; ++w) {
                if (w < wave) before[v] += red[v][w];
                total[v] += red[v][w];
            }
        }
    }
    const bool lead = blockIdx.x == 0;
    for (int i = i0; i < i1; ++i) {
        if (s_key[i] == 0xffffffffu) break;
        const int r = (int)(s_key[i] & 0xfff);
        s_at[r] = (int)before[0];
        if (first(i)) {
            if (lead) {
                a.groups[before[1]] = (int)(s_key[i] >> 12);
                a.group_starts[before[1]] = (int)before[0];
            }
            ++before[1];
        }
        before[0] += (uint32_t)count(r);
    }
    if (lead)
        for (int i = (int)total[1] + t; i <= n; i += kPrefixThreads) {
            if (i < n) a.groups[i] = -1;
            a.group_starts[i] = (int)total[0];
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (number(i) < n) s_key[number(i)] = (uint32_t)share[i];
    __syncthreads();

    // ---- the rows
    const int live = s_start[n], row0 = (int)blockIdx.x * kPrefixRows, n_own = min(a.max_rows - row0, kPrefixRows);
    for (int o = t; o < n_own; o += kPrefixThreads) {
        const int i = row0 + o, p = a.pos_in[i];
        int s = 0;
        if (i < live) {
            int lo = 0, hi = n;   // the last request that starts at row i or before
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_start[mid] <= i) lo = mid;
                else hi = mid;
            }
            const int at = i - s_start[lo];
            if (at >= 0 && at < count(lo)) {
                s = (int)s_key[lo];
                const uint32_t to = (uint32_t)s_at[lo] + (uint32_t)at;   // (below max_rows where starts ascend)
                if (s > 0 && to < (uint32_t)a.max_rows) a.order[to] = i;
            }
        }
        a.shared[i] = s;
        a.pos[i] = p >= 0 ? (int)min((int64_t)p + s, (int64_t)0x7fffffff) : p;
        if (i >= (int)total[0]) a.order[i] = -1;
    }
}

}  // namespace
}  // namespace bx

using namespace bx;

extern "C" {

int bx_prefix_plan(const int32_t* parent, const int32_t* shared_lens, const int32_t* starts, const int32_t* lens,
                   int n_req, const int32_t* pos_in, int32_t* pos, int32_t* shared, int32_t* order, int max_rows,
                   int32_t* groups, int32_t* group_starts, void* stream) {
    if (!parent || !shared_lens || !starts || !lens || !pos_in || !pos || !shared || !order || !groups || !group_starts)
        return fail(BX_EINVAL, "prefix_plan: null pointer");
    if (n_req <= 0 || max_rows <= 0) return fail(BX_EINVAL, "prefix_plan: bad shape");
    if (n_req > kPlanMaxReq) return fail(BX_EUNSUPPORTED, "prefix_plan: more than 4096 requests");
    const int32_t* const all[] = {pos, shared, order, groups, group_starts, parent, shared_lens, starts, lens, pos_in};
    for (int i = 0; i < 5; ++i)
        for (int j = i + 1; j < 10; ++j)
            if (all[i] == all[j] && !(i == 0 && j == 9))
                return fail(BX_EINVAL, "prefix_plan: only pos may lie over pos_in");
    PrefixArgs a{};
    a.parent = parent; a.shared_lens = shared_lens; a.starts = starts; a.lens = lens; a.pos_in = pos_in;
    a.n_req = n_req; a.max_rows = max_rows;
    a.slots = 64;
    while (a.slots < n_req) a.slots *= 2;
    a.pos = pos; a.shared = shared; a.order = order; a.groups = groups; a.group_starts = group_starts;
    const unsigned grid = ((unsigned)max_rows + kPrefixRows - 1) / kPrefixRows;
    hipStream_t st = as_stream(stream);
    if (a.slots <= kPrefixThreads) prefix_plan_kernel<1><<<grid, kPrefixThreads, 0, st>>>(a);
    else if (a.slots <= 2 * kPrefixThreads) prefix_plan_kernel<2><<<grid, kPrefixThreads, 0, st>>>(a);
    else prefix_plan_kernel<8><<<grid, kPrefixThreads, 0, st>>>(a);
    return launch_check("prefix_plan");
}

}  // extern "C"
