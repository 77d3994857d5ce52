// A mixture of 1-bit experts: the router's choice, the experts' linears over
// ragged groups of rows, and the weighted sum of what the experts give.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "b1_device.h"
#include "b1_internal.h"

namespace b1 {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));

// ------------------------------------------------- scans over a wave ----

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t old, uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)x, CTRL, ROWS, 0xf, false);
}
// Inclusive sums and maxima over the lanes before and a lane itself: within
// rows of 16 lanes by shifts, then the rows' last lanes onto the next rows.
__device__ __forceinline__ uint32_t scan_add(uint32_t x) {
    x += dpp<0x111>(0, x);
    x += dpp<0x112>(0, x);
    x += dpp<0x114>(0, x);
    x += dpp<0x118>(0, x);
    x += dpp<0x142, 0xa>(0, x);
    x += dpp<0x143, 0xc>(0, x);
    return x;
}
__device__ __forceinline__ uint32_t scan_max(uint32_t x) {
    x = max(x, dpp<0x111>(0, x));
    x = max(x, dpp<0x112>(0, x));
    x = max(x, dpp<0x114>(0, x));
    x = max(x, dpp<0x118>(0, x));
    x = max(x, dpp<0x142, 0xa>(0, x));
    x = max(x, dpp<0x143, 0xc>(0, x));
    return x;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t x, int lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) { return lane_value(scan_max(x), 63); }
template <class T>
__device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// ------------------------------------------------------------- router ----

constexpr int kRouteThreads = 1024, kRouteWaves = kRouteThreads / 64;

__device__ __forceinline__ float logit_at(const RouteArgs &a, int64_t i) {
    if (a.type == 2) return static_cast<const float *>(a.logits)[i];
    const uint16_t h = static_cast<const uint16_t *>(a.logits)[i];
    return a.type == 1 ? __builtin_bit_cast(float, (uint32_t)h << 16)
                       : (float)__builtin_bit_cast(_Float16, h);
}

// A token's experts and weights, by one wave; lane j < top_k returns the j-th
// expert (-1: none) and writes it and its weight.
//
// Lane l holds logits EL * l .. EL * l + EL - 1.  A choice is the largest key
// of all lanes (a scan of six steps), ties to the lowest lane, which holds the
// lowest experts.  Keys are the logits as integers of the same order, or,
// where a bias makes a score's rounding count (WIDE), the 64-bit scores +
// bias, compared by their high words first.  Key 0 is never chosen: -inf and
// what is chosen already.  NaN comes behind every number (and makes the row's
// weights NaN).  Up to four experts a lane are sorted once, so that a choice
// only moves the lane's next one up.
constexpr uint32_t kNanKey = 1;
template <int EL, bool WIDE>
__device__ __forceinline__ int route_token(const RouteArgs &a, int token) {
    constexpr bool SORTED = EL > 1 && EL <= 4;
    const int lane = threadIdx.x & 63;
    float x[EL];
    uint32_t hi[EL], lo[WIDE ? EL : 1];
    int id[EL];
    const int64_t row = (int64_t)token * a.ld;
    uint32_t top = 0; // the largest logit, as a key
    bool nan = false;
    auto key_of = [](float v) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f); // -0 is 0
        return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    };
    auto value_of = [](uint32_t key) {
        return __builtin_bit_cast(float, key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
    };
#pragma unroll
    for (int i = 0; i < EL; ++i) {
        const int e = lane * EL + i;
        id[i] = e;
        x[i] = e < a.experts ? logit_at(a, row + e) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < EL; ++i) {
        nan |= x[i] != x[i];
        hi[i] = x[i] > -INFINITY ? key_of(x[i]) : x[i] != x[i] ? kNanKey : 0u;
        top = max(top, hi[i]);
    }
    top = wave_max(top);
    const float peak = value_of(top);
    float all = 0.f; // softmax over all experts
    if (!a.sigmoid && !a.renormalize) {
#pragma unroll
        for (int i = 0; i < EL; ++i) all += x[i] > -INFINITY ? expf(x[i] - peak) : 0.f;
        all = wave_sum(all);
    }
    if constexpr (WIDE) {
        double z[EL], sum = 0.0;
#pragma unroll
        for (int i = 0; i < EL; ++i) {
            if (a.sigmoid) {
                z[i] = 1.0 / (1.0 + exp(-(double)x[i]));
            } else {
                z[i] = x[i] > -INFINITY ? exp((double)x[i] - (double)peak) : 0.0;
                sum += z[i];
            }
        }
        if (!a.sigmoid) sum = wave_sum(sum);
        // an infinite logit: weights NaN, chosen by the logits of those not off
        nan |= !a.sigmoid && peak == INFINITY;
        const bool by_score = a.sigmoid || sum < (double)INFINITY;
#pragma unroll
        for (int i = 0; i < EL; ++i) {
            lo[i] = 0;
            if (id[i] >= a.experts) continue;
            const float bias = a.bias[id[i]];
            if (bias == -INFINITY) hi[i] = 0; // off, whatever its logit
            if (!by_score || hi[i] <= kNanKey) continue;
            const double k = (a.sigmoid ? z[i] : z[i] / sum) + (double)bias + 0.0;
            const uint64_t b = __builtin_bit_cast(uint64_t, k);
            const uint64_t key = b ^ ((b >> 63) ? ~0ull : 1ull << 63);
            nan |= k != k;
            hi[i] = k > -(double)INFINITY ? (uint32_t)(key >> 32) : k != k ? kNanKey : 0u;
            lo[i] = k == k ? (uint32_t)key : 0u;
        }
    }
    const bool any_nan = __ballot(nan) != 0;
    auto above = [&](int i, int j) { // i's key is larger than j's
        if constexpr (WIDE) return hi[i] > hi[j] || (hi[i] == hi[j] && lo[i] > lo[j]);
        return hi[i] > hi[j];
    };
    if constexpr (SORTED) {
#pragma unroll
        for (int n = 1; n < EL; ++n)
#pragma unroll
            for (int i = n; i > 0; --i) {
                const bool swap = above(i, i - 1);
                const uint32_t h = hi[i];
                hi[i] = swap ? hi[i - 1] : h;
                hi[i - 1] = swap ? h : hi[i - 1];
                const int e = id[i];
                id[i] = swap ? id[i - 1] : e;
                id[i - 1] = swap ? e : id[i - 1];
                if constexpr (WIDE) {
                    const uint32_t l = lo[i];
                    lo[i] = swap ? lo[i - 1] : l;
                    lo[i - 1] = swap ? l : lo[i - 1];
                }
            }
    }
    int mine = -1;
    for (int j = 0; j < a.top_k; ++j) {
        uint32_t m = hi[0], ml = 0;
        int e = id[0];
        if constexpr (WIDE) ml = lo[0];
        if constexpr (!SORTED) { // the lane's largest, the first of equals
#pragma unroll
            for (int i = 1; i < EL; ++i) {
                bool more = hi[i] > m;
                if constexpr (WIDE) more = more || (hi[i] == m && lo[i] > ml);
                m = more ? hi[i] : m;
                e = more ? id[i] : e;
                if constexpr (WIDE) ml = more ? lo[i] : ml;
            }
        }
        const uint32_t best = wave_max(m);
        if (best == 0) break;
        bool same = m == best;
        if constexpr (WIDE) {
            const uint32_t best_lo = wave_max(same ? ml : 0u);
            same = same && ml == best_lo;
        }
        const int l = __builtin_ctzll(__ballot(same));
        const int chosen = __builtin_amdgcn_readlane(e, l);
        if (lane == j) mine = chosen;
        if (lane == l) {
            if constexpr (SORTED) {
#pragma unroll
                for (int i = 0; i + 1 < EL; ++i) {
                    hi[i] = hi[i + 1];
                    id[i] = id[i + 1];
                    if constexpr (WIDE) lo[i] = lo[i + 1];
                }
                hi[EL - 1] = 0;
            } else {
#pragma unroll
                for (int i = 0; i < EL; ++i) hi[i] = id[i] == chosen ? 0u : hi[i];
            }
        }
    }
    const float mine_x = mine >= 0 ? logit_at(a, row + mine) : -INFINITY;
    float weight;
    if (a.sigmoid) {
        // in 64 bits: scores of far logits stay apart from zero
        double s = mine >= 0 ? 1.0 / (1.0 + exp(-(double)mine_x)) : 0.0;
        if (a.renormalize) {
            const double sum = wave_sum(s);
            s = sum > 0.0 ? s / sum : 0.0;
        }
        weight = (float)(s * (double)a.scale);
    } else {
        // divided by their sum the chosen weights do not depend on what is
        // subtracted: the largest chosen logit (without a bias the largest of
        // all), so that none far above, left out by its bias, takes them to 0
        float from = peak;
        if constexpr (WIDE)
            if (a.renormalize) from = value_of(wave_max(mine_x > -INFINITY ? key_of(mine_x) : 0u));
        const float p = mine >= 0 ? expf(mine_x - from) : 0.f;
        weight = p / (a.renormalize ? wave_sum(p) : all) * a.scale;
    }
    if (any_nan) weight = __builtin_nanf("");
    if (mine < 0) weight = 0.f;
    if (lane < a.top_k) {
        a.expert[(int64_t)token * a.top_k + lane] = mine;
        a.weight[(int64_t)token * a.top_k + lane] = weight;
    }
    return lane < a.top_k ? mine : -1;
}

// Exclusive prefix sums of v[0 .. n) in LDS, by the first wave; returns (in
// that wave) the total.
__device__ __forceinline__ uint32_t lds_prefix(uint32_t *v, int n) {
    const int lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (int e0 = 0; e0 < n; e0 += 64) {
        const uint32_t x = e0 + lane < n ? v[e0 + lane] : 0u;
        const uint32_t s = scan_add(x);
        if (e0 + lane < n) v[e0 + lane] = before + s - x;
        before += lane_value(s, 63);
    }
    return before;
}

// Orders the accesses of a wave's lanes to what they share, before it and
// behind it (no instruction by itself: a wave's LDS accesses run in order).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Places of slots [s0, s1) of `expert` by a whole work-group: slot s of expert
// e goes to row base[e] + the number of e's slots before s.  A wave takes a
// contiguous part; counts[wave][expert] (LDS) become the parts' first rows.
__device__ __forceinline__ void route_place(const RouteArgs &a, int64_t s0, int64_t s1, const uint32_t *base,
                                            uint32_t *counts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = a.experts;
    for (int i = threadIdx.x; i < kRouteWaves * E; i += kRouteThreads) counts[i] = 0;
    const int64_t part = (s1 - s0 + 64 * kRouteWaves - 1) / (64 * kRouteWaves) * 64;
    const int64_t p0 = s0 + wave * part, p1 = min(p0 + part, s1);
    uint32_t *mine = counts + wave * E;
    __syncthreads();
    for (int64_t s = p0 + lane; s < p1; s += 64) {
        const int e = a.expert[s];
        if (e >= 0) atomicAdd(&mine[e], 1u);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) {
        uint32_t at = base[e];
        for (int w = 0; w < kRouteWaves; ++w) {
            const uint32_t n = counts[w * E + e];
            counts[w * E + e] = at;
            at += n;
        }
    }
    __syncthreads();
    const int bits = 32 - __builtin_clz(E);
    for (int64_t s = p0; s < p1; s += 64) {
        const int64_t slot = s + lane;
        const int e = slot < p1 ? a.expert[slot] : -1;
        // the lanes of the same expert
        uint64_t same = __ballot(e >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t one = __ballot((e >> b) & 1);
            same &= (e >> b) & 1 ? one : ~one;
        }
        // all of them read the expert's next row before their first moves it on,
        // and the next turn reads it behind that
        const int before = __popcll(same & ((1ull << lane) - 1));
        const int at = e >= 0 ? (int)(mine[e] + (uint32_t)before) : -1;
        wave_sync();
        if (e >= 0 && before == 0) mine[e] = (uint32_t)at + (uint32_t)__popcll(same);
        wave_sync();
        if (e >= 0) a.order[at] = (int)slot;
        if (slot < p1) a.place[slot] = at;
    }
}

// The whole router in one work-group: few tokens, or no workspace.
template <int EL, bool WIDE>
__global__ __launch_bounds__(kRouteThreads) void b1_route_kernel(RouteArgs a) {
    extern __shared__ uint32_t route_lds[];
    uint32_t *count = route_lds, *counts = route_lds + a.experts;
    __shared__ uint32_t total;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) count[e] = 0;
    __syncthreads();
    for (int t = wave; t < a.tokens; t += kRouteWaves) {
        const int e = route_token<EL, WIDE>(a, t);
        if (e >= 0) atomicAdd(&count[e], 1u);
    }
    __syncthreads();
    if (wave == 0) {
        const uint32_t n = lds_prefix(count, a.experts);
        if (lane == 0) total = n;
    }
    __syncthreads();
    const int64_t slots = (int64_t)a.tokens * a.top_k;
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) a.start[e] = (int)count[e];
    if (threadIdx.x == 0) a.start[a.experts] = (int)total;
    route_place(a, 0, slots, count, counts);
    for (int64_t r = (int64_t)total + threadIdx.x; r < slots; r += kRouteThreads) a.order[r] = -1;
}

// Many tokens, in two launches: each work-group chooses for `per` tokens and
// counts their experts (16 bits: a token has an expert once; rows of a
// multiple of 4 counts); then each finds its first row of every expert from
// all the counts and places its slots.  Bound by the choice's chain of scans
// and, in the second launch, by the round trips to the counts: 8192 tokens of
// 128 experts 8.7 + 6.3 us traced, where the logits' bytes would take 1 (with
// unsorted lanes and 32-bit counts 9.3 + 7.6; 13.4 in a graph).
__host__ __device__ constexpr int count_row(int experts) { return (experts + 3) / 4 * 4; }

template <int EL, bool WIDE>
__global__ __launch_bounds__(kRouteThreads) void b1_route_choose_kernel(RouteArgs a, int per, uint16_t *counts) {
    extern __shared__ uint32_t route_lds[];
    const int wave = threadIdx.x >> 6, E = count_row(a.experts);
    for (int e = threadIdx.x; e < E; e += kRouteThreads) route_lds[e] = 0;
    __syncthreads();
    const int t1 = min((int)(blockIdx.x + 1) * per, a.tokens);
    for (int t = blockIdx.x * per + wave; t < t1; t += kRouteWaves) {
        const int e = route_token<EL, WIDE>(a, t);
        if (e >= 0) atomicAdd(&route_lds[e], 1u);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) counts[(size_t)blockIdx.x * E + e] = (uint16_t)route_lds[e];
}

__global__ __launch_bounds__(kRouteThreads) void b1_route_place_kernel(RouteArgs a, int per, const uint16_t *counts) {
    extern __shared__ uint32_t route_lds[];
    const int E = count_row(a.experts), quads = E / 4, lane = threadIdx.x & 63;
    uint32_t *base = route_lds, *total = route_lds + E, *parts = route_lds + 2 * E;
    __shared__ uint32_t all;
    for (int e = threadIdx.x; e < E; e += kRouteThreads) base[e] = total[e] = 0;
    __syncthreads();
    // a thread takes four experts of every `groups`-th work-group
    const int groups = kRouteThreads / quads, g = threadIdx.x / quads, q = threadIdx.x - g * quads;
    if (g < groups) {
        uint32_t before[4] = {}, sum[4] = {};
#pragma unroll 8
        for (int w = g; w < (int)gridDim.x; w += groups) {
            const u32x2 n = *reinterpret_cast<const u32x2 *>(counts + (size_t)w * E + 4 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c = (n[i / 2] >> (16 * (i & 1))) & 0xffffu;
                sum[i] += c;
                before[i] += w < (int)blockIdx.x ? c : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (before[i]) atomicAdd(&base[4 * q + i], before[i]);
            if (sum[i]) atomicAdd(&total[4 * q + i], sum[i]);
        }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t n = lds_prefix(total, a.experts);
        if (lane == 0) all = n;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) {
        base[e] += total[e];
        if (blockIdx.x == 0) a.start[e] = (int)total[e];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.start[a.experts] = (int)all;
    __syncthreads();
    const int64_t slots = (int64_t)a.tokens * a.top_k;
    const int64_t s0 = (int64_t)blockIdx.x * per * a.top_k;
    route_place(a, s0, min(s0 + (int64_t)per * a.top_k, slots), base, parts);
    for (int64_t r = (int64_t)all + (int64_t)blockIdx.x * kRouteThreads + threadIdx.x; r < slots;
         r += (int64_t)gridDim.x * kRouteThreads)
        a.order[r] = -1;
}

// ------------------------------------------------------ groups of rows ----

// How many groups of up to BM rows of one expert there are, counting through
// the experts in order, and lane l's share: experts l * each .. of them, the
// first's rows from edge[0] on and its groups `before` the next lane's.  By a
// whole wave.  With starts out of order or range every row of the call is the
// first expert's, so that any contents of `start` give groups within the rows,
// apart from one another, no more of them than group_bound() says, and none of
// the rows that become NaN is left out.  Up to 256 experts a lane keeps its
// experts' edges (its loads all on their way at once), with more it reads them
// again in find_group().
constexpr int kEdges = 4;
struct Groups {
    uint32_t edge[kEdges + 1], before, total;
    int each;
    bool bad; // starts out of order or of range
};
template <int BM>
__device__ __forceinline__ Groups count_groups(const int32_t *start, int experts, int routes) {
    const int lane = threadIdx.x & 63;
    Groups g;
    g.each = (experts + 63) / 64;
    const int e0 = min(lane * g.each, experts), e1 = min(e0 + g.each, experts);
    auto groups = [&](uint32_t rows) { return (rows + BM - 1) / BM; };
    bool bad;
    uint32_t n = 0;
    if (g.each <= kEdges) {
        int v[kEdges + 1];
#pragma unroll
        for (int i = 0; i <= kEdges; ++i) v[i] = start[min(e0 + i, e1)];
        bad = v[0] < 0 || v[kEdges] > routes;
#pragma unroll
        for (int i = 0; i < kEdges; ++i) bad |= v[i + 1] < v[i];
        g.edge[0] = (uint32_t)v[0];
#pragma unroll
        for (int i = 1; i <= kEdges; ++i) g.edge[i] = (uint32_t)v[i];
    } else {
        int last = start[e0];
        bad = last < 0;
        g.edge[0] = (uint32_t)last;
        for (int e = e0; e < e1; ++e) {
            const int v = start[e + 1];
            bad |= v < last;
            n += groups((uint32_t)v - (uint32_t)last);
            last = v;
        }
        bad |= last > routes;
    }
    g.bad = __ballot(bad) != 0;
    if (g.bad) {
        g.edge[0] = lane ? (uint32_t)routes : 0u;
#pragma unroll
        for (int i = 1; i <= kEdges; ++i) g.edge[i] = (uint32_t)routes;
        n = groups((uint32_t)routes - g.edge[0]);
    }
    // (behind the check: one token's up projections 6.4 us, beside it 6.6)
    if (!g.bad && g.each <= kEdges) {
#pragma unroll
        for (int i = 0; i < kEdges; ++i) n += groups(g.edge[i + 1] - g.edge[i]);
    }
    g.before = scan_add(n);
    g.total = lane_value(g.before, 63);
    g.before -= n;
    return g;
}

// The t-th of them (t < total).
struct Group {
    int expert, row0, rows;
};
template <int BM>
__device__ __forceinline__ Group find_group(const Groups &g, const int32_t *start, int experts, int routes, int t) {
    // the last lane with no more groups before it that has some itself
    const uint64_t who = __ballot(g.before <= (uint32_t)t);
    const int l = 63 - __builtin_clzll(who);
    uint32_t left = (uint32_t)t - lane_value(g.before, l), row = lane_value(g.edge[0], l), end = row;
    int e = l * g.each;
    if (g.each <= kEdges) {
#pragma unroll
        for (int i = 0; i < kEdges; ++i) {
            const uint32_t to = lane_value(g.edge[i + 1], l), n = (to - row + BM - 1) / BM;
            if (left < n) {
                end = to;
                break;
            }
            left -= n;
            row = to;
            ++e;
        }
    } else {
        for (;; ++e) {
            end = (uint32_t)(g.bad ? routes : start[e + 1]);
            const uint32_t n = (end - row + BM - 1) / BM;
            if (left < n || e + 1 >= experts) break;
            left -= n;
            row = end;
        }
    }
    row += left * BM;
    // (wave-uniform: scalar registers)
    return Group{__builtin_amdgcn_readfirstlane(e), __builtin_amdgcn_readfirstlane((int)row),
                 __builtin_amdgcn_readfirstlane((int)min(end - row, (uint32_t)BM))};
}

// Groups of up to bm rows that `routes` rows of `experts` experts can have.
int64_t group_bound(int routes, int experts, int bm) {
    return routes / bm + std::min(routes, experts);
}

// This wave's LDS writes are done, and every wave's are seen behind it.
__device__ __forceinline__ void lds_publish() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    lds_barrier();
}

__device__ __forceinline__ floatx4 nan4() {
    const float n = __builtin_nanf("");
    return floatx4{n, n, n, n};
}

// A buffer offset past any buffer: reads zeros.
constexpr uint32_t kNowhere = 0x80000000u;

// silu(x) = x / (1 + 2^(-x log2 e)) by the hardware's exponential and
// reciprocal, which feed an fp16 rounding: the exponent is rounded once and so
// is its factor, the instructions are off by a step each: within 1.5 |x| + 7
// half steps of fp32 from x = -87 on.  Below, the reciprocal leaves the normal
// numbers and becomes 0 (as the exponential becomes infinite): off by less than
// 87 e^-87 < 1.5e-36, which no finite value (below 2^49 from fp16 inputs, scales
// and 2^16 products) brings near fp16's smallest 2^-24.
__device__ __forceinline__ float silu_fast(float x) {
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * x));
}

// The scheduler's order: M times an MFMA, D LDS reads and V vector operations.
template <int M, int V, int D>
__device__ __forceinline__ void interleave() {
    if constexpr (M > 0) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if constexpr (D > 0) __builtin_amdgcn_sched_group_barrier(0x100, D, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, V, 0);
        interleave<M - 1, V, D>();
    }
}

// ------------------------------------------------ few rows an expert ----

// y = W a for up to 16 rows of one expert and `per` steps of 64 weight rows.
//
// The weights are read once a group (6 bytes a block of 32); 64 blocks, one a
// lane, take 27 vector operations and four MFMAs.  512 rows over 128 experts,
// K = 2048, 1536 weight rows (75 MB) 24.5 us, the same loads and sums without
// expansion or MFMAs 16.5, the arithmetic without the loads 22.6.  What bounds
// it is that little runs beside anything else: by its counters a SIMD's matrix
// unit is busy 18 % of the time and its vector unit 38 %, with 2 waves on it
// that wait for data 37 % of theirs and 37 % to issue.  Expanding a block
// beside the MFMAs of the one before in a fixed order, two MFMA chains, two
// steps of loads ahead: no gain.  The sums of each step by another wave first:
// spread over all of them it took 1.4 us more.  Eight waves of four 256s and
// fp32 rows spill 4 registers a step, nothing else does.
//
// MFMA 16x16x32 with 16 weight rows as the A operand and the rows of
// activations as the B operand.  A wave takes U * 256 of K and lane (li, g)
// two blocks (12 bytes) of weight row li for every 256: MFMA (b, c) of the 256
// multiplies chunk c (8 values in packed order) of block 2 g + b, so that a
// lane expands just what it has loaded and the activations' fragments stay in
// registers over all steps.  The waves' partial sums meet in LDS.
template <int NW, int U, int OUT>
__global__ __launch_bounds__(NW * 64, 2) void b1_experts_few_kernel(ExpertArgs a, int parts, int per) {
    constexpr int BM = 16, RS = 68; // floats a row of partial sums
    __shared__ float red[2][NW][BM][RS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, g = lane >> 4;
    const int bid = blockIdx.x;
    const int slot = bid / parts, part = bid - slot * parts;
    const Groups all = count_groups<BM>(a.start, a.experts, a.routes);
    if (bid == 0 && threadIdx.x == 0 && all.bad && a.bad) atomicAdd(a.bad, 1);
    if (slot >= (int)all.total) return;
    const Group gr = find_group<BM>(all, a.start, a.experts, a.routes, slot);

    const uint32_t rs = (uint32_t)(a.K / 32) * 6;
    const __amdgpu_buffer_rsrc_t wrs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t *>(a.w) + (size_t)gr.expert * a.N * rs, (short)0, (int)((uint32_t)a.N * rs), kBufferFlags);
    const __amdgpu_buffer_rsrc_t none = __builtin_amdgcn_make_buffer_rsrc(nullptr, (short)0, 0, kBufferFlags);
    const int pairs = a.K / 64; // of blocks, 12 bytes of a weight row
    uint32_t woff[U]; // of this lane's pair within a weight row
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int pair = (wave * U + u) * 4 + g;
        woff[u] = pair < pairs ? 12u * (uint32_t)pair : kNowhere;
    }
    // weight rows of group nt of step s: 64 s + 16 nt, or 32 gates, then their 32 values
    auto weight_row = [&](int s, int nt) {
        if constexpr (OUT == 3) return 32 * s + 16 * (nt & 1) + (nt >> 1) * a.glu_h + li;
        return 64 * s + 16 * nt + li;
    };
    const int s0 = part * per, s1 = min(s0 + per, OUT == 3 ? a.glu_h / 32 : (a.N + 63) / 64);
    // (rows past the last read that again; behind the last step nothing is read)
    auto load = [&](int s, int u, int nt) {
        const uint32_t off = __umul24((uint32_t)min(weight_row(s, nt), a.N - 1), rs) + woff[u];
        return __builtin_bit_cast(u32x3, __builtin_amdgcn_raw_buffer_load_b96(s < s1 ? wrs : none, (int)off, 0, 0));
    };
    // a step's weights, each replaced by the next step's once it is expanded
    u32x3 w[4][U];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int u = 0; u < U; ++u) w[nt][u] = load(s0, u, nt);

    // the row's activations
    int64_t src = gr.row0 + li;
    bool there = li < gr.rows, wrong = false;
    if (a.order && there) {
        const int s = a.order[src];
        wrong = s < 0 || s >= a.routes;
        src = wrong ? 0 : s / a.top_k;
    }
    const uint32_t wrong_rows = all.bad ? 0xffffu : (uint32_t)__ballot(wrong) & 0xffffu;
    if (wrong_rows && !all.bad && a.bad && part == 0 && threadIdx.x == 0) atomicAdd(a.bad, __popc(wrong_rows));
    there = there && !wrong;
    half8 af[U][2][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int pair = (wave * U + u) * 4 + g;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                half8 v = {};
                if (there && pair < pairs)
                    v = *reinterpret_cast<const half8 *>(a.act + src * a.K + pair * 64 + b * 32 + c * 8);
                af[u][b][c] = v;
            }
    }
    int bad = 0;
    // block b of a pair's words as the operands of its four chunks
    auto expand = [&](const u32x3 &d, int b, u32x4 (&c)[4]) {
        const uint32_t sc = b ? dup_hi16(d[1]) : dup_lo16(d[0]);
        const uint32_t sign = b ? d[2] : __builtin_amdgcn_alignbit(d[1], d[0], 16);
        wpair_quads<0>(sign, sign >> 8, sc, c[0], c[2]);
        wpair_quads<1>(sign, sign >> 8, sc, c[1], c[3]);
    };
    for (int s = s0; s < s1; ++s) {
        floatx4 acc[4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            acc[nt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    u32x4 c[4];
                    expand(w[nt][u], b, c);
                    if (b == 1) w[nt][u] = load(s + 1, u, nt);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        acc[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, c[k]), af[u][b][k],
                                                                         acc[nt], 0, 0, 0);
                }
        }
        float(*const r)[BM][RS] = red[(s - s0) & 1];
        if (li < gr.rows)
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) *reinterpret_cast<floatx4 *>(&r[wave][li][16 * nt + 4 * g]) = acc[nt];
        lds_publish();
        auto sum4 = [&](int row, int col) {
            floatx4 v = *reinterpret_cast<const floatx4 *>(&r[0][row][col]);
#pragma unroll
            for (int k = 1; k < NW; ++k) {
                const floatx4 x = *reinterpret_cast<const floatx4 *>(&r[k][row][col]);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += x[i];
            }
            if ((wrong_rows >> row) & 1) v = nan4();
            return v;
        };
        auto count = [&](const floatx4 &v) {
#pragma unroll
            for (int i = 0; i < 4; ++i) bad += !__builtin_isfinite(v[i]);
        };
        const bool cnt = a.nonfinite != nullptr;
        // another wave first at each step: few rows are one wave's work, and
        // the others go on with the next step meanwhile
        const int item0 = (int)(threadIdx.x + 64 * (NW - (s - s0) % NW)) % (NW * 64);
        if constexpr (OUT == 0) {
            for (int i = item0; i < gr.rows * 16; i += NW * 64) {
                const int row = i >> 4, col = 64 * s + 4 * (i & 15);
                if (col >= a.N) continue;
                const floatx4 v = sum4(row, 4 * (i & 15));
                float *o = a.out + (size_t)(gr.row0 + row) * a.ldo + col;
                if (a.vec && col + 4 <= a.N) {
                    if (cnt) count(v);
                    *reinterpret_cast<floatx4 *>(o) = v;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (col + k < a.N) {
                            bad += cnt && !__builtin_isfinite(v[k]);
                            o[k] = v[k];
                        }
                }
            }
        } else {
            // (row, 32-column block, quad of 4 dwords)
            constexpr int Q = OUT == 3 ? 4 : 8;
            for (int i = item0; i < gr.rows * Q; i += NW * 64) {
                const int row = i / Q, q = i % Q, dq = (q & 3) * 4, blk = q >> 2;
                const int col = (OUT == 3 ? 32 * s : 64 * s + 32 * blk);
                if (OUT != 3 && col >= a.N) continue;
                floatx4 lo = sum4(row, 32 * blk + dq), hi = sum4(row, 32 * blk + dq + 16);
                if (cnt) {
                    count(lo);
                    count(hi);
                }
                if constexpr (OUT == 3) {
                    const floatx4 vlo = sum4(row, 32 + dq), vhi = sum4(row, 48 + dq);
                    if (cnt) {
                        count(vlo);
                        count(vhi);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        lo[k] = mul_f32(silu_fast(lo[k]), vlo[k]);
                        hi[k] = mul_f32(silu_fast(hi[k]), vhi[k]);
                    }
                } else if constexpr (OUT == 2) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        lo[k] = gelu_tanh(lo[k]);
                        hi[k] = gelu_tanh(hi[k]);
                    }
                }
                u32x4 v;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = pack_f16_rounded(lo[k], hi[k]);
                *reinterpret_cast<u32x4 *>(a.pk + (size_t)(gr.row0 + row) * a.ldpw + col / 2 + dq) = v;
            }
        }
    }
    count_nonfinite(a.nonfinite, bad);
}

// ----------------------------------------------- many rows an expert ----

// Tiles of BM rows of one expert and BN = NWN * WN weight rows, by work-groups
// that stay and take tiles in turn: a tile's rows are looked up while the one
// before is computed, and its first stages are on their way while that one is
// stored.
//
// Bound by the matrix units: in the loop over K, 128-row tiles run at 1.4
// PFLOP/s counting the rows they do not have (clock about 1.8 GHz at the
// board's power limit, where a library product of 8192^3 runs at 1.29 to 1.35
// by board); over the whole call the matrix units are busy 64 % of the time
// and the vector units 26 %.  65536 rows over 128 experts, K = 2048, 1536
// weight rows with SwiGLU: 361 to 381 us by board = 1.08 to 1.14 PFLOP/s of
// rows there are; one work-group a tile with its sums stored through LDS took
// 459.  Fp32 rows add their bytes' time (K = 768, 2048 columns, 537 MB: 287 to
// 302 us): the stores hold up the loads of the CU's other work-group, counted
// waits or not.
// Branches that skip the upper 64 rows of tiles without any saved what they
// cost.  One loop over all stages, the reads behind the last one wasted: with
// the last stages apart the compiler copied the sums between loops and spilled
// in them (405 us).  128-row tiles take all 256 registers: one value is stored
// to memory once a work-group and read once a tile; the loop itself spills
// none.
//
// MFMA, 16 weight rows as the A operand, rows of activations as the
// B operand.  A stage is 64 of K: BM rows of 128 bytes, shared by the waves,
// their 16-byte chunks at c ^ row / 2 so that the 16 rows of a fragment read
// cover all banks; and a wave's own WN columns of weights, 12 bytes a column
// and stage, loaded L stages at once so that L lanes take adjacent bytes of a
// row (a slice of WN / L columns a stage, a group of L stages ahead).  R
// stages of activations in a ring, copied straight to LDS.
template <int BM_, int WN_, int NWN_, int R_, int L_, int OCC_, int SETS_>
struct ExpertTile {
    static constexpr int BM = BM_, WN = WN_, NWN = NWN_, R = R_, L = L_, OCC = OCC_, SETS = SETS_;
    static constexpr int NT = NWN * 64, BN = WN * NWN, MT = BM / 16, NTL = WN / 16;
    static constexpr int ASZ = BM * 128;                 // bytes of a stage's activations
    static constexpr int AW = ASZ / 1024 / NWN;          // loads of them a wave
    static constexpr int WSL = WN * 16, WGRP = L * WSL;  // a slice, a group (16 bytes a lane's 12)
    // groups kept: stage s + R's loads fill a slice of group (s + R) / L + 1
    // while stage s + 1 of this and every later group is still to be read
    static constexpr int groups() {
        int g = 0;
        for (int s = 0; s < 4 * L; ++s) g = (s + R) / L + 1 - (s + 1) / L > g ? (s + R) / L + 1 - (s + 1) / L : g;
        return g + 1;
    }
    static constexpr int RW = groups();
    static constexpr int WBASE = R * ASZ, LDS = WBASE + NWN * RW * WGRP;
    static constexpr int LOADS = AW + 1;                 // a wave and stage
    static constexpr int TOK = (BM + 63) / 64;           // of a lane
    static_assert(ASZ % (1024 * NWN) == 0 && WN % 64 == 0 && WN % L == 0 && WN / L * L <= 64, "loads of whole waves");
    static_assert(LDS <= 160 * 1024 && (R - 1) * LOADS < 64, "gfx950 LDS, vmcnt");
};

// Waits until at most `later` stages' loads are outstanding (later <= MAXL).
template <int LOADS, int MAXL>
__device__ __forceinline__ void wait_stages(int later) {
    if constexpr (MAXL == 0) {
        wait_vmcnt<0>();
    } else {
        if (later >= MAXL)
            wait_vmcnt<LOADS * MAXL>();
        else
            wait_stages<LOADS, MAXL - 1>(later);
    }
}

template <class C, int OUT>
__global__ __launch_bounds__(C::NT, C::OCC) void b1_experts_tile_kernel(ExpertArgs a, int tiles_n) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wn = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, g = lane >> 4;
    const Groups all = count_groups<C::BM>(a.start, a.experts, a.routes);
    if (blockIdx.x == 0 && tid == 0 && all.bad && a.bad) atomicAdd(a.bad, 1);
    // contiguous tiles an XCD, its work-groups taking them in turn
    const int tiles = (int)all.total * tiles_n;
    const int xcd = blockIdx.x & 7, each = gridDim.x >> 3;
    const int share = tiles >> 3, more = tiles & 7;
    const int first = xcd * share + min(xcd, more) + ((int)blockIdx.x >> 3);
    const int last = xcd * share + min(xcd, more) + share + (xcd < more ? 1 : 0);
    if (first >= last) return;

    const int K = a.K, n = K / 64;
    const uint32_t rs = (uint32_t)(K / 32) * 6;
    const __amdgpu_buffer_rsrc_t none = __builtin_amdgcn_make_buffer_rsrc(nullptr, (short)0, 0, kBufferFlags);
    __amdgpu_buffer_rsrc_t ars = none, wrs = none;
    uint32_t aoff[C::AW], boff[C::L];
    int expert, row0, rows, n0; // of the tile
    uint64_t wrong[C::TOK];

    // slots of a tile's rows, on their way while the one before is computed
    int slots[C::TOK];
    int expert_next = 0, row0_next = 0, rows_next = 0, n0_next = 0;
    auto look_up = [&](int t) {
        const int GM = 8, tg = t / (GM * tiles_n), first_m = tg * GM;
        const int size = min(GM, (int)all.total - first_m), in = t - first_m * tiles_n;
        const Group gr = find_group<C::BM>(all, a.start, a.experts, a.routes, first_m + in % size);
        expert_next = gr.expert;
        row0_next = gr.row0;
        rows_next = gr.rows;
        n0_next = in / size * C::BN;
        if (a.order)
#pragma unroll
            for (int i = 0; i < C::TOK; ++i) slots[i] = a.order[row0_next + min(64 * i + lane, rows_next - 1)];
    };
    auto swz = [](int row) { return (row >> 1) & 7; };
    auto swl = [](int c) { return C::L == 4 ? (c >> 2) & 3 : C::L == 2 ? (c >> 3) & 1 : 0; };
    // the weight row of a tile column
    auto weight_row = [&](int tc) {
        const int c = n0 + tc;
        if constexpr (OUT == 3) {
            // 32 gates, then their 32 values
            const int j = min(c >> 6, a.glu_h / 32 - 1) * 32 + (c & 31);
            return (c & 32 ? a.glu_h : 0) + j;
        }
        return min(c, a.N - 1);
    };
    // the addresses of the tile that was looked up
    auto aim = [&]() {
        expert = expert_next;
        row0 = row0_next;
        rows = rows_next;
        n0 = n0_next;
        int token[C::TOK];
#pragma unroll
        for (int i = 0; i < C::TOK; ++i) {
            token[i] = min(64 * i + lane, rows - 1);
            bool is = false;
            if (a.order) {
                is = slots[i] < 0 || slots[i] >= a.routes;
                token[i] = is ? 0 : slots[i] / a.top_k;
            }
            wrong[i] = __ballot(is && 64 * i + lane < rows);
        }
        const uint16_t *act = a.act;
        uint32_t bytes = (uint32_t)a.act_rows * (uint32_t)K * 2u;
        if (!a.order) {
            act += (size_t)row0 * K;
            bytes = (uint32_t)rows * (uint32_t)K * 2u;
        }
        ars = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(act), (short)0, (int)bytes, kBufferFlags);
        wrs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.w) + (size_t)expert * a.N * rs, (short)0,
                                                (int)((uint32_t)a.N * rs), kBufferFlags);
#pragma unroll
        for (int i = 0; i < C::AW; ++i) {
            const int row = 8 * (wn * C::AW + i) + lane / 8;
            int tok = __shfl(token[0], row & 63);
            if constexpr (C::TOK == 2) tok = row < 64 ? tok : __shfl(token[1], row & 63);
            aoff[i] = ((uint32_t)tok * (uint32_t)K + (uint32_t)((lane % 8) ^ swz(row)) * 8) * 2;
        }
#pragma unroll
        for (int i = 0; i < C::L; ++i) {
            const int c = i * (C::WN / C::L) + lane / C::L;
            boff[i] = (uint32_t)weight_row(wn * C::WN + c) * rs + 12u * (uint32_t)((lane % C::L) ^ swl(c));
        }
    };
    const int last_group = (n - 1) / C::L;
    uint8_t *const sw0 = smem + C::WBASE + wn * (C::RW * C::WGRP);
    int wfill;
    auto load_slice = [&](int at, int group) {
        // (a group's stages past K are the next row's, or zeros past the buffer,
        // whose end the lanes' offsets are checked against; never used)
        dma_buf_lds12s(wrs, sw0 + at, boff[0] + (uint32_t)(min(group, last_group) * C::L * 12), 0);
        const uint32_t b0 = boff[0];
#pragma unroll
        for (int i = 0; i + 1 < C::L; ++i) boff[i] = boff[i + 1];
        boff[C::L - 1] = b0;
    };
    auto issue = [&](int s, int slot) {
        uint8_t *sa = smem + slot + wn * C::AW * 1024;
#pragma unroll
        for (int i = 0; i < C::AW; ++i) dma_buf_lds16s(ars, sa + i * 1024, aoff[i], (uint32_t)s * 128u);
        load_slice(wfill, s / C::L + 1);
        wfill = wfill + C::WSL == C::RW * C::WGRP ? 0 : wfill + C::WSL;
    };
    // the first stages of a tile
    auto begin = [&]() {
#pragma unroll
        for (int i = 0; i < C::L; ++i) load_slice(i * C::WSL, 0);
        wfill = C::WGRP;
#pragma unroll
        for (int s = 0; s < C::R; ++s)
            if (s < n) issue(s, s * C::ASZ);
    };

    typedef __attribute__((address_space(3))) uint8_t lds_u8;
    typedef const __attribute__((address_space(3))) uint32_t lds_u32;
    typedef __attribute__((address_space(3))) half8 lds_half8;
    lds_u8 *const lbase = (lds_u8 *)smem;
    lds_u8 *fa[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) fa[j] = lbase + li * 128 + (((4 * j + g) ^ swz(li)) * 16);
    lds_u8 *const qw = lbase + C::WBASE + wn * (C::RW * C::WGRP) + li * (C::L * 16);
    const int qsw = swl(li) * 16;
    int rgrp, rsub;
    floatx4 acc[C::MT][C::NTL];
    uint32_t d[C::NTL][3], s2[C::NTL], wg[C::NTL];
    half8 af[C::SETS][C::MT];
    auto read_weights = [&]() {
        lds_u8 *const qp = qw + rgrp + (rsub ^ qsw);
        rsub += 16;
        if (rsub == 16 * C::L) {
            rsub = 0;
            rgrp = rgrp + C::WGRP == C::RW * C::WGRP ? 0 : rgrp + C::WGRP;
        }
#pragma unroll
        for (int nt = 0; nt < C::NTL; ++nt) {
            lds_u32 *q = (lds_u32 *)(qp + nt * (C::L * 256));
            d[nt][0] = q[0];
            d[nt][1] = q[1];
            d[nt][2] = q[2];
        }
    };
    auto read_rows = [&](int slot, int j) {
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) af[j][mt] = *(const lds_half8 *)(fa[j] + slot + mt * 16 * 128);
    };
    // the scale pairs of block j and its sign words, the lane's last pair at
    // the sign bits, from the stage's words
    auto scales = [&](int j) {
#pragma unroll
        for (int nt = 0; nt < C::NTL; ++nt) {
            if (j == 0) {
                s2[nt] = dup_lo16(d[nt][0]);
                wg[nt] = __builtin_amdgcn_alignbit(d[nt][1], d[nt][0], 4 + 4 * g);
            } else {
                s2[nt] = dup_hi16(d[nt][1]);
                wg[nt] = d[nt][2] << (12 - 4 * g);
            }
        }
    };
    // Every wave's part of the next stage is in LDS (its loads waited for
    // before) and this one's reads are done, so that its slot can be filled.
    auto publish = [&]() {
        wait_lgkmcnt0();
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto next = [&](int slot) { return slot + C::ASZ == C::R * C::ASZ ? 0 : slot + C::ASZ; };
    // A stage: its two blocks, 16 weight rows at a time.  What the next MFMAs
    // need (fragments, packed words, the next 16 rows as fp16) is read and
    // expanded while the MFMAs at hand run, a few vector operations behind
    // each: an MFMA holds its SIMD's matrix unit for 16 cycles and the issue
    // for 4, and what stands behind a row of MFMAs waits for all of them.
    u32x4 bo;
    auto stage = [&](int slot, auto &&advance) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (j == 1) { // (behind the last stage reads what is not used)
                advance();
                read_weights();
            }
            const int slot_ahead = j == 0 ? slot : next(slot);
            if (C::SETS == 2) read_rows(slot_ahead, 1 - j);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int nt = 0; nt < C::NTL; ++nt) {
                u32x4 ahead = bo;
                if (nt + 1 < C::NTL) {
                    ahead = wpair4(wg[nt + 1], s2[nt + 1]);
                } else {
                    scales(1 - j);
                    ahead = wpair4(wg[0], s2[0]);
                }
#pragma unroll
                for (int mt = 0; mt < C::MT; ++mt) {
                    acc[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        __builtin_bit_cast(half8, bo), af[C::SETS == 2 ? j : 0][mt], acc[mt][nt], 0, 0, 0);
                    // each fragment makes room for the next block's
                    if (C::SETS == 1 && nt + 1 == C::NTL)
                        af[0][mt] = *(const lds_half8 *)(fa[1 - j] + slot_ahead + mt * 16 * 128);
                }
                constexpr int V = (8 + C::MT - 1) / C::MT;
                if (nt + 1 < C::NTL)
                    interleave<C::MT, V, 0>();
                else
                    interleave<C::MT, 2 * V, C::SETS == 1>();
                __builtin_amdgcn_sched_barrier(0);
                bo = ahead;
            }
        }
    };

    look_up(first);
    aim();
    begin();
    int bad = 0;
    for (int t = first; t < last; t += each) {
        if (t + each < last) look_up(t + each);
        wait_stages<C::LOADS, C::R - 1>(n - 1);
        publish();
        rgrp = rsub = 0;
        read_weights();
        read_rows(0, 0);
        scales(0);
        bo = wpair4(wg[0], s2[0]);
#pragma unroll
        for (int i = 0; i < C::MT; ++i)
#pragma unroll
            for (int j = 0; j < C::NTL; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
        int slot = 0;
        for (int s = 0; s < n; ++s) {
            stage(slot, [&]() {
                if (s + C::R < n) {
                    wait_vmcnt<(C::R - 2) * C::LOADS>();
                    publish();
                    issue(s + C::R, slot);
                } else if (s + 1 < n) {
                    wait_stages<C::LOADS, C::R - 2>(n - 2 - s);
                    publish();
                }
            });
            slot = next(slot);
        }

        // the next tile's first loads, then what this one leaves
        const int my_row0 = row0, my_rows = rows;
        const int c0 = n0 + wn * C::WN;
        uint64_t nans[C::TOK];
#pragma unroll
        for (int i = 0; i < C::TOK; ++i) nans[i] = all.bad ? ~0ull : wrong[i];
        if (n0 == 0 && wn == 0 && lane == 0 && a.bad && !all.bad) {
            int bad_rows = 0;
#pragma unroll
            for (int i = 0; i < C::TOK; ++i) bad_rows += __popcll(wrong[i]);
            if (bad_rows) atomicAdd(a.bad, bad_rows);
        }
        if (t + each < last) {
            aim();
            publish(); // no wave reads the stages any more
            begin();
        }
        const bool cnt = a.nonfinite != nullptr;
        auto count4 = [&](const floatx4 &v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) bad += !__builtin_isfinite(v[e]);
        };
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
            const int row = 16 * mt + li;
            if (row >= my_rows) continue;
            if ((nans[mt / 4] >> (row & 63)) & 1)
#pragma unroll
                for (int nt = 0; nt < C::NTL; ++nt) acc[mt][nt] = nan4();
            if constexpr (OUT == 0) {
                float *const o = a.out + (size_t)(my_row0 + row) * a.ldo;
#pragma unroll
                for (int nt = 0; nt < C::NTL; ++nt) {
                    const int col = c0 + 16 * nt + 4 * g;
                    const floatx4 v = acc[mt][nt];
                    if (a.vec && col + 4 <= a.N) {
                        if (cnt) count4(v);
                        *reinterpret_cast<floatx4 *>(o + col) = v;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (col + e < a.N) {
                                bad += cnt && !__builtin_isfinite(v[e]);
                                o[col + e] = v[e];
                            }
                    }
                }
            } else {
                uint32_t *const o = a.pk + (size_t)(my_row0 + row) * a.ldpw + 4 * g;
#pragma unroll
                for (int nt = 0; nt < C::NTL; nt += OUT == 3 ? 4 : 2) {
                    const int col = c0 + 16 * nt; // of the weight rows
                    if (col >= a.N) continue;
                    floatx4 lo = acc[mt][nt], hi = acc[mt][nt + 1];
                    if (cnt) {
                        count4(lo);
                        count4(hi);
                    }
                    if constexpr (OUT == 3) {
                        const floatx4 vlo = acc[mt][nt + 2], vhi = acc[mt][nt + 3];
                        if (cnt) {
                            count4(vlo);
                            count4(vhi);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            lo[e] = mul_f32(silu_fast(lo[e]), vlo[e]);
                            hi[e] = mul_f32(silu_fast(hi[e]), vhi[e]);
                        }
                    } else if constexpr (OUT == 2) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            lo[e] = gelu_tanh(lo[e]);
                            hi[e] = gelu_tanh(hi[e]);
                        }
                    }
                    u32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = pack_f16_rounded(lo[e], hi[e]);
                    *reinterpret_cast<u32x4 *>(o + col / (OUT == 3 ? 4 : 2)) = v;
                }
            }
        }
    }
    count_nonfinite(a.nonfinite, bad);
}

// ------------------------------------------------------------ combine ----

// out[t] = residual[t] + sum_j weight[t][j] y[place[t][j]], 4 columns a
// thread; bound by HBM (4 bytes a value of y, the residual and out: 8192
// tokens of 8 rows of 2048 134 us, 5.0 TB/s, the rate of a large copy).
__global__ __launch_bounds__(256) void b1_combine_kernel(CombineArgs a) {
    const int token = blockIdx.x, col = (blockIdx.y * 256 + threadIdx.x) * 4;
    const int32_t *place = a.place + (int64_t)token * a.top_k;
    const float *weight = a.weight + (int64_t)token * a.top_k;
    bool wrong = false;
    for (int j = 0; j < a.top_k; ++j) wrong |= place[j] < -1 || place[j] >= a.routes;
    if (wrong && a.bad && threadIdx.x == 0 && blockIdx.y == 0) atomicAdd(a.bad, 1);
    if (col >= a.H) return;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < a.top_k; ++j) {
        const int p = place[j];
        if (p < 0 || p >= a.routes) continue;
        const floatx4 x = *reinterpret_cast<const floatx4 *>(a.y + (int64_t)p * a.ldy + col);
        const float w = weight[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(w, x[i], v[i]);
    }
    if (a.residual) v += *reinterpret_cast<const floatx4 *>(a.residual + (int64_t)token * a.ldr + col);
    if (wrong) v = nan4();
    *reinterpret_cast<floatx4 *>(a.out + (int64_t)token * a.ldo + col) = v;
}

// ---------------------------------------------------------- launchers ----

// Tokens of a single work-group (128 experts: 16 tokens 5.9 us, 32 8.3, 64 12.6;
// two launches 9.0).
constexpr int kRouteOneGroup = 32;

// Tokens a work-group of the two-launch router: 256 work-groups and one at most.
int route_per(int tokens) { return std::min(std::max(kRouteWaves, (tokens + 255) / 256), 65535); }

template <class F>
hipError_t with_route(const RouteArgs &a, F f) {
    auto wide = [&](auto el) {
        return a.bias ? f(el, std::true_type{}) : f(el, std::false_type{});
    };
    if (a.experts <= 64) return wide(std::integral_constant<int, 1>{});
    if (a.experts <= 128) return wide(std::integral_constant<int, 2>{});
    if (a.experts <= 256) return wide(std::integral_constant<int, 4>{});
    if (a.experts <= 512) return wide(std::integral_constant<int, 8>{});
    return wide(std::integral_constant<int, 16>{});
}

} // namespace

size_t route_workspace_bytes(const RouteArgs &a) {
    if (a.tokens <= kRouteOneGroup) return 0;
    const int per = route_per(a.tokens);
    return (size_t)((a.tokens + per - 1) / per) * count_row(a.experts) * 2;
}

// More than 64 KB of LDS is for the asking.
template <class K>
static hipError_t allow_lds(K kernel, size_t bytes) {
    return bytes <= (64u << 10) ? hipSuccess
                                : hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

hipError_t launch_route(const RouteArgs &a, void *ws, size_t ws_bytes, hipStream_t s) {
    const size_t need = route_workspace_bytes(a);
    const size_t row = (size_t)count_row(a.experts) * 4;
    if (need == 0 || !ws || ws_bytes < need)
        return with_route(a, [&](auto el, auto wide) {
            auto kernel = &b1_route_kernel<decltype(el)::value, decltype(wide)::value>;
            const size_t lds = row * (1 + kRouteWaves);
            const hipError_t e = allow_lds(kernel, lds);
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL(kernel, dim3(1), dim3(kRouteThreads), lds, s, a);
            return hipGetLastError();
        });
    const int per = route_per(a.tokens), groups = (a.tokens + per - 1) / per;
    uint16_t *counts = static_cast<uint16_t *>(ws);
    const hipError_t e = with_route(a, [&](auto el, auto wide) {
        hipLaunchKernelGGL((b1_route_choose_kernel<decltype(el)::value, decltype(wide)::value>), dim3(groups),
                           dim3(kRouteThreads), row, s, a, per, counts);
        return hipGetLastError();
    });
    if (e != hipSuccess) return e;
    const size_t lds = row * (2 + kRouteWaves);
    const hipError_t e2 = allow_lds(&b1_route_place_kernel, lds);
    if (e2 != hipSuccess) return e2;
    hipLaunchKernelGGL(b1_route_place_kernel, dim3(groups), dim3(kRouteThreads), lds, s, a, per, counts);
    return hipGetLastError();
}

// ------------------------------------------------ the experts' linears ----

namespace {

// Groups of up to bm rows of one expert that evenly spread routes make.
double likely_groups(const ExpertArgs &a, int bm) {
    const double mean = (double)a.routes / a.experts;
    return a.experts * (1.0 - std::exp(-mean) + std::max(0.0, mean / bm - 0.5));
}

// Which kernel a call takes, by models of their microseconds.  They are fitted
// to 4563 shapes of 2 to 256 experts, 0.5 to 600 rows an expert, K 128 to 8192
// and N 512 to 8192 on 256 CUs, each run with all four (the median shape within
// 4 %; the kernel chosen takes 1.4 % more than the fastest of them on average,
// 10 % at the 95th percentile, where one kernel by rows an expert alone takes
// 18 % and 90 %): a fixed time, and for tiles the longer of what the rounds of
// a CU's resident work-groups take one after another and what all its tiles
// take of its matrix units, for few rows a work-group's steps beside the
// others on its CU.
struct FewPlan {
    int waves, units, parts, per; // 256s of K a wave; work-groups a group of rows, steps each
    double us;
};

FewPlan plan_few(const ExpertArgs &a, int num_cus) {
    const int units = (a.K + 255) / 256;
    FewPlan f = {};
    f.waves = units <= 3 || (units > 4 && units <= 6) ? 3 : units <= 8 ? 4 : 8;
    f.units = units <= 4 ? 1 : units <= 16 ? 2 : 4;
    const int steps = a.kind == 3 ? a.glu_h / 32 : (a.N + 63) / 64;
    // work-groups a CU, by their registers
    const int resident = (f.units == 1 ? 16 : f.units == 2 ? 12 : 8) / f.waves;
    const double groups = likely_groups(a, 16);
    double best = 1e30;
    int per = steps;
    for (int p = 1; p <= steps; p = per > 1 ? (steps + per - 2) / (per - 1) : steps + 1) { // the parts of each size
        per = (steps + p - 1) / p;
        const double wgs = std::ceil(groups * p / num_cus), beside = std::min(wgs, (double)resident);
        const double rounds = std::ceil(wgs / resident), cost = rounds * (3.0 + per * (beside + 1.0));
        if (cost < best) {
            best = cost;
            f.parts = p;
            f.per = per;
            const double wave = f.units * f.waves / 4.0;
            f.us = a.kind == 0 ? 4.9 + rounds * (per * (0.85 * wave * beside + 0.12 * f.units) - 1.3)
                               : 5.7 + rounds * (per * (0.80 * wave * beside + 0.20 * f.units) - 1.7);
        }
    }
    return f;
}

//                      BM  WN NWN R  L OCC SETS
using E32 = ExpertTile<32, 64, 4, 3, 2, 4, 2>;
using E64 = ExpertTile<64, 64, 4, 3, 2, 3, 1>;
using E128 = ExpertTile<128, 64, 4, 2, 4, 2, 1>;

struct TileTimes {
    double fixed, round, round_k, tile, tile_k; // us; _k: a stage
};
template <class C>
double tile_us(const ExpertArgs &a, int num_cus, const TileTimes &packed, const TileTimes &rows) {
    const TileTimes &t = a.kind == 0 ? rows : packed;
    const double tiles = likely_groups(a, C::BM) * ((a.N + C::BN - 1) / C::BN) / num_cus, n = a.K / 64;
    return t.fixed + std::max(std::ceil(tiles / C::OCC) * (t.round + t.round_k * n),
                              std::ceil(tiles) * (t.tile + t.tile_k * n));
}

// 0: few rows; else the tiles' rows
int plan_experts(const ExpertArgs &a, int num_cus, FewPlan *few) {
    const double us[3] = {
        tile_us<E32>(a, num_cus, {3.9, 0.48, 0.42, 0.51, 0.30}, {3.7, 0.63, 0.43, 0.91, 0.31}),
        tile_us<E64>(a, num_cus, {3.5, 1.1, 0.53, 0.82, 0.42}, {2.7, 2.1, 0.53, 1.8, 0.43}),
        tile_us<E128>(a, num_cus, {3.8, 1.7, 0.76, 1.4, 0.68}, {3.5, 0.0, 0.35, 2.2, 0.76})};
    const int best = (int)(std::min_element(us, us + 3) - us);
    if (a.K <= kFewMaxK) {
        *few = plan_few(a, num_cus);
        const int64_t threads = group_bound(a.routes, a.experts, 16) * few->parts * few->waves * 64;
        if (few->us < us[best] && threads < ((int64_t)1 << 31)) return 0;
    }
    return 32 << best;
}

template <int NW, int U>
hipError_t launch_few(const ExpertArgs &a, const FewPlan &f, hipStream_t s) {
    const dim3 grid((unsigned)(group_bound(a.routes, a.experts, 16) * f.parts));
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(NW * 64), 0, s, a, f.parts, f.per);
        return hipGetLastError();
    };
    switch (a.kind) {
    case 0: return run(b1_experts_few_kernel<NW, U, 0>);
    case 1: return run(b1_experts_few_kernel<NW, U, 1>);
    case 2: return run(b1_experts_few_kernel<NW, U, 2>);
    default: return run(b1_experts_few_kernel<NW, U, 3>);
    }
}

template <class C>
hipError_t launch_tiles(const ExpertArgs &a, int num_cus, hipStream_t s) {
    const int tiles_n = (a.N + C::BN - 1) / C::BN;
    const int64_t tiles = group_bound(a.routes, a.experts, C::BM) * tiles_n;
    // a multiple of the XCDs
    const unsigned grid = (unsigned)(std::min<int64_t>((int64_t)num_cus * C::OCC, tiles + 7) / 8 * 8);
    auto run = [&](auto kernel) {
        const hipError_t e = allow_lds(kernel, C::LDS);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, dim3(std::max(grid, 8u)), dim3(C::NT), C::LDS, s, a, tiles_n);
        return hipGetLastError();
    };
    switch (a.kind) {
    case 0: return run(&b1_experts_tile_kernel<C, 0>);
    case 1: return run(&b1_experts_tile_kernel<C, 1>);
    case 2: return run(&b1_experts_tile_kernel<C, 2>);
    default: return run(&b1_experts_tile_kernel<C, 3>);
    }
}

} // namespace

extern "C" int b1_experts_plan(int routes, int experts, int K, int N, int kind, int num_cus, int *waves, int *units) {
    ExpertArgs a{};
    a.routes = routes;
    a.experts = experts;
    a.K = K;
    a.N = N;
    a.kind = kind;
    a.glu_h = N / 2;
    FewPlan f = {};
    const int rows = plan_experts(a, num_cus, &f);
    *waves = rows ? 0 : f.waves;
    *units = rows ? 0 : f.units;
    return rows;
}

hipError_t launch_experts(const ExpertArgs &a, int num_cus, hipStream_t s) {
    FewPlan f = {};
    switch (plan_experts(a, num_cus, &f)) {
    case 0: break;
    case 32: return launch_tiles<E32>(a, num_cus, s);
    case 64: return launch_tiles<E64>(a, num_cus, s);
    default: return launch_tiles<E128>(a, num_cus, s);
    }
    if (f.units == 1) return f.waves == 3 ? launch_few<3, 1>(a, f, s) : launch_few<4, 1>(a, f, s);
    if (f.units == 2 && f.waves == 3) return launch_few<3, 2>(a, f, s);
    if (f.units == 2) return f.waves == 4 ? launch_few<4, 2>(a, f, s) : launch_few<8, 2>(a, f, s);
    return launch_few<8, 4>(a, f, s);
}

hipError_t launch_combine(const CombineArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(b1_combine_kernel, dim3(a.tokens, (a.H / 4 + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError();
}

} // namespace b1
