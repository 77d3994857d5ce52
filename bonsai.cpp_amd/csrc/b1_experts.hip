// A mixture of 1-bit experts: the router's choice, the experts' linears over
// ragged groups of rows, and the weighted sum of what the experts give.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "b1_device.h"
#include "b1_internal.h"

namespace b1 {
namespace {

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
// Lane l holds logits l, l + 64, ...  (EL of them).  A choice is the largest
// key of all lanes, ties to the lowest expert: keys are the logits as
// integers of the same order, or, where a bias makes a score's rounding count
// (WIDE), the 64-bit scores + bias, compared by their high words first.  Key
// 0 is never chosen: -inf and what is chosen already.  NaN comes behind every
// number (and makes the row's weights NaN).
constexpr uint32_t kNanKey = 1;
template <int EL, bool WIDE>
__device__ __forceinline__ int route_token(const RouteArgs &a, int token) {
    const int lane = threadIdx.x & 63;
    float x[EL];
    uint32_t hi[EL], lo[WIDE ? EL : 1];
    const int64_t row = (int64_t)token * a.ld;
    uint32_t top = 0; // the largest logit, as a key
    bool nan = false;
    auto key_of = [](float v) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f); // -0 is 0
        return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    };
#pragma unroll
    for (int i = 0; i < EL; ++i) {
        const int e = lane + 64 * i;
        x[i] = e < a.experts ? logit_at(a, row + e) : -INFINITY;
        nan |= x[i] != x[i];
        hi[i] = x[i] > -INFINITY ? key_of(x[i]) : x[i] != x[i] ? kNanKey : 0u;
        top = max(top, hi[i]);
    }
    top = wave_max(top);
    const float peak = __builtin_bit_cast(float, top ^ ((top >> 31) ? 0x80000000u : 0xffffffffu));
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
        // an infinite logit: weights NaN, chosen by the logits
        if (a.sigmoid || sum < (double)INFINITY) {
#pragma unroll
            for (int i = 0; i < EL; ++i) {
                const int e = lane + 64 * i;
                if (e >= a.experts || hi[i] <= kNanKey) {
                    lo[i] = 0;
                    continue;
                }
                const double k = (a.sigmoid ? z[i] : z[i] / sum) + (double)a.bias[e] + 0.0;
                const uint64_t b = __builtin_bit_cast(uint64_t, k);
                const uint64_t key = b ^ ((b >> 63) ? ~0ull : 1ull << 63);
                nan |= k != k;
                hi[i] = k > -(double)INFINITY ? (uint32_t)(key >> 32) : k != k ? kNanKey : 0u;
                lo[i] = k == k ? (uint32_t)key : 0u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < EL; ++i) lo[i] = 0;
        }
    }
    const bool any_nan = __ballot(nan) != 0;
    int mine = -1;
    float mine_x = -INFINITY;
    for (int j = 0; j < a.top_k; ++j) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < EL; ++i) m = max(m, hi[i]);
        m = wave_max(m);
        if (m == 0) break;
        uint32_t ml = 0;
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < EL; ++i) ml = max(ml, hi[i] == m ? lo[i] : 0u);
            ml = wave_max(ml);
        }
        bool found = false;
#pragma unroll
        for (int i = 0; i < EL; ++i) {
            bool same = hi[i] == m;
            if constexpr (WIDE) same = same && lo[i] == ml;
            const uint64_t who = __ballot(same);
            if (!found && who) { // wave-uniform
                found = true;
                const int l = __builtin_ctzll(who);
                const float v = __builtin_bit_cast(float, lane_value(__builtin_bit_cast(uint32_t, x[i]), l));
                if (lane == l) hi[i] = 0;
                if (lane == j) {
                    mine = l + 64 * i;
                    mine_x = v;
                }
            }
        }
    }
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
        const float p = mine >= 0 ? expf(mine_x - peak) : 0.f;
        float sum = p;
        if (!a.renormalize) {
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < EL; ++i) sum += x[i] > -INFINITY ? expf(x[i] - peak) : 0.f;
        }
        weight = p / wave_sum(sum) * a.scale;
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
        int at = -1;
        if (e >= 0) {
            const int before = __popcll(same & ((1ull << lane) - 1));
            at = (int)(mine[e] + (uint32_t)before);
            if (before == 0) mine[e] = (uint32_t)at + (uint32_t)__popcll(same);
            a.order[at] = (int)slot;
        }
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
// counts their experts; then each finds its first row of every expert from
// all the counts and places its slots.
template <int EL, bool WIDE>
__global__ __launch_bounds__(kRouteThreads) void b1_route_choose_kernel(RouteArgs a, int per, uint32_t *counts) {
    extern __shared__ uint32_t route_lds[];
    const int wave = threadIdx.x >> 6, E = a.experts;
    for (int e = threadIdx.x; e < E; e += kRouteThreads) route_lds[e] = 0;
    __syncthreads();
    const int t1 = min((int)(blockIdx.x + 1) * per, a.tokens);
    for (int t = blockIdx.x * per + wave; t < t1; t += kRouteWaves) {
        const int e = route_token<EL, WIDE>(a, t);
        if (e >= 0) atomicAdd(&route_lds[e], 1u);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) counts[(size_t)blockIdx.x * E + e] = route_lds[e];
}

__global__ __launch_bounds__(kRouteThreads) void b1_route_place_kernel(RouteArgs a, int per, const uint32_t *counts) {
    extern __shared__ uint32_t route_lds[];
    uint32_t *base = route_lds, *total = route_lds + a.experts, *parts = route_lds + 2 * a.experts;
    __shared__ uint32_t all;
    const int E = a.experts, lane = threadIdx.x & 63;
    for (int e = threadIdx.x; e < E; e += kRouteThreads) base[e] = total[e] = 0;
    __syncthreads();
    // threads e, e + E', ... of an expert take the work-groups in turn
    const int groups = max(1, kRouteThreads / E);
    const int g = threadIdx.x / E;
    if (g < groups) {
        for (int e = threadIdx.x - g * E; e < E; e += kRouteThreads) {
            uint32_t before = 0, sum = 0;
#pragma unroll 8
            for (int w = g; w < (int)gridDim.x; w += groups) {
                const uint32_t n = counts[(size_t)w * E + e];
                sum += n;
                before += w < (int)blockIdx.x ? n : 0u;
            }
            if (before) atomicAdd(&base[e], before);
            if (sum) atomicAdd(&total[e], sum);
        }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t n = lds_prefix(total, E);
        if (lane == 0) all = n;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) {
        base[e] += total[e];
        if (blockIdx.x == 0) a.start[e] = (int)total[e];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.start[E] = (int)all;
    __syncthreads();
    const int64_t slots = (int64_t)a.tokens * a.top_k;
    const int64_t s0 = (int64_t)blockIdx.x * per * a.top_k;
    route_place(a, s0, min(s0 + (int64_t)per * a.top_k, slots), base, parts);
    for (int64_t r = (int64_t)all + (int64_t)blockIdx.x * kRouteThreads + threadIdx.x; r < slots;
         r += (int64_t)gridDim.x * kRouteThreads)
        a.order[r] = -1;
}

// ------------------------------------------------------ groups of rows ----

// Rows of an expert: up to `most` of them from row0 on.
struct Group {
    int expert, row0, rows;
    bool bad; // the starts of the experts' rows are out of order or of range
};

// The t-th group of up to BM rows of one expert, counting through the experts
// in order, and how many groups there are (*groups); by a whole wave.  Starts
// are brought into range and order first, so that any contents of `start` give
// groups within the rows, apart from one another, and no more of them than
// group_bound() says.
template <int BM>
__device__ __forceinline__ Group find_group(const int32_t *start, int experts, int routes, int t, int *groups) {
    const int lane = threadIdx.x & 63;
    Group found = {0, 0, 0, false};
    uint32_t before = 0, floor = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
        const int e = min(e0 + lane, experts - 1);
        const int a = start[e], b = start[e + 1];
        const bool there = e0 + lane < experts;
        found.bad |= __ballot(a < 0 || b < a || b > routes) != 0;
        uint32_t s0 = (uint32_t)min(max(a, 0), routes), s1 = (uint32_t)min(max(b, 0), routes);
        if (found.bad) { // no start before an earlier one
            s0 = scan_max(max(s0, floor));
            s1 = scan_max(max(s1, s0));
            floor = lane_value(s1, 63);
        }
        const uint32_t rows = there ? s1 - s0 : 0u, n = (rows + BM - 1) / BM;
        const uint32_t end = before + scan_add(n);
        const uint64_t who = __ballot((uint32_t)t >= end - n && (uint32_t)t < end);
        if (who) {
            const int l = __builtin_ctzll(who);
            const uint32_t first = lane_value(end - n, l);
            const uint32_t at = ((uint32_t)t - first) * BM;
            found.expert = e0 + l;
            found.row0 = (int)(lane_value(s0, l) + at);
            found.rows = (int)min(lane_value(rows, l) - at, (uint32_t)BM);
        }
        before = lane_value(end, 63);
    }
    *groups = (int)before;
    return found;
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

// ------------------------------------------------ few rows an expert ----

// y = W a for up to 16 rows of one expert and `per` steps of 64 weight rows.
//
// Bound by the weights, read once a group (6 bytes a block of 32), and by the
// shifts and selects that make fp16 of them, about 7 a lane and 8 weights.
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
    int groups;
    const int slot = bid / parts, part = bid - slot * parts;
    const Group gr = find_group<BM>(a.start, a.experts, a.routes, slot, &groups);
    if (bid == 0 && threadIdx.x == 0 && gr.bad && a.bad) atomicAdd(a.bad, 1);
    if (slot >= groups) return;

    // the row's activations
    int64_t src = gr.row0 + li;
    bool there = li < gr.rows, wrong = false;
    if (a.order && there) {
        const int s = a.order[src];
        wrong = s < 0 || s >= a.routes;
        src = wrong ? 0 : s / a.top_k;
    }
    const uint32_t wrong_rows = gr.bad ? 0xffffu : (uint32_t)__ballot(wrong) & 0xffffu;
    if (wrong_rows && !gr.bad && a.bad && part == 0 && threadIdx.x == 0) atomicAdd(a.bad, __popc(wrong_rows));
    there = there && !wrong;
    const int pairs = a.K / 64; // of blocks, 12 bytes of a weight row
    half8 af[U][2][4];
    uint32_t woff[U]; // of this lane's pair within a weight row
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int pair = (wave * U + u) * 4 + g;
        woff[u] = pair < pairs ? 12u * (uint32_t)pair : kNowhere;
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
    const uint32_t rs = (uint32_t)(a.K / 32) * 6;
    const __amdgpu_buffer_rsrc_t wrs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t *>(a.w) + (size_t)gr.expert * a.N * rs, (short)0, (int)((uint32_t)a.N * rs), kBufferFlags);
    // weight rows of group nt of step s: 64 s + 16 nt, or 32 gates, then their 32 values
    auto weight_row = [&](int s, int nt) {
        if constexpr (OUT == 3) return 32 * s + 16 * (nt & 1) + (nt >> 1) * a.glu_h + li;
        return 64 * s + 16 * nt + li;
    };
    const int s0 = part * per, s1 = min(s0 + per, OUT == 3 ? a.glu_h / 32 : (a.N + 63) / 64);
    u32x3 w[U][4], next[U][4];
    auto load = [&](u32x3 (&to)[U][4], int s) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                const int row = weight_row(s, nt);
                const uint32_t off = row < a.N && woff[u] != kNowhere ? (uint32_t)row * rs + woff[u] : kNowhere;
                to[u][nt] = __builtin_bit_cast(u32x3, __builtin_amdgcn_raw_buffer_load_b96(wrs, (int)off, 0, 0));
            }
    };
    int bad = 0;
    if (s0 < s1) load(w, s0);
    for (int s = s0; s < s1; ++s) {
        if (s + 1 < s1) load(next, s + 1);
        floatx4 acc[4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            acc[nt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const u32x3 d = w[u][nt];
                    const uint32_t sc = b ? dup_hi16(d[1]) : dup_lo16(d[0]);
                    const uint32_t sign = b ? d[2] : __builtin_amdgcn_alignbit(d[1], d[0], 16);
                    u32x4 c[4];
                    wpair_quads<0>(sign, sign >> 8, sc, c[0], c[2]);
                    wpair_quads<1>(sign, sign >> 8, sc, c[1], c[3]);
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
        if constexpr (OUT == 0) {
            for (int i = threadIdx.x; i < gr.rows * 16; i += NW * 64) {
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
            for (int i = threadIdx.x; i < gr.rows * Q; i += NW * 64) {
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
                        lo[k] = mul_f32(silu_f32(lo[k]), vlo[k]);
                        hi[k] = mul_f32(silu_f32(hi[k]), vhi[k]);
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
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) w[u][nt] = next[u][nt];
    }
    count_nonfinite(a.nonfinite, bad);
}

// ------------------------------------------------------------ combine ----

// out[t] = residual[t] + sum_j weight[t][j] y[place[t][j]], 4 columns a
// thread; bound by HBM (4 bytes a value of y, the residual and out).
__global__ __launch_bounds__(256) void b1_combine_kernel(CombineArgs a) {
    const int token = blockIdx.x, col = (blockIdx.y * 256 + threadIdx.x) * 4;
    const int32_t *place = a.place + (int64_t)token * a.top_k;
    const float *weight = a.weight + (int64_t)token * a.top_k;
    bool wrong = false;
    for (int j = 0; j < a.top_k; ++j) wrong |= place[j] < -1 || place[j] >= a.routes;
    if (wrong && a.bad && threadIdx.x == 0 && blockIdx.y == 0) atomicAdd(a.bad, 1);
    if (col >= a.H) return;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    if (a.residual) v = *reinterpret_cast<const floatx4 *>(a.residual + (int64_t)token * a.ldr + col);
    for (int j = 0; j < a.top_k; ++j) {
        const int p = place[j];
        if (p < 0 || p >= a.routes) continue;
        const floatx4 x = *reinterpret_cast<const floatx4 *>(a.y + (int64_t)p * a.ldy + col);
        const float w = weight[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(w, x[i], v[i]);
    }
    if (wrong) v = nan4();
    *reinterpret_cast<floatx4 *>(a.out + (int64_t)token * a.ldo + col) = v;
}

// ---------------------------------------------------------- launchers ----

constexpr int kRouteOneGroup = 64; // tokens

// Tokens a work-group of the two-launch router: at most 256 work-groups.
int route_per(int tokens) { return std::max(kRouteWaves, (tokens + 255) / 256); }

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
    return (size_t)((a.tokens + per - 1) / per) * a.experts * 4;
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
    const size_t row = (size_t)a.experts * 4;
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
    uint32_t *counts = static_cast<uint32_t *>(ws);
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

namespace {

template <int NW, int U>
hipError_t launch_few(const ExpertArgs &a, int num_cus, hipStream_t s) {
    const int steps = a.kind == 3 ? a.glu_h / 32 : (a.N + 63) / 64;
    const int64_t slots = group_bound(a.routes, a.experts, 16);
    // two work-groups a CU at a time, some rounds of them
    const int64_t want = std::max<int64_t>(1, 4 * (int64_t)num_cus / slots);
    const int per = (int)std::max<int64_t>(1, (steps + want - 1) / want), parts = (steps + per - 1) / per;
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(slots * parts)), dim3(NW * 64), 0, s, a, parts, per);
        return hipGetLastError();
    };
    switch (a.kind) {
    case 0: return run(b1_experts_few_kernel<NW, U, 0>);
    case 1: return run(b1_experts_few_kernel<NW, U, 1>);
    case 2: return run(b1_experts_few_kernel<NW, U, 2>);
    default: return run(b1_experts_few_kernel<NW, U, 3>);
    }
}

} // namespace

hipError_t launch_experts(const ExpertArgs &a, int num_cus, hipStream_t s) {
    const int units = (a.K + 255) / 256;
    if (units <= 4) return launch_few<4, 1>(a, num_cus, s);
    if (units <= 8) return launch_few<8, 1>(a, num_cus, s);
    if (units <= 16) return launch_few<8, 2>(a, num_cus, s);
    return launch_few<8, 4>(a, num_cus, s);
}

hipError_t launch_combine(const CombineArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(b1_combine_kernel, dim3(a.tokens, (a.H / 4 + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError();
}

} // namespace b1
