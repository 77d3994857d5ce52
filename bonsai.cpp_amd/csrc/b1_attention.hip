// Attention over packed sequences, with contiguous or paged keys:
//
//   out[i] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i k_j - max_j)
//
// over the keys j that row i sees (causal: none past its own position,
// window: only the last `window` of those), in one pass over the keys with a
// running maximum and sum.  The heads that share a key head are rows of one
// tile (row = token * group + head in the group), so a tile's keys are read
// once for all of them.
#include <hip/hip_runtime.h>

#include <limits.h>

#include "b1_seqs.h"

namespace b1 {
namespace {


// Below every score, and finite: a masked score is -inf, and -inf minus this
// is -inf (weight 0), where -inf - -inf would be NaN.
constexpr float kLowest = -3.4028235e38f;
constexpr float kInf = __builtin_inff();

template <bool BF>
__device__ __forceinline__ floatx16 mfma32(u32x4 x, u32x4 y, floatx16 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), c, 0,
                                                      0, 0);
}

template <bool BF>
__device__ __forceinline__ floatx4 mfma16(u32x4 x, u32x4 y, floatx4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), c, 0,
                                                      0, 0);
}

// v of the lane and of the same lane of the wave's other half, in an order
// that both halves share.  The copy is hidden from the compiler: of a swap
// whose operands it knows to be equal it used one result for both.
__device__ __forceinline__ float2v halves(float v) {
    uint32_t x = __builtin_bit_cast(uint32_t, v), y = x;
    asm("" : "+v"(y));
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    return float2v{__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
__device__ __forceinline__ float halves_max(float v) {
    const float2v r = halves(v);
    return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float halves_sum(float v) {
    const float2v r = halves(v);
    return r[0] + r[1];
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4_t;
// Transposed read of 16-bit values from LDS.  Each group of 16 lanes reads a
// 4 x 16 block, lane i its row i / 4, columns 4 (i % 4) .. + 3 at p; lane i
// receives column i, rows 0 .. 3 (layout checked on gfx950).
__device__ __forceinline__ u32x2 read_columns(const void *p) {
    return __builtin_bit_cast(u32x2,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)const_cast<void *>(p)));
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < kInf; }

// One key head's keys (or values) of one sequence.
struct KeyRows {
    const uint16_t *base; // contiguous: the sequence's first row
    int64_t page, row;    // element strides
};

template <bool PAGED>
__device__ __forceinline__ KeyRows key_rows(const uint16_t *p, int64_t page, int64_t row, int64_t head, int kvh,
                                            const Seq &s) {
    KeyRows r;
    r.base = p + kvh * head;
    if (!PAGED) r.base += s.kv0 * row;
    r.page = page;
    r.row = row;
    return r;
}

template <bool PAGED>
__device__ __forceinline__ int64_t key_at(const AttnArgs &a, const KeyRows &r, int b, int j, bool &bad) {
    if constexpr (PAGED) {
        const int p = page_of(a.seqs, b, j, bad);
        return p * r.page + (j & ((1 << a.seqs.page_shift) - 1)) * r.row;
    } else {
        return j * r.row;
    }
}

// The keys [lo, hi] that token i of a sequence sees.
__device__ __forceinline__ void visible(const AttnArgs &a, const Seq &s, int i, int &lo, int &hi) {
    lo = 0;
    hi = s.nk - 1;
    if (a.causal) {
        hi = s.nk - s.nq + i; // < nk
        if (a.window) lo = max(0, hi - a.window + 1);
    }
}

// One row in fp32 over the visible keys of [j0, j1), without matrix
// instructions: what a tile falls back to for a row that came out
// non-finite.  There a product of weight 0 and a masked key's infinity or NaN
// may have reached it, or a sum of weights above 1 times large values may
// have left fp32's range; here masked keys are never read, and the weights
// are divided by their sum before they meet a value (l is then 1, and m the
// maximum that goes with it).
template <bool BF, int D, bool PAGED, class Add>
__device__ void row_fp32(const AttnArgs &a, const KeyRows &kr, const KeyRows &vr, int b, const uint16_t *q, int j0,
                         int j1, float scale2, float &m, float &l, Add add) {
    bool bad = false; // reported by the tile
    auto score = [&](int j) {
        const uint16_t *k = kr.base + key_at<PAGED>(a, kr, b, j, bad);
        float s = 0.f;
        for (int c = 0; c < D; c += 8) {
            const u32x4 x = *reinterpret_cast<const u32x4 *>(q + c), y = *reinterpret_cast<const u32x4 *>(k + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s += to_f32<BF>((uint16_t)x[e]) * to_f32<BF>((uint16_t)y[e]);
                s += to_f32<BF>((uint16_t)(x[e] >> 16)) * to_f32<BF>((uint16_t)(y[e] >> 16));
            }
        }
        return s * scale2;
    };
    m = kLowest;
    l = 0.f;
    for (int j = j0; j < j1; ++j) m = fmaxf(m, score(j));
    for (int j = j0; j < j1; ++j) l += __builtin_amdgcn_exp2f(score(j) - m);
    if (l == 0.f) return;
    const float inv = 1.0f / l;
    for (int j = j0; j < j1; ++j)
        add(vr.base + key_at<PAGED>(a, vr, b, j, bad), __builtin_amdgcn_exp2f(score(j) - m) * inv);
    m += __builtin_amdgcn_logf(l); // base 2
    l = l == l ? 1.f : l;
}

// ---- tiles of 128 rows ------------------------------------------------------

constexpr int kRows = 128, kKeys = 64;

// Swizzle of a row's 16-byte chunks in LDS.  A K fragment reads one chunk
// column of 32 consecutive rows and a V fragment two neighbouring columns of
// 4 consecutive rows; without it all rows of D >= 128 (256 bytes, one sweep
// of the banks) share their banks.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
    if constexpr (D == 64)
        return ((row >> 1) & 3) << 1 | ((row >> 3) & 1);
    else
        return (row & 7) << 1 | ((row >> 3) & 1);
}

// The rows of tile t (of kRows) and the range of 64-key tiles they see.
struct TileKeys {
    int r0, rows; // first row, rows there (<= kRows)
    int t0, t1;   // key tiles
};
__device__ __forceinline__ TileKeys tile_keys(const AttnArgs &a, const Seq &s, int group, int t) {
    TileKeys k;
    k.r0 = t * kRows;
    k.rows = min(kRows, s.nq * group - k.r0);
    int lo, hi, x;
    visible(a, s, k.r0 / group, lo, x);
    visible(a, s, (k.r0 + k.rows - 1) / group, x, hi);
    k.t0 = lo / kKeys;
    k.t1 = hi < lo ? k.t0 : hi / kKeys + 1;
    return k;
}
// Key tiles of each of the ranges a row tile's keys are split into: at least
// four, so that a range's fixed costs stay small beside its keys.
__device__ __forceinline__ int tiles_a_range(const TileKeys &k, int splits) {
    return max(4, (k.t1 - k.t0 + splits - 1) / splits);
}

// The sequence and row tile of work item t, by the whole wave; b = -1: none.
__device__ __forceinline__ int find_tile(const AttnArgs &a, int group, int t, int &local) {
    const int lane = threadIdx.x & 63;
    int run = 0;
    for (int b0 = 0; b0 < a.seqs.n_seqs; b0 += 64) {
        const int b = b0 + lane;
        int n = 0;
        if (b < a.seqs.n_seqs) n = (seq_of(a.seqs, b).nq * group + kRows - 1) / kRows;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o);
            if (lane >= o) incl += v;
        }
        const uint64_t past = __ballot(run + incl > t);
        if (past) {
            const int l = __builtin_ctzll(past);
            local = t - run - __shfl(incl - n, l);
            return b0 + l;
        }
        run += __shfl(incl, 63);
    }
    return -1;
}

// A range-checked resource over `bytes` from p (at most 2^32 - 1): reads at
// or past its end give zeros and touch no memory.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t key_buffer(const uint16_t *p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(p), 0,
                                             (int)(uint32_t)min(bytes, (int64_t)0xffffffffu), kBufferFlags);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <bool BF, int D, bool PAGED>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void b1_attn_tile_kernel(AttnArgs a) {
    constexpr int ST = D / 16, DT = D / 32, CH = D / 8;
    // two tiles of keys and values, as four objects: the compiler then knows
    // that the copies into one tile do not concern the reads of the other,
    // and does not wait for them before these
    __shared__ __align__(1024) uint8_t k0[kKeys * D * 2], k1[kKeys * D * 2], v0[kKeys * D * 2], v1[kKeys * D * 2];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int l31 = lane & 31, h = lane >> 5;
    const int group = a.heads / a.kv_heads;
    if (a.bad && blockIdx.x == 0 && wave == 0) report_seqs(a.seqs, a.bad);

    // work item: key head, row tile, key range
    int item = blockIdx.x;
    const int split = item % a.splits;
    item /= a.splits;
    const int kvh = item % a.kv_heads;
    int t;
    const int b = uniform(find_tile(a, group, item / a.kv_heads, t));
    if (b < 0) return;
    Seq s = seq_of(a.seqs, b);
    s.q0 = uniform(s.q0), s.nq = uniform(s.nq), s.kv0 = uniform(s.kv0), s.nk = uniform(s.nk);
    // the last tiles of a causal sequence have the most keys: first
    t = uniform((s.nq * group + kRows - 1) / kRows - 1 - t);
    const TileKeys tk = tile_keys(a, s, group, t);
    const int per = tiles_a_range(tk, a.splits);
    const int ranges = uniform(max(1, (tk.t1 - tk.t0 + per - 1) / per));
    if (split >= ranges) return;
    const int t0 = uniform(tk.t0 + split * per), t1 = uniform(min(t0 + per, tk.t1));

    // this lane's row; rows past the tile's last repeat it and store nothing
    const int r = tk.r0 + min(wave * 32 + l31, tk.rows - 1);
    const bool mine = wave * 32 + l31 < tk.rows;
    const int token = s.q0 + r / group, head = kvh * group + r % group;
    int lo, hi;
    visible(a, s, r / group, lo, hi);
    // the wave's rows: keys that some see, keys that all see
    const bool wave_on = wave * 32 < tk.rows;
    int first_lo, first_hi, last_lo, last_hi;
    visible(a, s, (tk.r0 + min(wave * 32, tk.rows - 1)) / group, first_lo, first_hi);
    visible(a, s, (tk.r0 + min(wave * 32 + 31, tk.rows - 1)) / group, last_lo, last_hi);
    first_lo = uniform(first_lo), first_hi = uniform(first_hi), last_lo = uniform(last_lo), last_hi = uniform(last_hi);

    const uint16_t *qrow = a.q + token * a.q_row + head * a.q_head;
    const KeyRows kr = key_rows<PAGED>(a.k, a.k_page, a.k_row, a.k_head, kvh, s);
    const KeyRows vr = key_rows<PAGED>(a.v, a.v_page, a.v_row, a.v_head, kvh, s);
    bool bad = s.bad;

    // Copies a tile of keys and values.  A wave's instruction copies the
    // 512 / D rows that lie in 1 KiB; lane i lands at 16 i, so the swizzle is
    // in which chunk of the row it reads.  Rows past the last key read zeros.
    // Paged: `page` is the page of key kb + lane, and rows of more than one
    // page (of fewer than 512 / D keys) take an instruction a page.
    constexpr int NR = 512 / D;
    auto load = [&](int kb, int page, uint8_t *ks, uint8_t *vs) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int at = wave * (D / 32) + i, row0 = at * NR;
            const int row = row0 + lane / CH;
            const int chunk = ((lane % CH) ^ swizzle<D>(row)) * 16;
            if constexpr (PAGED) {
                const int size = 1 << a.seqs.page_shift, span = min(size, NR);
                for (int sub = 0; sub < NR; sub += span) {
                    const int id = __builtin_amdgcn_readlane(page, row0 + sub);
                    const int first = (kb + row0 + sub) & -size;         // the page's first key
                    const int64_t keys = max(0, min(size, s.nk - first)); // keys there
                    const uint32_t off = (uint32_t)((kb + row) & (size - 1));
                    if (NR == span || (unsigned)(lane / CH - sub) < (unsigned)span) {
                        dma_buf_lds16(key_buffer(kr.base + id * kr.page, keys * kr.row * 2), ks + at * 1024,
                                      off * (uint32_t)(kr.row * 2) + chunk);
                        dma_buf_lds16(key_buffer(vr.base + id * vr.page, keys * vr.row * 2), vs + at * 1024,
                                      off * (uint32_t)(vr.row * 2) + chunk);
                    }
                }
            } else {
                const int64_t keys = s.nk - kb;
                dma_buf_lds16(key_buffer(kr.base + kb * kr.row, keys * kr.row * 2), ks + at * 1024,
                              (uint32_t)row * (uint32_t)(kr.row * 2) + chunk);
                dma_buf_lds16(key_buffer(vr.base + kb * vr.row, keys * vr.row * 2), vs + at * 1024,
                              (uint32_t)row * (uint32_t)(vr.row * 2) + chunk);
            }
        }
    };
    auto pages = [&](int kb) {
        if constexpr (PAGED)
            return page_of(a.seqs, b, min(kb + lane, s.nk - 1), bad);
        else
            return 0;
    };

    u32x4 qf[ST];
#pragma unroll
    for (int i = 0; i < ST; ++i) qf[i] = *reinterpret_cast<const u32x4 *>(qrow + 16 * i + 8 * h);
    floatx16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = floatx16{};
    float m = kLowest, l = 0.f;
    const float scale2 = a.scale * 1.44269504f; // exp(x) = exp2(x log2 e)

    int next = 0; // pages of the tile after the one that is being copied
    if (t0 < t1) {
        load(t0 * kKeys, pages(t0 * kKeys), k0, v0);
        next = pages((t0 + 1) * kKeys);
    }
    auto tile = [&](int tt, const uint8_t *ks, const uint8_t *vs, uint8_t *ks2, uint8_t *vs2) {
        const int kb = tt * kKeys;
        wait_vmcnt<0>();
        wait_lgkmcnt0();
        lds_barrier();
        if (tt + 1 < t1) {
            load(kb + kKeys, next, ks2, vs2);
            next = pages(kb + 2 * kKeys);
        }
        if (!wave_on || kb > last_hi || kb + kKeys - 1 < first_lo) return;
        // scores, transposed: column = row of q, register i of half h = key
        // 8 (i / 4) + 4 h + i % 4
        floatx16 sc[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            sc[kt] = floatx16{};
            const int row = kt * 32 + l31;
#pragma unroll
            for (int i = 0; i < ST; ++i) {
                const u32x4 kf = *reinterpret_cast<const u32x4 *>(ks + row * (D * 2) +
                                                                  (((2 * i + h) ^ swizzle<D>(row)) << 4));
                sc[kt] = mfma32<BF>(kf, qf[i], sc[kt]);
            }
        }
        if (kb + kKeys - 1 > first_hi || kb < last_lo) {
            const int top = hi - kb - 4 * h, bot = lo - kb - 4 * h;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int c = 32 * kt + 8 * (i / 4) + i % 4;
                    sc[kt][i] = c <= top && c >= bot ? sc[kt][i] : -kInf;
                }
        }
        float mx = -kInf;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kt][i]);
        mx = halves_max(mx) * scale2;
        // the maximum is only moved when some row's grew by 2^8: until then
        // its weights are up to 256, which fp16 and the fp32 sums hold
        if (__any(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= alpha;
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sc[kt][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kt][i], scale2, -m));
                l += sc[kt][i];
            }
        // o (transposed) += v (transposed) p: 16 keys a step, in the order
        // the scores' registers hold them
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                u32x4 pf;
#pragma unroll
                for (int e = 0; e < 4; ++e) pf[e] = pack_16<BF>(sc[kt][8 * u + 2 * e], sc[kt][8 * u + 2 * e + 1]);
                const int row = kt * 32 + 16 * u + 4 * h + (lane & 15) / 4;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const int chunk = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
                    auto at = [&](int rw) {
                        return vs + rw * (D * 2) + ((chunk ^ swizzle<D>(rw)) << 4) + (lane & 1) * 8;
                    };
                    const u32x2 x = read_columns(at(row)), y = read_columns(at(row + 8));
                    o[dt] = mfma32<BF>(u32x4{x[0], x[1], y[0], y[1]}, pf, o[dt]);
                }
            }
    };
    for (int tt = t0; tt < t1; tt += 2) {
        tile(tt, k0, v0, k1, v1);
        if (tt + 1 < t1) tile(tt + 1, k1, v1, k0, v0);
    }
    l = halves_sum(l);

    if (__syncthreads_or(bad)) {
        bad = true;
        if (a.bad && threadIdx.x == 0) atomicAdd(a.bad, 1);
    }
    if (!wave_on) return;
    float inv = l == 0.f ? 0.f : 1.0f / l;
    if (bad) {
        inv = l = __builtin_nanf("");
    } else {
        int odd = 0;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) odd |= !finite(o[i][e] * inv);
        odd |= __shfl_xor(odd, 32);
        if (odd) {
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] = floatx16{};
            row_fp32<BF, D, PAGED>(a, kr, vr, b, qrow, max(lo, t0 * kKeys), min(hi + 1, t1 * kKeys), scale2, m, l,
                                   [&](const uint16_t *v, float p) {
#pragma unroll
                                       for (int i = 0; i < DT; ++i)
#pragma unroll
                                           for (int e = 0; e < 16; ++e)
                                               o[i][e] += p * to_f32<BF>(v[32 * i + 8 * (e / 4) + 4 * h + e % 4]);
                                   });
            inv = l == 0.f ? 0.f : 1.0f / l;
        }
    }
    if (!mine) return;
    if (ranges > 1) {
        const int64_t at = ((int64_t)split * a.seqs.tokens + token) * a.heads + head;
        float *po = a.part_o + at * D;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<floatx4 *>(po + 32 * i + 8 * g + 4 * h) =
                    floatx4{o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]};
        if (h == 0) *reinterpret_cast<float2v *>(a.part_ml + 2 * at) = float2v{m, l};
        if (h == 0 && split == 0) a.part_n[token * a.heads + head] = ranges;
        return;
    }
    if (a.splits > 1 && h == 0) a.part_n[token * a.heads + head] = 1;
    uint16_t *orow = a.out + token * a.ldo + head * D;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        o[i] *= inv;
        if (a.packed) {
            // words d .. d + 3 of the block: columns d and d + 16
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pack_f16(o[i][4 * g + e], o[i][4 * g + e + 8]);
                *reinterpret_cast<u32x4 *>(orow + 32 * i + 16 * g + 8 * h) = w;
            }
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<u32x2 *>(orow + 32 * i + 8 * g + 4 * h) =
                    u32x2{pack_16<BF>(o[i][4 * g], o[i][4 * g + 1]), pack_16<BF>(o[i][4 * g + 2], o[i][4 * g + 3])};
        }
    }
}

// ---- few rows a sequence ----------------------------------------------------

constexpr int kFewRows = 16, kFewKeys = 32, kWaves = 4;

// The keys that any token of a sequence sees, and into how many ranges of
// how many keys they are split so that all sequences together make about
// a.target work-groups.  A range is a multiple of what the four waves take
// at once.
struct FewPlan {
    int at, ranges, keys;
};
__device__ __forceinline__ int few_len(const AttnArgs &a, const Seq &s, int &at) {
    at = 0;
    if (s.nq == 0) return 0;
    int hi;
    visible(a, s, 0, at, hi);
    at = min(at, s.nk);
    return s.nk - at;
}
// Keys a range, from the lengths of all sequences (by the whole wave).
__device__ __forceinline__ int few_unit(const AttnArgs &a) {
    constexpr int step = kFewKeys * kWaves;
    if (a.splits == 1) return INT_MAX;
    const int lane = threadIdx.x & 63;
    float total = 0.f; // a split size needs no more
    for (int b = lane; b < a.seqs.n_seqs; b += 64) {
        int at;
        total += (float)few_len(a, seq_of(a.seqs, b), at);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) total += __shfl_xor(total, o);
    const int want = (int)fminf(total * (float)a.kv_heads / (float)a.target, 1.9e9f);
    return (want / step + 1) * step;
}
__device__ __forceinline__ FewPlan few_plan(const AttnArgs &a, const Seq &s, int unit) {
    constexpr int step = kFewKeys * kWaves;
    FewPlan p;
    const int len = few_len(a, s, p.at);
    p.ranges = s.nq == 0 ? 0 : min(a.splits, max(1, len / unit + (len % unit != 0)));
    p.keys = p.ranges <= 1 ? len : (len / p.ranges + step) / step * step;
    if (p.ranges > 1) p.ranges = (len + p.keys - 1) / p.keys;
    return p;
}

// The final values of D / 16 columns from c0 on of one row by 16 lanes.
template <bool BF, int D>
__device__ __forceinline__ void store_row(const AttnArgs &a, int token, int head, int c0, const float (&o)[D / 16],
                                          bool mine) {
    constexpr int E = D / 16, apart = 16 / E; // lanes between columns d and d + 16
    uint16_t *orow = a.out + token * a.ldo + head * D;
    if (a.packed) {
        float other[E];
#pragma unroll
        for (int e = 0; e < E; ++e) other[e] = __shfl_xor(o[e], apart);
        const int block = c0 / 32, d = c0 % 32;
        if (mine && d < 16) {
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                u32x4 w;
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = pack_f16(o[e + k], other[e + k]);
                *reinterpret_cast<u32x4 *>(orow + 32 * block + 2 * (d + e)) = w;
            }
        }
    } else if (mine) {
#pragma unroll
        for (int e = 0; e < E; e += 4)
            *reinterpret_cast<u32x2 *>(orow + c0 + e) =
                u32x2{pack_16<BF>(o[e], o[e + 1]), pack_16<BF>(o[e + 2], o[e + 3])};
    }
}

template <bool BF, int D, bool PAGED>
__global__ __launch_bounds__(256) void b1_attn_few_kernel(AttnArgs a) {
    constexpr int E = D / 16, ST = D / 32, PAD = D + 4;
    __shared__ __align__(16) float so[kWaves][kFewRows][PAD];
    __shared__ float sml[kWaves][kFewRows][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int group = a.heads / a.kv_heads;
    const int kvh = blockIdx.x % a.kv_heads, item = blockIdx.x / a.kv_heads;
    if (a.bad && blockIdx.x == 0 && wave == 0) report_seqs(a.seqs, a.bad);

    // work item -> sequence and key range
    const int unit = few_unit(a);
    int b = -1, range = 0, run = 0;
    for (int b0 = 0; b0 < a.seqs.n_seqs && b < 0; b0 += 64) {
        int n = 0;
        if (b0 + lane < a.seqs.n_seqs) n = few_plan(a, seq_of(a.seqs, b0 + lane), unit).ranges;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o);
            if (lane >= o) incl += v;
        }
        const uint64_t past = __ballot(run + incl > item);
        if (past) {
            const int w = __builtin_ctzll(past);
            range = item - run - __shfl(incl - n, w);
            b = b0 + w;
        }
        run += __shfl(incl, 63);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    if (b < 0) return;
    const Seq s = seq_of(a.seqs, b);
    const FewPlan plan = few_plan(a, s, unit);
    const int j0 = plan.at + range * plan.keys, j1 = min(j0 + plan.keys, s.nk);

    const KeyRows kr = key_rows<PAGED>(a.k, a.k_page, a.k_row, a.k_head, kvh, s);
    const KeyRows vr = key_rows<PAGED>(a.v, a.v_page, a.v_row, a.v_head, kvh, s);
    const float scale2 = a.scale * 1.44269504f;
    const int rows = s.nq * group;
    bool any_bad = s.bad;

    for (int r0 = 0; r0 < rows; r0 += kFewRows) {
        bool bad = s.bad;
        const int r = min(r0 + c, rows - 1);
        const uint16_t *qrow = a.q + (s.q0 + r / group) * a.q_row + (kvh * group + r % group) * a.q_head;
        int lo, hi;
        visible(a, s, r / group, lo, hi);
        u32x4 qf[ST];
#pragma unroll
        for (int i = 0; i < ST; ++i) qf[i] = *reinterpret_cast<const u32x4 *>(qrow + 32 * i + 8 * g);
        floatx4 o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = floatx4{};
        float m = kLowest, l = 0.f;

        for (int kb = j0 + wave * kFewKeys; kb < j1; kb += kWaves * kFewKeys) {
            u32x4 kf[2][ST];
            uint32_t vw[8][E / 2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const int j = min(kb + 16 * kt + c, s.nk - 1);
                const uint16_t *p = kr.base + key_at<PAGED>(a, kr, b, j, bad) + 8 * g;
#pragma unroll
                for (int i = 0; i < ST; ++i) kf[kt][i] = *reinterpret_cast<const u32x4 *>(p + 32 * i);
            }
            // lane (c, g): columns E c .. of the 8 keys its scores are about
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = min(kb + 16 * (i / 4) + 4 * g + i % 4, s.nk - 1);
                const uint16_t *p = vr.base + key_at<PAGED>(a, vr, b, j, bad) + E * c;
                if constexpr (E == 4) {
                    const u32x2 x = *reinterpret_cast<const u32x2 *>(p);
                    vw[i][0] = x[0], vw[i][1] = x[1];
                } else {
#pragma unroll
                    for (int k = 0; k < E / 8; ++k) {
                        const u32x4 x = *reinterpret_cast<const u32x4 *>(p + 8 * k);
#pragma unroll
                        for (int y = 0; y < 4; ++y) vw[i][4 * k + y] = x[y];
                    }
                }
            }
            floatx4 sc[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                sc[kt] = floatx4{};
#pragma unroll
                for (int i = 0; i < ST; ++i) sc[kt] = mfma16<BF>(kf[kt][i], qf[i], sc[kt]);
            }
            float mx = -kInf;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = kb + 16 * kt + 4 * g + i;
                    sc[kt][i] = j <= hi && j >= lo && j < j1 ? sc[kt][i] * scale2 : -kInf;
                    mx = fmaxf(mx, sc[kt][i]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mn = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= alpha;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[kt][i] = __builtin_amdgcn_exp2f(sc[kt][i] - m);
                    l += sc[kt][i];
                }
            const u32x4 pf = {pack_16<BF>(sc[0][0], sc[0][1]), pack_16<BF>(sc[0][2], sc[0][3]),
                              pack_16<BF>(sc[1][0], sc[1][1]), pack_16<BF>(sc[1][2], sc[1][3])};
            // matrix row c of product e is column E c + e
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                u32x4 vf;
#pragma unroll
                for (int k = 0; k < 4; ++k) vf[k] = __builtin_amdgcn_perm(vw[2 * k + 1][e / 2], vw[2 * k][e / 2], sel);
                o[e] = mfma16<BF>(vf, pf, o[e]);
            }
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        // the four waves' shares; register i of product e: column E (4 g + i) + e
        if (r0 > 0) __syncthreads(); // the last rows' are read
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<floatx4 *>(&so[wave][c][E * (4 * g + i) + e]) =
                    floatx4{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
        if (g == 0) sml[wave][c][0] = m, sml[wave][c][1] = l;
        bad = __syncthreads_or(bad);
        any_bad |= bad;

        // 16 threads a row, E columns each
        const int row = threadIdx.x / 16, c0 = (threadIdx.x & 15) * E;
        const int rr = min(r0 + row, rows - 1);
        const bool mine = r0 + row < rows;
        const int token = s.q0 + rr / group, head = kvh * group + rr % group;
        float acc[E];
        float M = kLowest, L = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sml[w][row][0]);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(sml[w][row][0] - M);
            L += f * sml[w][row][1];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f * so[w][row][c0 + e];
        }
        float inv = L == 0.f ? 0.f : 1.0f / L;
        if (bad) {
            inv = L = __builtin_nanf("");
        } else {
            int odd = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) odd |= !finite(acc[e] * inv);
#pragma unroll
            for (int x = 8; x >= 1; x >>= 1) odd |= __shfl_xor(odd, x); // the row's threads alike
            if (odd) {
                int rlo, rhi;
                visible(a, s, rr / group, rlo, rhi);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = 0.f;
                row_fp32<BF, D, PAGED>(a, kr, vr, b, a.q + token * a.q_row + head * a.q_head, max(rlo, j0),
                                       min(rhi + 1, j1), scale2, M, L, [&](const uint16_t *v, float p) {
#pragma unroll
                                           for (int e = 0; e < E; ++e) acc[e] += p * to_f32<BF>(v[c0 + e]);
                                       });
                inv = L == 0.f ? 0.f : 1.0f / L;
            }
        }
        if (plan.ranges > 1) {
            if (mine) {
                const int64_t at = ((int64_t)range * a.seqs.tokens + token) * a.heads + head;
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    *reinterpret_cast<floatx4 *>(a.part_o + at * D + c0 + e) =
                        floatx4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
                if (c0 == 0) *reinterpret_cast<float2v *>(a.part_ml + 2 * at) = float2v{M, L};
                if (c0 == 0 && range == 0) a.part_n[token * a.heads + head] = plan.ranges;
            }
        } else {
            if (a.splits > 1 && mine && c0 == 0) a.part_n[token * a.heads + head] = 1;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] *= inv;
            store_row<BF, D>(a, token, head, c0, acc, mine);
        }
    }
    if (any_bad && a.bad && threadIdx.x == 0) atomicAdd(a.bad, 1);
}

// ---- joining the ranges -----------------------------------------------------

// P groups of 16 lanes take a row, each every P-th of its ranges; rows whose
// keys were not split are there already.  Bound by latency: a row's sequence
// and number of ranges are one read deep, the maxima and sums of all ranges
// are read at once by the 16 lanes.
template <bool BF, int D, int P>
__global__ __launch_bounds__(256) void b1_attn_join_kernel(AttnArgs a) {
    constexpr int E = D / 16, ROWS = 16 / P; // rows a work-group
    __shared__ __align__(16) float so[16][D + 4];
    const int all = a.seqs.tokens * a.heads;
    const int lane16 = threadIdx.x & 15, at16 = threadIdx.x >> 4;
    const int row = blockIdx.x * ROWS + at16 / P, part = at16 % P, c0 = lane16 * E;
    int ranges = row < all ? a.part_n[row] : 0; // of a row of no sequence: anything
    // the sequences of the wave's rows, each by the whole wave
    const int wave_row = uniform(row);
    int last = -1, there = 0, mask = 0;
#pragma unroll
    for (int k = 0; k < (P < 4 ? 4 / P : 1); ++k) {
        const int tk = (wave_row + k) / a.heads;
        if (wave_row + k < all && tk != last) {
            there = seq_of_token(a.seqs, tk) >= 0;
            last = tk;
        }
        mask |= there << k;
    }
    const bool mine = row < all && (mask >> (row - wave_row) & 1) && ranges > 1 && ranges <= a.splits;
    if (!mine) ranges = 0;
    float M = kLowest, L = 0.f;
    for (int i = lane16; i < ranges; i += 16) M = fmaxf(M, a.part_ml[2 * ((int64_t)i * all + row)]);
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
    for (int i = lane16; i < ranges; i += 16) {
        const float2v ml = *reinterpret_cast<const float2v *>(a.part_ml + 2 * ((int64_t)i * all + row));
        L += __builtin_amdgcn_exp2f(ml[0] - M) * ml[1];
    }
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1) L += __shfl_xor(L, x);
    // weights that add up to at most 1 before they meet a sum of values
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
    for (int i = part; i < ranges; i += P) {
        const int64_t at = (int64_t)i * all + row;
        const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * at] - M) * inv;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const floatx4 v = *reinterpret_cast<const floatx4 *>(a.part_o + at * D + c0 + e);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[e + k] += f * v[k];
        }
    }
    if constexpr (P > 1) {
#pragma unroll
        for (int e = 0; e < E; e += 4)
            *reinterpret_cast<floatx4 *>(&so[at16][c0 + e]) = floatx4{o[e], o[e + 1], o[e + 2], o[e + 3]};
        __syncthreads();
        if (part == 0) {
#pragma unroll
            for (int k = 1; k < P; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += so[at16 + k][c0 + e];
        }
    }
    store_row<BF, D>(a, row / a.heads, row % a.heads, c0, o, mine && part == 0);
}

// ---- which kernel, how many ranges -------------------------------------------

struct AttnPlan {
    bool few;
    int splits, target, grid;
};

int ceil_div(int64_t a, int64_t b) {
    const int64_t v = (a + b - 1) / b;
    return v > INT_MAX ? INT_MAX : (int)v;
}

AttnPlan attn_plan(const AttnArgs &a, int num_cus, bool split) {
    AttnPlan p{};
    const int group = a.heads / a.kv_heads;
    const int n = a.seqs.n_seqs;
    const int64_t rows = (int64_t)a.seqs.tokens * group; // a key head
    const int64_t most = a.seqs.pages ? (int64_t)a.seqs.max_pages << a.seqs.page_shift : a.seqs.kv_tokens;
    p.few = rows <= (int64_t)kFewRows * n;
    if (p.few) {
        p.target = 4 * num_cus;
        const int64_t units = (int64_t)n * a.kv_heads;
        int64_t s = 4 * ((p.target + units - 1) / units);
        s = s < 256 ? s : 256;
        const int64_t fit = (most + kFewKeys * kWaves - 1) / (kFewKeys * kWaves);
        if (s > fit) s = fit;
        p.splits = split && s > 1 ? (int)s : 1;
    } else {
        const int64_t tiles = (rows / kRows + n) * a.kv_heads;
        int64_t s = tiles < 2 * num_cus ? (2 * num_cus + tiles - 1) / tiles : 1;
        const int64_t fit = most / (4 * kKeys);
        if (s > fit) s = fit;
        p.splits = split && s > 1 ? (int)s : 1;
    }
    // partial results no larger than 1 GiB
    const int64_t each = (int64_t)a.seqs.tokens * a.heads * (a.head_dim + 2) * 4;
    if ((int64_t)p.splits * each > (int64_t)1 << 30) p.splits = (int)(((int64_t)1 << 30) / each);
    if (p.splits < 1) p.splits = 1;
    if (p.few) {
        // sum over sequences of ceil(len / unit) <= n + target / kv_heads
        int64_t items = n + (p.splits > 1 ? p.target / a.kv_heads + 1 : 0);
        const int64_t cap = (int64_t)n * p.splits;
        if (items > cap) items = cap;
        p.grid = ceil_div(items * a.kv_heads, 1);
    } else {
        p.grid = ceil_div((rows / kRows + n) * a.kv_heads * p.splits, 1);
    }
    return p;
}

size_t round_256(size_t b) { return (b + 255) & ~(size_t)255; }

size_t part_bytes(const AttnArgs &a, int splits) {
    if (splits <= 1) return 0;
    const size_t rows = (size_t)splits * a.seqs.tokens * a.heads;
    return round_256(rows * a.head_dim * 4) + round_256(rows * 8) + (size_t)a.seqs.tokens * a.heads * 4;
}

template <bool BF, int D>
hipError_t launch(const AttnArgs &a, const AttnPlan &p, hipStream_t s) {
    const dim3 grid(p.grid), block(256);
    if (p.few) {
        if (a.seqs.pages)
            hipLaunchKernelGGL((b1_attn_few_kernel<BF, D, true>), grid, block, 0, s, a);
        else
            hipLaunchKernelGGL((b1_attn_few_kernel<BF, D, false>), grid, block, 0, s, a);
    } else {
        if (a.seqs.pages)
            hipLaunchKernelGGL((b1_attn_tile_kernel<BF, D, true>), grid, block, 0, s, a);
        else
            hipLaunchKernelGGL((b1_attn_tile_kernel<BF, D, false>), grid, block, 0, s, a);
    }
    if (p.splits > 1) {
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        const int64_t rows = (int64_t)a.seqs.tokens * a.heads;
        if (p.splits <= 4)
            hipLaunchKernelGGL((b1_attn_join_kernel<BF, D, 1>), dim3(ceil_div(rows, 16)), block, 0, s, a);
        else if (p.splits <= 16)
            hipLaunchKernelGGL((b1_attn_join_kernel<BF, D, 4>), dim3(ceil_div(rows, 4)), block, 0, s, a);
        else
            hipLaunchKernelGGL((b1_attn_join_kernel<BF, D, 16>), dim3(rows), block, 0, s, a);
    }
    return hipGetLastError();
}

} // namespace

size_t attn_workspace_bytes(const AttnArgs &a, int num_cus) {
    return part_bytes(a, attn_plan(a, num_cus, true).splits);
}

hipError_t launch_attn(const AttnArgs &args, int num_cus, void *ws, size_t ws_bytes, hipStream_t s) {
    AttnArgs a = args;
    AttnPlan p = attn_plan(a, num_cus, true);
    if (p.splits > 1 && (!ws || ws_bytes < part_bytes(a, p.splits))) p = attn_plan(a, num_cus, false);
    a.splits = p.splits;
    a.target = p.target;
    if (p.splits > 1) {
        a.part_o = static_cast<float *>(ws);
        const size_t rows = (size_t)p.splits * a.seqs.tokens * a.heads;
        uint8_t *at = static_cast<uint8_t *>(ws) + round_256(rows * a.head_dim * 4);
        a.part_ml = reinterpret_cast<float *>(at);
        a.part_n = reinterpret_cast<int32_t *>(at + round_256(rows * 8));
    }
    switch (a.head_dim) {
    case 64: return a.bf16 ? launch<true, 64>(a, p, s) : launch<false, 64>(a, p, s);
    case 128: return a.bf16 ? launch<true, 128>(a, p, s) : launch<false, 128>(a, p, s);
    case 256: return a.bf16 ? launch<true, 256>(a, p, s) : launch<false, 256>(a, p, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace b1
