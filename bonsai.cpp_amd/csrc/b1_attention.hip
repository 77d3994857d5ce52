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

#include <algorithm>
#include <type_traits>
#include <vector>

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

// x / group for 0 <= x < 2^28 (AttnArgs::div_m and div_s).
__host__ __device__ __forceinline__ int div_group(const AttnArgs &a, int x) {
    const uint32_t hi = (uint32_t)(((uint64_t)(uint32_t)x * a.div_m) >> 32);
    return (int)((hi + (uint32_t)x) >> a.div_s);
}

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
__host__ __device__ __forceinline__ void visible(const AttnArgs &a, const Seq &s, int i, int &lo, int &hi) {
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
        s *= scale2;
        asm("" : "+v"(s)); // rounded: past fp32's range infinity, whose weight is NaN
        return s;
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

// l + the two values of a pair.
template <bool BF>
__device__ __forceinline__ float add_pair(uint32_t p, float l) {
    if constexpr (BF)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), __builtin_bit_cast(bf16x2, 0x3f803f80u),
                                               l, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, p), __builtin_bit_cast(half2v, 0x3c003c00u), l,
                                      false);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---- tiles of 128 rows ------------------------------------------------------

constexpr int kRows = 128;
// Keys in LDS at a time (a stage), waves a SIMD (= work-groups a CU) and
// stages in LDS, by head dim.  Three work-groups hide one another's waits:
// at D = 128 that takes stages of 32 keys (4608 tokens x 24 heads 299 us, of
// 64 keys and two work-groups 310; 4096 causal tokens x 32 heads 156, 167);
// at D = 64 stages of 64 fit too (168, 179 of 32 keys).  At D = 256 the
// registers of a row's sums leave one (690 TFLOP/s, 520 of two that spill),
// and LDS has room for four stages of 32 keys (4608 tokens x 12 heads 375 us,
// two of 64 keys 385).  Two stages at D = 128 against three: chunks over a
// paged cache 156 us, 164, others alike; three at D = 64 against two: 8191
// causal tokens 178, 179.
template <int D>
struct TileShapeOf {
    static constexpr int keys = D == 64 ? 64 : 32;
    static constexpr int waves = D == 256 ? 1 : 3;
    static constexpr int stages = D == 64 ? 3 : D == 128 ? 2 : 4;
};
// A range of a split tile has at least this many keys, so that its fixed
// costs (queries, partial sums out and in) stay small beside them.
constexpr int kLeastKeys = 256;

// Swizzles of a row's 16-byte chunks in LDS (64 banks of 4 bytes: two rows of
// D = 64, one of 128 a sweep).  A K fragment reads one chunk column of 16
// consecutive rows in a sweep; a V fragment a block of four chunks of four
// consecutive rows.  Each swizzle spreads its own pattern over all banks.
template <int D>
__device__ __forceinline__ int swizzle_k(int row) {
    if constexpr (D == 64)
        return ((row >> 1) & 3) << 1 | ((row >> 3) & 1);
    else
        return (row & 7) << 1 | ((row >> 3) & 1);
}
template <int D>
__device__ __forceinline__ int swizzle_v(int row) {
    if constexpr (D == 64)
        return ((row >> 1) & 1) << 2;
    else
        return (row & 3) << 2;
}

// The rows of tile t of a sequence and the keys [k0, k1) that they see.
struct TileKeys {
    int r0, rows; // first row, rows there (<= kRows)
    int k0, k1;
};
__host__ __device__ __forceinline__ TileKeys tile_keys(const AttnArgs &a, const Seq &s, int group, int t) {
    TileKeys k;
    k.r0 = t * kRows;
    k.rows = min(kRows, s.nq * group - k.r0);
    int lo, hi, x;
    visible(a, s, div_group(a, k.r0), lo, x);
    visible(a, s, div_group(a, k.r0 + k.rows - 1), x, hi);
    k.k0 = lo;
    k.k1 = max(hi + 1, lo);
    return k;
}
__host__ __device__ __forceinline__ int seq_tiles(const Seq &s, int group) {
    return (s.nq * group + kRows - 1) / kRows;
}

// Sum over the wave.
__device__ __forceinline__ int wave_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false); // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false); // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false); // row_bcast:31
    return __builtin_amdgcn_readlane(v, 63);
}

// Keys a range: a tile with more is split (into at most a.splits ranges), so
// that no range outlasts the rest of the call.
//
// Splitting pays where the longest tile takes longer than everything at the
// rate of a full device and the partial sums' way out and in.  In us at D =
// 128, measured: a 32-key step of a tile 0.72 with one work-group a CU, 1.15
// with two, 1.5 with three; a partial tile 0.026.  Split against whole (us):
// 128 tiles over 4096 keys 59 / 104, 8 over 4000 24 / 102, 128 over 1000
// 36 / 33, 256 over 1024 (causal) 41 / 33, 480 over 2560 126 / 97.
// (Without contraction: the two kernels that build a plan from the lengths,
// and the host, compute the same values.)
struct SeqWork {
    int tiles;   // of a key head
    int most;    // keys of a tile, no tile has more
    float total; // keys of all tiles
};
// A tile's rows are of at most `span` tokens, so that a window leaves it
// window + span - 1 keys at most; a last tile of fewer rows has fewer.
__host__ __device__ __forceinline__ SeqWork seq_work(const AttnArgs &a, const Seq &s, int group) {
#pragma clang fp contract(off)
    SeqWork w = {seq_tiles(s, group), 0, 0.f};
    if (w.tiles > 0) {
        const int span = min(s.nq, (kRows - 2 + 2 * group) / group);
        w.most = a.window ? min(s.nk, a.window + span - 1) : s.nk;
        const TileKeys x = tile_keys(a, s, group, 0);
        w.total = (float)w.tiles * 0.5f * ((float)(x.k1 - x.k0) + (float)w.most);
    }
    return w;
}
// Of a call's sequences: the keys of all tiles, as they are and if each had
// its sequence's most, the longest tile's, and the tiles (of a key head).
struct CallWork {
    float total, reach, longest;
    int tiles;
};
__host__ __device__ __forceinline__ CallWork call_work(const SeqWork &w) {
    return CallWork{w.total, (float)w.tiles * (float)w.most, (float)w.most, w.tiles};
}
__host__ __device__ __forceinline__ void add_work(CallWork &c, const CallWork &w) {
#pragma clang fp contract(off)
    c.total += w.total;
    c.reach += w.reach;
    c.longest = fmaxf(c.longest, w.longest);
    c.tiles += w.tiles;
}
constexpr int kWhole = INT_MAX / 2; // a unit that splits nothing
__host__ __device__ __forceinline__ int tile_unit(const AttnArgs &a, const CallWork &w) {
#pragma clang fp contract(off)
    const float total = w.total * (float)a.kv_heads, reach = w.reach * (float)a.kv_heads;
    const float tiles = (float)w.tiles * (float)a.kv_heads;
    const float target = (float)a.target;
    const float cus = target * (a.head_dim == 256 ? 1.f / TileShapeOf<256>::waves : 1.f / TileShapeOf<128>::waves);
    const float scale = (float)a.head_dim * (1.f / 128);
    const float whole = w.longest * (1.f / 32) * scale * (tiles <= cus ? 0.72f : tiles <= 2 * cus ? 1.15f : 1.5f);
    const float parts = tiles + fminf(target, total * (1.f / kLeastKeys));
    const float split = (total * (1.f / 32) * 1.7f / target + 0.026f * parts) * scale + 8.f;
    if (whole < 1.2f * split) return kWhole;
    // so that tiles x ceil(most keys / unit) <= tiles + target, which the
    // grid has room for
    return (int)fminf(fmaxf((float)kLeastKeys, reach / target + 1.f), (float)kWhole);
}
__host__ __device__ __forceinline__ int key_ranges(const AttnArgs &a, int keys, int unit) {
    return max(1, min(a.splits, (keys + unit - 1) / unit));
}
// A larger unit where the items (of a key head, at the unit so far) are more
// than the device holds at once, by as much: those left over would run after
// all others.  (Ranges are whole, so a few may still be.)
__host__ __device__ __forceinline__ int fit_unit(const AttnArgs &a, int unit, int items) {
#pragma clang fp contract(off)
    const float have = (float)items * (float)a.kv_heads;
    return have <= (float)a.target ? unit : (int)fminf((float)unit * have / (float)a.target, (float)kWhole) + 1;
}
// The unit of the only sequence of a call, of its last tiles where the first
// a.solo are whole.
__host__ __device__ __forceinline__ int one_seq_unit(const AttnArgs &a, const SeqWork &w) {
    if (a.solo > 0) return max(1, (w.most + a.splits - 1) / a.splits);
    if (a.splits == 1) return kWhole;
    const int unit = tile_unit(a, call_work(w));
    return unit < kWhole ? fit_unit(a, unit, w.tiles * key_ranges(a, w.most, unit)) : unit;
}

// A work item: key head, row tile and range of one of the sequences.  The
// first a.solo items are whole tiles; behind them a sequence's n tiles (key
// heads counted) have as many items each as one of its most keys has ranges,
// the tiles' first ranges before their second ones: neighbouring items run on different
// XCDs, and each is to have its share of those that have something to do.
// The partial sums of range i of the tile are number part + i * apart.
struct TileItem {
    int b, kvh, t, range, unit, part, apart;
    Seq s;
};
// Item g of a sequence's (its tile alone, where whole), whose partial sums
// begin at number `base`, behind a.solo whole tiles.
__host__ __device__ __forceinline__ void place_item(const AttnArgs &a, const SeqWork &w, int g, int base, bool whole,
                                                    TileItem &r) {
    if (!whole) {
        r.range = r.apart > 0 ? g / r.apart : 0;
        g -= r.range * r.apart;
    }
    r.part = base + g;
    g += a.solo;
    const int q = g / a.kv_heads;
    r.kvh = g - q * a.kv_heads;
    r.t = w.tiles - 1 - q;
}
// Finds item i (or, of whole tiles, the i-th tile behind the solo ones), by
// the whole wave; b = -1: none.  Unsplit tiles come in the order of their
// keys, the most first, so that the last work-groups to start are short: of
// up to 64 causal sequences by levels, the tile's place behind the keys
// before the sequence's first token, counted in tiles.
__device__ __forceinline__ TileItem find_item(const AttnArgs &a, int group, int i, bool whole) {
    TileItem r;
    const int lane = threadIdx.x & 63;
    r.b = -1;
    r.range = 0;
    r.part = 0;
    r.apart = 1;
    r.unit = kWhole;
    r.s = Seq{};
    r.t = 0;
    if (a.seqs.n_seqs == 1) {
        r.s = seq_of(a.seqs, 0);
        const SeqWork w = seq_work(a, r.s, group);
        if (whole || i >= a.solo) {
            r.apart = w.tiles * a.kv_heads - a.solo;
            r.unit = one_seq_unit(a, w);
            place_item(a, w, whole ? i : i - a.solo, 0, whole, r);
        } else {
            const int q = i / a.kv_heads;
            r.kvh = i - q * a.kv_heads;
            r.t = w.tiles - 1 - q;
        }
        if (r.t >= 0) r.b = 0;
    } else {
        // the first 64 sequences stay in registers
        const Seq mine = lane < a.seqs.n_seqs ? seq_of(a.seqs, lane) : Seq{};
        const SeqWork work = seq_work(a, mine, group);
        if (a.splits > 1) {
            CallWork c = call_work(work);
            for (int b = 64 + lane; b < a.seqs.n_seqs; b += 64)
                add_work(c, call_work(seq_work(a, seq_of(a.seqs, b), group)));
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1)
                add_work(c, CallWork{__shfl_xor(c.total, o), __shfl_xor(c.reach, o), __shfl_xor(c.longest, o),
                                     __shfl_xor(c.tiles, o)});
            r.unit = tile_unit(a, c);
            for (int k = 0; k < 2 && r.unit < kWhole && a.seqs.n_seqs <= 64; ++k)
                r.unit = fit_unit(a, r.unit, wave_sum(work.tiles * key_ranges(a, work.most, r.unit)));
        }
        int l = -1;
        Seq s = mine;
        if (a.causal && a.splits == 1 && a.seqs.n_seqs <= 64) {
            const int q = i / a.kv_heads;
            r.kvh = i - q * a.kv_heads;
            const int off = (int)min((int64_t)max(0, mine.nk - mine.nq) * group / kRows, (int64_t)1 << 29);
            // tiles at a level or above it
            auto from = [&](int level) { return min(work.tiles, max(0, work.tiles - max(0, level - off))); };
            if (wave_sum(work.tiles) > q) {
                int top = work.tiles > 0 ? off + work.tiles : 0;
#pragma unroll
                for (int o = 32; o >= 1; o >>= 1) top = max(top, __shfl_xor(top, o));
                int low = 0, high = uniform(top); // the tile's level is in [low, high)
                while (high - low > 1) {
                    const int mid = (low + high) >> 1;
                    if (wave_sum(from(mid)) > q)
                        low = mid;
                    else
                        high = mid;
                }
                // the q-th tile is one of those at this level, a sequence's each
                const bool here = from(low) > from(low + 1);
                const int above = wave_sum(from(low + 1));
                const uint64_t at = __ballot(here);
                const bool it = here && __popcll(at & ((1ull << lane) - 1)) == q - above;
                l = __builtin_ctzll(__ballot(it));
                r.b = l;
                r.t = __shfl(low - off, l);
            }
        } else {
            int tiles0 = 0, items0 = 0;
            for (int b0 = 0; b0 < a.seqs.n_seqs && r.b < 0; b0 += 64) {
                SeqWork w = work;
                if (b0 > 0) {
                    s = b0 + lane < a.seqs.n_seqs ? seq_of(a.seqs, b0 + lane) : Seq{};
                    w = seq_work(a, s, group);
                }
                const int n = w.tiles * a.kv_heads, c = key_ranges(a, w.most, r.unit);
                int tiles = n, items = n * c;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int x = __shfl_up(tiles, o), y = __shfl_up(items, o);
                    if (lane >= o) tiles += x, items += y;
                }
                const uint64_t past = __ballot((whole ? tiles0 + tiles : items0 + items) > i);
                if (past) {
                    l = __builtin_ctzll(past);
                    r.b = b0 + l;
                    r.apart = __shfl(n, l);
                    const int base = items0 + __shfl(items - n * c, l);
                    w.tiles = __shfl(w.tiles, l);
                    place_item(a, w, i - (whole ? tiles0 + __shfl(tiles - n, l) : base), base, whole, r);
                }
                tiles0 += __shfl(tiles, 63);
                items0 += __shfl(items, 63);
            }
        }
        if (l >= 0) {
            r.s.q0 = __shfl(s.q0, l);
            r.s.nq = __shfl(s.nq, l);
            r.s.kv0 = __shfl(s.kv0, l);
            r.s.nk = __shfl(s.nk, l);
            r.s.bad = __shfl((int)s.bad, l);
        }
    }
    if (r.b < 0) return r;
    r.b = uniform(r.b);
    r.s.q0 = uniform(r.s.q0);
    r.s.nq = uniform(r.s.nq);
    r.s.kv0 = uniform(r.s.kv0);
    r.s.nk = uniform(r.s.nk);
    r.kvh = uniform(r.kvh);
    r.t = uniform(r.t);
    r.range = uniform(r.range);
    r.part = uniform(r.part);
    r.apart = uniform(r.apart);
    r.unit = uniform(r.unit);
    return r;
}
// The stages [t0, t1) of a tile's range, and how many ranges it has.
struct TileRange {
    int t0, t1, ranges;
};
template <int D>
__host__ __device__ __forceinline__ TileRange tile_range(const AttnArgs &a, const TileKeys &k, const TileItem &it) {
    constexpr int KK = TileShapeOf<D>::keys;
    const int first = k.k0 / KK, last = (k.k1 + KK - 1) / KK, n = last - first;
    TileRange r;
    r.ranges = key_ranges(a, k.k1 - k.k0, it.unit);
    const int per = r.ranges == 1 ? n : (n + r.ranges - 1) / r.ranges;
    if (r.ranges > 1) r.ranges = (n + per - 1) / per; // none empty
    r.t0 = first + it.range * per;
    r.t1 = min(r.t0 + per, last);
    return r;
}

// A buffer resource over `bytes` from p (uniform; none where it is negative,
// as for keys past the last): reads at or past its end give zeros and touch
// no memory.
__device__ __forceinline__ u32x4 key_buffer(const uint16_t *p, int bytes) {
    const uint64_t v = (uint64_t)p;
    return u32x4{(uint32_t)v, (uint32_t)(v >> 32) & 0xffffu, (uint32_t)max(0, bytes), (uint32_t)kBufferFlags};
}

// 16 bytes a lane from byte `off` of a resource to lds + 16 * lane (uniform
// lds).  In assembly so that the compiler does not wait for the copy before
// reads of LDS that other copies filled, as it does for its own builtin
// where it cannot tell the two apart; there is no output register.  The
// reader waits with wait_vmcnt and a barrier.  (The compiler's own counted
// waits stay right: copies that it does not count only make them longer.)
__device__ __forceinline__ void copy_to_lds(u32x4 rsrc, uint8_t *lds, uint32_t off) {
    const uint32_t at = (uint32_t)(uintptr_t)(lds_void_t *)lds;
    uint32_t m0; // the compiler's, kept
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
                 "buffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "s"(at), "v"(off), "s"(rsrc)
                 : "memory");
}

// Order for the scheduler: the LDS reads (PER each) of AHEAD products (USES
// instructions each), then N products with a read PER each behind them while
// there are any.
template <int AHEAD, int PER, int N, int USES = 1>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * PER, 0); // LDS reads
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, USES, 0); // matrix instructions
        __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, AHEAD * USES, 0);
}

// One pass over the keys: S^T = K Q^T by 32x32x16 products leaves a lane the
// scores of one row, whose maximum and sum then need one exchange between the
// wave's halves; O^T += V^T P^T takes the weights in the registers and the key
// order they are in.  Four waves of 32 rows share a stage's keys and values.
//
// Bound by the matrix units together with the vector instructions of the
// softmax (a 32 x 32 block of scores is 8 products of 32 cycles at D = 128,
// as many for the values, and about 80 vector instructions, 16 of them
// exponentials), and by how well three independent work-groups a CU hide one
// another's LDS reads, barriers and copies.  Left out in turn at D = 128, 8192
// tokens (1103 us, 1.0 PFLOP/s): reads of keys 21 %, softmax 15 %, copies 10
// %, reads of values 9 %; matrix units busy 63 % of the cycles, no bank
// conflicts.  0.96 PFLOP/s at 4608 tokens x 24 heads of 128, 0.8 at 8191
// causal tokens x 16 heads of 64.
//
// FINE, for bf16 inputs and fp16 output (packed): the weights are two products'
// worth of bf16, 2^-16 in place of 2^-8, which is eight times as coarse as the
// output (error against 64 bits 1.00 of that of fp32 weights, 3.5 to 5 times
// with one product).  Half as many matrix instructions again: 6000 causal
// tokens x 16 heads of 128 241 us, with one product 178; of 64 147, 116; of
// 256 503, 422.  fp16 weights are as fine as the output, and bf16 output as
// coarse as the weights: one product (1.07 to 1.29 times).
template <bool BF, int D, bool PAGED, bool FINE>
__global__ __launch_bounds__(256, TileShapeOf<D>::waves) void b1_attn_tile_kernel(AttnArgs a) {
    constexpr int ST = D / 16, DT = D / 32, CH = D / 8, KK = TileShapeOf<D>::keys, KT = KK / 32,
                  S = TileShapeOf<D>::stages, SB = KK * D * 2;
    __shared__ __align__(1024) uint8_t sk[S][SB], sv[S][SB];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int l31 = lane & 31, h = lane >> 5;
    const int group = a.heads / a.kv_heads;
    if (a.bad && blockIdx.x == 0 && wave == 0) report_seqs(a.seqs, a.bad);

    const TileItem it = find_item(a, group, blockIdx.x, false);
    const int b = uniform(it.b), kvh = uniform(it.kvh);
    if (b < 0) return;
    Seq s = it.s;
    s.q0 = uniform(s.q0), s.nq = uniform(s.nq), s.kv0 = uniform(s.kv0), s.nk = uniform(s.nk);
    const TileKeys tk = tile_keys(a, s, group, it.t);
    const TileRange tr = tile_range<D>(a, tk, it);
    const int ranges = uniform(tr.ranges), t0 = uniform(tr.t0), t1 = uniform(tr.t1);
    const int first_key = uniform(tk.k0);
    if (it.range >= ranges) return;

    // this lane's row; rows past the tile's last repeat it and store nothing
    const int wrow = wave * 32 + l31;
    const int r = tk.r0 + min(wrow, tk.rows - 1);
    const bool mine = wrow < tk.rows;
    const int ri = div_group(a, r), token = s.q0 + ri, head = kvh * group + r - ri * group;
    int lo, hi;
    visible(a, s, ri, lo, hi);
    // the wave's rows: keys that some see, keys that all see
    const bool wave_on = wave * 32 < tk.rows;
    int first_lo, first_hi, last_lo, last_hi;
    visible(a, s, div_group(a, tk.r0 + min(wave * 32, tk.rows - 1)), first_lo, first_hi);
    visible(a, s, div_group(a, tk.r0 + min(wave * 32 + 31, tk.rows - 1)), last_lo, last_hi);
    first_lo = uniform(first_lo), first_hi = uniform(first_hi), last_lo = uniform(last_lo), last_hi = uniform(last_hi);

    const uint16_t *qrow = a.q + token * a.q_row + head * a.q_head;
    const KeyRows kr = key_rows<PAGED>(a.k, a.k_page, a.k_row, a.k_head, kvh, s);
    const KeyRows vr = key_rows<PAGED>(a.v, a.v_page, a.v_row, a.v_head, kvh, s);
    bool bad = s.bad;

    // Copies a stage.  A wave's instruction copies the NR rows that lie in 1
    // KiB; lane i lands at 16 i, so the swizzle is in which chunk of the row
    // it reads.  Rows past the last key read zeros.  Paged: keys and values
    // lie alike, `page` holds the page of each instruction's first row, and
    // rows of more than one page (of fewer than NR keys) take an instruction
    // a page.
    constexpr int NR = 512 / D, NI = SB / 4096;
    struct Pages {
        int id[PAGED ? NI : 1];
    };
    auto page_at = [&](int j) __attribute__((always_inline)) {
        // a scalar read: it does not wait for the copies under way
        typedef const __attribute__((address_space(4))) int32_t *scalar_ptr;
        const scalar_ptr table = (scalar_ptr)(uintptr_t)(a.seqs.pages + b * a.seqs.ld_pages);
        return table[min(j, s.nk - 1) >> a.seqs.page_shift];
    };
    auto pages = [&](int kb) __attribute__((always_inline)) {
        Pages p;
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < NI; ++i) p.id[i] = page_at(kb + (wave * NI + i) * NR);
        }
        return p;
    };
    auto load = [&](int kb, const Pages &page, int to, bool begin) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int at = wave * NI + i, row0 = at * NR;
            const int row = row0 + lane / CH;
            const int ck = ((lane % CH) ^ swizzle_k<D>(row)) * 16, cv = ((lane % CH) ^ swizzle_v<D>(row)) * 16;
            uint8_t *const ks = sk[to] + at * 1024, *const vs = sv[to] + at * 1024;
            if constexpr (PAGED) {
                const int size = 1 << a.seqs.page_shift, bytes = (int)kr.row * 2;
                const uint32_t off = (uint32_t)((kb + row) & (size - 1)) * (uint32_t)bytes;
                auto copy = [&](int id, int j) __attribute__((always_inline)) {
                    // keys of the page up to the sequence's last; none of a
                    // page that a window leaves behind, whose entry may be
                    // anything (only in a tile's first stage)
                    int keys = min(size, s.nk - (j & -size));
                    if (begin && (j | (size - 1)) < first_key) keys = 0, id = 0;
                    if ((unsigned)id >= (unsigned)a.seqs.n_pages) bad = true, id = 0;
                    copy_to_lds(key_buffer(kr.base + id * kr.page, keys * bytes), ks, off + ck);
                    copy_to_lds(key_buffer(vr.base + id * vr.page, keys * bytes), vs, off + cv);
                };
                if (size >= NR) {
                    copy(page.id[i], kb + row0);
                } else {
                    for (int sub = 0; sub < NR; sub += size) {
                        const int id = page_at(kb + row0 + sub);
                        if ((unsigned)(lane / CH - sub) < (unsigned)size) copy(id, kb + row0 + sub);
                    }
                }
            } else {
                const int keys = min(KK, s.nk - kb), kbytes = (int)kr.row * 2, vbytes = (int)vr.row * 2;
                copy_to_lds(key_buffer(kr.base + kb * kr.row, keys * kbytes), ks, row * kbytes + ck);
                copy_to_lds(key_buffer(vr.base + kb * vr.row, keys * vbytes), vs, row * vbytes + cv);
            }
        }
    };

    // this lane's places in a stage: chunk 2 i + h of key row l31, and its
    // share of the value columns 32 dt .. of 4 keys.  Opaque, so that they
    // stay one register each beside a constant offset.
    uint32_t ka[ST], va[DT];
#pragma unroll
    for (int i = 0; i < ST; ++i) {
        ka[i] = l31 * (D * 2) + (((2 * i + h) ^ swizzle_k<D>(l31)) << 4);
        asm("" : "+v"(ka[i]));
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        const int row = 4 * h + (lane & 15) / 4, chunk = 4 * i + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
        va[i] = row * (D * 2) + ((chunk ^ swizzle_v<D>(row)) << 4) + (lane & 1) * 8;
        asm("" : "+v"(va[i]));
    }

    u32x4 qf[ST];
#pragma unroll
    for (int i = 0; i < ST; ++i) qf[i] = *reinterpret_cast<const u32x4 *>(qrow + 16 * i + 8 * h);
    floatx16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = floatx16{};
    float m = kLowest, l = 0.f;
    const float scale2 = a.scale * 1.44269504f; // exp(x) = exp2(x log2 e)

    // S - 1 stages are being copied while one is read
    Pages next = {}; // of the stage to copy next
    if (t0 < t1) {
#pragma unroll
        for (int i = 0; i < S - 1; ++i)
            if (t0 + i < t1) load((t0 + i) * KK, pages((t0 + i) * KK), i, i == 0);
        next = pages((t0 + S - 1) * KK);
        // the queries too, so that no wait for them remains in the loop
        wait_vmcnt<0>();
    }
    auto stage = [&](int tt, int at) __attribute__((always_inline)) {
        const int kb = tt * KK;
        const uint8_t *const ks = sk[at], *const vs = sv[at];
        // every wave's copies of this stage are there (those of the next ones
        // may be under way), and its reads of the last one done
        if (S > 2 && tt + S - 2 < t1)
            wait_vmcnt<2 * NI * (S - 2)>();
        else
            wait_vmcnt<0>();
        wait_lgkmcnt0();
        lds_barrier();
        if (tt + S - 1 < t1) {
            load(kb + (S - 1) * KK, next, (at + S - 1) % S, false);
            next = pages(kb + S * KK);
        }
        if (!wave_on || kb > last_hi || kb + KK - 1 < first_lo) return;
        // scores, transposed: column = row of q, register i of half h = key
        // 8 (i / 4) + 4 h + i % 4
        floatx16 sc[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            sc[kt] = floatx16{};
#pragma unroll
            for (int i = 0; i < ST; ++i)
                sc[kt] = mfma32<BF>(*reinterpret_cast<const u32x4 *>(ks + 32 * kt * (D * 2) + ka[i]), qf[i], sc[kt]);
        }
        // three reads ahead of the products (1.03 of the compiler's own order)
        reads_ahead<3, 1, KT * ST>();
        if (kb + KK - 1 > first_hi || kb < last_lo) {
            const int top = hi - kb - 4 * h, bot = lo - kb - 4 * h;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int c = 32 * kt + 8 * (i / 4) + i % 4;
                    sc[kt][i] = c <= top && c >= bot ? sc[kt][i] : -kInf;
                }
        }
        float mx = -kInf;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
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
        // weights, rounded to the inputs' type for the product and summed as
        // rounded, or (FINE) with another product for what the rounding left;
        // o (transposed) += v (transposed) p, 16 keys a product, in
        // the order the scores' registers hold them
#pragma unroll
        for (int x = 0; x < 2 * KT; ++x) {
            u32x4 pf, pr;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 8 * (x & 1) + 2 * e;
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x / 2][i], scale2, -m));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x / 2][i + 1], scale2, -m));
                pf[e] = pack_16<BF>(p0, p1);
                if constexpr (FINE) {
                    l += p0 + p1;
                    pr[e] = pack_16<BF>(p0 - to_f32<BF>((uint16_t)pf[e]), p1 - to_f32<BF>((uint16_t)(pf[e] >> 16)));
                } else {
                    l = add_pair<BF>(pf[e], l);
                }
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const uint8_t *at = vs + 16 * x * (D * 2) + va[dt];
                const u32x2 y = read_columns(at), z = read_columns(at + 8 * (D * 2));
                const u32x4 vf = {y[0], y[1], z[0], z[1]};
                o[dt] = mfma32<BF>(vf, pf, o[dt]);
                if constexpr (FINE) o[dt] = mfma32<BF>(vf, pr, o[dt]);
            }
        }
        reads_ahead<2, 2, 2 * KT * DT, FINE ? 2 : 1>();
    };
    for (int tt = t0; tt < t1; tt += S) {
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (tt + i < t1) stage(tt + i, i);
    }
    l = halves_sum(l);
    // A scaled score past fp32's range: its weight is exp2 of the product less
    // the maximum, in one instruction that does not round the product, and so
    // 0 in place of infinity less infinity.
    if (m == kInf) l = __builtin_nanf("");

    if (__syncthreads_or(bad)) {
        bad = true;
        if (a.bad && threadIdx.x == 0) atomicAdd(a.bad, 1);
    }
    if (!wave_on) return;
    if (bad) l = __builtin_nanf("");
    float inv = l == 0.f ? 0.f : 1.0f / l;
    // columns 32 i .. of the row: register e of half h = column 8 (e / 4) +
    // 4 h + e % 4
    const int64_t part = ((int64_t)it.range * it.apart + it.part) * kRows + wrow;
    auto store = [&](int i, floatx16 v) __attribute__((always_inline)) {
        if (!mine) return;
        if (ranges > 1) {
            float *po = a.part_o + part * D + 32 * i + 4 * h;
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<floatx4 *>(po + 8 * g) = floatx4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
            return;
        }
        v *= inv;
        uint16_t *orow = a.out + token * a.ldo + head * D + 32 * i;
        if (a.packed) {
            // words d .. d + 3 of the block: columns d and d + 16
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pack_f16(v[4 * g + e], v[4 * g + e + 8]);
                *reinterpret_cast<u32x4 *>(orow + 16 * g + 8 * h) = w;
            }
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<u32x2 *>(orow + 8 * g + 4 * h) =
                    u32x2{pack_16<BF>(v[4 * g], v[4 * g + 1]), pack_16<BF>(v[4 * g + 2], v[4 * g + 3])};
        }
    };
    int odd = 0;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) odd |= !finite(o[i][e] * inv);
    odd |= __shfl_xor(odd, 32);
    if (odd && !bad) {
#pragma unroll 1
        for (int i = 0; i < DT; ++i) {
            floatx16 v = {};
            row_fp32<BF, D, PAGED>(a, kr, vr, b, qrow, max(lo, t0 * KK), min(hi + 1, t1 * KK), scale2, m, l,
                                   [&](const uint16_t *x, float p) {
#pragma unroll
                                       for (int e = 0; e < 16; ++e)
                                           v[e] += p * to_f32<BF>(x[32 * i + 8 * (e / 4) + 4 * h + e % 4]);
                                   });
            inv = l == 0.f ? 0.f : 1.0f / l;
            store(i, v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < DT; ++i) store(i, o[i]);
    }
    if (ranges > 1 && mine && h == 0) *reinterpret_cast<float2v *>(a.part_ml + 2 * part) = float2v{m, l};
}

// ---- few rows a sequence ----------------------------------------------------
//
// Up to 16 rows of a key head take one 16x16x32 product's columns; keys and
// values go from memory to registers once, each lane the 16 bytes that its
// matrix operand needs (values are put together from two keys' words), so
// that a wave's 32 keys of both are in flight together.  The weights of bf16
// inputs are two products' worth of bf16 (the value and what its rounding
// left): 2^-16 in place of 2^-8, for a product that costs nothing beside the
// reads; those of fp16 inputs are rounded once, 2^-11 (two products: no time
// at D = 64 and 128, 3 to 6 % at 256; the output's own rounding is as large).
// Bound by HBM: 64 bf16 caches of 60 to 8100 keys, 1.04 GB, 210 us,
// 4.9 TB/s (the rate of a large copy); one of 32700 keys, 134 MB, 27 us and a
// join of 5.6, latency at both ends.
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
// Keys a range, from the lengths of all sequences (by the whole wave).  None
// is split where a CU's share of all keys is twice the longest's or more (64
// sequences of 2000 keys, 8 key heads: 102 us, split 111; 100 of 60 to 4000
// keys 188, split 161, and 64 of 60 to 8100 keys 268, split 217: their
// longest is more than half a share).
__device__ __forceinline__ int few_unit(const AttnArgs &a) {
    constexpr int step = kFewKeys * kWaves;
    if (a.splits == 1) return INT_MAX;
    const int lane = threadIdx.x & 63;
    float total = 0.f, longest = 0.f; // a split size needs no more
    for (int b = lane; b < a.seqs.n_seqs; b += 64) {
        int at;
        const float len = (float)few_len(a, seq_of(a.seqs, b), at);
        total += len;
        longest = fmaxf(longest, len);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        total += __shfl_xor(total, o);
        longest = fmaxf(longest, __shfl_xor(longest, o));
    }
    total *= (float)a.kv_heads;
    if (2.f * longest * (float)a.cus <= total) return INT_MAX;
    const int want = (int)fminf(total / (float)a.target, 1.9e9f);
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
    if (a.splits == 1) b = item;
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
    if (plan.ranges == 0) return; // no tokens
    const int j0 = plan.at + range * plan.keys, j1 = min(j0 + plan.keys, s.nk);

    const KeyRows kr = key_rows<PAGED>(a.k, a.k_page, a.k_row, a.k_head, kvh, s);
    const KeyRows vr = key_rows<PAGED>(a.v, a.v_page, a.v_row, a.v_head, kvh, s);
    const float scale2 = a.scale * 1.44269504f;
    const int rows = s.nq * group;
    bool any_bad = s.bad;

    for (int r0 = 0; r0 < rows; r0 += kFewRows) {
        bool bad = s.bad;
        const int r = min(r0 + c, rows - 1);
        const int ri = div_group(a, r);
        const uint16_t *qrow = a.q + (s.q0 + ri) * a.q_row + (kvh * group + r - ri * group) * a.q_head;
        int lo, hi;
        visible(a, s, ri, lo, hi);
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
                    // (a product past fp32's range is infinity and its weight
                    // NaN: the choice keeps it apart from the difference below)
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
            u32x4 pf, pr;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float p0 = sc[k / 2][2 * (k & 1)], p1 = sc[k / 2][2 * (k & 1) + 1];
                pf[k] = pack_16<BF>(p0, p1);
                if (BF) // what the rounding to 8 bits left
                    pr[k] = pack_16<BF>(p0 - to_f32<BF>((uint16_t)pf[k]), p1 - to_f32<BF>((uint16_t)(pf[k] >> 16)));
            }
            // matrix row c of product e is column E c + e
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                u32x4 vf;
#pragma unroll
                for (int k = 0; k < 4; ++k) vf[k] = __builtin_amdgcn_perm(vw[2 * k + 1][e / 2], vw[2 * k][e / 2], sel);
                o[e] = mfma16<BF>(vf, pf, o[e]);
                if (BF) o[e] = mfma16<BF>(vf, pr, o[e]);
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
        const int rri = div_group(a, rr), token = s.q0 + rri, head = kvh * group + rr - rri * group;
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
                visible(a, s, rri, rlo, rhi);
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

// The joined sums of a row's ranges, by 16 lanes with E columns each: from
// `first` on every `step`-th of `ranges`, partial sums `apart` rows apart,
// with the weights of all ranges.
template <int E>
__device__ __forceinline__ void join_ranges(const float *part_o, const float *part_ml, int64_t row, int64_t apart,
                                            int ranges, int first, int step, int c0, float (&o)[E]) {
    const int lane16 = threadIdx.x & 15;
    auto sums = [&](int i, int c) {
        return *reinterpret_cast<const floatx4 *>(part_o + (row + i * apart) * (16 * E) + c0 + c);
    };
    // the first sums are on their way while the maxima are joined
    constexpr int PRE = 4;
    floatx4 pre[PRE][E / 4];
#pragma unroll
    for (int k = 0; k < PRE; ++k)
#pragma unroll
        for (int c = 0; c < E / 4; ++c) {
            pre[k][c] = floatx4{};
            if (first + k * step < ranges) pre[k][c] = sums(first + k * step, 4 * c);
        }
    // lane i: range i, i + 16, ..
    const float2v none = {kLowest, 0.f};
    const float2v mine =
        lane16 < ranges ? *reinterpret_cast<const float2v *>(part_ml + 2 * (row + lane16 * apart)) : none;
    float M = mine[0];
    for (int i = lane16 + 16; i < ranges; i += 16) M = fmaxf(M, part_ml[2 * (row + i * apart)]);
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
    float L = __builtin_amdgcn_exp2f(mine[0] - M) * mine[1];
    for (int i = lane16 + 16; i < ranges; i += 16) {
        const float2v ml = *reinterpret_cast<const float2v *>(part_ml + 2 * (row + i * apart));
        L += __builtin_amdgcn_exp2f(ml[0] - M) * ml[1];
    }
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1) L += __shfl_xor(L, x);
    // weights that add up to at most 1 before they meet a sum of values
    const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    auto add = [&](float m, floatx4 v, int c) {
        const float f = __builtin_amdgcn_exp2f(m - M) * inv;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[4 * c + k] += f * v[k];
    };
#pragma unroll
    for (int k = 0; k < PRE; ++k) {
        const int i = first + k * step;
        const float m = i < 16       ? __shfl(mine[0], (threadIdx.x & 48) + (i & 15))
                        : i < ranges ? part_ml[2 * (row + i * apart)]
                                     : 0.f;
        if (i < ranges)
#pragma unroll
            for (int c = 0; c < E / 4; ++c) add(m, pre[k][c], c);
    }
#pragma unroll 4
    for (int i = first + PRE * step; i < ranges; i += step) {
        const float m = part_ml[2 * (row + i * apart)];
#pragma unroll
        for (int c = 0; c < E / 4; ++c) add(m, sums(i, 4 * c), c);
    }
}

// Rows of split tiles: W work-groups a tile, each every W-th 16 of its rows.
template <bool BF, int D>
__global__ __launch_bounds__(256) void b1_attn_tile_join_kernel(AttnArgs a, int W) {
    constexpr int E = D / 16;
    const int group = a.heads / a.kv_heads;
    const int tile = blockIdx.x / W;
    const TileItem it = find_item(a, group, tile, true);
    if (it.b < 0) return;
    const Seq &s = it.s;
    const TileKeys tk = tile_keys(a, s, group, it.t);
    const int ranges = tile_range<D>(a, tk, it).ranges, c0 = (threadIdx.x & 15) * E;
    // (partial sums past the launched items: of sequences that overlap, which
    // no plan counts)
    if (ranges <= 1 || (int64_t)(ranges - 1) * it.apart + it.part >= a.items) return;
    for (int r0 = (blockIdx.x - tile * W) * 16; r0 < tk.rows; r0 += W * 16) {
        const int row = r0 + (threadIdx.x >> 4), there = min(row, tk.rows - 1);
        const int r = tk.r0 + there, ri = div_group(a, r);
        float o[E];
        join_ranges<E>(a.part_o, a.part_ml, (int64_t)it.part * kRows + there, (int64_t)it.apart * kRows, ranges, 0, 1,
                       c0, o);
        store_row<BF, D>(a, s.q0 + ri, it.kvh * group + r - ri * group, c0, o, row < tk.rows);
    }
}

// Rows of the few-rows kernel: P groups of 16 lanes take a row, each every
// P-th of its ranges; rows whose keys were not split are there already.
// Bound by latency: a row's sequence and number of ranges are one read deep,
// the maxima and sums of all ranges are read at once by the 16 lanes.
template <bool BF, int D, int P>
__global__ __launch_bounds__(256) void b1_attn_few_join_kernel(AttnArgs a) {
    constexpr int E = D / 16, ROWS = 16 / P; // rows a work-group
    __shared__ __align__(16) float so[16][D + 4];
    const int all = a.seqs.tokens * a.heads;
    const int at16 = threadIdx.x >> 4;
    const int row = blockIdx.x * ROWS + at16 / P, part = at16 % P, c0 = (threadIdx.x & 15) * E;
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
    float o[E];
    join_ranges<E>(a.part_o, a.part_ml, mine ? row : 0, all, mine ? ranges : 0, part, P, c0, o);
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
    int splits, target, solo;
    int64_t grid, tiles; // work-groups; tiles that may be split
};

// Calls whose sequences have up to 16 rows a key head on average run the
// few-rows kernel, others tiles (8 sequences over 3000 keys, 8 key heads, us:
// 16 rows 27.3, as tiles 32.0; 24 rows 42.1, 32.8; 32 sequences over 2000: 16
// rows 52.0, 50.0; 24 rows 89.8, 50.5; all of equal sequences: a long chunk
// among single tokens is far from both, 63 tokens and one of 190 over 6000
// keys 4105, apart 282 and 49).  Tiles of few rounds of the device are split
// where that pays; of more equal ones (one sequence, every key seen) the part
// of the last round that would leave most of the device idle.
AttnPlan attn_plan(const AttnArgs &a, int num_cus, bool split) {
    AttnPlan p{};
    const int group = a.heads / a.kv_heads;
    const int64_t n = a.seqs.n_seqs;
    const int64_t rows = (int64_t)a.seqs.tokens * group; // a key head
    const int64_t most = a.seqs.pages ? (int64_t)a.seqs.max_pages << a.seqs.page_shift : a.seqs.kv_tokens;
    p.few = rows <= kFewRows * n;
    p.splits = 1;
    if (p.few) {
        // Two work-groups a CU fit (one at D = 256, whose second round runs
        // after the first).  Where the sequences themselves make few, exactly
        // two (32 heads over 32700 keys: 38 us, 45 with 4 a CU);
        // else small pieces, so that none outlasts the rest (64 sequences of
        // 60 to 8100 keys: 215 us, 245 with 2).  Four rounds of whole sequences
        // even out by themselves (256 of 60 to 4000 keys, 8 key heads: 379 us,
        // split 393; 1024 of them 1413, 1543; 128 of them 225, 210), and with
        // a work-group a CU short ones cost less than a join (33 of 500 keys:
        // 20 us, split 32; of 2000 keys 52, 64, but of 60 to 4000 93, 73).
        const int64_t step = kFewKeys * kWaves, units = n * a.kv_heads;
        split = split && units < 8 * num_cus && (units < num_cus || most > 1024);
        const int64_t target = (units <= num_cus ? 2 : 6) * num_cus;
        int64_t s = std::min<int64_t>({4 * ((target + units - 1) / units), 256, (most + step - 1) / step});
        // partial results no larger than 1 GiB
        s = std::min(s, ((int64_t)1 << 30) / ((int64_t)a.seqs.tokens * a.heads * (a.head_dim + 2) * 4));
        if (split && s > 1) p.splits = (int)s, p.target = (int)target;
        // sum over sequences of ceil(len / unit) <= n + target / kv_heads
        p.grid = std::min(n * p.splits, n + (p.splits > 1 ? target / a.kv_heads + 1 : 0)) * a.kv_heads;
        return p;
    }
    const int64_t slots = (int64_t)num_cus * (a.head_dim == 256 ? TileShapeOf<256>::waves : TileShapeOf<128>::waves);
    p.tiles = (n == 1 ? (rows + kRows - 1) / kRows : rows / kRows + n) * a.kv_heads;
    p.grid = p.tiles;
    if (!split || most <= 2 * kLeastKeys) return p;
    if (p.tiles >= slots && n == 1 && !a.causal) {
        // equal tiles: the last round's
        const int64_t rest = p.tiles % slots;
        const int64_t s = rest ? std::min<int64_t>(slots / rest, most / (2 * kLeastKeys)) : 1;
        if (s > 1) {
            p.solo = (int)(p.tiles - rest);
            p.splits = (int)s;
            p.tiles = rest;
            p.grid = p.solo + rest * s;
        }
    } else if (p.tiles < slots) { // the kernel decides
        p.splits = (int)std::min<int64_t>(most / kLeastKeys, 64);
        p.target = (int)slots;
        p.grid = std::min(p.tiles * p.splits, p.tiles + slots + 1);
    }
    return p;
}

// For a call's launch: where the kernels get what the plan says.
void set_plan(AttnArgs *a, const AttnPlan &p, int num_cus) {
    a->splits = p.splits;
    a->target = p.target;
    a->solo = p.solo;
    a->cus = num_cus;
    a->items = (int)(p.grid - p.solo);
    // x / group by a multiplication (x < 2^31): s = ceil(log2 group), m =
    // floor(2^32 (2^s - group) / group) + 1, x / group = (hi(x m) + x) >> s
    const uint32_t group = (uint32_t)(a->heads / a->kv_heads);
    a->div_s = 0;
    while ((1u << a->div_s) < group) ++a->div_s;
    a->div_m = (uint32_t)(((((uint64_t)1 << a->div_s) - group) << 32) / group) + 1;
}

// find_item of a split call on the host, from the sequences themselves.
TileItem find_split_item(const AttnArgs &a, const Seq *seqs, int i, bool whole) {
    const int group = a.heads / a.kv_heads, n_seqs = a.seqs.n_seqs;
    TileItem r{};
    r.b = -1;
    r.unit = kWhole;
    r.apart = 1;
    if (n_seqs == 1) {
        const SeqWork w = seq_work(a, seqs[0], group);
        r.s = seqs[0];
        r.apart = w.tiles * a.kv_heads - a.solo;
        r.unit = one_seq_unit(a, w);
        place_item(a, w, whole ? i : i - a.solo, 0, whole, r);
        if (r.t >= 0) r.b = 0;
        return r;
    }
    CallWork c[64] = {};
    for (int b = 0; b < n_seqs; ++b) add_work(c[b % 64], call_work(seq_work(a, seqs[b], group)));
    for (int o = 32; o >= 1; o >>= 1)
        for (int l = 0; l < o; ++l) add_work(c[l], c[l + o]);
    r.unit = tile_unit(a, c[0]);
    for (int k = 0; k < 2 && r.unit < kWhole && n_seqs <= 64; ++k) {
        int items = 0;
        for (int b = 0; b < n_seqs; ++b) {
            const SeqWork w = seq_work(a, seqs[b], group);
            items += w.tiles * key_ranges(a, w.most, r.unit);
        }
        r.unit = fit_unit(a, r.unit, items);
    }
    int tiles = 0, items = 0;
    for (int b = 0; b < n_seqs; ++b) {
        const SeqWork w = seq_work(a, seqs[b], group);
        const int n = w.tiles * a.kv_heads, all = n * key_ranges(a, w.most, r.unit);
        if ((whole ? tiles + n : items + all) > i) {
            r.b = b;
            r.s = seqs[b];
            r.apart = n;
            place_item(a, w, i - (whole ? tiles : items), items, whole, r);
            return r;
        }
        tiles += n;
        items += all;
    }
    return r;
}

size_t round_256(size_t b) { return (b + 255) & ~(size_t)255; }

// Partial results of a plan: their rows, and bytes of the three areas (sums
// of values, maxima and sums of weights, ranges of a row).
int64_t part_rows(const AttnArgs &a, const AttnPlan &p) {
    if (p.splits <= 1) return 0;
    return p.few ? (int64_t)p.splits * a.seqs.tokens * a.heads : (p.grid - p.solo) * kRows;
}
size_t part_bytes(const AttnArgs &a, const AttnPlan &p) {
    const size_t rows = (size_t)part_rows(a, p);
    if (rows == 0) return 0;
    return round_256(rows * a.head_dim * 4) + round_256(rows * 8) + (p.few ? (size_t)a.seqs.tokens * a.heads * 4 : 0);
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
        auto run = [&](auto fine) {
            constexpr bool FINE = decltype(fine)::value;
            if (a.seqs.pages)
                hipLaunchKernelGGL((b1_attn_tile_kernel<BF, D, true, FINE>), grid, block, 0, s, a);
            else
                hipLaunchKernelGGL((b1_attn_tile_kernel<BF, D, false, FINE>), grid, block, 0, s, a);
        };
        if (BF && a.packed)
            run(std::bool_constant<BF>());
        else
            run(std::false_type());
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits <= 1) return e;
    const int64_t rows = (int64_t)a.seqs.tokens * a.heads;
    if (!p.few) {
        // Few tiles take a work-group for every 16 rows (60 rows over 32000
        // keys 60 us in all, with 2 a tile 76), many have work-groups enough,
        // each of which looks its tile up or, where the kernel decided against
        // splitting, only finds that out (368 tiles 152 us, with 8 157; 2048
        // causal tokens 61, 67).
        const int w = p.solo > 0 || p.tiles < 256 ? kRows / 16 : 2;
        hipLaunchKernelGGL((b1_attn_tile_join_kernel<BF, D>), dim3(p.tiles * w), block, 0, s, a, w);
    } else if (p.splits <= 4)
        hipLaunchKernelGGL((b1_attn_few_join_kernel<BF, D, 1>), dim3((rows + 15) / 16), block, 0, s, a);
    else if (p.splits <= 16)
        hipLaunchKernelGGL((b1_attn_few_join_kernel<BF, D, 4>), dim3((rows + 3) / 4), block, 0, s, a);
    else
        hipLaunchKernelGGL((b1_attn_few_join_kernel<BF, D, 16>), dim3(rows), block, 0, s, a);
    return hipGetLastError();
}

} // namespace

extern "C" int64_t b1_attention_items(const int32_t *q_len, const int32_t *kv_len, int n_seqs, int most, int heads,
                                      int kv_heads, int head_dim, int causal, int window, int num_cus, int join,
                                      int32_t *items, int64_t room, int64_t *rows) {
    AttnArgs a{};
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.causal = causal;
    a.window = window;
    a.seqs.n_seqs = n_seqs;
    a.seqs.kv_tokens = most;
    std::vector<Seq> seqs(n_seqs);
    int64_t kv0 = 0;
    for (int b = 0; b < n_seqs; ++b) {
        seqs[b] = Seq{a.seqs.tokens, q_len[b], (int)kv0, kv_len[b], false};
        a.seqs.tokens += q_len[b];
        kv0 += kv_len[b];
    }
    if (a.seqs.tokens == 0) return 0;
    const AttnPlan p = attn_plan(a, num_cus, true);
    if (p.few || p.splits <= 1) return 0;
    set_plan(&a, p, num_cus);
    *rows = part_rows(a, p);
    const int group = heads / kv_heads;
    const int64_t n = join ? p.tiles : p.grid - p.solo;
    for (int64_t i = 0; i < std::min(n, room); ++i) {
        const TileItem it = find_split_item(a, seqs.data(), (int)(join ? i : p.solo + i), join != 0);
        TileRange r{};
        if (it.b >= 0) {
            const TileKeys k = tile_keys(a, it.s, group, it.t);
            r = head_dim == 64 ? tile_range<64>(a, k, it) : head_dim == 128 ? tile_range<128>(a, k, it)
                                                                            : tile_range<256>(a, k, it);
        }
        const int32_t row[] = {it.b, it.kvh, it.t, it.range, r.ranges, r.t0, r.t1, it.part, it.apart};
        std::copy(row, row + 9, items + 9 * i);
    }
    return n;
}

size_t attn_workspace_bytes(const AttnArgs &a, int num_cus) { return part_bytes(a, attn_plan(a, num_cus, true)); }

hipError_t launch_attn(const AttnArgs &args, int num_cus, void *ws, size_t ws_bytes, hipStream_t s) {
    AttnArgs a = args;
    AttnPlan p = attn_plan(a, num_cus, true);
    if (p.splits > 1 && (!ws || ws_bytes < part_bytes(a, p))) p = attn_plan(a, num_cus, false);
    set_plan(&a, p, num_cus);
    if (p.splits > 1) {
        const size_t rows = (size_t)part_rows(a, p);
        uint8_t *at = static_cast<uint8_t *>(ws);
        a.part_o = reinterpret_cast<float *>(at);
        at += round_256(rows * a.head_dim * 4);
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
