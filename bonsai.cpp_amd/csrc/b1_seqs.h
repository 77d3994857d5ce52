// Device helpers shared by the kernels that work on packed sequences and
// paged keys (b1_block.hip, b1_attention.hip).  Indexes that lie in device
// memory cannot be checked on the host: every one is brought into range
// here before it addresses anything, and what was out of range is reported.
#pragma once

#include "b1_device.h"
#include "b1_internal.h"

namespace b1 {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Two fp32 values as a pair of 16-bit ones, round to nearest even.
template <bool BF>
__device__ __forceinline__ uint32_t pack_16(float lo, float hi) {
    if constexpr (BF) {
        const float2v v = {lo, hi};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    } else {
        return pack_f16(lo, hi);
    }
}

template <bool BF>
__device__ __forceinline__ float to_f32(uint16_t x) {
    if constexpr (BF)
        return __builtin_bit_cast(float, (uint32_t)x << 16);
    else
        return (float)__builtin_bit_cast(_Float16, x);
}

// A sequence's tokens (rows q0 .. q0 + nq), its keys (rows kv0 .. kv0 + nk of
// contiguous keys, places 0 .. nk of its pages), and whether an index had to
// be brought into range.
struct Seq {
    int q0, nq, kv0, nk;
    bool bad;
};

// [start[b], start[b + 1]) within [0, n]; NULL: all of [0, n].
__device__ __forceinline__ void seq_rows(const int32_t *start, int b, int n, int &at, int &len, bool &bad) {
    if (!start) {
        at = 0;
        len = n;
        return;
    }
    const int s = start[b], e = start[b + 1];
    at = min(max(s, 0), n);
    const int end = min(max(e, at), n);
    len = end - at;
    bad |= at != s || end != e;
}

__device__ __forceinline__ Seq seq_of(const KvSeqs &s, int b) {
    Seq r;
    r.bad = false;
    seq_rows(s.q_start, b, s.tokens, r.q0, r.nq, r.bad);
    if (s.pages) {
        const int n = s.kv_len[b];
        const int64_t room = (int64_t)s.max_pages << s.page_shift;
        r.kv0 = 0;
        r.nk = (int)min((int64_t)max(n, 0), room);
        r.bad |= r.nk != n;
    } else {
        seq_rows(s.kv_start, b, s.kv_tokens, r.kv0, r.nk, r.bad);
    }
    return r;
}

// Reports starts and lengths out of range, those of sequences without rows
// among them (no other work-group sees these).  For one wave of a launch.
__device__ __forceinline__ void report_seqs(const KvSeqs &s, int32_t *bad) {
    int n = 0;
    for (int b = threadIdx.x & 63; b < s.n_seqs; b += 64) n |= seq_of(s, b).bad;
    if (__any(n) && (threadIdx.x & 63) == 0) atomicAdd(bad, 1);
}

// The page that holds place j of sequence b; page 0, and bad, where the
// table's entry names none.  j < max_pages << page_shift.
__device__ __forceinline__ int page_of(const KvSeqs &s, int b, int j, bool &bad) {
    const int p = s.pages[b * s.ld_pages + (j >> s.page_shift)];
    if ((unsigned)p < (unsigned)s.n_pages) return p;
    bad = true;
    return 0;
}

// The sequence of a token, by the whole wave: the number of sequences that
// end at or before it.  -1 for a token before the first sequence or behind
// the last.
__device__ __forceinline__ int seq_of_token(const KvSeqs &s, int token) {
    if (!s.q_start) return 0;
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b = lane; b < s.n_seqs; b += 64) before += min(s.q_start[b + 1], s.tokens) <= token;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) before += __shfl_xor(before, o);
    if (before >= s.n_seqs || s.q_start[before] > token) return -1;
    return before;
}

} // namespace
} // namespace b1
