// The element-wise operators around a block's linears and attention: RMS
// norm with the residual's addition, and the q/k/v columns' head norm,
// rotary embedding and store.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "b1_seqs.h"

namespace b1 {
namespace {

// Sum over groups of W consecutive lanes.
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = W / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// y = h / sqrt(mean(h^2) + eps) * w over rows of h = x + add.
//
// Bound by HBM: x, add and h at 4 bytes a value, y at 4 or (packed) 2, so a
// row is read once and kept in registers between the sum and the scaling
// (8192 rows of 4096 with add: 84 us, 5.6 TB/s).
// T threads take a row (a work-group has 256 threads or T), U units of 8
// values each (4 + 4 values 16 columns apart: the halves of a packed word
// quad); U = 0 reads wider rows twice.  The sum is fp32, at most 8 U values a
// thread and then a tree.
template <int T, int U>
__global__ __launch_bounds__(T < 256 ? 256 : T) void b1_rms_norm_kernel(
    const float *x, int64_t ldx, const float *add, int64_t lda, int H, int rows, const float *__restrict__ w,
    float eps, float *h, int64_t ldh, float *__restrict__ y, int64_t ldy, uint32_t *__restrict__ packed) {
    constexpr int ROWS = T < 256 ? 256 / T : 1; // a work-group
    __shared__ float part[T / 64];
    const int t = threadIdx.x % T;
    const int row = blockIdx.x * ROWS + threadIdx.x / T;
    if (T == 64 && row >= rows) return; // whole wave; others have a row a work-group
    const float *xr = x + (size_t)row * ldx;
    const float *ar = add ? add + (size_t)row * lda : nullptr;
    float *hr = h ? h + (size_t)row * ldh : nullptr;
    const int units = H / 8;
    auto col = [](int u) { return (u >> 2) * 32 + (u & 3) * 4; };
    auto load = [&](int c) {
        floatx4 v = *reinterpret_cast<const floatx4 *>(xr + c);
        if (ar) v += *reinterpret_cast<const floatx4 *>(ar + c);
        return v;
    };
    auto squares = [](floatx4 v) { return (v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3]); };
    auto total = [&](float s) {
        s = lanes_sum<64>(s);
        if constexpr (T > 64) {
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
            __syncthreads();
            s = lanes_sum<T / 64>(part[threadIdx.x & (T / 64 - 1)]);
        }
        return 1.0f / sqrtf(s / (float)H + eps);
    };
    auto store = [&](floatx4 lo, floatx4 hi, int u, float r) {
        const int c = col(u);
        lo *= r;
        hi *= r;
        if (w) {
            lo *= *reinterpret_cast<const floatx4 *>(w + c);
            hi *= *reinterpret_cast<const floatx4 *>(w + c + 16);
        }
        if (packed) {
            u32x4 p;
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = pack_f16_rounded(lo[j], hi[j]);
            *reinterpret_cast<u32x4 *>(packed + (size_t)row * (H / 2) + 4 * u) = p;
        } else {
            float *yr = y + (size_t)row * ldy + c;
            *reinterpret_cast<floatx4 *>(yr) = lo;
            *reinterpret_cast<floatx4 *>(yr + 16) = hi;
        }
    };
    float s = 0.f;
    if constexpr (U > 0) {
        floatx4 lo[U], hi[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = t + T * i;
            lo[i] = hi[i] = floatx4{0.f, 0.f, 0.f, 0.f};
            if (u < units) {
                lo[i] = load(col(u));
                hi[i] = load(col(u) + 16);
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) s += squares(lo[i]) + squares(hi[i]);
        const float r = total(s);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = t + T * i;
            if (u >= units) continue;
            if (hr) {
                *reinterpret_cast<floatx4 *>(hr + col(u)) = lo[i];
                *reinterpret_cast<floatx4 *>(hr + col(u) + 16) = hi[i];
            }
            store(lo[i], hi[i], u, r);
        }
    } else {
        for (int u = t; u < units; u += T) {
            const floatx4 lo = load(col(u)), hi = load(col(u) + 16);
            s += squares(lo) + squares(hi);
        }
        const float r = total(s);
        // a thread's own values again, each read before h (which may be x or
        // add) is written there
        for (int u = t; u < units; u += T) {
            const floatx4 lo = load(col(u)), hi = load(col(u) + 16);
            if (hr) {
                *reinterpret_cast<floatx4 *>(hr + col(u)) = lo;
                *reinterpret_cast<floatx4 *>(hr + col(u) + 16) = hi;
            }
            store(lo, hi, u, r);
        }
    }
}

// Head norm, rotary embedding and store of a token's q, k and v heads.
//
// Bound by HBM (4 bytes read, 2 written a value; 4608 tokens of 72 heads of
// 128: 54 us, 4.8 TB/s, the rate of a large copy).  D / 4 lanes take a head,
// 4 columns each: the norm's sum is a tree over those lanes, and a rotation's
// partner column is in the lane itself (pairs) or rope_dim / 8 lanes away
// (halves).  A work-group takes `per` of a token's heads, so that its rotary
// row, its position and its page are looked up once.
template <bool BF, int D>
__global__ __launch_bounds__(256) void b1_qkv_kernel(QkvArgs a, int per) {
    constexpr int L = D / 4; // lanes a head
    const int token = blockIdx.x;
    const int col = (threadIdx.x % L) * 4;
    // the token's position and its keys' place
    int pos = token;
    int64_t kv_at = (int64_t)token * a.kv_row;
    bool bad = false, stored = true;
    if (a.seqs.pages) {
        if (a.bad && token == 0 && blockIdx.y == 0 && threadIdx.x < 64) report_seqs(a.seqs, a.bad);
        const int b = seq_of_token(a.seqs, token);
        if (b < 0) return; // a row of no sequence
        const Seq s = seq_of(a.seqs, b);
        pos = s.nk - s.nq + (token - s.q0);
        // more tokens than places; starts that do not ascend, which can give a
        // token to a sequence that does not hold it
        bad = s.bad || pos < 0 || pos >= s.nk;
        if (pos >= 0 && pos < s.nk) {
            const int page = page_of(a.seqs, b, pos, bad);
            kv_at = page * a.kv_page + (pos & ((1 << a.seqs.page_shift) - 1)) * a.kv_row;
        }
        stored = !bad;
    }
    if (a.positions) pos = a.positions[token];
    if (a.rope && (unsigned)pos >= (unsigned)a.rope_rows) {
        bad = true;
        stored = stored && !a.seqs.pages; // rows of NaN, or nothing in a cache
        pos = 0;
    }
    floatx4 c = {1.f, 1.f, 1.f, 1.f}, sn = {0.f, 0.f, 0.f, 0.f};
    const int half = a.rope_dim / 2;
    if (a.rope && col < a.rope_dim) {
        const float *r = a.rope + (size_t)pos * a.rope_dim;
        if (a.interleaved) {
            const float2v cc = *reinterpret_cast<const float2v *>(r + col / 2);
            const float2v ss = *reinterpret_cast<const float2v *>(r + half + col / 2);
            c = floatx4{cc[0], cc[0], cc[1], cc[1]};
            sn = floatx4{-ss[0], ss[0], -ss[1], ss[1]};
        } else {
            const int f = col < half ? col : col - half;
            c = *reinterpret_cast<const floatx4 *>(r + f);
            sn = *reinterpret_cast<const floatx4 *>(r + half + f);
            if (col < half) sn = -sn;
        }
    }
    // the lane (of this wave) that holds the other half's columns
    const int lane = threadIdx.x & 63;
    const int partner = !a.rope || col >= a.rope_dim ? lane : col < half ? lane + half / 4 : lane - half / 4;
    const floatx4 one = {1.f, 1.f, 1.f, 1.f};
    const floatx4 qw = a.q_weight ? *reinterpret_cast<const floatx4 *>(a.q_weight + col) : one;
    const floatx4 kw = a.k_weight ? *reinterpret_cast<const floatx4 *>(a.k_weight + col) : one;
    const int all = a.heads + 2 * a.kv_heads;
    const int first = blockIdx.y * per, last = min(first + per, all);
    for (int hd0 = first; hd0 < last; hd0 += 256 / L) {
        const int hd = hd0 + threadIdx.x / L;
        const bool there = hd < last;
        const bool is_q = hd < a.heads, is_k = !is_q && hd < a.heads + a.kv_heads;
        const int at = is_q ? hd : is_k ? hd - a.heads : hd - a.heads - a.kv_heads;
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
        if (there) {
            const float *src = is_q ? a.q + (size_t)token * a.ldq : is_k ? a.k + (size_t)token * a.ldk
                                                                        : a.v + (size_t)token * a.ldv;
            x = *reinterpret_cast<const floatx4 *>(src + (size_t)at * D + col);
        }
        const float ss = lanes_sum<L>((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]));
        if (is_q ? a.q_weight != nullptr : is_k && a.k_weight != nullptr) {
            const float r = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
            x *= r;
            x *= is_q ? qw : kw;
        }
        floatx4 other;
        if (a.interleaved) {
            other = floatx4{x[1], x[0], x[3], x[2]};
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) other[j] = __shfl(x[j], partner);
        }
        if (a.rope && (is_q || is_k) && col < a.rope_dim) x = x * c + other * sn;
        if (!there) continue;
        if (bad) x = floatx4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        const u32x2 p = {pack_16<BF>(x[0], x[1]), pack_16<BF>(x[2], x[3])};
        uint16_t *dst = is_q ? a.q_out + (size_t)token * a.q_row + (size_t)at * D
                             : (is_k ? a.k_out : a.v_out) + kv_at + at * a.kv_head;
        if (is_q || stored) *reinterpret_cast<u32x2 *>(dst + col) = p;
    }
    if (bad && a.bad && threadIdx.x == 0 && blockIdx.y == 0) atomicAdd(a.bad, 1);
}

// Calls f(kernel, its threads a work-group, its rows a work-group) for rows
// of H values.
//
// Few units a thread and as many threads as that takes: all of a row's
// loads are on their way at once, with few registers held.  Measured (us
// of a norm of x + add into h and packed): 32768 x 512 40.7 (256 threads
// a row 47.3), 8192 x 2048 41.2 (a wave a row 50.8), 8192 x 4096 86.4
// (256 threads 93.8), 4096 x 8192 88.0 (512 threads 94.9, 256 98.3),
// 2048 x 16384 96.8 = 4.9 TB/s (256 threads 117), 2048 x 32768 188 (row
// read twice 303).
template <class F>
auto with_rms_kernel(int H, F f) {
    if (H <= 512) return f(b1_rms_norm_kernel<64, 1>, 256, 4);
    if (H <= 2048) return f(b1_rms_norm_kernel<256, 1>, 256, 1);
    if (H <= 4096) return f(b1_rms_norm_kernel<512, 1>, 512, 1);
    if (H <= 8192) return f(b1_rms_norm_kernel<1024, 1>, 1024, 1);
    if (H <= 16384) return f(b1_rms_norm_kernel<1024, 2>, 1024, 1);
    if (H <= 32768) return f(b1_rms_norm_kernel<1024, 4>, 1024, 1);
    return f(b1_rms_norm_kernel<1024, 0>, 1024, 1);
}

// The rows of a launch: work-groups of 2^31 threads (a launch has less than
// 2^32).
int64_t rms_launch_rows(int threads, int per) { return ((int64_t)1 << 31) / threads * per; }

} // namespace

extern "C" int64_t b1_rms_norm_launch(int H, int *threads, int *per) {
    return with_rms_kernel(H, [&](auto, int t, int p) {
        *threads = t;
        *per = p;
        return rms_launch_rows(t, p);
    });
}

hipError_t launch_rms_norm(const float *x, int64_t ldx, const float *add, int64_t lda, int H, int rows,
                           const float *w, float eps, float *h, int64_t ldh, float *y, int64_t ldy, void *packed,
                           hipStream_t s) {
    uint32_t *pk = static_cast<uint32_t *>(packed);
    return with_rms_kernel(H, [&](auto kernel, int threads, int per) {
        const int64_t most = rms_launch_rows(threads, per);
        for (int64_t r0 = 0; r0 < rows; r0 += most) {
            const int n = (int)std::min<int64_t>(most, rows - r0);
            hipLaunchKernelGGL(kernel, dim3((unsigned)(((int64_t)n + per - 1) / per)), dim3(threads), 0, s,
                               x + r0 * ldx, ldx, add ? add + r0 * lda : nullptr, lda, H, n, w, eps,
                               h ? h + r0 * ldh : nullptr, ldh, y ? y + r0 * ldy : nullptr, ldy,
                               pk ? pk + r0 * (H / 2) : nullptr);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    });
}

hipError_t launch_qkv(const QkvArgs &a, hipStream_t s) {
    const int all = a.heads + 2 * a.kv_heads, round = 1024 / a.head_dim; // heads a pass of a work-group
    // all of a token's heads to a work-group (4608 tokens of 72 heads 50 us,
    // 4.9 TB/s; a pass of heads each 75), or one pass where the tokens alone
    // would leave CUs idle (64 tokens of 48 heads 3.9 us, all of them 6.8;
    // 640 tokens 9.0 and 9.7, 768 tokens 10.1 and 9.7)
    const int per = a.tokens < 700 ? round : (all + round - 1) / round * round;
    const dim3 grid(a.tokens, (all + per - 1) / per);
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, per);
        return hipGetLastError();
    };
    switch (a.head_dim) {
    case 64: return a.bf16 ? run(b1_qkv_kernel<true, 64>) : run(b1_qkv_kernel<false, 64>);
    case 128: return a.bf16 ? run(b1_qkv_kernel<true, 128>) : run(b1_qkv_kernel<false, 128>);
    case 256: return a.bf16 ? run(b1_qkv_kernel<true, 256>) : run(b1_qkv_kernel<false, 256>);
    default: return hipErrorInvalidValue;
    }
}

} // namespace b1
