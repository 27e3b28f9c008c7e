// What the attention kernels share: operands, query rows, partial states.
#pragma once
#include "kv_device.hpp"
#include "kv_launch.hpp"

namespace mgq {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;    // tokens of a tile
constexpr float kTop = 14.0f;  // w is 2^14 at the running maximum
constexpr float kLeastScale = 0x1p-90f;  // smaller scales of V count as this

struct AttnArgs {
    const float *q;
    void *out;
    int64_t q_stride, out_stride;
    int group;  // query heads of a kv head
    int out_f16;
    // softcap off: scale * log2 e; on: scale / softcap, and softcap * log2 e
    float scale, softcap;
    int window;
    float *ws;
};

// What a running maximum is compared with and taken from: w = 2^(t - ref). Where
// numbers as large as M lie 4 and more apart, M - kTop may be off by more than f16 has
// room for (2^15 to 2^16): ref is M there.
__device__ __forceinline__ bool outgrown(float top, float M) { return top - M > 1.0f; }
__device__ __forceinline__ float reference_of(float M) {
    const float r = M - kTop;
    return M == -INFINITY ? 0.0f : M - r > kTop + 0.5f ? M : r;
}

// l = sum of w_j / vs_j = 2^(s_j - ref) moves with V's scales, by 2^211 between a page of
// 2^121 and one of kLeastScale: more than a power of two in f32, and more than w_j have
// that vanish below 2^-126. So l is multiplied by the power in two factors, 2^(x/2)
// each, and
constexpr float kLoudScale = 0x1p26f;
struct Exp2 {
    float h, f;  // f = h * h = 2^x, 0 below f32
    __device__ __forceinline__ explicit Exp2(float x) : h(__builtin_amdgcn_exp2f(0.5f * x)), f(h * h) {}
    __device__ __forceinline__ float times(float l) const { return l * h * h; }
};
// where the largest t of a lane's tokens is so far below ref, their w are summed
// relative to that largest. This is looked at once a page above kLoudScale has been
// seen: without one they are within 2^116 of each other, and what vanishes is below
// l's own rounding. (4096 tokens of 28 heads with f32 results: heads of 64 4 % longer, of 96
// 2.5 %, of 128 1.3 %, others the same.)
__device__ __forceinline__ bool vanishing(float top, float ref) { return top < ref - 100.0f && top > -INFINITY; }

// kv_attn_wide.hip: many query rows of a sequence.
hipError_t kv_attn_wide_launch(const KvView &c, int dim, int fmt, const AttnArgs &a, hipStream_t stream);
size_t kv_attn_wide_workspace(int dim, int group, int hkv, int n_seqs, int max_new, int64_t cap);

template <int FMT>
__device__ __forceinline__ half8 kv_half8(uint32_t lo, uint32_t hi) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    half2v r[4];
    if constexpr (FMT == kFmtI8) {
        // 0x6400 | u is 1024 + u in f16; u = b + 128 after the sign flip
        const uint32_t x[2] = {lo ^ 0x80808080u, hi ^ 0x80808080u};
        const half2v bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x[i / 2], i % 2 ? 0x04030402u : 0x04010400u)) + bias;
    } else {
        r[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
        r[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
        r[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
        r[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    }
    return half8{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}

__device__ __forceinline__ f32x4 mfma16(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float ldexp2(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }

// The larger of each of the 4 lanes l, l^16, l^32, l^48.
__device__ __forceinline__ float max_groups(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t h0 = h[0], h1 = h[1];  // a bit cast of an element would take the first
    x = fmaxf(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1));
    const uint32_t v = __builtin_bit_cast(uint32_t, x);
    const auto q = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t q0 = q[0], q1 = q[1];
    return fmaxf(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
}

// tanh(x) for |x| < kCapNear, good to 2^-22: its series.
constexpr float kCapNear = 0.35f;
__device__ __forceinline__ float tanh_near(float x) {
    const float y = x * x;
    float p = fmaf(y, -0.008863235529902197f, 0.021869488536155203f);
    p = fmaf(y, p, -0.05396825396825397f);
    p = fmaf(y, p, 0.13333333333333333f);
    p = fmaf(y, p, -0.3333333333333333f);
    return fmaf(x * y, p, x);
}
// cap * log2 e * tanh(x): the series where the exponential's form would cancel.
__device__ __forceinline__ float softcap_log2(float x, float cap_log2e) {
    const float e = __builtin_amdgcn_exp2f(x * 2.8853900817779268f);  // exp(2x)
    const float big = 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
    return cap_log2e * (fabsf(x) < kCapNear ? tanh_near(x) : big);
}

__device__ __forceinline__ i32x4 mfma16(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// A lane's D/4 floats of a query row.
template <int D>
__device__ __forceinline__ void read_query(const float *qp, float (&v)[D / 4]) {
#pragma unroll
    for (int i = 0; i < D / 4; i += 4) {
        const f32x4 x = ld_f32x4(qp + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i + e] = x[e];
    }
}

// A query row's dims grp*KB .. +KB-1 (KB = D/4) as f16 hi + lo pairs of the row
// times 2^ex, the largest of the row in [2^13, 2^14): 22 bits of every value
// that is not 2^-24 of the largest. Lanes l, l^16, l^32, l^48 share a row.
// Returns scale * 2^-ex: 2^-ex by itself is 0 for the smallest rows.
template <int D>
__device__ __forceinline__ float split_query(float scale, const float (&v)[D / 4], half8 (&qh)[D / 32],
                                             half8 (&ql)[D / 32]) {
    constexpr int KB = D / 4;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < KB; ++i) top = fmaxf(top, fabsf(v[i]));
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int ex = 0;
    if (top > 0.0f && top < INFINITY) ex = 14 - __builtin_amdgcn_frexp_expf(top);
#pragma unroll
    for (int i = 0; i < KB; ++i) {
        const float x = ldexp2(v[i], ex);
        const _Float16 hi = (_Float16)x;
        qh[i / 8][i % 8] = hi;
        ql[i / 8][i % 8] = (_Float16)(x - (float)hi);
    }
    return ldexp2(scale, -ex);
}

// The same row as N signed digits of 8 bits, 16 dims to a register quad: the
// row times a factor that takes its largest to 0x7F7F.. (all digits 127),
// rounded to whole numbers; for the int8 matrix cores, whose products with an
// 8-bit K and their sums are exact. Returns scale over the factor (the power of two
// first, so that neither the smallest nor the largest rows leave f32 on the way); a
// row with a NaN or infinity returns NaN.
template <int D, int N>
__device__ __forceinline__ float split_query(float scale, const float (&v)[D / 4], i32x4 (&qd)[N][D / 64]) {
    constexpr int KB = D / 4;
    constexpr float kMost = (float)(N == 2 ? 0x7F7F : 0x7F7F7F);
    float top = 0.0f, bad = 0.0f;
#pragma unroll
    for (int i = 0; i < KB; ++i) {
        top = fmaxf(top, fabsf(v[i]));
        bad += v[i] * 0.0f;
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    bad += __shfl_xor(bad, 16, 64);
    bad += __shfl_xor(bad, 32, 64);
    int ex = 0;
    float mant = 1.0f;  // top = mant * 2^ex
    if (top > 0.0f && top < INFINITY) {
        ex = __builtin_amdgcn_frexp_expf(top);
        mant = __builtin_amdgcn_frexp_mantf(top);
    }
    const float f = kMost / mant;
#pragma unroll
    for (int i = 0; i < KB; i += 4) {
        uint32_t w[N] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int q = (int)rintf(fminf(fmaxf(ldexp2(v[i + e], -ex) * f, -kMost), kMost));
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int d = n + 1 < N ? (int)(int8_t)q : q;
                w[n] |= (uint32_t)(d & 0xFF) << (8 * e);
                q = (q - d) >> 8;
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) qd[n][i / 16][i / 4 % 4] = (int)w[n];
    }
    constexpr int kBits = 8 * N - 1;  // kMost is just below 2^kBits
    return ldexp2(scale, ex - kBits) * (mant * ((float)(1 << kBits) / kMost)) + bad;
}

// The first nv of a lane's 16 tokens of V kept, the bytes of the others (they
// may be NaN codes) zero. u: which 8 of them x holds.
__device__ __forceinline__ u32x2 kv_keep(u32x2 x, int nv, int u) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int k = nv - 8 * u - 4 * e;
        x[e] = k >= 4 ? x[e] : k <= 0 ? 0u : x[e] & (0xFFFFFFFFu >> (32 - 8 * k));
    }
    return x;
}

// A partial state of R query rows: O[R][D] unnormalized, then (M, l)[R].
template <int D>
constexpr int state_floats(int rows) {
    return rows * (D + 2);
}

// The states of one query row, in `n` slots (slot(i) -> its first float), joined
// by a work-group of 256 threads: D/4 threads a state, so that (M, l) and O of
// 1024/D states load at once; each such group of threads joins every 1024/D-th
// state as it comes, then the groups join through LDS. The row's dims 4d .. on
// thread d < D/4.
template <int D, class Slot>
__device__ __forceinline__ f32x4 join_row(int n, int rows, int row, Slot slot) {
    constexpr int L = D / 4, W = 256 / L, U = 4;  // threads of a state, states at once, loads ahead
    __shared__ f32x4 sO[W * L];
    __shared__ float2 sML[W];
    const int d = threadIdx.x % L, k = threadIdx.x / L;
    float M = -INFINITY, l = 0.0f;
    f32x4 o = {};
    for (int i0 = k; i0 < n && k < W; i0 += U * W) {
        float2 ml[U];
        f32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float *s = slot(min(i0 + u * W, n - 1));
            ml[u] = *reinterpret_cast<const float2 *>(s + rows * D + 2 * row);
            x[u] = *reinterpret_cast<const f32x4 *>(s + row * D + 4 * d);
            if (i0 + u * W >= n) ml[u] = make_float2(-INFINITY, 0.0f);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (ml[u].x == -INFINITY && ml[u].y == 0.0f) continue;  // of nothing; scores of NaN have a NaN l
            const float m = fmaxf(M, ml[u].x);
            const Exp2 f(M - m), g(ml[u].x - m);
            M = m;
            l = f.times(l) + g.times(ml[u].y);
            o = o * f.f + x[u] * g.f;
        }
    }
    if (k < W) sO[k * L + d] = o;
    if (k < W && d == 0) sML[k] = make_float2(M, l);
    __syncthreads();
    M = sML[0].x;
#pragma unroll
    for (int i = 1; i < W; ++i) M = fmaxf(M, sML[i].x);
    l = 0.0f;
    o = f32x4{};
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const Exp2 f(sML[i].x == -INFINITY ? -INFINITY : sML[i].x - M);
        l += f.times(sML[i].y);
        o += sO[i * L + d] * f.f;
    }
    return o * (l == 0.0f ? 0.0f : 1.0f / l);
}

// 4 neighbouring values of a result row.
__device__ __forceinline__ void put_out4(const AttnArgs &a, int64_t token, int head_dim0, f32x4 o) {
    const int64_t to = token * a.out_stride + head_dim0;
    if (a.out_f16) {
        typedef _Float16 half4 __attribute__((ext_vector_type(4)));
        const half4 x = {(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
        *reinterpret_cast<u32x2_a1 *>(static_cast<_Float16 *>(a.out) + to) = __builtin_bit_cast(u32x2, x);
    } else {
        *reinterpret_cast<f32x4_a4 *>(static_cast<float *>(a.out) + to) = o;
    }
}

}  // namespace mgq
