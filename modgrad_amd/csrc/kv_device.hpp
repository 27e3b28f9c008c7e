// Device-side helpers of the rotary and key/value-cache kernels (gfx950).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "q4k_device.hpp"

namespace mgq {

// A paged 8-bit cache as the kernels see it. One (page, kv head) block is
// page_tokens * D contiguous bytes: K as [token][dim], V as [dim][token], the
// order in which the matrix cores take each as an operand with the tokens (K:
// rows; V: the summed index) where a lane reads them as one contiguous load.
struct KvView {
    uint8_t *k, *v;
    float *ks, *vs;    // [page][kv head]
    const int *table;  // [sequence][max_pages]
    const int *len;    // [sequence]: tokens with the new ones
    const int *cu;     // [sequence + 1] or null: one new token per sequence
    int64_t page_stride;
    int n_pages, page_shift, hkv, n_seqs, max_pages;
    int n_tokens, max_new;  // rows of q / k / v, most new tokens of a sequence
};

// The new tokens of sequence b: rows t0 .. t0+n-1, at positions pos0 .. ;
// `len` tokens of the cache are behind the table. cu, len and the table are
// device data the host has not seen: rows that fall or do not lie in the call's
// are none (a clamped range could be another sequence's rows too, which both
// would then write), n is clamped to what the launch covers, and pos0 to 2^30
// either way (a sequence holds fewer tokens), so that no index leaves a buffer and
// no position wraps whatever they hold.
struct SeqInfo {
    int t0, n, pos0, len;
};
__host__ __device__ __forceinline__ SeqInfo kv_seq(const KvView &c, int b) {
    SeqInfo s;
    const int len = c.len[b];
    s.t0 = b;
    int end = b + 1;
    if (c.cu) {
        s.t0 = c.cu[b];
        end = c.cu[b + 1];
    }
    int n = s.t0 >= 0 && s.t0 <= end && end <= c.n_tokens ? end - s.t0 : 0;
    const int cap = c.max_pages << c.page_shift;
    constexpr int64_t kFar = INT64_C(1) << 30;
    const int64_t pos = (int64_t)len - n;
    s.pos0 = (int)(pos < -kFar ? -kFar : pos > kFar ? kFar : pos);
    s.len = len < 0 ? 0 : (len < cap ? len : cap);
    s.n = n > c.max_new ? c.max_new : n;
    return s;
}

constexpr int kFmtI8 = 0, kFmtE4M3 = 1;

template <int FMT>
constexpr double kv_most() {
    return FMT == kFmtI8 ? 127.0 : 448.0;
}

// A value in units of its scale -> the 8-bit code: nearest, ties to even,
// saturating, NaN as 0. In 64 bits, so that the code is that of the exact
// quotient wherever a 32-bit one would land on the wrong side of a tie.
template <int FMT>
__device__ __forceinline__ uint32_t kv_code(double x) {
    if (!(x == x)) return 0u;
    const double a = fmin(fabs(x), kv_most<FMT>());
    if constexpr (FMT == kFmtI8) {
        const int q = (int)rint(a);
        return (uint32_t)(x < 0.0 ? -q : q) & 0xFFu;
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, a);
        uint32_t q;
        if (a < 0x1p-6) {
            q = (uint32_t)(int)rint(a * 512.0);  // subnormals are multiples of 2^-9
        } else {
            // 3 of 52 fraction bits stay; the carry of the rounding runs into
            // the exponent, which moves from bias 1023 to bias 7
            const uint64_t r = u + ((1ull << 48) - 1) + ((u >> 49) & 1);
            q = (uint32_t)(r >> 49) - ((1023u - 7u) << 3);
        }
        return q | (x < 0.0 ? 0x80u : 0u);
    }
}

template <int FMT>
__device__ __forceinline__ float kv_value(uint32_t code) {
    if constexpr (FMT == kFmtI8) {
        return (float)(int8_t)code;
    } else {
        const uint32_t e = (code >> 3) & 15u, f = code & 7u;
        const float m = e == 0 ? (float)f * 0x1p-9f
                               : __builtin_bit_cast(float, ((e + 120u) << 23) | (f << 20));
        return (code & 0x80u) ? -m : m;
    }
}

// Rotation of a pair by a table row (cos, sin). The products of two f32 are
// exact in f64, so the sum is rounded once, fused or not.
__device__ __forceinline__ void rope_pair(double &a, double &b, float c, float s) {
    const double x = a, y = b;
    a = x * c - y * s;
    b = x * s + y * c;
}

// A unit of a head's dims as one thread rotates it. Wide units (VEC) are 8
// dims: two quads that hold four pairs (the pairs (i, i + rot/2), or four
// neighbouring pairs), or 8 dims past the rotated ones; narrow ones are one
// pair. Unit u of a head covers dims d0 .. and d1 .. (N/2 each).
template <bool VEC>
struct RopeUnit {
    static constexpr int N = VEC ? 8 : 2;
    int d0, d1;
    bool rot;
    __device__ __forceinline__ RopeUnit(int u, int rot_dim, bool half) {
        constexpr int H = N / 2;
        rot = u * N < rot_dim;
        if (rot && half) {
            d0 = u * H;
            d1 = rot_dim / 2 + u * H;
        } else {
            d0 = u * N;
            d1 = d0 + H;
        }
    }
    __device__ __forceinline__ void load(const float *x, double (&v)[N]) const {
        if constexpr (VEC) {
            const f32x4 a = ld_f32x4(x + d0), b = ld_f32x4(x + d1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = a[i];
                v[4 + i] = b[i];
            }
        } else {
            v[0] = x[d0];
            v[1] = x[d1];
        }
    }
    // row: the position's (cos, sin) pairs
    __device__ __forceinline__ void turn(const float *row, bool half, double (&v)[N]) const {
        if (!rot) return;
        if constexpr (VEC) {
            const int p = half ? d0 : d0 / 2;
            const f32x4 a = ld_f32x4(row + 2 * p), b = ld_f32x4(row + 2 * p + 4);
            if (half) {
                rope_pair(v[0], v[4], a[0], a[1]);
                rope_pair(v[1], v[5], a[2], a[3]);
                rope_pair(v[2], v[6], b[0], b[1]);
                rope_pair(v[3], v[7], b[2], b[3]);
            } else {
                rope_pair(v[0], v[1], a[0], a[1]);
                rope_pair(v[2], v[3], a[2], a[3]);
                rope_pair(v[4], v[5], b[0], b[1]);
                rope_pair(v[6], v[7], b[2], b[3]);
            }
        } else {
            const int p = half ? d0 : d0 / 2;
            rope_pair(v[0], v[1], row[2 * p], row[2 * p + 1]);
        }
    }
    __device__ __forceinline__ void store(float *y, const double (&v)[N]) const {
        if constexpr (VEC) {
            typedef f32x4_a4 V;
            V a, b;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = (float)v[i];
                b[i] = (float)v[4 + i];
            }
            *reinterpret_cast<V *>(y + d0) = a;
            *reinterpret_cast<V *>(y + d1) = b;
        } else {
            y[d0] = (float)v[0];
            y[d1] = (float)v[1];
        }
    }
};

// Whether heads of `dim` with `rot` rotated dims split into wide units.
__host__ __device__ inline bool rope_wide(int dim, int rot) { return rot % 8 == 0 && dim % 8 == 0; }

}  // namespace mgq
