// The norms around a block of a decoder layer, with what lies between them:
//
//   z  = x * r(x) * post_w   (post_w null: x),   r(a) = 1 / sqrt(mean(a^2) + eps)
//   h' = h_scale * h + x_scale * gate * z
//   y  = h' * r(h') * norm_w, f32 or f16
//
// in one pass: a row of x and h is read once and stays in registers over both
// sums. The squares are summed in 64 bits (a row of 1e20 has a square that f32 does
// not), each product of factors is taken in 64 bits and rounded once, to h' and to
// y; y is that of the h' that was stored. The conversions and 64-bit operations,
// some 12 a value, take a tenth of the time that its 16 bytes do.
#include "q4k_device.hpp"
#include "q4k_launch.hpp"

namespace mgq {

constexpr int kNormThreads = 256;

// NT threads a row (64: a wavefront each, kNormThreads / 64 rows a work-group), V
// quads of neighbouring values a thread.
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
template <int NT>
__device__ __forceinline__ double row_sum(double v, double *part) {
    v = wave_sum(v);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) v += part[w];
    }
    return v;
}
// 1 / sqrt(s): the instruction's 26 bits and one correction, which is left out where
// it is no number (s infinite or zero).
__device__ __forceinline__ double inv_sqrt(double s) {
    const double r = __builtin_amdgcn_rsq(s), e = fma(-s * r, r, 1.0);
    return fabs(e) < 1.0 ? fma(0.5 * e, r, r) : r;
}

// Quad c of a row of n values; values past the row's end are 0.
__device__ __forceinline__ f32x4 ld_quad(const float *row, int c, int n) {
    if (4 * c + 4 <= n) return ld_f32x4(row + 4 * c);
    f32x4 v = {};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (4 * c + e < n) v[e] = row[4 * c + e];
    return v;
}
__device__ __forceinline__ void st_quad(float *row, int c, int n, const float (&v)[4]) {
    if (4 * c + 4 <= n) {
        *reinterpret_cast<f32x4_a4 *>(row + 4 * c) = f32x4_a4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * c + e < n) row[4 * c + e] = v[e];
    }
}
__device__ __forceinline__ void st_quad(_Float16 *row, int c, int n, const float (&v)[4]) {
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    const half4 x = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    if (4 * c + 4 <= n) {
        *reinterpret_cast<u32x2_a1 *>(row + 4 * c) = __builtin_bit_cast(u32x2, x);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * c + e < n) row[4 * c + e] = x[e];
    }
}

template <int NT, int V>
__global__ __launch_bounds__(NT < kNormThreads ? kNormThreads : NT) void block_norm_kernel(BlockNorm a) {
    constexpr int ROWS = NT < kNormThreads ? kNormThreads / NT : 1;
    // of this row and the one before, which a slower wavefront may still be reading
    __shared__ double part[2][2][NT / 64];
    const int tid = threadIdx.x % NT, n = a.hidden;
    f32x4 pv[V], nv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        pv[i] = a.post_w ? ld_quad(a.post_w, tid + i * NT, n) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
        nv[i] = a.norm_w ? ld_quad(a.norm_w, tid + i * NT, n) : f32x4{};
    }
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
        const float *h = a.h + row * a.h_stride, *x = a.x ? a.x + row * a.x_stride : nullptr;
        const float *gate = a.gate ? a.gate + row * a.gate_stride : nullptr;
        f32x4 xv[V], hv[V], gv[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = tid + i * NT;
            xv[i] = x ? ld_quad(x, c, n) : f32x4{};
            hv[i] = ld_quad(h, c, n);
            gv[i] = gate ? ld_quad(gate, c, n) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
        }
        double r = a.x_scale;
        if (a.post_w) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fma((double)xv[i][e], (double)xv[i][e], s);
            r *= inv_sqrt(row_sum<NT>(s, part[turn][0]) / n + a.eps);
        }
        double s = 0.0;
        float *ho = a.h_out ? a.h_out + row * a.h_out_stride : nullptr;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = tid + i * NT;
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double z = (double)xv[i][e] * r * pv[i][e] * gv[i][e];
                o[e] = (float)(x ? fma((double)a.h_scale, (double)hv[i][e], z) : (double)a.h_scale * hv[i][e]);
                hv[i][e] = o[e];
                s = fma((double)o[e], (double)o[e], s);
            }
            if (ho) st_quad(ho, c, n, o);
        }
        if (a.y) {
            r = inv_sqrt(row_sum<NT>(s, part[turn][1]) / n + a.eps);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = tid + i * NT;
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = (float)((double)hv[i][e] * r * nv[i][e]);
                if (a.y_f16) st_quad(static_cast<_Float16 *>(a.y) + row * a.y_stride, c, n, o);
                else st_quad(static_cast<float *>(a.y) + row * a.y_stride, c, n, o);
            }
        }
        turn ^= 1;
    }
}

// Rows that no work-group's registers hold: each thread goes through its quads three
// times (h' through h_out, or computed again where it is not kept).
constexpr int kLongThreads = 1024;

__global__ __launch_bounds__(kLongThreads) void block_norm_long_kernel(BlockNorm a) {
    constexpr int NT = kLongThreads;
    __shared__ double part[2][2][NT / 64];
    const int tid = threadIdx.x, n = a.hidden, quads = (n + 3) / 4;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float *h = a.h + row * a.h_stride, *x = a.x ? a.x + row * a.x_stride : nullptr;
        const float *gate = a.gate ? a.gate + row * a.gate_stride : nullptr;
        double r = a.x_scale;
        if (a.post_w) {
            double s = 0.0;
#pragma unroll 4
            for (int c = tid; c < quads; c += NT) {
                const f32x4 v = ld_quad(x, c, n);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fma((double)v[e], (double)v[e], s);
            }
            r *= inv_sqrt(row_sum<NT>(s, part[turn][0]) / n + a.eps);
        }
        const auto value = [&](int c, float (&o)[4]) {
            const f32x4 hv = ld_quad(h, c, n);
            if (!x) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = (float)((double)a.h_scale * hv[e]);
                return;
            }
            const f32x4 one = {1.0f, 1.0f, 1.0f, 1.0f}, xv = ld_quad(x, c, n);
            const f32x4 pv = a.post_w ? ld_quad(a.post_w, c, n) : one, gv = gate ? ld_quad(gate, c, n) : one;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double z = (double)xv[e] * r * pv[e] * gv[e];
                o[e] = (float)fma((double)a.h_scale, (double)hv[e], z);
            }
        };
        float *ho = a.h_out ? a.h_out + row * a.h_out_stride : nullptr;
        double s = 0.0;
#pragma unroll 2
        for (int c = tid; c < quads; c += NT) {
            float o[4];
            value(c, o);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fma((double)o[e], (double)o[e], s);
            if (ho) st_quad(ho, c, n, o);
        }
        if (!a.y) {
            turn ^= 1;
            continue;
        }
        const double ry = inv_sqrt(row_sum<NT>(s, part[turn][1]) / n + a.eps);
#pragma unroll 2
        for (int c = tid; c < quads; c += NT) {
            float o[4];
            if (ho) {  // what this thread has stored (h may be h_out)
                const f32x4 v = ld_quad(ho, c, n);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = v[e];
            } else {
                value(c, o);
            }
            const f32x4 nv = ld_quad(a.norm_w, c, n);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (float)((double)o[e] * ry * nv[e]);
            if (a.y_f16) st_quad(static_cast<_Float16 *>(a.y) + row * a.y_stride, c, n, o);
            else st_quad(static_cast<float *>(a.y) + row * a.y_stride, c, n, o);
        }
        turn ^= 1;
    }
}

// Work-groups go through the rows in strides of the grid: 2^20 and 1024 threads are
// within what a launch counts.
static unsigned norm_grid(int64_t groups) { return (unsigned)std::min<int64_t>(groups, 1 << 20); }

template <int NT, int V>
static hipError_t norm_run(const BlockNorm &a, hipStream_t stream) {
    constexpr int ROWS = NT < kNormThreads ? kNormThreads / NT : 1, THREADS = NT * ROWS;
    block_norm_kernel<NT, V><<<norm_grid(((int64_t)a.rows + ROWS - 1) / ROWS), THREADS, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t block_norm_launch(const BlockNorm &a, hipStream_t stream) {
    const int quads = (a.hidden + 3) / 4;
    const bool few = a.rows < 4 * device_cus();
    if (few ? quads <= 64 : quads <= 256) return quads <= 64 ? norm_run<64, 1>(a, stream) : norm_run<64, 4>(a, stream);
    if (few ? quads <= 256 : quads <= 1024) return quads <= 256 ? norm_run<256, 1>(a, stream) : norm_run<256, 4>(a, stream);
    if (quads <= 1024) return norm_run<1024, 1>(a, stream);
    if (quads <= 4096) return norm_run<1024, 4>(a, stream);
    block_norm_long_kernel<<<norm_grid(a.rows), kLongThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace mgq
