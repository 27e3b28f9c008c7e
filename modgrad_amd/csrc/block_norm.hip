// The norms around a block of a decoder layer, with what lies between them:
//
//   z  = x * r(x) * post_w   (post_w null: x),   r(a) = 1 / sqrt(mean(a^2) + eps)
//   h' = h_scale * h + x_scale * gate * z
//   y  = h' * r(h') * norm_w, f32 or f16; of the h' that was stored
//
// in one pass: a row of x and h is read once and stays in registers over both sums. The
// squares are summed in 64 bits (a row of 1e25 has squares that f32 does not), the
// factor r is a mantissa and a power of two, and everything else is f32: with its
// products in 64 bits too, a value took 12 conversions at a quarter of the rate (4096
// rows of 3584, f16 results: 55 us, 46 so).
//
// Many rows are bound by their bytes: 256 threads of 4 quads a row of 3584 (206 MB, 46 us,
// 4.5 TB/s; a copy reaches 5.1), a wavefront a row up to 1024 values (16384 rows of 896:
// 4.8 TB/s). 512 threads of 2 quads: 50 us; registers for 5 or 6 wavefronts a SIMD
// instead of 4: 65 and 104 (spills). Rows that end inside a quad cost more: 4096 of 3585
// values 63 us (2 wavefronts a SIMD), of 12001 256 (36 registers spilled; 12000: 163). Few
// rows are bound by latency: a quad a thread.
#include "q4k_device.hpp"
#include "q4k_launch.hpp"

#include <climits>

namespace mgq {

constexpr int kNormThreads = 256;

template <class T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// The sum of a row's NT threads, on each (64: a wavefront each, kNormThreads / 64 rows a
// work-group).
template <int NT, class T>
__device__ __forceinline__ T row_sum(T v, T *part) {
    v = wave_sum(v);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0;
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
// A factor of any size on f32 values.
struct Factor {
    float m;
    int e;
    __device__ __forceinline__ explicit Factor(double r) : m((float)__builtin_amdgcn_frexp_mant(r)), e(__builtin_amdgcn_frexp_exp(r)) {}
    __device__ __forceinline__ float operator*(float x) const { return __builtin_amdgcn_ldexpf(x, e) * m; }
};

// Quad c of a row of n values; values past the row's end are 0.
__device__ __forceinline__ f32x4 ld_quad(const float *row, int c, int n) {
    if (4 * c + 4 <= n) return ld_f32x4(row + 4 * c);
    f32x4 v = {};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (4 * c + e < n) v[e] = row[4 * c + e];
    return v;
}
__device__ __forceinline__ void st_quad(float *row, int c, int n, f32x4 v) {
    if (4 * c + 4 <= n) {
        *reinterpret_cast<f32x4_a4 *>(row + 4 * c) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * c + e < n) row[4 * c + e] = v[e];
    }
}
__device__ __forceinline__ void st_quad(_Float16 *row, int c, int n, f32x4 v) {
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
// V quads of neighbouring values a thread; TAIL: rows end inside a quad.
template <int NT, int V, bool TAIL>
__global__ __launch_bounds__(NT < kNormThreads ? kNormThreads : NT) void block_norm_kernel(BlockNorm a) {
    constexpr int ROWS = NT < kNormThreads ? kNormThreads / NT : 1;
    // of this row and the one before, which a slower wavefront may still be reading
    __shared__ double part[2][2][NT / 64];
    const int tid = threadIdx.x % NT, n = a.hidden;
    const auto get = [&](const float *row, int i) {
        const int c = tid + i * NT;
        if (TAIL) return ld_quad(row, c, n);
        return 4 * c < n ? ld_f32x4(row + 4 * c) : f32x4{};
    };
    const auto put = [&](auto *row, int i, f32x4 v) {
        const int c = tid + i * NT;
        if (TAIL || 4 * c < n) st_quad(row, c, TAIL ? n : INT_MAX, v);
    };
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
        turn ^= 1;
        const float *h = a.h + row * a.h_stride, *x = a.x ? a.x + row * a.x_stride : nullptr;
        const float *gate = a.gate ? a.gate + row * a.gate_stride : nullptr;
        f32x4 xv[V], hv[V];
#pragma unroll
        for (int i = 0; i < V; ++i) xv[i] = x ? get(x, i) : f32x4{};
#pragma unroll
        for (int i = 0; i < V; ++i) hv[i] = get(h, i);
        // one quad a thread: few rows, whose time is latency, and room for the weights ahead
        // of the sums (37 rows of 896: 3.8 -> 3.3 us)
        f32x4 early[3] = {};
        if constexpr (V == 1) {
            if (a.post_w) early[0] = get(a.post_w, 0);
            if (gate) early[1] = get(gate, 0);
            if (a.y) early[2] = get(a.norm_w, 0);
        }
        if (a.post_w) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fma((double)xv[i][e], (double)xv[i][e], s);
            const Factor r(inv_sqrt(row_sum<NT>(s, part[turn][0]) / n + a.eps));
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const f32x4 w = V == 1 ? early[0] : get(a.post_w, i);
#pragma unroll
                for (int e = 0; e < 4; ++e) xv[i][e] = r * xv[i][e] * w[e];
            }
        }
        if (gate) {
#pragma unroll
            for (int i = 0; i < V; ++i) xv[i] *= V == 1 ? early[1] : get(gate, i);
        }
        double s = 0.0;
        float *ho = a.h_out ? a.h_out + row * a.h_out_stride : nullptr;
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hv[i][e] = a.h_scale * hv[i][e];
                if (x) hv[i][e] = fmaf(xv[i][e], a.x_scale, hv[i][e]);
                s = fma((double)hv[i][e], (double)hv[i][e], s);
            }
            if (ho) put(ho, i, hv[i]);
        }
        if (!a.y) continue;
        const Factor r(inv_sqrt(row_sum<NT>(s, part[turn][1]) / n + a.eps));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const f32x4 w = V == 1 ? early[2] : get(a.norm_w, i);
#pragma unroll
            for (int e = 0; e < 4; ++e) hv[i][e] = r * hv[i][e] * w[e];
            if (a.y_f16) put(static_cast<_Float16 *>(a.y) + row * a.y_stride, i, hv[i]);
            else put(static_cast<float *>(a.y) + row * a.y_stride, i, hv[i]);
        }
    }
}

// Rows that no work-group's registers hold: each thread goes through its own quads three
// times; h' comes back through h_out, or is computed again where it is not kept.
constexpr int kLongThreads = 1024;
__global__ __launch_bounds__(kLongThreads) void block_norm_long_kernel(BlockNorm a) {
    constexpr int NT = kLongThreads;
    __shared__ double part[2][2][NT / 64];
    const int tid = threadIdx.x, n = a.hidden, quads = (n + 3) / 4;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        turn ^= 1;
        const float *h = a.h + row * a.h_stride, *x = a.x ? a.x + row * a.x_stride : nullptr;
        const float *gate = a.gate ? a.gate + row * a.gate_stride : nullptr;
        float *ho = a.h_out ? a.h_out + row * a.h_out_stride : nullptr;
        double mean = 1.0;
        if (a.post_w) {
            double s = 0.0;
#pragma unroll 4
            for (int c = tid; c < quads; c += NT) {
                const f32x4 v = ld_quad(x, c, n);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fma((double)v[e], (double)v[e], s);
            }
            mean = row_sum<NT>(s, part[turn][0]) / n + a.eps;
        }
        const Factor rx(a.post_w ? inv_sqrt(mean) : 1.0);
        const auto value = [&](int c) {
            f32x4 o = a.h_scale * ld_quad(h, c, n);
            if (!x) return o;
            f32x4 z = ld_quad(x, c, n);
            if (a.post_w) {
                const f32x4 w = ld_quad(a.post_w, c, n);
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = rx * z[e] * w[e];
            }
            if (gate) z *= ld_quad(gate, c, n);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(z[e], a.x_scale, o[e]);
            return o;
        };
        double s = 0.0;
#pragma unroll 2
        for (int c = tid; c < quads; c += NT) {
            const f32x4 o = value(c);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fma((double)o[e], (double)o[e], s);
            if (ho) st_quad(ho, c, n, o);
        }
        if (!a.y) continue;
        const Factor r(inv_sqrt(row_sum<NT>(s, part[turn][1]) / n + a.eps));
#pragma unroll 2
        for (int c = tid; c < quads; c += NT) {
            f32x4 o = ho ? ld_quad(ho, c, n) : value(c);
            const f32x4 w = ld_quad(a.norm_w, c, n);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = r * o[e] * w[e];
            if (a.y_f16) st_quad(static_cast<_Float16 *>(a.y) + row * a.y_stride, c, n, o);
            else st_quad(static_cast<float *>(a.y) + row * a.y_stride, c, n, o);
        }
    }
}

// Work-groups go through the rows in strides of the grid: 2^20 and 1024 threads are
// within what a launch counts.
static unsigned norm_grid(int64_t groups) { return (unsigned)std::min<int64_t>(groups, 1 << 20); }

template <int NT, int V>
static hipError_t norm_run(const BlockNorm &a, hipStream_t stream) {
    constexpr int ROWS = NT < kNormThreads ? kNormThreads / NT : 1, THREADS = NT * ROWS;
    const unsigned grid = norm_grid(((int64_t)a.rows + ROWS - 1) / ROWS);
    if (a.hidden % 4) block_norm_kernel<NT, V, true><<<grid, THREADS, 0, stream>>>(a);
    else block_norm_kernel<NT, V, false><<<grid, THREADS, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t block_norm_launch(const BlockNorm &a, hipStream_t stream) {
    const int quads = (a.hidden + 3) / 4;
    const bool few = a.rows < 4 * device_cus();
    if (few ? quads <= 64 : quads <= 256) return quads <= 64 ? norm_run<64, 1>(a, stream) : norm_run<64, 4>(a, stream);
    if (few ? quads <= 256 : quads <= 1024) return quads <= 256 ? norm_run<256, 1>(a, stream) : norm_run<256, 4>(a, stream);
    if (quads <= 1024) return norm_run<1024, 1>(a, stream);
    if (quads <= 2048) return norm_run<1024, 2>(a, stream);
    if (quads <= 4096) return norm_run<1024, 4>(a, stream);
    block_norm_long_kernel<<<norm_grid(a.rows), kLongThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace mgq
