// Rotary positions: the table of cosines and sines, and its application.
//
// Table: entry (p, i) is mscale * (cos, sin)(p * t_i) with the frequencies t_i
// of mgq_rope_scaling. p * t_i reaches 1e5 radians, where f32 has no correct
// digit left after the point, so the angles are 64-bit and each entry is
// rounded once. A 64-bit sine costs ~150 operations, a table entry is 8 bytes:
// the work-group takes one sine and cosine per pair and run of J positions
// and turns them on by the angle addition (4 fused operations a step; 32 steps
// add < 1e-14), which leaves the kernel bound by its stores: 131072 positions of
// 128 dims, 67 MB, 13 us (5.2 TB/s; filling them with one value takes 11).
#include "kv_device.hpp"
#include "kv_launch.hpp"

namespace mgq {

struct RopeFreq {
    double base, freq_scale, ext_factor, lo, hi, mscale;
    const float *factors;
};

__device__ __forceinline__ double rope_freq(const RopeFreq &f, int i, int rot_dim) {
    double t = pow(f.base, -2.0 * i / rot_dim);
    if (f.factors) t /= (double)f.factors[i];
    double s = t * f.freq_scale;
    if (f.ext_factor != 0.0) {
        const double r = fmin(fmax((i - f.lo) / fmax(f.hi - f.lo, 0.001), 0.0), 1.0);
        const double keep = f.ext_factor * (1.0 - r);
        s = s * (1.0 - keep) + t * keep;
    }
    return s;
}

constexpr int kTableRun = 32;  // most positions per sine

__global__ __launch_bounds__(256) void rope_table_kernel(float *__restrict__ out, int n_pos, int first, int rot_dim,
                                                         int run, RopeFreq f) {
    __shared__ double th[256], co[256], si[256];
    const int pairs = rot_dim / 2;
    if ((int)threadIdx.x < pairs) {
        const double t = rope_freq(f, threadIdx.x, rot_dim);
        th[threadIdx.x] = t;
        sincos(t, &si[threadIdx.x], &co[threadIdx.x]);
    }
    __syncthreads();
    const int groups = 256 / pairs;  // runs of positions this work-group writes
    const int g = threadIdx.x / pairs, i = threadIdx.x % pairs;
    if (g >= groups) return;
    const int64_t p0 = ((int64_t)blockIdx.x * groups + g) * run;
    if (p0 >= n_pos) return;
    const int n = (int)(n_pos - p0 < run ? n_pos - p0 : run);
    double c, s;
    sincos((double)(first + p0) * th[i], &s, &c);
    const double c1 = co[i], s1 = si[i];
    float *o = out + 2 * (p0 * pairs + i);
    for (int j = 0; j < n; ++j) {
        *reinterpret_cast<float2 *>(o) = make_float2((float)(f.mscale * c), (float)(f.mscale * s));
        const double x = c * c1 - s * s1;
        s = c * s1 + s * c1;
        c = x;
        o += 2 * pairs;
    }
}

hipError_t rope_table_launch(float *table, int n_pos, int first, int rot_dim, const mgq_rope_scaling &s,
                             hipStream_t stream) {
    RopeFreq f;
    f.base = s.base;
    f.freq_scale = s.freq_scale;
    f.ext_factor = s.ext_factor;
    f.factors = s.factors;
    f.mscale = s.attn_factor;
    f.lo = f.hi = 0.0;
    if (s.ext_factor != 0.0) {
        const auto dim = [&](double turns) {
            return rot_dim * std::log(s.orig_ctx / (turns * 6.283185307179586)) / (2.0 * std::log(s.base));
        };
        f.lo = std::max(0.0, std::floor(dim(s.beta_fast)));
        f.hi = std::min(rot_dim - 1.0, std::ceil(dim(s.beta_slow)));
        f.mscale *= 1.0 + 0.1 * std::log(1.0 / s.freq_scale);
    }
    const int groups = 256 / (rot_dim / 2);
    // the longest run that still leaves two work-groups a CU
    int run = kTableRun;
    while (run > 4 && (int64_t)n_pos < (int64_t)run * groups * 2 * device_cus()) run /= 2;
    const int64_t per = (int64_t)run * groups;
    rope_table_kernel<<<(unsigned)((n_pos + per - 1) / per), 256, 0, stream>>>(table, n_pos, first, rot_dim, run, f);
    return hipGetLastError();
}

// y = x with the first rot_dim dims of each head turned by the table row of the
// token's position. Bound by x and y: one thread per unit of dims, a token's
// heads next to one another, so the row (rot * 4 bytes) comes from the cache
// for all heads but the first. 4096 tokens of 28 heads of 128, 118 MB: 24 us from
// memory (4.9 TB/s, a large copy's rate), 19 where the Infinity Cache holds them (a
// copy of them 17).
template <bool VEC>
__global__ __launch_bounds__(256) void rope_kernel(const float *x, float *y, const int *__restrict__ pos,
                                                   const float *__restrict__ table, int n_pos, int rot_dim, int half,
                                                   int n_tokens, int heads, int dim, int64_t x_stride,
                                                   int64_t y_stride) {
    typedef RopeUnit<VEC> U;
    const unsigned per_head = dim / U::N, per_token = per_head * heads;
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (uint64_t)per_token * n_tokens) return;
    const unsigned t = (unsigned)(i / per_token), r = (unsigned)(i % per_token), h = r / per_head;
    const U u(r % per_head, rot_dim, half);
    double v[U::N];
    u.load(x + t * x_stride + (int64_t)h * dim, v);
    const int p = pos[t];
    if (p >= 0 && p < n_pos) {
        u.turn(table + (int64_t)p * rot_dim, half, v);
    } else {
#pragma unroll
        for (int e = 0; e < U::N; ++e) v[e] = __builtin_nan("");
    }
    u.store(y + t * y_stride + (int64_t)h * dim, v);
}

hipError_t rope_launch(const float *x, float *y, const int *pos, const mgq_rope &r, int n_tokens, int heads, int dim,
                       int64_t x_stride, int64_t y_stride, hipStream_t stream) {
    const bool vec = rope_wide(dim, r.rot_dim);
    const uint64_t units = (uint64_t)n_tokens * heads * (dim / (vec ? 8 : 2));
    const unsigned grid = (unsigned)((units + 255) / 256);
    const int half = r.style == MGQ_ROPE_HALF;
    if (vec)
        rope_kernel<true><<<grid, 256, 0, stream>>>(x, y, pos, r.table, r.n_pos, r.rot_dim, half, n_tokens, heads, dim,
                                                    x_stride, y_stride);
    else
        rope_kernel<false><<<grid, 256, 0, stream>>>(x, y, pos, r.table, r.n_pos, r.rot_dim, half, n_tokens, heads,
                                                     dim, x_stride, y_stride);
    return hipGetLastError();
}

}  // namespace mgq
