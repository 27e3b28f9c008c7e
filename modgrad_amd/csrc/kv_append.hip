// Appending keys and values to the paged 8-bit cache, the keys rotated on the
// way and the queries with them; and the cache's pages back as f32.
//
// A scale belongs to a (page, kv head), so the tokens a call adds to a page
// are quantized together and, where they are louder than what the page holds,
// the held ones are brought to the new scale: s = max(s_old, f32(amax / M)),
// q -> Q(q * s_old / s), new ones Q(x / s), all in 64 bits (see kv_code).
//
// One work-group has one page of one kv head of K or of V. K's rotated rows stay
// in registers between the largest and the codes where they fit (4 units of 8
// dims a thread: 64 tokens of 128), else are read and turned twice; V's, at most
// 128 x 256 floats, are read twice, the second time from L2. The queries are
// rotated by further work-groups of the same launch. A single token per sequence
// is bound by latency (length -> page -> old scale -> store: 64 sequences, 28 + 2*4
// heads of 128, 4.8 us); a prompt by its floats, mostly the queries' (4096 tokens, 162 MB:
// 31-35 us, 4.9 TB/s). At positions of several axes: 33 single tokens 4.7 us; 3 ragged
// prompts of 3593 tokens together on e4m3 34, 3.6 TB/s (their query work-groups are as many as
// for three prompts of the longest one's 2500, so half of 3282 have nothing to do, and
// positions and table entries are read again for each head).
#include "kv_device.hpp"
#include "kv_launch.hpp"

namespace mgq {

struct AppendGrid {
    int page_blocks;  // most pages of a sequence that the new tokens touch
    int kv_groups;    // work-groups of the K and V part, which come first
    int q_blocks;     // work-groups of a sequence in the query part
};
constexpr int kQueryUnits = 4;

// The largest of a work-group's values, on every thread.
template <int NT>
__device__ __forceinline__ double group_max(double m) {
    __shared__ double part[NT / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmax(m, __shfl_xor(m, o, 64));
    if (NT > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) m = fmax(m, part[w]);
    }
    return m;
}

__device__ __forceinline__ double finite_abs(double v) {
    const double a = fabs(v);
    return a <= 1.7976931348623157e308 ? a : 0.0;  // NaN and inf do not count
}

// x / s for one s > 0 and many x: the product with the reciprocal, corrected by
// its remainder, is the rounded quotient (ties of the code to come among them),
// at a fifth of a division's operations.
struct Divider {
    double s, r;
    __device__ __forceinline__ explicit Divider(float scale) : s(scale), r(1.0 / scale) {}
    __device__ __forceinline__ double operator()(double x) const {
        const double q = x * r;
        return fabs(q) < 1e300 ? fma(fma(-q, s, x), r, q) : q;  // infinities and NaN as they are
    }
};

template <int D, int FMT, bool VEC, int NT, class Rope>
__global__ __launch_bounds__(NT) void kv_append_kernel(KvView c, KvAppend a, Rope rope, AppendGrid gr) {
    const int rot = rope.rot, half = rope.half;
    typedef RopeUnit<VEC> U;
    constexpr int kUnits = D / U::N;
    const int tid = threadIdx.x;
    const int page = 1 << c.page_shift;
    if ((int)blockIdx.x >= gr.kv_groups) {
        // ---- queries: 4 units a thread, their loads side by side
        const int w = blockIdx.x - gr.kv_groups, b = w / gr.q_blocks;
        const SeqInfo s = kv_seq(c, b);
        const unsigned per_token = kUnits * a.hq, units = (unsigned)s.n * per_token;
        const unsigned first = (unsigned)(w % gr.q_blocks) * (kQueryUnits * NT) + tid;
        if (first >= units) return;
        unsigned t[kQueryUnits], r[kQueryUnits];  // token, unit in it
#pragma unroll
        for (int k = 0; k < kQueryUnits; ++k) {
            const unsigned i = min(first + k * NT, units - 1);
            t[k] = i / per_token;
            r[k] = i - t[k] * per_token;
        }
        double v[kQueryUnits][U::N];
#pragma unroll
        for (int k = 0; k < kQueryUnits; ++k)
            U(r[k] % kUnits, rot, half).load(a.q + (s.t0 + (int64_t)t[k]) * a.q_stride + (r[k] / kUnits) * D, v[k]);
#pragma unroll
        for (int k = 0; k < kQueryUnits; ++k)
            rope.turn(U(r[k] % kUnits, rot, half), s.pos0 + (int)t[k], s.t0 + (int64_t)t[k], v[k]);
#pragma unroll
        for (int k = 0; k < kQueryUnits; ++k)
            if (first + k * NT < units)
                U(r[k] % kUnits, rot, half).store(a.q_out + (s.t0 + (int64_t)t[k]) * a.q_out_stride + (r[k] / kUnits) * D, v[k]);
        return;
    }
    // ---- one page of one kv head, K or V
    int w = blockIdx.x;
    const int h = w % c.hkv;
    w /= c.hkv;
    const bool is_v = w & 1;
    w >>= 1;
    const SeqInfo s = kv_seq(c, w / gr.page_blocks);
    const int slot = (max(s.pos0, 0) >> c.page_shift) + w % gr.page_blocks;
    if (slot >= c.max_pages) return;
    const int begin = max(max(s.pos0, 0), slot << c.page_shift);
    const int end = min(s.pos0 + s.n, (slot + 1) << c.page_shift);
    if (begin >= end) return;
    const int n = end - begin, off = begin & (page - 1);
    const float *x = (is_v ? a.v : a.k) + (s.t0 + begin - s.pos0) * a.kv_stride + h * D;

    // K's rotated units tid + e * NT, kBatch of them with their loads side by side:
    // all of the page's, which then stay in registers, or (`once` false) as many as
    // there are, one batch after another
    constexpr int kBatch = VEC ? 4 : NT == 64 ? D / 128 + 1 : 2;
    const int total = n * kUnits;
    const bool once = total <= kBatch * NT;
    double kv[kBatch][U::N];
    const auto load_keys = [&](int i0) {
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int i = min(i0 + e * NT, total - 1);
            U(i % kUnits, rot, half).load(x + (int64_t)(i / kUnits) * a.kv_stride, kv[e]);
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int i = min(i0 + e * NT, total - 1);
            const int p = begin + i / kUnits;
            rope.turn_key(U(i % kUnits, rot, half), p, s.t0 + (int64_t)p - s.pos0, kv[e]);
        }
    };
    const auto each_key = [&](int i0, auto f) {
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int i = i0 + e * NT;
            if (i < total) f(i / kUnits, U(i % kUnits, rot, half), kv[e]);
        }
    };

    // the page's id loads beside the rows
    const int id = c.table[(int64_t)(w / gr.page_blocks) * c.max_pages + slot];
    double m = 0.0;
    if (is_v) {
        constexpr int Q = D / 4, B = 8;
        float top = 0.0f;
        for (int i0 = tid; i0 < n * Q; i0 += B * NT) {
            f32x4 y[B];
#pragma unroll
            for (int e = 0; e < B; ++e) {
                const int i = min(i0 + e * NT, n * Q - 1);
                y[e] = ld_f32x4(x + (int64_t)(i / Q) * a.kv_stride + i % Q * 4);
            }
#pragma unroll
            for (int e = 0; e < B; ++e)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float z = fabsf(y[e][k]);
                    top = z <= 3.4028235e38f && z > top ? z : top;
                }
        }
        m = top;
    } else {
        for (int i0 = tid; i0 < total; i0 += kBatch * NT) {
            load_keys(i0);
            each_key(i0, [&](int, const U &, const double (&v)[U::N]) {
#pragma unroll
                for (int e = 0; e < U::N; ++e) m = fmax(m, finite_abs(v[e]));
            });
        }
    }
    if (id < 0 || id >= c.n_pages) return;
    float *sp = (is_v ? c.vs : c.ks) + (int64_t)id * c.hkv + h;
    uint8_t *blk = (is_v ? c.v : c.k) + id * c.page_stride + (int64_t)h * page * D;
    const float old = off > 0 ? *sp : 0.0f;
    m = group_max<NT>(m);
    const float now = fmaxf(old, (float)(m / kv_most<FMT>()));
    if (tid == 0) *sp = now;  // every thread has `old`: group_max's barrier, or one wavefront
    const Divider div(now);

    if (now > old && off > 0) {  // the held tokens to the new scale
        const double held = old;
        if (is_v) {
            const int tg = (off + 3) / 4;
            for (int i = tid; i < D * tg; i += NT) {
                const int d = i % D, t0 = (i / D) * 4;
                uint8_t *p = blk + (int64_t)d * page + t0;
                const int k = min(4, off - t0);
                for (int e = 0; e < k; ++e) p[e] = (uint8_t)kv_code<FMT>(div((double)kv_value<FMT>(p[e]) * held));
            }
        } else {
            for (int i = tid; i < off * (D / 4); i += NT) {
                uint32_t *p = reinterpret_cast<uint32_t *>(blk) + i;
                const uint32_t q = *p;
                uint32_t r = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    r |= kv_code<FMT>(div((double)kv_value<FMT>((q >> (8 * e)) & 0xFFu) * held)) << (8 * e);
                *p = r;
            }
        }
    }

    const auto code = [&](double v) { return now > 0.0f ? kv_code<FMT>(div(v)) : 0u; };
    if (is_v) {
        // a thread has one dim of up to 16 neighbouring tokens: 16 bytes of the
        // [dim][token] block
        const int g0 = off >> 4, gn = ((off + n - 1) >> 4) - g0 + 1;
        for (int i = tid; i < gn * D; i += NT) {
            const int d = i % D, t0 = (g0 + i / D) * 16 - off;  // first token, counted from `begin`
            uint8_t *p = blk + (int64_t)d * page + off + t0;
            if (t0 >= 0 && t0 + 16 <= n) {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = x[(t0 + e) * a.kv_stride + d];
                u32x4 q;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    q[e] = code(v[4 * e]) | code(v[4 * e + 1]) << 8 | code(v[4 * e + 2]) << 16 | code(v[4 * e + 3]) << 24;
                *reinterpret_cast<u32x4 *>(p) = q;
            } else {
                for (int e = max(0, -t0); e < min(16, n - t0); ++e) p[e] = (uint8_t)code(x[(t0 + e) * a.kv_stride + d]);
            }
        }
    } else {
        for (int i0 = tid; i0 < total; i0 += kBatch * NT) {
            if (!once) load_keys(i0);
            each_key(i0, [&](int t, const U &u, const double (&v)[U::N]) {
                uint8_t *p = blk + (off + t) * D;
                if constexpr (VEC) {
                    *reinterpret_cast<uint32_t *>(p + u.d0) =
                        code(v[0]) | code(v[1]) << 8 | code(v[2]) << 16 | code(v[3]) << 24;
                    *reinterpret_cast<uint32_t *>(p + u.d1) =
                        code(v[4]) | code(v[5]) << 8 | code(v[6]) << 16 | code(v[7]) << 24;
                } else {
                    p[u.d0] = (uint8_t)code(v[0]);
                    p[u.d1] = (uint8_t)code(v[1]);
                }
            });
        }
    }
}

template <int D, int FMT, bool VEC, int NT, class Rope>
static hipError_t append_run(const KvView &c, const Rope &rope, const KvAppend &a, hipStream_t stream) {
    const int page = 1 << c.page_shift;
    AppendGrid g;
    g.page_blocks = (c.max_new + page - 2) / page + 1;
    g.kv_groups = c.n_seqs * g.page_blocks * 2 * c.hkv;
    const int64_t units = (int64_t)c.max_new * a.hq * (D / RopeUnit<VEC>::N);
    g.q_blocks = a.q ? (int)((units + kQueryUnits * NT - 1) / (kQueryUnits * NT)) : 0;
    const int64_t grid = g.kv_groups + (int64_t)c.n_seqs * g.q_blocks;
    kv_append_kernel<D, FMT, VEC, NT, Rope><<<(unsigned)grid, NT, 0, stream>>>(c, a, rope, g);
    return hipGetLastError();
}

template <int D, int FMT, class Rope>
static hipError_t append_dim(const KvView &c, const Rope &rope, const KvAppend &a, hipStream_t stream) {
    // a single token has one pair for each lane; wide units are for rows of work
    if (c.max_new == 1) return append_run<D, FMT, false, 64>(c, rope, a, stream);
    if (rope_wide(D, rope.rot)) return append_run<D, FMT, true, 256>(c, rope, a, stream);
    return append_run<D, FMT, false, 256>(c, rope, a, stream);
}

template <class Rope>
static hipError_t append_any(const KvView &c, int dim, int fmt, const Rope &rope, const KvAppend &a, hipStream_t stream) {
    const bool i8 = fmt == MGQ_KV_I8;
    switch (dim) {
    case 64: return i8 ? append_dim<64, kFmtI8>(c, rope, a, stream) : append_dim<64, kFmtE4M3>(c, rope, a, stream);
    case 96: return i8 ? append_dim<96, kFmtI8>(c, rope, a, stream) : append_dim<96, kFmtE4M3>(c, rope, a, stream);
    case 128: return i8 ? append_dim<128, kFmtI8>(c, rope, a, stream) : append_dim<128, kFmtE4M3>(c, rope, a, stream);
    default: return i8 ? append_dim<256, kFmtI8>(c, rope, a, stream) : append_dim<256, kFmtE4M3>(c, rope, a, stream);
    }
}

hipError_t kv_append_launch(const KvView &c, int dim, int fmt, const mgq_rope *rope, const mgq_rope_axes *axes,
                            const KvAppend &a, hipStream_t stream) {
    if (axes) return append_any(c, dim, fmt, rope_many(*rope, *axes), a, stream);
    // no table: rows are copied, wherever they are
    RopeLine line = {nullptr, 0, 0, 0xFFFFFFFFu};
    if (rope) line = {rope->table, rope->rot_dim, rope->style == MGQ_ROPE_HALF, (unsigned)(rope->n_pos - 1)};
    return append_any(c, dim, fmt, line, a, stream);
}

// Pages of the cache as f32, K and V both [page][kv head][token][dim]. One
// work-group per (page, kv head) and K or V, bound by its stores; V's 16 bytes
// per lane are 16 tokens of one dim, stored with the lanes along the dims.
template <int D, int FMT>
__global__ __launch_bounds__(256) void kv_dequant_kernel(KvView c, const int *__restrict__ pages,
                                                         float *__restrict__ k_out, float *__restrict__ v_out) {
    const int page = 1 << c.page_shift;
    int w = blockIdx.x;
    const bool is_v = w & 1;
    w >>= 1;
    const int h = w % c.hkv, i0 = w / c.hkv;
    float *o = (is_v ? v_out : k_out) + ((int64_t)i0 * c.hkv + h) * page * D;
    const int id = pages[i0];
    if (id < 0 || id >= c.n_pages) {  // names no page
        for (int i = threadIdx.x; i < page * D; i += 256) o[i] = 0.0f;
        return;
    }
    const float s = (is_v ? c.vs : c.ks)[(int64_t)id * c.hkv + h];
    const uint8_t *blk = (is_v ? c.v : c.k) + id * c.page_stride + (int64_t)h * page * D;
    if (is_v) {
        for (int i = threadIdx.x; i < D * (page / 16); i += 256) {
            const int d = i % D, t = (i / D) * 16;
            const u32x4 q = *reinterpret_cast<const u32x4 *>(blk + (int64_t)d * page + t);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[(t + e) * D + d] = kv_value<FMT>((q[e / 4] >> (8 * (e % 4))) & 0xFFu) * s;
        }
    } else {
        for (int i = threadIdx.x; i < page * D / 4; i += 256) {
            const uint32_t q = reinterpret_cast<const uint32_t *>(blk)[i];
            f32x4_a4 r;
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = kv_value<FMT>((q >> (8 * e)) & 0xFFu) * s;
            *reinterpret_cast<f32x4_a4 *>(o + 4 * i) = r;
        }
    }
}

hipError_t kv_dequant_launch(const KvView &c, int dim, int fmt, const int *pages, int n, float *k_out, float *v_out,
                             hipStream_t stream) {
    const unsigned grid = (unsigned)(2 * n * c.hkv);
    const bool i8 = fmt == MGQ_KV_I8;
#define MGQ_KV_DEQUANT(D)                                                                              \
    if (i8) kv_dequant_kernel<D, kFmtI8><<<grid, 256, 0, stream>>>(c, pages, k_out, v_out);            \
    else kv_dequant_kernel<D, kFmtE4M3><<<grid, 256, 0, stream>>>(c, pages, k_out, v_out)
    switch (dim) {
    case 64: MGQ_KV_DEQUANT(64); break;
    case 96: MGQ_KV_DEQUANT(96); break;
    case 128: MGQ_KV_DEQUANT(128); break;
    default: MGQ_KV_DEQUANT(256); break;
    }
#undef MGQ_KV_DEQUANT
    return hipGetLastError();
}

}  // namespace mgq
