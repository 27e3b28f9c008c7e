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
    int window, sinks;  // sinks: 0 without a window
    float *ws;
    // a prefix that the sequences share: its tiles (0: none), the blocks of kWideRows
    // query rows that go through them, the places that a block has in the row of all
    // tiles (some at its end may be empty), the tiles of a work-group, and its states
    int shared, prefix_blocks, prefix_span, prefix_run;
    // few query rows: blocks of kRows of them, each block's tiles in `prefix_cuts` parts of
    // prefix_run tiles (0: many rows)
    int prefix_cuts;
    int prefix_two;  // whether a run may have tiles of two blocks, and so two states
    float *prefix;
    int row_blocks;  // of kWideRows, of all sequences, that the call's rows can make (no prefix: any number)
};
constexpr int kRows = 16;       // query rows of a work-group's row of tiles
constexpr int kWideRows = 128;  // query rows that share a tile through LDS

// Which tiles a run of query rows goes through, by number: those of the first tokens
// that stay visible, then from the window of the first row on.
struct TileList {
    int head, gap;  // tiles of the first tokens, tiles passed over behind them
    __device__ __forceinline__ int at(int t) const { return t + (t < head ? 0 : gap); }
    // tiles up to position `hi`; one at least, so that a row that sees nothing has its zeros written
    __device__ __forceinline__ int count(int hi) const { return max(max((hi + kTile - 1) / kTile - gap, head), 1); }
};
// Tiles of the prefix that all rows of a sequence see.
__device__ __forceinline__ int shared_tiles(const AttnArgs &a, const SeqInfo &s) {
    return min(a.shared, max(s.pos0 + 1, 0) / kTile);
}
__device__ __forceinline__ TileList tile_list(const AttnArgs &a, const SeqInfo &s, int first_pos) {
    TileList l;
    if (a.shared > 0) {
        l.head = 0;
        l.gap = shared_tiles(a, s);
        return l;
    }
    const int first = (a.window > 0 ? max(first_pos - a.window + 1, 0) : 0) / kTile;
    l.head = min((a.sinks + kTile - 1) / kTile, first);
    l.gap = first - l.head;
    return l;
}
// Which of 16 neighbouring tokens from position `first` on the row at `pos` sees, as
// bits: those up to its own of the nv that exist, in its window or among the first.
__device__ __forceinline__ uint32_t low_bits(int n) { return (1u << min(max(n, 0), 16)) - 1u; }
__device__ __forceinline__ uint32_t seen_tokens(const AttnArgs &a, int pos, int first, int nv) {
    uint32_t m = low_bits(min(pos + 1 - first, nv));
    if (a.window > 0) m &= ~low_bits(pos - a.window + 1 - first) | low_bits(a.sinks - first);
    return m;
}

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
// ... and of that of any call no larger than this one, behind a shared prefix or not.
size_t kv_attn_wide_room(int dim, int group, int hkv, int n_seqs, int n_tokens, int max_new, int64_t cap, bool shared);
// Its launches: row blocks of all kv heads, splits of each, work-groups of the join (0: none)
// and which of the two joins that is.
struct WideGrid {
    int64_t items;
    int splits;
    int64_t join;
    bool few;
};
// Row blocks that the sequences' rows make at most, where their ranges do not overlap: each
// begins at most one that is not full.
inline int64_t most_row_blocks(int group, int n_seqs, int n_tokens, int max_new) {
    const int64_t each = ((int64_t)max_new * group + kWideRows - 1) / kWideRows;
    return std::min(each * n_seqs, (int64_t)n_tokens * group / kWideRows + n_seqs);
}
WideGrid kv_attn_wide_grid(int dim, int hkv, int n_seqs, int max_new, int64_t cap, const AttnArgs &a);
// All query rows over the tiles of a prefix that they share, and how many of its
// work-groups are resident at once.
int kv_attn_prefix_slots(int dim, int fmt, bool out_f16);
hipError_t kv_attn_prefix_launch(const KvView &c, int dim, int fmt, const AttnArgs &a, hipStream_t stream);

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
    // q + 0x80 in every digit's place has the digits, each plus 128, as its bytes: they
    // are brought together by bytes and lose the 128 by their sign bit
    constexpr int kBias = N == 2 ? 0x8080 : 0x808080;
#pragma unroll
    for (int i = 0; i < KB; i += 4) {
        uint32_t q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            q[e] = (uint32_t)((int)rintf(fminf(fmaxf(ldexp2(v[i + e], -ex) * f, -kMost), kMost)) + kBias);
        // bytes 0 and 1 of two values each, then of four; perm's bytes 0 to 3 are of its
        // second operand, 4 to 7 of the first
        const uint32_t a = __builtin_amdgcn_perm(q[1], q[0], 0x05010400u), b = __builtin_amdgcn_perm(q[3], q[2], 0x05010400u);
        qd[0][i / 16][i / 4 % 4] = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
        qd[1][i / 16][i / 4 % 4] = (int)(__builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u);
        if constexpr (N == 3) {
            const uint32_t x = __builtin_amdgcn_perm(q[1], q[0], 0x0C0C0602u), y = __builtin_amdgcn_perm(q[3], q[2], 0x0C0C0602u);
            qd[2][i / 16][i / 4 % 4] = (int)(__builtin_amdgcn_perm(y, x, 0x05040100u) ^ 0x80808080u);
        }
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

// Where a query row's partial state lies.
struct RowState {
    const float *o, *ml;
};
template <int D>
__device__ __forceinline__ RowState row_state(const float *state, int rows, int row) {
    return {state + row * D, state + rows * D + 2 * row};
}
// A shared prefix's states. Many rows: run r of a kv head has state 2r for a row block
// that an earlier run begins, 2r + 1 for one that it begins, and state r where runs are
// parts of one block. Few: every part has one.
inline int64_t prefix_runs(const AttnArgs &a) {
    return ((int64_t)a.prefix_blocks * a.prefix_span + a.prefix_run - 1) / a.prefix_run;
}
template <int D>
__device__ __forceinline__ float *prefix_slot(const KvView &c, const AttnArgs &a, int h, int run, bool begins) {
    return a.prefix + ((a.prefix_two ? 2 * (int64_t)run + begins : run) * c.hkv + h) * state_floats<D>(kWideRows);
}
template <int D>
__device__ __forceinline__ float *prefix_part(const KvView &c, const AttnArgs &a, int h, int block, int k) {
    return a.prefix + (((int64_t)block * a.prefix_cuts + k) * c.hkv + h) * state_floats<D>(kRows);
}
// Row `row` of all the call's query rows of a kv head: the states that its sequence's
// share of the prefix is in.
struct PrefixParts {
    int first, n;  // many rows: the first run
    int64_t row;
    template <int D>
    __device__ __forceinline__ RowState state(const KvView &c, const AttnArgs &a, int h, int i) const {
        if (a.prefix_cuts > 0)
            return row_state<D>(prefix_part<D>(c, a, h, (int)(row / kRows), i), kRows, (int)(row % kRows));
        return row_state<D>(prefix_slot<D>(c, a, h, first + i, i == 0), kWideRows, (int)(row % kWideRows));
    }
};
__device__ __forceinline__ PrefixParts prefix_parts(const AttnArgs &a, const SeqInfo &s, int64_t row) {
    PrefixParts p = {0, 0, row};
    const int tiles = a.shared > 0 ? shared_tiles(a, s) : 0;
    if (tiles > 0) {
        const int64_t at = a.prefix_cuts > 0 ? 0 : row / kWideRows * a.prefix_span;
        p.first = (int)(at / a.prefix_run);
        p.n = (int)((at + tiles - 1) / a.prefix_run) - p.first + 1;
    }
    return p;
}
// What tokens t0 .. t1-1 of the call, whichever sequence's they are, see of the prefix:
// lim gets the tiles of each (0: a row of no sequence), for a work-group of `threads`.
// The pages are those of the sequence that sees most (the first such), which the others'
// lists begin with: `best` has its tiles, and its number's complement.
__device__ __forceinline__ void prefix_limits(const KvView &c, const AttnArgs &a, int t0, int t1, int threads, int *lim,
                                              unsigned long long &best) {
    if (threadIdx.x == 0) best = 0;
    for (int i = threadIdx.x; i < t1 - t0; i += threads) lim[i] = 0;
    __syncthreads();
    // without row starts a token is its own sequence's
    for (int i = threadIdx.x + (c.cu ? 0 : t0); i < (c.cu ? c.n_seqs : t1); i += threads) {
        const SeqInfo s = kv_seq(c, i);
        const int lo = max(s.t0, t0), hi = min(s.t0 + s.n, t1), n = shared_tiles(a, s);
        for (int t = lo; t < hi; ++t) atomicMax(&lim[t - t0], n);
        if (lo < hi) atomicMax(&best, (unsigned long long)n << 32 | (0xFFFFFFFFu - (unsigned)i));
    }
    __syncthreads();
}

// The states of one query row, `n` of them (slot(i) -> the i-th), joined by a
// work-group of 256 threads: D/4 threads a state, so that (M, l) and O of
// 1024/D states load at once; each such group of threads joins every 1024/D-th
// state as it comes, then the groups join through LDS. The row's dims 4d .. on
// thread d < D/4.
template <int D, class Slot>
__device__ __forceinline__ f32x4 join_row(int n, Slot slot) {
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
            const RowState s = slot(min(i0 + u * W, n - 1));
            ml[u] = *reinterpret_cast<const float2 *>(s.ml);
            x[u] = *reinterpret_cast<const f32x4 *>(s.o + 4 * d);
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
