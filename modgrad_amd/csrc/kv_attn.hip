// Attention of the new tokens' queries over the paged 8-bit cache.
//
//   s_j = scale * q . k_j (or softcap * tanh(s_j / softcap)),
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j), j <= pos, j > pos - window
//
// k_j = ks[page] * K8_j, v_j = vs[page] * V8_j. The 8-bit values of either
// format are exact in f16, so both products run on the f16 matrix cores with
// f32 accumulation (v_mfma_f32_16x16x32_f16), and what has more than 11 bits,
// the queries and the probabilities, goes in as two halves (hi + lo, 22 bits):
// results stay within f32's own rounding of the sums.
//
// Operands. The product of a tile of 64 tokens is taken as S^T = K Q^T: 4
// blocks of 16 tokens (matrix rows) against 16 query rows (columns), so that a
// lane's 16 scores are all of ONE query row (column lane % 16) and of 16
// NEIGHBOURING tokens (16 * (lane / 16) + 0..15; block t's row 4j + i is token
// 16j + 4t + i). They are the B operand of O^T = V^T P^T as they stand: no
// score ever moves between lanes. 16 neighbouring tokens lie in one page
// (pages are 16 tokens or more), so a lane needs one K and one V scale a tile.
// V^T's operand is 16 tokens of one dim, 16 contiguous bytes of the
// [dim][token] block; K's is D/4 contiguous bytes of a token (the order of the
// summed dims is free, so lane group j takes bytes j*D/4 ..). Every operand
// byte goes from memory to its lane's registers by 8- and 16-byte loads,
// without shared memory.
//
// Softmax in base 2 with V's scale in the exponent: t_j = s_j log2 e +
// log2(vs), M the running maximum of t, w_j = 2^(t_j - M + 14) = p_j * vs *
// const, O += w_j V8_j, l += w_j / vs. So w_j <= 2^14 whatever the scales are:
// its f16 hi + lo pair keeps 22 bits down to 2^-24 of the largest. M, l and O
// are f32.
//
// Split. All (sequence, kv head, 16 query rows) rows of tiles laid end to end
// are cut into equal runs, one for each work-group, so ragged batches and one
// long sequence balance alike. The 4 wavefronts of a work-group take tiles in
// turn, each with its own softmax state, joined through LDS at the end of a
// row; a row that a cut goes through leaves partial states in the workspace,
// which kv_attn_join_kernel joins.
#include "kv_attn.hpp"

namespace mgq {

constexpr int kRows = 16;       // query rows of a work-group's row of tiles
constexpr int kAttnGroups = 512;  // work-groups: two per CU
constexpr int kMinTiles = 4;    // least tiles of a run: one for each wavefront

// A row's tiles: rows of (sequence, kv head, row block), kv head and row block
// within the sequence.
struct AttnSeq {
    SeqInfo s;
    int tile0, tiles, blocks;  // first tile, tiles of a row, row blocks
};
__device__ __forceinline__ AttnSeq attn_seq(const KvView &c, const AttnArgs &a, int b) {
    AttnSeq r;
    r.s = kv_seq(c, b);
    // tiles that some row sees: from the first one's window to the length
    const int lo = a.window > 0 ? max(r.s.pos0 - a.window + 1, 0) : 0;
    r.tile0 = lo / kTile;
    const int hi = min(r.s.len, max(r.s.pos0 + r.s.n, 0));
    // at least one: a row that sees nothing has its zeros written
    r.tiles = max((hi + kTile - 1) / kTile - r.tile0, 1);
    r.blocks = (r.s.n * a.group + kRows - 1) / kRows;
    return r;
}
__device__ __forceinline__ int attn_units(const KvView &c, const AttnArgs &a, int b) {
    const AttnSeq r = attn_seq(c, a, b);
    return r.tiles * r.blocks * c.hkv;
}

// Sum of v over the work-group (256 threads) and the sum over lower threads.
__device__ __forceinline__ int group_scan(int v, int *part, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(s, o, 64);
        if (lane >= o) s += t;
    }
    if (lane == 63) part[w] = s;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int k = 0; k < 4; ++k) {
        if (k < w) before += part[k];
        total += part[k];
    }
    __syncthreads();
    return before + s - v;
}

// All units, and where unit `at(total)` lies: its sequence and that one's first
// unit. One pass over the sequences where they are no more than the threads.
struct AttnPlace {
    int total, b, base;
};
template <class At>
__device__ __forceinline__ AttnPlace attn_place(const KvView &c, const AttnArgs &a, int *part, int *found, At at) {
    AttnPlace p = {0, 0, 0};
    if (c.n_seqs == 1) {
        p.total = attn_units(c, a, 0);
        return p;
    }
    if (c.n_seqs > 256)
        for (int b0 = 0; b0 < c.n_seqs; b0 += 256) {
            int t;
            group_scan(b0 + (int)threadIdx.x < c.n_seqs ? attn_units(c, a, b0 + threadIdx.x) : 0, part, t);
            p.total += t;
        }
    int before = 0;
    for (int b0 = 0; b0 < c.n_seqs; b0 += 256) {
        const int i = b0 + threadIdx.x;
        const int u = i < c.n_seqs ? attn_units(c, a, i) : 0;
        int t;
        const int start = before + group_scan(u, part, t);
        before += t;
        if (c.n_seqs <= 256) p.total = t;
        const int x = at(p.total);
        if (x >= start && x < start + u) {
            found[0] = i;
            found[1] = start;
        }
    }
    __syncthreads();
    p.b = found[0];
    p.base = found[1];
    return p;
}
__device__ __forceinline__ int attn_run(int total, int groups) {
    return max((total + groups - 1) / groups, kMinTiles);
}

// Workspace of run w: slot 0 for a row begun by an earlier run, slot 1 for one
// that this run begins.
template <int D, int FMT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv_attn_kernel(KvView c, AttnArgs a) {
    constexpr int KB = D / 4;    // bytes of a token that a lane group has
    constexpr int KS = D / 32;   // summed steps of S
    constexpr int DB = D / 16;   // blocks of 16 dims of O
    constexpr int OP = D + 4;    // LDS row of O
    __shared__ float sO[4 * kRows * OP];
    __shared__ float sM[4][kRows], sL[4][kRows];
    __shared__ int part[4], found[2];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 15, grp = lane >> 4;
    const int page = 1 << c.page_shift;

    const AttnPlace place = attn_place(
        c, a, part, found, [&](int total) { return (int)blockIdx.x * attn_run(total, gridDim.x); });
    const int run = attn_run(place.total, gridDim.x);
    int at = blockIdx.x * run;
    const int stop = min(at + run, place.total);
    if (at >= stop) return;
    int b = place.b, base = place.base;
    AttnSeq q = attn_seq(c, a, b);

    while (at < stop) {
        while (at - base >= q.tiles * q.blocks * c.hkv) {  // the next sequence with rows
            base += q.tiles * q.blocks * c.hkv;
            q = attn_seq(c, a, ++b);
        }
        const int row = (at - base) / q.tiles, t0 = (at - base) % q.tiles;
        const int t1 = min(q.tiles, t0 + stop - at);
        at += t1 - t0;
        const int h = row % c.hkv, r0 = (row / c.hkv) * kRows;  // kv head, first query row of the block
        const int rows = q.s.n * a.group;

        // ---- this lane's query row, as hi + lo halves of a normalized row
        const int r = r0 + col;
        const bool live = r < rows;
        const int tq = live ? r / a.group : 0, hd = live ? r % a.group : 0;
        const int pos = live ? q.s.pos0 + tq : -1;
        half8 qh[KS], ql[KS];
        float qv[KB];
        read_query<D>(a.q + (int64_t)(q.s.t0 + tq) * a.q_stride + (h * a.group + hd) * D + grp * KB, qv);
        const float kscale = a.scale * split_query<D>(qv, qh, ql);

        f32x4 O[DB] = {};
        float M = -INFINITY, l = 0.0f;

        const int tile_end = q.tile0 + t1;
        const int kgrp = col >> 2;  // the 16 tokens that this lane's K rows are of
        u32x4 vreg[DB];
        uint32_t kreg[4][KB / 4];
        float ksv, vsv;
        int nv;  // of this lane group's 16 tokens, those that exist
        const int *tab = c.table + (int64_t)b * c.max_pages;
        const auto fetch = [&](int tile) {
            // a page that the table does not name, or past the length, is read
            // as page 0 and counts as no tokens
            const int pk = tile * kTile + 16 * kgrp, pv = tile * kTile + 16 * grp;
            int ik = pk < q.s.len ? tab[pk >> c.page_shift] : -1;
            int iv = pv < q.s.len ? tab[pv >> c.page_shift] : -1;
            const bool okv = iv >= 0 && iv < c.n_pages;
            if (ik < 0 || ik >= c.n_pages) ik = 0;
            if (!okv) iv = 0;
            nv = okv ? min(q.s.len - pv, 16) : 0;
            ksv = c.ks[(int64_t)iv * c.hkv + h];
            vsv = c.vs[(int64_t)iv * c.hkv + h];
            const uint8_t *kp = c.k + ik * c.page_stride + ((int64_t)h * page + (pk & (page - 1)) + (col & 3)) * D + grp * KB;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < KB / 8; ++i) {
                    const u32x2 x = *reinterpret_cast<const u32x2 *>(kp + 4 * t * D + 8 * i);
                    kreg[t][2 * i] = x[0];
                    kreg[t][2 * i + 1] = x[1];
                }
            const uint8_t *vp = c.v + iv * c.page_stride + ((int64_t)h * D + col) * page + (pv & (page - 1));
#pragma unroll
            for (int d = 0; d < DB; ++d) vreg[d] = *reinterpret_cast<const u32x4 *>(vp + (int64_t)16 * d * page);
        };

        for (int tile = q.tile0 + t0 + wave; tile < tile_end; tile += 4) {
            fetch(tile);
            f32x4 S[4] = {};
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const half8 x = kv_half8<FMT>(kreg[t][2 * k], kreg[t][2 * k + 1]);
                    S[t] = mfma16(x, qh[k], S[t]);
                    S[t] = mfma16(x, ql[k], S[t]);
                }
            // a page of zeros has scale 0: its tokens still count in l
            const float vs = fmaxf(vsv, kLeastScale);
            const float lv = __log2f(vs), ks = kscale * ksv;
            const int first = tile * kTile + 16 * grp;
            const int see = min(pos + 1 - first, nv);  // tokens of the 16 up to the row's own
            const int skip = a.window > 0 ? pos - a.window + 1 - first : 0;
            float top = M;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float s = S[t][i] * ks;
                    if (a.softcap > 0.0f) s = softcap_log2(s, a.softcap);
                    s += lv;
                    const int e = 4 * t + i;
                    s = (e < see && e >= skip) ? s : -INFINITY;
                    S[t][i] = s;
                    top = fmaxf(top, s);
                }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float ref = top == -INFINITY ? 0.0f : top - kTop;
            const float fac = M == -INFINITY ? 0.0f : exp2f(M - top);
            M = top;
            float sum = 0.0f;
            half8 ph[2], pl[2];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = exp2f(S[t][i] - ref);
                    sum += w;
                    const _Float16 hi = (_Float16)w;
                    ph[t / 2][4 * (t % 2) + i] = hi;
                    pl[t / 2][4 * (t % 2) + i] = (_Float16)(w - (float)hi);
                }
            l = l * fac + sum / vs;
#pragma unroll
            for (int d = 0; d < DB; ++d) O[d] *= fac;
            if (nv < 16) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const u32x2 x = kv_keep(u32x2{vreg[d][2 * u], vreg[d][2 * u + 1]}, nv, u);
                        vreg[d][2 * u] = x[0];
                        vreg[d][2 * u + 1] = x[1];
                    }
            }
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const half8 x = kv_half8<FMT>(vreg[d][2 * u], vreg[d][2 * u + 1]);
                    O[d] = mfma16(x, ph[u], O[d]);
                    O[d] = mfma16(x, pl[u], O[d]);
                }
        }

        // ---- the 4 wavefronts' states into one
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        __syncthreads();
        if (grp == 0) sM[wave][col] = M;
        __syncthreads();
        const float all = fmaxf(fmaxf(sM[0][col], sM[1][col]), fmaxf(sM[2][col], sM[3][col]));
        const float fac = M == -INFINITY ? 0.0f : exp2f(M - all);
        if (grp == 0) sL[wave][col] = l * fac;
#pragma unroll
        for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4 *>(&sO[(wave * kRows + col) * OP + 16 * d + 4 * grp]) = O[d] * fac;
        __syncthreads();
        const bool whole = t0 == 0 && t1 == q.tiles;
        float *slot = a.ws + ((int64_t)blockIdx.x * 2 + (t0 == 0)) * state_floats<D>(kRows);
        for (int i = tid; i < kRows * D; i += 256) {
            const int rr = i / D, d = i % D;
            if (r0 + rr >= rows) break;
            float o = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) o += sO[(w * kRows + rr) * OP + d];
            const float s = (sL[0][rr] + sL[1][rr]) + (sL[2][rr] + sL[3][rr]);
            if (whole) {
                put_out(a, q.s.t0 + (r0 + rr) / a.group, (h * a.group + (r0 + rr) % a.group) * D + d,
                        s == 0.0f ? 0.0f : o / s);
            } else {
                slot[i] = o;
                if (d == 0) {
                    slot[kRows * D + 2 * rr] = fmaxf(fmaxf(sM[0][rr], sM[1][rr]), fmaxf(sM[2][rr], sM[3][rr]));
                    slot[kRows * D + 2 * rr + 1] = s;
                }
            }
        }
        __syncthreads();
    }
}

// Joins the partial states of query rows that a cut went through: one
// work-group per (sequence, row block, kv head, query row).
template <int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvView c, AttnArgs a, int groups, int max_blocks,
                                                           int block_rows) {
    __shared__ int part[4], found[2];
    __shared__ float f[kMostStates], red[8 + 256];
    int w = blockIdx.x;
    const int rr = w % block_rows;
    w /= block_rows;
    const int h = w % c.hkv;
    w /= c.hkv;
    const int blk = w % max_blocks, b = w / max_blocks;
    const AttnSeq q = attn_seq(c, a, b);
    const int r = blk * kRows + rr;
    if (blk >= q.blocks || r >= q.s.n * a.group) return;
    int total, base = (blk * c.hkv + h) * q.tiles;
    if (c.n_seqs == 1) {
        total = q.tiles * q.blocks * c.hkv;
    } else {
        total = 0;
        for (int b0 = 0; b0 < c.n_seqs; b0 += 256) {
            const int i = b0 + threadIdx.x;
            int t;
            const int before = total + group_scan(i < c.n_seqs ? attn_units(c, a, i) : 0, part, t);
            if (i == b) found[0] = before;
            total += t;
        }
        __syncthreads();
        base += found[0];
    }
    const int run = attn_run(total, groups);
    const int g0 = base / run, g1 = (base + q.tiles - 1) / run;
    if (g0 == g1) return;  // one run had the whole row and has written it
    const auto slot = [&](int i) {
        return a.ws + ((int64_t)(g0 + i) * 2 + (i == 0)) * state_floats<D>(kRows);
    };
    const float o = join_row<D>(g1 - g0 + 1, kRows, rr, slot, f, red);
    if ((int)threadIdx.x < D)
        put_out(a, q.s.t0 + r / a.group, (h * a.group + r % a.group) * D + threadIdx.x, o);
}

// Rows of a kv head above which kv_attn_wide.hip takes the call.
constexpr int kNarrowRows = 16;

size_t kv_attn_workspace(int dim, int hq, int hkv, int n_seqs, int max_new, int64_t capacity) {
    const size_t narrow = (size_t)kAttnGroups * 2 * kRows * (dim + 2) * sizeof(float);
    if (max_new * (hq / hkv) <= kNarrowRows) return narrow;
    return std::max<size_t>(16, kv_attn_wide_workspace(dim, hq / hkv, hkv, n_seqs, max_new, capacity));
}

template <int D, int FMT>
static hipError_t attn_run_dim(const KvView &c, const AttnArgs &a, hipStream_t stream) {
    const int max_blocks = (c.max_new * a.group + kRows - 1) / kRows;
    const int64_t cap = (int64_t)c.max_pages << c.page_shift;
    const int64_t most = (int64_t)c.n_seqs * c.hkv * max_blocks * ((cap + kTile - 1) / kTile);
    const int groups = (int)std::min<int64_t>(kAttnGroups, (most + kMinTiles - 1) / kMinTiles);
    kv_attn_kernel<D, FMT><<<(unsigned)groups, 256, 0, stream>>>(c, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || groups == 1) return e;
    const int block_rows = std::min(kRows, c.max_new * a.group);
    kv_attn_join_kernel<D><<<(unsigned)(c.n_seqs * max_blocks * c.hkv * block_rows), 256, 0, stream>>>(
        c, a, groups, max_blocks, block_rows);
    return hipGetLastError();
}

hipError_t kv_attn_launch(const KvView &c, int dim, int fmt, const KvAttn &x, hipStream_t stream) {
    AttnArgs a;
    a.q = x.q;
    a.out = x.out;
    a.q_stride = x.q_stride;
    a.out_stride = x.out_stride;
    a.group = x.hq / c.hkv;
    a.out_f16 = x.out_f16;
    a.scale = x.softcap > 0.0f ? x.scale / x.softcap : x.scale * 1.4426950408889634f;
    a.softcap = x.softcap * 1.4426950408889634f;
    a.window = x.window;
    a.ws = x.ws;
    if (c.max_new * a.group > kNarrowRows) return kv_attn_wide_launch(c, dim, fmt, a, stream);
    const bool i8 = fmt == MGQ_KV_I8;
    switch (dim) {
    case 64: return i8 ? attn_run_dim<64, kFmtI8>(c, a, stream) : attn_run_dim<64, kFmtE4M3>(c, a, stream);
    case 96: return i8 ? attn_run_dim<96, kFmtI8>(c, a, stream) : attn_run_dim<96, kFmtE4M3>(c, a, stream);
    case 128: return i8 ? attn_run_dim<128, kFmtI8>(c, a, stream) : attn_run_dim<128, kFmtE4M3>(c, a, stream);
    default: return i8 ? attn_run_dim<256, kFmtI8>(c, a, stream) : attn_run_dim<256, kFmtE4M3>(c, a, stream);
    }
}

}  // namespace mgq
