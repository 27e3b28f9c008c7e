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
// const, O += w_j V8_j, l += w_j / vs. M may lag by 1, so w_j < 2^15 whatever the
// scales are: its f16 hi + lo pair keeps 22 bits down to 2^-17 of the largest, and
// is off by less than 2^-38 of the largest below. M, l and O are f32.
//
// int8 K skips the conversion: q goes in as three digits of 8 bits on the int8
// matrix cores (v_mfma_i32_16x16x64_i8), whose sums are exact.
//
// Loads. K's registers are free for the next tile after S, V's after O, and the
// page ids are a tile ahead of both: 64 tokens' 16 KiB (D = 128) are on their way
// for each wavefront while it computes.
//
// Split. The tiles of a (sequence, kv head, 16 query rows) make a row. Much work:
// all rows laid end to end are cut into equal runs, one for each resident
// work-group, so ragged batches and one long sequence balance alike. Little work
// (under kRunTiles tiles a work-group): each row is cut into equal parts by
// itself, a work-group each, since every further row that a run touches costs its
// latencies again (~7 us: page ids, loads, join through LDS); rows of kSoloTiles
// and less are one part. The wavefronts of a work-group take tiles in turn, each
// with its own softmax state, joined through LDS; a row in several parts leaves
// their states in the workspace for kv_attn_join_kernel.
//
// Bound by the cache's bytes (28 heads on 4 of 128): 32 ragged sequences to 32 Ki
// tokens, e4m3, 380 MB: 81 us + 4.8 for the join, 4.7 TB/s; 200 000 tokens, int8,
// 205 MB: 42 + 5 us. A sequence of 1000 tokens is latency: 9 + 3 us.
#include "kv_attn.hpp"

namespace mgq {

constexpr int kRows = 16;         // query rows of a work-group's row of tiles
constexpr int kAttnGroups = 512;  // work-groups: two of 4 wavefronts per CU
constexpr int NW = 4;             // wavefronts of a work-group
// A row of 512 tokens is not cut (2 tiles a wavefront cost less than the joining
// launch), a part has a tile for each wavefront.
constexpr int kSoloTiles = 2 * NW, kPartTiles = NW, kRunTiles = 4 * NW;

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
// Sum of v over the work-group (NW wavefronts) and the sum over lower threads.
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
    for (int k = 0; k < NW; ++k) {
        if (k < w) before += part[k];
        total += part[k];
    }
    __syncthreads();
    return before + s - v;
}

// The cut. Runs: a unit is a tile, `run` of them a work-group's. Parts: a unit is
// a part of at most `part` tiles. Where no row can have more than kSoloTiles
// tiles (`most` 0) every row is one part, however many there are: no join follows.
struct AttnPlace {
    int total, run, part;  // part 0: runs
    int at, b, base;       // first unit, its sequence, that one's first unit
    AttnSeq q;             // the sequence
    __device__ __forceinline__ int parts(const AttnSeq &s) const {
        return s.tiles <= kSoloTiles ? 1 : (s.tiles + part - 1) / part;
    }
    // units of a sequence
    __device__ __forceinline__ int units(const AttnSeq &s, int hkv) const {
        return s.blocks * hkv * (part ? parts(s) : s.tiles);
    }
    __device__ __forceinline__ void cut(int tiles, int most) {
        if (most == 0) part = kSoloTiles;
        else part = tiles < most * kRunTiles ? max(kPartTiles, (tiles + most - 1) / most) : 0;
    }
    __device__ __forceinline__ void deal(int units, int most) {
        const int groups = part ? (int)gridDim.x : min(most, (int)gridDim.x);
        total = units;
        run = (total + groups - 1) / groups;
        at = (int)blockIdx.x < groups ? (int)blockIdx.x * run : total;
    }
};
__device__ __forceinline__ AttnPlace attn_place(const KvView &c, const AttnArgs &a, int most, int *part, int *found) {
    constexpr int NT = 64 * NW;
    AttnPlace p = {};
    if (c.n_seqs == 1) {
        p.q = attn_seq(c, a, 0);
        p.cut(p.q.blocks * c.hkv * p.q.tiles, most);
        p.deal(p.units(p.q, c.hkv), most);
        return p;
    }
    // all tiles, then all units, then the sequence that `at` lies in; the
    // sequence of a thread is kept where there are no more than threads
    AttnSeq q = {};
    int tiles = 0, units = 0, before = 0, t;
    for (int b0 = 0; b0 < c.n_seqs; b0 += NT) {
        q.blocks = 0;
        if (b0 + (int)threadIdx.x < c.n_seqs) q = attn_seq(c, a, b0 + threadIdx.x);
        tiles += q.blocks * c.hkv * q.tiles;
    }
    group_scan(tiles, part, t);
    p.cut(t, most);
    int start;
    if (c.n_seqs <= NT) {
        units = p.units(q, c.hkv);
        start = group_scan(units, part, t);
    } else {
        for (int b = threadIdx.x; b < c.n_seqs; b += NT) units += p.units(attn_seq(c, a, b), c.hkv);
        group_scan(units, part, t);
    }
    p.deal(t, most);
    for (int b0 = 0; b0 < c.n_seqs; b0 += NT) {
        if (c.n_seqs > NT) {
            units = b0 + (int)threadIdx.x < c.n_seqs ? p.units(attn_seq(c, a, b0 + threadIdx.x), c.hkv) : 0;
            start = before + group_scan(units, part, t);
            before += t;
        }
        if (p.at >= start && p.at < start + units) {
            found[0] = b0 + threadIdx.x;
            found[1] = start;
        }
    }
    __syncthreads();
    if (p.at < p.total) {
        p.b = found[0];
        p.base = found[1];
        p.q = attn_seq(c, a, p.b);
    }
    return p;
}

// Workspace: states, then for every row its first state's number and how many
// it has, written by the row's first work-group. Runs: run w has state 2w for a
// row that an earlier run begins, 2w + 1 for one it begins (the number of states
// is negative then). Parts: a state has its unit's number.
template <int D>
__device__ __forceinline__ int2 *row_states(const AttnArgs &a, int states) {
    return reinterpret_cast<int2 *>(a.ws + (int64_t)states * state_floats<D>(kRows));
}

template <int D, int FMT>
__global__ __launch_bounds__(64 * NW, D == 256 ? 1 : 2) void kv_attn_kernel(KvView c, AttnArgs a, int max_blocks, int most,
                                                                               int states) {
    constexpr bool I8 = FMT == kFmtI8 && D % 64 == 0;
    constexpr int KB = D / 4;               // bytes of a token that a lane group has
    constexpr int KS = I8 ? D / 64 : D / 32;  // summed steps of S
    constexpr int DB = D / 16;              // blocks of 16 dims of O
    constexpr int OP = D + 4;               // LDS row of O
    constexpr int NT = 64 * NW;
    __shared__ float sO[NW * kRows * OP];
    __shared__ float sM[NW][kRows], sL[NW][kRows];
    __shared__ int part[NW], found[2];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 15, grp = lane >> 4;
    const int page = 1 << c.page_shift;

    const AttnPlace place = attn_place(c, a, most, part, found);
    int at = place.at;
    const int stop = min(at + place.run, place.total);
    if (at >= stop) return;
    int b = place.b, base = place.base;
    AttnSeq q = place.q;

    while (at < stop) {
        while (at - base >= place.units(q, c.hkv)) {  // the next sequence with rows
            base += place.units(q, c.hkv);
            q = attn_seq(c, a, ++b);
        }
        const int first_unit = at, cuts = place.part ? place.parts(q) : q.tiles;
        const int k = (at - base) % cuts, row = (at - base) / cuts;
        int t0, t1;
        if (place.part) {
            t0 = (int)((int64_t)q.tiles * k / cuts);
            t1 = (int)((int64_t)q.tiles * (k + 1) / cuts);
            ++at;
        } else {
            t0 = k;
            t1 = min(q.tiles, t0 + stop - at);
            at += t1 - t0;
        }
        const int h = row % c.hkv, blk = row / c.hkv, r0 = blk * kRows;  // kv head, row block, its first query row
        const int rows = q.s.n * a.group;

        // ---- this lane's query row
        const int r = r0 + col;
        const bool live = r < rows;
        const int tq = live ? r / a.group : 0, hd = live ? r % a.group : 0;
        const int pos = live ? q.s.pos0 + tq : -1;
        // ---- loads
        const int tile_end = q.tile0 + t1;
        const int kgrp = col >> 2;  // the 16 tokens that this lane's K rows are of
        u32x4 vreg[DB];
        u32x4 kreg[4][(KB + 15) / 16];
        float ks_n = 0.0f, vs_n = 1.0f;
        int nv_n = 0;         // of this lane group's 16 tokens, those that exist
        int ik = -1, iv = -1;  // page ids of the next tile to load
        const int *tab = c.table + (int64_t)b * c.max_pages;
        const auto look = [&](int tile) {
            const int pk = tile * kTile + 16 * kgrp, pv = tile * kTile + 16 * grp;
            ik = pk < q.s.len ? tab[pk >> c.page_shift] : -1;
            iv = pv < q.s.len ? tab[pv >> c.page_shift] : -1;
        };
        // a page that the table does not name, or past the length, is read as
        // page 0 and counts as no tokens; its scales may be anything
        const auto load_k = [&](int tile) {
            const int p = tile * kTile + 16 * kgrp, id = ik < 0 || ik >= c.n_pages ? 0 : ik;
            const uint8_t *kp = c.k + id * c.page_stride + ((int64_t)h * page + (p & (page - 1)) + (col & 3)) * D + grp * KB;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if constexpr (KB % 16 == 0) {
#pragma unroll
                    for (int i = 0; i < KB / 16; ++i)
                        kreg[t][i] = *reinterpret_cast<const u32x4 *>(kp + 4 * t * D + 16 * i);
                } else {  // 24 bytes at a multiple of 8
#pragma unroll
                    for (int i = 0; i < KB / 8; ++i) {
                        const u32x2 x = *reinterpret_cast<const u32x2 *>(kp + 4 * t * D + 8 * i);
                        kreg[t][i / 2][2 * (i % 2)] = x[0];
                        kreg[t][i / 2][2 * (i % 2) + 1] = x[1];
                    }
                }
            }
        };
        const auto load_v = [&](int tile) {
            const int p = tile * kTile + 16 * grp;
            const bool ok = iv >= 0 && iv < c.n_pages;
            const int id = ok ? iv : 0;
            nv_n = ok ? min(q.s.len - p, 16) : 0;
            ks_n = ok ? c.ks[(int64_t)id * c.hkv + h] : 0.0f;
            vs_n = ok ? c.vs[(int64_t)id * c.hkv + h] : 1.0f;
            const uint8_t *vp = c.v + id * c.page_stride + ((int64_t)h * D + col) * page + (p & (page - 1));
#pragma unroll
            for (int d = 0; d < DB; ++d) vreg[d] = *reinterpret_cast<const u32x4 *>(vp + 16 * d * page);
        };
        int tile = q.tile0 + t0 + wave;
        // loads come back in order: the page ids first, which the others wait for
        look(tile);
        __builtin_amdgcn_sched_barrier(0);
        float qv[KB];
        read_query<D>(a.q + (int64_t)(q.s.t0 + tq) * a.q_stride + (h * a.group + hd) * D + grp * KB, qv);
        if (tile < tile_end) {
            load_k(tile);
            load_v(tile);
            look(tile + NW);
        }

        half8 qh[I8 ? 1 : KS], ql[I8 ? 1 : KS];
        i32x4 qd[3][I8 ? KS : 1];
#pragma unroll
        for (int i = 0; i < KB; ++i) qv[i] = live ? qv[i] : 0.0f;
        float kscale;
        if constexpr (I8) kscale = split_query<D, 3>(a.scale, qv, qd);
        else kscale = split_query<D>(a.scale, qv, qh, ql);

        f32x4 O[DB] = {};
        float M = -INFINITY, l = 0.0f;
        bool loud = false;
        for (; tile < tile_end; tile += NW) {
            const float ks = kscale * ks_n, vs = fmaxf(vs_n, kLeastScale);
            const int nv = nv_n;
            f32x4 S[4] = {};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if constexpr (I8) {
                    i32x4 d[3] = {};
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int n = 0; n < 3; ++n)
                            d[n] = mfma16(__builtin_bit_cast(i32x4, kreg[t][k]), qd[n][k], d[n]);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        S[t][e] = fmaf((float)(d[2][e] * 256 + d[1][e]), 256.0f, (float)d[0][e]);
                } else {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const half8 x = kv_half8<FMT>(kreg[t][k / 2][2 * (k % 2)], kreg[t][k / 2][2 * (k % 2) + 1]);
                        S[t] = mfma16(x, qh[k], S[t]);
                        S[t] = mfma16(x, ql[k], S[t]);
                    }
                }
            }
            const bool more = tile + NW < tile_end;
            if (more) load_k(tile + NW);

            const float lv = __log2f(vs);
            const int first = tile * kTile + 16 * grp;
            const int see = min(pos + 1 - first, nv);  // tokens of the 16 up to the row's own
            const int skip = a.window > 0 ? pos - a.window + 1 - first : 0;
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float s = S[t][i] * ks;
                    if (a.softcap > 0.0f) s = softcap_log2(s, a.softcap);
                    const int e = 4 * t + i;
                    s = e < see && e >= skip ? s + lv : -INFINITY;
                    S[t][i] = s;
                    top = fmaxf(top, s);
                }
            const float own = top;
            loud = loud || __any(vs > kLoudScale);
            top = max_groups(top);
            float per = __builtin_amdgcn_rcpf(vs);
            if (loud || __any(outgrown(top, M))) {  // the maximum may lag by 1: w stays below 2^15
                const float m = fmaxf(M, top);
                const Exp2 f(M == -INFINITY ? -INFINITY : M - m);
                M = m;
                l = f.times(l);
#pragma unroll
                for (int d = 0; d < DB; ++d) O[d] *= f.f;
                const float ref = reference_of(m);
                if (loud && vanishing(own, ref)) {
                    float near = 0.0f;
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) near += __builtin_amdgcn_exp2f(S[t][i] - own);
                    l += Exp2(own - ref - lv).times(near);
                    per = 0.0f;
                }
            }
            const float ref = reference_of(M);
            float sum = 0.0f;
            half8 ph[2], pl[2];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = __builtin_amdgcn_exp2f(S[t][i] - ref);
                    sum += w;
                    const _Float16 hi = (_Float16)w;
                    ph[t / 2][4 * (t % 2) + i] = hi;
                    pl[t / 2][4 * (t % 2) + i] = (_Float16)(w - (float)hi);
                }
            l += sum * per;
            if (__any(nv < 16)) {
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
            if (more) {
                load_v(tile + NW);
                look(tile + 2 * NW);
            }
        }

        // ---- the wavefronts' states into one
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (grp == 0) sM[wave][col] = M;
        __syncthreads();
        float all = sM[0][col];
#pragma unroll
        for (int w = 1; w < NW; ++w) all = fmaxf(all, sM[w][col]);
        const Exp2 f(M == -INFINITY ? -INFINITY : M - all);
        const float fac = f.f;
        if (grp == 0) sL[wave][col] = f.times(l);
        if (live) {
#pragma unroll
            for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4 *>(&sO[(wave * kRows + col) * OP + 16 * d + 4 * grp]) = O[d] * fac;
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == q.tiles;
        float *slot = a.ws + (int64_t)(place.part ? first_unit : 2 * (int)blockIdx.x + (t0 == 0)) * state_floats<D>(kRows);
        const int mine = min(kRows, rows - r0);
        for (int i = tid; i < mine * (D / 4); i += NT) {
            const int rr = i / (D / 4), d = 4 * (i % (D / 4));
            f32x4 o = {};
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                o += *reinterpret_cast<const f32x4 *>(&sO[(w * kRows + rr) * OP + d]);
                s += sL[w][rr];
            }
            if (whole) {
                put_out4(a, q.s.t0 + (r0 + rr) / a.group, (h * a.group + (r0 + rr) % a.group) * D + d,
                         o * (s == 0.0f ? 0.0f : 1.0f / s));
            } else {
                *reinterpret_cast<f32x4 *>(slot + rr * D + d) = o;
                if (d == 0) {
                    float m = sM[0][rr];
#pragma unroll
                    for (int w = 1; w < NW; ++w) m = fmaxf(m, sM[w][rr]);
                    *reinterpret_cast<float2 *>(slot + kRows * D + 2 * rr) = make_float2(m, s);
                }
            }
        }
        if (tid == 0 && t0 == 0) {
            int2 st = {first_unit, cuts};
            if (whole) st.y = 1;
            else if (!place.part) st = {(int)blockIdx.x, (int)blockIdx.x - 1 - (first_unit + q.tiles - 1) / place.run};
            row_states<D>(a, states)[((int64_t)b * max_blocks + blk) * c.hkv + h] = st;
        }
        __syncthreads();
    }
}

// Joins the partial states of query rows that a cut went through: one
// work-group per (sequence, row block, kv head, query row).
template <int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvView c, AttnArgs a, int max_blocks, int block_rows, int states) {
    int w = blockIdx.x;
    const int rr = w % block_rows;
    w /= block_rows;
    const int h = w % c.hkv;
    w /= c.hkv;
    const int blk = w % max_blocks, b = w / max_blocks;
    const int2 st = row_states<D>(a, states)[((int64_t)b * max_blocks + blk) * c.hkv + h];
    const SeqInfo s = kv_seq(c, b);
    const int r = blk * kRows + rr;
    if (r >= s.n * a.group) return;  // no such row, and nobody has written its states' numbers
    if (st.y == 1) return;  // the whole row was one work-group's, which has written it
    const auto slot = [&](int i) {
        return a.ws + (int64_t)(st.y > 0 ? st.x + i : 2 * (st.x + i) + (i == 0)) * state_floats<D>(kRows);
    };
    const f32x4 o = join_row<D>(abs(st.y), kRows, rr, slot);
    if ((int)threadIdx.x < D / 4)
        put_out4(a, s.t0 + r / a.group, (h * a.group + r % a.group) * D + 4 * threadIdx.x, o);
}

// Query rows of a kv head up to which this kernel takes the call, in blocks of
// 16 that each read the cache, and above which kv_attn_wide.hip does. Measured
// (28 heads on 4 of 128, int8): 28 rows x 16 sequences of 4000 tokens 29 us here,
// 46 there; 63 rows x 8 of 8000 56 and 51. Heads of 256: 24 rows 25 and 29, 48
// rows 57 and 40.
bool kv_attn_is_wide(int dim, int64_t rows) { return rows > (dim == 256 ? 32 : 48); }

// Most tiles of a row: the table's, or the window's.
static int64_t most_tiles(int64_t cap, int max_new, int window) {
    if (window > 0) cap = std::min<int64_t>(cap, (int64_t)window + max_new - 1 + kTile - 1);
    return (cap + kTile - 1) / kTile;
}

// States: a run has two, a part one, and with the parts' least size given by
// `most` there are no more parts than `most` and one for every row.
static int64_t most_states(int64_t rows) { return kAttnGroups + std::max<int64_t>(rows, kAttnGroups); }

size_t kv_attn_workspace(int dim, int hq, int hkv, int n_seqs, int max_new, int64_t capacity) {
    const int64_t rows = (int64_t)max_new * (hq / hkv), blocks = (rows + kRows - 1) / kRows;
    if (kv_attn_is_wide(dim, rows)) return std::max<size_t>(16, kv_attn_wide_workspace(dim, hq / hkv, hkv, n_seqs, max_new, capacity));
    const int64_t all = (int64_t)n_seqs * blocks * hkv;
    return (size_t)most_states(all) * kRows * (dim + 2) * sizeof(float) + (size_t)all * sizeof(int2);
}

template <int D, int FMT>
static hipError_t attn_run_dim(const KvView &c, const AttnArgs &a, hipStream_t stream) {
    const int max_blocks = (c.max_new * a.group + kRows - 1) / kRows;
    const int64_t tiles = most_tiles((int64_t)c.max_pages << c.page_shift, c.max_new, a.window);
    const int64_t rows = (int64_t)c.n_seqs * c.hkv * max_blocks;
    const bool solo = tiles <= kSoloTiles;  // no row can be longer
    const int most = D == 256 ? kAttnGroups / 2 : kAttnGroups;  // resident at once
    const int groups = (int)(solo ? rows : std::min(rows * ((tiles + kPartTiles - 1) / kPartTiles), most + rows));
    const int states = (int)most_states(rows);
    kv_attn_kernel<D, FMT><<<(unsigned)groups, 64 * NW, 0, stream>>>(c, a, max_blocks, solo ? 0 : most, states);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || solo) return e;
    const int block_rows = std::min(kRows, c.max_new * a.group);
    kv_attn_join_kernel<D><<<(unsigned)(rows * block_rows), 256, 0, stream>>>(c, a, max_blocks, block_rows, states);
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
    a.window = std::min(x.window, 1 << 30);  // all of any sequence; pos0 - window stays in 32 bits
    a.ws = x.ws;
    if (kv_attn_is_wide(dim, c.max_new * a.group)) return kv_attn_wide_launch(c, dim, fmt, a, stream);
    const bool i8 = fmt == MGQ_KV_I8;
    switch (dim) {
    case 64: return i8 ? attn_run_dim<64, kFmtI8>(c, a, stream) : attn_run_dim<64, kFmtE4M3>(c, a, stream);
    case 96: return i8 ? attn_run_dim<96, kFmtI8>(c, a, stream) : attn_run_dim<96, kFmtE4M3>(c, a, stream);
    case 128: return i8 ? attn_run_dim<128, kFmtI8>(c, a, stream) : attn_run_dim<128, kFmtE4M3>(c, a, stream);
    default: return i8 ? attn_run_dim<256, kFmtI8>(c, a, stream) : attn_run_dim<256, kFmtE4M3>(c, a, stream);
    }
}

}  // namespace mgq
