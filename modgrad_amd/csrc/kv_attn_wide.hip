// Attention over the paged 8-bit cache for many query rows of a sequence (a
// prompt, a piece of one): the same operands and softmax as kv_attn.hip, with
// a tile's K and V shared by a work-group through LDS.
//
// A work-group has 128 query rows of one (sequence, kv head): row r is new token
// r / group, head r % group of the group, so the rows of a group's heads share
// the tile. 4 wavefronts of 32 rows (two sets of 16 columns of S^T), or 8 of 16.
// Each tile of 64 tokens is converted to f16 ONCE on its way into LDS (V, and K
// unless it is int8: a 4-byte word costs 5 operations, shared by the wavefronts),
// as the operands the matrix cores take: 16 bytes of each of 64 lanes one after
// another, so every LDS access is a contiguous 1 KiB. One operand read feeds a
// set's two or three digits or halves of q, and one (f16 result) or two (f32) of p.
//
// Tile i+2's bytes load into registers and tile i+1's go to the other LDS
// buffer while tile i multiplies; one barrier a tile, which does not wait for
// the loads. Bound by the softmax's exponentials and conversions on the vector
// ALU, which issues in 71 % of the cycles of a 4096-token prompt of 28 heads of
// 128 on int8 with f16 results (151 us, 797 TFLOP/s counted as 4 D a pair), beside
// the matrix cores (34 %): the second wavefront of each SIMD overlaps the two. With f32
// results, three digits of q and two halves of p, 255 us (66 and 35 %). Pieces of up to 250
// tokens over 9000, 16 heads of 256 on e4m3 with f32 results and a softcap: 97 us, a
// tenth of it the join, the products twice a plain f16 attention's (50 and 39 %).
//
// Causal work is dealt longest first; work-groups of one kv head are neighbours
// modulo the number of kv heads, so an XCD's L2 holds few heads' caches. With
// too few rows to fill the chip, a row block's tiles are split and the partial
// states joined by a second kernel.
#include "kv_attn.hpp"

namespace mgq {

// Work-groups that a call's splits are made for: those resident at once, of 4 wavefronts
// two a CU and of 8 one. By the head alone: heads of 128 with one set of rows (int8,
// f32 results) have 8 wavefronts too and so twice as many splits as fit at once.
__host__ __device__ constexpr int wide_slots(int dim) { return dim == 256 ? 256 : 512; }
constexpr int kWideChunk = 4;  // least tiles of a split: a work-group's start costs about as much

struct WideBlock {
    SeqInfo s;
    int r0, rows;            // first query row, rows of the sequence
    TileList list;
    int tiles, chunk;        // tiles, tiles of a split
};
__device__ __forceinline__ bool wide_block(const KvView &c, const AttnArgs &a, int b, int rt, int splits, WideBlock &w) {
    w.s = kv_seq(c, b);
    w.rows = w.s.n * a.group;
    w.r0 = rt * kWideRows;
    if (w.r0 >= w.rows) return false;
    const int first = w.s.pos0 + w.r0 / a.group, last = w.s.pos0 + (min(w.r0 + kWideRows, w.rows) - 1) / a.group;
    const int hi = min(w.s.len, max(last + 1, 0));
    w.list = tile_list(a, w.s, first);
    w.tiles = w.list.count(hi);
    w.chunk = max((w.tiles + splits - 1) / splits, splits > 1 ? kWideChunk : 1);
    return true;
}

// Row block `at` of those that are there (sequence by sequence, each from its
// last, longest one), found by every wavefront for itself; and the splits of
// every block: as many as fill the chip's slots once, which only the device
// knows. Work-groups without a block have the last numbers: the dispatcher
// deals numbers to the shader engines in turn and waits for the one whose turn
// it is, so empty numbers among the others leave engines idle.
struct WidePlace {
    int b, rt;      // rt < 0: none
    int split, splits;
    int64_t state;  // number of the block's state, the kv head aside
    int total;      // row blocks
};
template <int D>
__device__ __forceinline__ WidePlace wide_place(const KvView &c, const AttnArgs &a, int id, int most_splits) {
    const int lane = threadIdx.x & 63;
    const auto blocks = [&](int b) { return b < c.n_seqs ? (kv_seq(c, b).n * a.group + kWideRows - 1) / kWideRows : 0; };
    WidePlace p = {0, -1, 0, 1, 0, 0};
    if (c.n_seqs == 1) {
        p.total = blocks(0);
        p.splits = most_splits;  // made for all its blocks
        p.split = id / max(1, p.total);
        if (p.split >= p.splits) return p;
        p.state = id - p.split * p.total;
        p.rt = p.total - 1 - (int)p.state;
        return p;
    }
    int n = blocks(lane);
    if (most_splits > 1) {
        int sum = n;
        for (int b = lane + 64; b < c.n_seqs; b += 64) sum += blocks(b);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        p.total = min(__builtin_amdgcn_readfirstlane(sum), a.row_blocks);  // overlapping ranges: those that have a place
        p.splits = max(1, min(most_splits, wide_slots(D) / max(1, p.total * c.hkv)));
        p.split = id / max(1, p.total);
        if (p.split >= p.splits) return p;
        id -= p.split * p.total;
    }
    p.state = id;
    int before = 0;
    for (int b0 = 0; b0 < c.n_seqs; b0 += 64) {
        if (b0 > 0) n = blocks(b0 + lane);
        int s = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(s, o, 64);
            if (lane >= o) s += t;
        }
        const uint64_t past = __ballot(before + s > id);  // lanes whose blocks reach beyond id
        if (past) {
            const int l = __builtin_ctzll(past);
            p.b = b0 + l;
            p.rt = before + __shfl(s, l, 64) - 1 - id;
            p.b = __builtin_amdgcn_readfirstlane(p.b);
            p.rt = __builtin_amdgcn_readfirstlane(p.rt);
            return p;
        }
        before += __builtin_amdgcn_readlane(s, 63);
    }
    return p;
}

// A shared prefix: block rt of all the call's query rows.
struct PrefixRows {
    int lim[kWideRows];
    unsigned long long best;
};
__device__ __forceinline__ void prefix_block(const KvView &c, const AttnArgs &a, int rt, PrefixRows &p, int &b, WideBlock &w) {
    w.rows = c.n_tokens * a.group;
    w.r0 = rt * kWideRows;
    prefix_limits(c, a, w.r0 / a.group, (min(w.r0 + kWideRows, w.rows) - 1) / a.group + 1, blockDim.x, p.lim, p.best);
    w.tiles = (int)(p.best >> 32);
    b = w.tiles > 0 ? (int)(0xFFFFFFFFu - (unsigned)p.best) : 0;
    w.s = {0, c.n_tokens, 0, w.tiles * kTile};
    w.list = {0, 0};
    w.chunk = 0;
}

__device__ __forceinline__ void wide_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
}

// Compile-time shape of the kernel. int8 K goes into the int8 matrix cores as it
// is, q as digits of 8 bits: 16 bits for an f16 result, 24 for f32 (heads of 96
// are no multiple of the 64 dims of such a product).
// SETS of 16 query rows a wavefront: two sets and 4 wavefronts read LDS half as
// often; one and 8 wavefronts where two spill more than that is worth. Measured when
// it was chosen (two, one; us for 4096 tokens of 28 heads): heads of 64 to f32 166, 197, on e4m3
// to f16 129, 157; of 96 156, 198; of 128 on e4m3 to f32 239, 248, on int8 to f32
// 449, 250; pieces of heads of 256 to f32 192, 126.
template <int D, int FMT, bool LO>
struct WideShape {
    static constexpr bool I8 = FMT == kFmtI8 && D % 64 == 0;
    static constexpr int SETS = D == 256 || (D == 128 && LO && FMT == kFmtI8) ? 1 : 2;
    static constexpr int NW = kWideRows / (16 * SETS);      // wavefronts
    static constexpr int kThreads = 64 * NW, kPerSimd = 2;
    static constexpr int KS = I8 ? D / 64 : D / 32;         // summed steps of S
    static constexpr int DB = D / 16;                       // blocks of 16 dims of O
    static constexpr int NK = 4 * KS / NW;                  // pieces of K a wavefront stages: 64 lanes x 16 bytes of LDS
    static constexpr int NV = 2 * DB / NW;                  // pieces of V
    // of a prefix's kernel, its rows' limits behind the buffers
    template <bool PREFIX>
    static constexpr size_t lds_bytes() {
        return 2 * kBuf * sizeof(half8) + (PREFIX ? sizeof(PrefixRows) : 0);
    }
    static_assert(4 * KS % NW == 0 && 2 * DB % NW == 0, "each wavefront stages as many pieces");
    static constexpr int kOfV = 4 * KS * 64, kBuf = kOfV + 2 * DB * 64;  // 16-byte units of a buffer: K, then V
};

// Tiles t0 .. t1-1 of the rows of one (row block, kv head). LO: the probabilities as hi +
// lo pairs. PREFIX: over the tiles of a shared prefix, to a state always.
template <int D, int FMT, bool LO, bool PREFIX>
__device__ __forceinline__ void wide_rows(const KvView &c, const AttnArgs &a, half8 *lds, const WideBlock &w, int h, int b,
                                          int t0, int t1, float *st, bool whole) {
    typedef WideShape<D, FMT, LO> W;
    constexpr bool I8 = W::I8;
    constexpr int SETS = W::SETS, KS = W::KS, DB = W::DB, NK = W::NK, NV = W::NV;
    constexpr int ND = LO ? 3 : 2;  // digits of q
    constexpr int KB = D / 4;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15,
              grp = lane >> 4;
    const int page = 1 << c.page_shift;
    const PrefixRows &rows = *reinterpret_cast<const PrefixRows *>(lds + 2 * W::kBuf);  // PREFIX only

    // ---- query rows; those past the last repeat it and are not written
    half8 qh[SETS][I8 ? 1 : KS], ql[SETS][I8 ? 1 : KS];
    i32x4 qd[SETS][ND][I8 ? KS : 1];
    float qs[SETS], qv[SETS][KB];
    int pos[SETS];
    const int wr0 = w.r0 + 16 * SETS * wave;  // the wavefront's first row
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        const int r = min(wr0 + 16 * s + col, w.rows - 1);
        const int tq = r / a.group;
        pos[s] = PREFIX ? rows.lim[tq - w.r0 / a.group] * kTile - 1 : w.s.pos0 + tq;
        read_query<D>(a.q + (int64_t)(w.s.t0 + tq) * a.q_stride + (h * a.group + r % a.group) * D + grp * KB, qv[s]);
    }
    const bool live = wr0 < w.rows;
    // positions of the wavefront's first and last row
    int pos_lo = w.s.pos0 + min(wr0, w.rows - 1) / a.group;
    int pos_hi = w.s.pos0 + min(wr0 + 16 * SETS - 1, w.rows - 1) / a.group;
    if constexpr (PREFIX) {  // the least and the most of its rows
        pos_lo = pos[0];
        pos_hi = pos[0];
#pragma unroll
        for (int s = 1; s < SETS; ++s) {
            pos_lo = min(pos_lo, pos[s]);
            pos_hi = max(pos_hi, pos[s]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            pos_lo = min(pos_lo, __shfl_xor(pos_lo, o, 64));
            pos_hi = max(pos_hi, __shfl_xor(pos_hi, o, 64));
        }
        pos_lo = __builtin_amdgcn_readfirstlane(pos_lo);
        pos_hi = __builtin_amdgcn_readfirstlane(pos_hi);
    }

    // ---- staging
    const int kgrp = col >> 2;
    const int *tab = c.table + (int64_t)b * c.max_pages;
    const int last = t1 - 1;
    // page ids of the tile after the staged one, a tile ahead of their use: -1
    // past the length
    int ik_n, iv_n;
    const auto look = [&](int t) {
        const int at = w.list.at(min(t, last)) * kTile, pk = at + 16 * kgrp, pv = at + 16 * grp;
        ik_n = pk < w.s.len ? tab[pk >> c.page_shift] : -1;
        iv_n = pv < w.s.len ? tab[pv >> c.page_shift] : -1;
    };
    u32x4 kst[NK];  // I8: 16 bytes a piece, else 8
    u32x2 vst[NV];
    float ks_n, vs_n;  // scales and count of the tile in the staging registers
    int nv_n;
    const auto fetch = [&](int t) {  // past the last tile, the last again
        const int at = w.list.at(min(t, last)) * kTile, pk = at + 16 * kgrp, pv = at + 16 * grp;
        int ik = ik_n, iv = iv_n;
        const bool okv = iv >= 0 && iv < c.n_pages;
        if (ik < 0 || ik >= c.n_pages) ik = 0;
        if (!okv) iv = 0;
        nv_n = okv ? min(w.s.len - pv, 16) : 0;
        look(t + 1);
        // what lies in a page's place that is none of the sequence's may be anything
        ks_n = okv ? c.ks[(int64_t)iv * c.hkv + h] : 0.0f;
        vs_n = okv ? c.vs[(int64_t)iv * c.hkv + h] : 1.0f;
        const uint8_t *kp = c.k + ik * c.page_stride + ((int64_t)h * page + (pk & (page - 1)) + (col & 3)) * D + grp * KB;
        const uint8_t *vp = c.v + iv * c.page_stride + ((int64_t)h * D + col) * page + (pv & (page - 1));
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int p = wave * NK + i, bt = p / KS, k = p % KS;
            if constexpr (I8) {
                kst[i] = *reinterpret_cast<const u32x4 *>(kp + 4 * bt * D + 16 * k);
            } else {
                const u32x2 x = *reinterpret_cast<const u32x2 *>(kp + 4 * bt * D + 8 * k);
                kst[i][0] = x[0];
                kst[i][1] = x[1];
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = wave * NV + i;  // dims 16 (p/2) .., tokens 8 (p%2) ..
            vst[i] = *reinterpret_cast<const u32x2 *>(vp + 16 * (p >> 1) * page + 8 * (p & 1));
        }
    };
    const auto stage = [&](half8 *buf) {
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int p = wave * NK + i;
            if constexpr (I8) reinterpret_cast<u32x4 *>(buf)[p * 64 + lane] = kst[i];
            else buf[p * 64 + lane] = kv_half8<FMT>(kst[i][0], kst[i][1]);
        }
        if (__any(nv_n < 16)) {
#pragma unroll
            for (int i = 0; i < NV; ++i) vst[i] = kv_keep(vst[i], nv_n, (wave * NV + i) & 1);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) buf[W::kOfV + (wave * NV + i) * 64 + lane] = kv_half8<FMT>(vst[i][0], vst[i][1]);
    };

    f32x4 O[SETS][DB] = {};
    float M[SETS], l[SETS];
    bool loud = false;
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        M[s] = -INFINITY;
        l[s] = 0.0f;
    }

    look(t0);
    fetch(t0);
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        if constexpr (I8) qs[s] = split_query<D, ND>(a.scale, qv[s], qd[s]);
        else qs[s] = split_query<D>(a.scale, qv[s], qh[s], ql[s]);
    }
    stage(lds);
    float ks_c = ks_n, vs_c = vs_n;
    int nv_c = nv_n;
    fetch(t0 + 1);
    for (int t = t0; t < t1; ++t) {
        wide_barrier();  // tile t is in its buffer, the other one is free
        const half8 *buf = lds + ((t - t0) & 1) * W::kBuf;
        const float ks = ks_c, vsv = vs_c;
        const int nv = nv_c;
        i32x4 kx[4][I8 ? KS : 1];
        const auto read_k = [&] {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < KS; ++k) kx[i][k] = reinterpret_cast<const i32x4 *>(buf)[(i * KS + k) * 64 + lane];
        };
        if constexpr (I8) {
            // K's operands on their way while the next tile is staged
            read_k();
            __builtin_amdgcn_sched_barrier(0);
        }
        stage(lds + ((t + 1 - t0) & 1) * W::kBuf);
        nv_c = nv_n;
        ks_c = ks_n;
        vs_c = vs_n;
        fetch(t + 2);
        const int first = w.list.at(t) * kTile;
        if (!live || first > pos_hi) continue;  // no row of the wavefront sees it

        f32x4 S[SETS][4] = {};
        if constexpr (I8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int s = 0; s < SETS; ++s) {
                    i32x4 d[ND] = {};
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int n = 0; n < ND; ++n) d[n] = mfma16(kx[i][k], qd[s][n][k], d[n]);
                    // two digits' sums stay below 2^31 and join as whole numbers, so that the
                    // score is rounded once, to f32; the third joins in f32
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (LO) S[s][i][e] = fmaf((float)(d[2][e] * 256 + d[1][e]), 256.0f, (float)d[0][e]);
                        else S[s][i][e] = (float)(d[1][e] * 256 + d[0][e]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const half8 x = buf[(i * KS + k) * 64 + lane];
#pragma unroll
                    for (int s = 0; s < SETS; ++s) {
                        S[s][i] = mfma16(x, qh[s][k], S[s][i]);
                        S[s][i] = mfma16(x, ql[s][k], S[s][i]);
                    }
                }
        }

        constexpr int G = 2;  // blocks of 16 dims read at once
        const half8 *vb = buf + W::kOfV;
        half8 vx[2][2 * G];
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) vx[0][i] = vb[i * 64 + lane];
        // a wavefront in its softmax goes before one whose matrix products only
        // wait for the matrix core (4096-token prompt 164 -> 155 us)
        __builtin_amdgcn_s_setprio(1);
        const float vs = fmaxf(vsv, kLeastScale), lv = __log2f(vs), rvs = __builtin_amdgcn_rcpf(vs);
        // all rows see all of the tile
        const bool clear = first + kTile - 1 <= pos_lo &&
                           (a.window == 0 || first > pos_hi - a.window || first + kTile <= a.sinks) && __all(nv == 16);
        half8 ph[SETS][2], pl[SETS][2];
        // (an f16 result is infinite before the page that makes others vanish is that loud)
        if (LO) loud = loud || __any(vs > kLoudScale);
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
            float sc = qs[s] * ks, add = lv;
            // scores that may reach 2^19: t is rounded once, below, so that no w passes
            // the largest. S is below 2^38 (three digits of q, 256 products with an int8
            // code), 2^30 (two) or 2^31 (q's halves below 2^14, e4m3 codes to 448).
            constexpr float kFarScale = !I8 ? 0x1p-12f : LO ? 0x1p-19f : 0x1p-11f;
            const bool exact = !clear || (a.softcap > 0.0f ? a.softcap > 0x1p19f : __any(sc >= kFarScale));
            if (a.softcap > 0.0f) {
                float far = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        S[s][i][e] *= sc;
                        far = fmaxf(far, fabsf(S[s][i][e]));
                    }
                if (!__any(far >= kCapNear)) {  // scores are rarely beyond a third of their bound
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) S[s][i][e] = a.softcap * tanh_near(S[s][i][e]);
                } else {
#pragma unroll 1
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = i == 0 ? S[s][0][e] : i == 1 ? S[s][1][e] : i == 2 ? S[s][2][e] : S[s][3][e];
                            const float y = softcap_log2(x, a.softcap);
                            S[s][0][e] = i == 0 ? y : S[s][0][e];
                            S[s][1][e] = i == 1 ? y : S[s][1][e];
                            S[s][2][e] = i == 2 ? y : S[s][2][e];
                            S[s][3][e] = i == 3 ? y : S[s][3][e];
                        }
                }
                sc = 1.0f;
            }
            if (exact) {
                const uint32_t seen = seen_tokens(a, pos[s], first + 16 * grp, nv);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        S[s][i][e] = seen >> (4 * i + e) & 1 ? fmaf(S[s][i][e], sc, lv) : -INFINITY;
                sc = 1.0f;
                add = 0.0f;
            }
            // the largest of t = S * sc + add: sc, a lane's own, is not negative
            float hi = S[s][0][0];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) hi = fmaxf(hi, S[s][i][e]);
            const float own = fmaf(hi, sc, add), top = max_groups(own);
            // the maximum may lag by 1: w stays below 2^15
            if (__any(outgrown(top, M[s]))) {
                const float m = fmaxf(M[s], top);
                float fac;
                if constexpr (LO) {
                    const Exp2 f(M[s] == -INFINITY ? -INFINITY : M[s] - m);
                    fac = f.f;
                    l[s] = f.times(l[s]);
                } else {
                    fac = M[s] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M[s] - m);
                    l[s] *= fac;
                }
                M[s] = m;
#pragma unroll
                for (int d = 0; d < DB; ++d) O[s][d] *= fac;
            }
            const float ref = reference_of(M[s]), off = add - ref;
            float per = rvs;
            if (loud && __any(vanishing(own, ref))) {
                float near = 0.0f;
#pragma unroll 1
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = i == 0 ? S[s][0][e] : i == 1 ? S[s][1][e] : i == 2 ? S[s][2][e] : S[s][3][e];
                        near += __builtin_amdgcn_exp2f(fmaf(x, sc, add - own));
                    }
                if (vanishing(own, ref)) {
                    l[s] += Exp2(own - ref - lv).times(near);
                    per = 0.0f;
                }
            }
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(S[s][i][e], sc, off));
                    sum += x;
                    const _Float16 xh = (_Float16)x;
                    ph[s][i / 2][4 * (i % 2) + e] = xh;
                    if (LO) pl[s][i / 2][4 * (i % 2) + e] = (_Float16)(x - (float)xh);
                }
            l[s] += sum * per;
        }
        __builtin_amdgcn_s_setprio(0);
        // V's operands a group ahead of their products
#pragma unroll
        for (int g = 0; g < DB / G; ++g) {
            if (g + 1 < DB / G) {
#pragma unroll
                for (int i = 0; i < 2 * G; ++i) vx[(g + 1) & 1][i] = vb[(2 * G * (g + 1) + i) * 64 + lane];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int s = 0; s < SETS; ++s) {
                        const int d = g * G + i;
                        O[s][d] = mfma16(vx[g & 1][2 * i + u], ph[s][u], O[s][d]);
                        if (LO) O[s][d] = mfma16(vx[g & 1][2 * i + u], pl[s][u], O[s][d]);
                    }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (!live) return;

#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        float sum = l[s];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const int r = wr0 + 16 * s + col, rr = r - w.r0;
        if (r >= w.rows) continue;
        if (whole) {
            const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int hd = (h * a.group + r % a.group) * D + 4 * grp;
#pragma unroll
            for (int d = 0; d < DB; ++d) put_out4(a, w.s.t0 + r / a.group, hd + 16 * d, O[s][d] * f);
        } else {
#pragma unroll
            for (int d = 0; d < DB; ++d)
                *reinterpret_cast<f32x4_a4 *>(st + rr * D + 16 * d + 4 * grp) = O[s][d];
            if (grp == 0) *reinterpret_cast<float2 *>(st + kWideRows * D + 2 * rr) = make_float2(M[s], sum);
        }
    }
}

template <int D, int FMT, bool LO>
__global__ __launch_bounds__((WideShape<D, FMT, LO>::kThreads), (WideShape<D, FMT, LO>::kPerSimd)) void kv_attn_wide_kernel(KvView c, AttnArgs a, int most_splits, int turn) {
    extern __shared__ half8 lds[];
    // the second work-groups of the CUs are dealt from the shorter end, beside the
    // longest ones (where a CU has one at a time they only come in another order)
    const int h = blockIdx.x % c.hkv;
    int id = blockIdx.x / c.hkv;
    if (id >= turn && id < 2 * turn) id = 3 * turn - 1 - id;
    const WidePlace place = wide_place<D>(c, a, id, most_splits);
    if (place.rt < 0) return;
    WideBlock w;
    if (!wide_block(c, a, place.b, place.rt, place.splits, w)) return;
    const int t0 = place.split * w.chunk, t1 = min(w.tiles, t0 + w.chunk);
    if (t0 >= t1) return;
    float *st = a.ws + ((place.split * (int64_t)place.total + place.state) * c.hkv + h) * state_floats<D>(kWideRows);
    wide_rows<D, FMT, LO, false>(c, a, lds, w, h, place.b, t0, t1, st, w.chunk >= w.tiles && a.shared == 0);
}

// A shared prefix: the tiles of a kv head's row blocks, laid end to end, are cut into
// equal runs, a work-group each, whatever the number of blocks. A run is no longer than
// a block's tiles, so it has the end of one block's and the beginning of the next one's
// at most, with a state for each.
//
// Bound like the prompt's by the softmax's vector work and, where runs are short, by their
// start (limits, query rows, page ids, first loads: 5 us) and the states: 64 tokens of 28 heads behind
// 12000, int8 with f32 results, 12 tiles a work-group: 36-38 us, 2.1 us a tile; 598
// tokens behind 10000 with f16 results, 41 tiles: 137-140 us (87 GFLOP, 630 TFLOP/s).
// Heads of 128 on e4m3 spill 18 registers (the plain kernel 6 to 9), on int8 with f16 results 3:
// those two calls on e4m3 take 66 and 190 us in all, on int8 61-65 and 156.
template <int D, int FMT, bool LO>
__global__ __launch_bounds__((WideShape<D, FMT, LO>::kThreads), (WideShape<D, FMT, LO>::kPerSimd)) void kv_attn_prefix_kernel(KvView c, AttnArgs a) {
    typedef WideShape<D, FMT, LO> W;
    extern __shared__ half8 lds[];
    PrefixRows &rows = *reinterpret_cast<PrefixRows *>(lds + 2 * W::kBuf);
    const int h = blockIdx.x % c.hkv, run = blockIdx.x / c.hkv;
    const int64_t stop = min((int64_t)(run + 1) * a.prefix_run, (int64_t)a.prefix_blocks * a.prefix_span);
    for (int64_t at = (int64_t)run * a.prefix_run; at < stop;) {
        const int rt = (int)(at / a.prefix_span), t0 = (int)(at - (int64_t)rt * a.prefix_span);
        const int t1 = (int)min((int64_t)a.prefix_span, t0 + stop - at);
        at += t1 - t0;
        __syncthreads();  // the run's other block has been read
        int b;
        WideBlock w;
        prefix_block(c, a, rt, rows, b, w);
        // tiles that no row of the block sees are left out; a state is of those that some does
        if (t0 < w.tiles)
            wide_rows<D, FMT, LO, true>(c, a, lds, w, h, b, t0, min(t1, w.tiles),
                                        prefix_slot<D>(c, a, h, run, t0 == 0), false);
    }
}

// Joins a split row block: one work-group per (row block, sequence, kv head, row).
template <int D>
__global__ __launch_bounds__(256) void kv_attn_wide_join_kernel(KvView c, AttnArgs a, int most_splits) {
    int id = blockIdx.x;
    const int rr = id % kWideRows;
    id /= kWideRows;
    const int h = id % c.hkv;
    id /= c.hkv;
    const WidePlace place = wide_place<D>(c, a, id, most_splits);
    if (place.rt < 0 || place.split > 0) return;
    WideBlock w;
    if (!wide_block(c, a, place.b, place.rt, place.splits, w)) return;
    const int r = w.r0 + rr;
    if (r >= w.rows || (w.chunk >= w.tiles && a.shared == 0)) return;
    const int n = (w.tiles + w.chunk - 1) / w.chunk;
    const PrefixParts ahead = prefix_parts(a, w.s, (int64_t)w.s.t0 * a.group + r);
    const auto slot = [&](int i) {
        if (i < ahead.n) return ahead.state<D>(c, a, h, i);
        return row_state<D>(a.ws + (((i - ahead.n) * (int64_t)place.total + id) * c.hkv + h) * state_floats<D>(kWideRows),
                            kWideRows, rr);
    };
    const f32x4 o = join_row<D>(ahead.n + n, slot);
    if ((int)threadIdx.x < D / 4)
        put_out4(a, w.s.t0 + r / a.group, (h * a.group + r % a.group) * D + 4 * threadIdx.x, o);
}

// The same for few splits: D/4 lanes a row. Behind a shared prefix every row is joined:
// latency bounds it, so that 4 states load at once, and the sum moves with the maximum.
constexpr int kJoinFew = 16;
template <int D, bool SHARED>
__global__ __launch_bounds__(256) void kv_attn_wide_join_few_kernel(KvView c, AttnArgs a, int most_splits) {
    constexpr int L = D / 4, PER = 256 / L, R = 8, STEPS = kWideRows / R;  // R rows a work-group
    int id = blockIdx.x;
    const int part = id % STEPS;
    id /= STEPS;
    const int h = id % c.hkv;
    id /= c.hkv;
    const WidePlace place = wide_place<D>(c, a, id, most_splits);
    if (place.rt < 0 || place.split > 0) return;
    WideBlock w;
    if (!wide_block(c, a, place.b, place.rt, place.splits, w)) return;
    if (w.chunk >= w.tiles && !SHARED) return;
    const int own = (w.tiles + w.chunk - 1) / w.chunk, d = 4 * (threadIdx.x % L);
    if ((int)threadIdx.x >= PER * L) return;
    const float *base = a.ws + ((int64_t)id * c.hkv + h) * state_floats<D>(kWideRows);
    const int64_t step = (int64_t)place.total * c.hkv * state_floats<D>(kWideRows);
    for (int rr = R * part + threadIdx.x / L; rr < R * part + R; rr += PER) {
        const int r = w.r0 + rr;
        if (r >= w.rows) break;
        PrefixParts ahead = {};
        if (SHARED) ahead = prefix_parts(a, w.s, (int64_t)w.s.t0 * a.group + r);
        const int n = ahead.n + own;
        const auto slot = [&](int i) {
            return SHARED && i < ahead.n ? ahead.state<D>(c, a, h, i) : row_state<D>(base + (i - ahead.n) * step, kWideRows, rr);
        };
        float M = -INFINITY, l = 0.0f;
        f32x4 o = {};
        if constexpr (SHARED) {
            constexpr int U = 4;
            for (int i0 = 0; i0 < n; i0 += U) {
                float2 ml[U];
                f32x4 x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const RowState s = slot(min(i0 + u, n - 1));
                    ml[u] = *reinterpret_cast<const float2 *>(s.ml);
                    x[u] = *reinterpret_cast<const f32x4 *>(s.o + d);
                    if (i0 + u >= n) ml[u] = make_float2(-INFINITY, 0.0f);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (ml[u].x == -INFINITY && ml[u].y == 0.0f) continue;  // of nothing; scores of NaN have a NaN l
                    const float m = fmaxf(M, ml[u].x);
                    const Exp2 f(M == -INFINITY ? -INFINITY : M - m), g(ml[u].x == -INFINITY ? -INFINITY : ml[u].x - m);
                    M = m;
                    l = f.times(l) + g.times(ml[u].y);
                    o = o * f.f + x[u] * g.f;
                }
            }
            put_out4(a, w.s.t0 + r / a.group, (h * a.group + r % a.group) * D + d, o * (l == 0.0f ? 0.0f : 1.0f / l));
            continue;
        }
        for (int i = 0; i < n; ++i) M = fmaxf(M, slot(i).ml[0]);
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const RowState s = slot(i);
            const float2 ml = *reinterpret_cast<const float2 *>(s.ml);
            const Exp2 f(ml.x == -INFINITY ? -INFINITY : ml.x - M);
            l += f.times(ml.y);
            o += f.f * *reinterpret_cast<const f32x4 *>(s.o + d);
        }
        put_out4(a, w.s.t0 + r / a.group, (h * a.group + r % a.group) * D + d, o * (l == 0.0f ? 0.0f : 1.0f / l));
    }
}

// Row blocks of a sequence and splits of a block, both at most: the grid stays
// within twice the slots, or has no splits.
static void wide_plan(int dim, int group, int hkv, int n_seqs, int max_new, int64_t cap, int &row_blocks, int &splits) {
    row_blocks = (max_new * group + kWideRows - 1) / kWideRows;
    const int64_t items = (int64_t)row_blocks * n_seqs * hkv, tiles = (cap + kTile - 1) / kTile;
    splits = (int)std::max<int64_t>(1, std::min(2 * wide_slots(dim) / items, (tiles + kWideChunk - 1) / kWideChunk));
    splits = std::min(splits, std::max(1, wide_slots(dim) / (row_blocks * hkv)));  // one sequence has all its blocks
}

size_t kv_attn_wide_workspace(int dim, int group, int hkv, int n_seqs, int max_new, int64_t cap) {
    int row_blocks, splits;
    wide_plan(dim, group, hkv, n_seqs, max_new, cap, row_blocks, splits);
    if (splits == 1) return 0;
    return (size_t)row_blocks * hkv * n_seqs * splits * kWideRows * (dim + 2) * sizeof(float);
}

// A split block's states are no more than twice the slots, nor a whole one's (behind a prefix
// they have one each) than the blocks: neither falls with the call.
size_t kv_attn_wide_room(int dim, int group, int hkv, int n_seqs, int n_tokens, int max_new, int64_t cap, bool shared) {
    int row_blocks, splits;
    wide_plan(dim, group, hkv, n_seqs, max_new, cap, row_blocks, splits);
    const int64_t tiles = (cap + kTile - 1) / kTile, most = (tiles + kWideChunk - 1) / kWideChunk;
    int64_t states = most > 1 ? std::min<int64_t>(2 * wide_slots(dim), (int64_t)row_blocks * hkv * n_seqs * most) : 0;
    if (shared) states = std::max(states, most_row_blocks(group, n_seqs, n_tokens, max_new) * hkv);
    return (size_t)states * kWideRows * (dim + 2) * sizeof(float);
}

// LDS past 64 KiB has to be allowed, per device.
template <int D, int FMT, bool LO, bool PREFIX = false>
static hipError_t wide_allow() {
    static std::atomic<int> state[64];
    if (WideShape<D, FMT, LO>::template lds_bytes<PREFIX>() <= 64 * 1024) return hipSuccess;
    if constexpr (PREFIX) return allow_full_lds(reinterpret_cast<const void *>(kv_attn_prefix_kernel<D, FMT, LO>), state);
    else return allow_full_lds(reinterpret_cast<const void *>(kv_attn_wide_kernel<D, FMT, LO>), state);
}

hipError_t kv_attn_prepare() {
    hipError_t e = hipSuccess;
    const auto all = [&](auto... f) { ((e = e == hipSuccess ? f() : e), ...); };
    all(wide_allow<128, kFmtI8, false>, wide_allow<128, kFmtI8, true>, wide_allow<128, kFmtE4M3, false>,
        wide_allow<128, kFmtE4M3, true>, wide_allow<256, kFmtI8, false>, wide_allow<256, kFmtI8, true>,
        wide_allow<256, kFmtE4M3, false>, wide_allow<256, kFmtE4M3, true>);
    all(wide_allow<128, kFmtI8, false, true>, wide_allow<128, kFmtI8, true, true>, wide_allow<128, kFmtE4M3, false, true>,
        wide_allow<128, kFmtE4M3, true, true>, wide_allow<256, kFmtI8, false, true>, wide_allow<256, kFmtI8, true, true>,
        wide_allow<256, kFmtE4M3, false, true>, wide_allow<256, kFmtE4M3, true, true>);
    return e;
}

WideGrid kv_attn_wide_grid(int dim, int hkv, int n_seqs, int max_new, int64_t cap, const AttnArgs &a) {
    WideGrid g;
    int row_blocks;
    wide_plan(dim, a.group, hkv, n_seqs, max_new, cap, row_blocks, g.splits);
    if (a.window > 0) {  // a row block's tokens, their windows and the first tokens
        const int64_t seen = (int64_t)a.window + kWideRows / a.group + 2 * kTile + (a.sinks > 0 ? a.sinks + kTile : 0);
        g.splits = (int)std::min<int64_t>(g.splits, (seen / kTile + kWideChunk - 1) / kWideChunk);
    }
    // behind a prefix every block is joined: the grid is of those that the rows can make
    // (64 sequences, one with 2048 tokens: 716 pairs of 28672), and of blocks that have a state
    g.items = (a.shared > 0 ? a.row_blocks : (int64_t)row_blocks * n_seqs) * hkv;
    g.few = g.splits + (a.shared > 0 ? (a.shared + a.prefix_run - 1) / a.prefix_run : 0) <= kJoinFew;
    g.join = g.splits == 1 && a.shared == 0 ? 0 : g.items * (g.few ? kWideRows / 8 : kWideRows);
    return g;
}

template <int D, int FMT, bool LO>
static hipError_t wide_run(const KvView &c, const AttnArgs &a, hipStream_t stream) {
    const WideGrid g = kv_attn_wide_grid(D, c.hkv, c.n_seqs, c.max_new, (int64_t)c.max_pages << c.page_shift, a);
    typedef WideShape<D, FMT, LO> W;
    constexpr size_t kLds = W::template lds_bytes<false>();
    const hipError_t allowed = wide_allow<D, FMT, LO>();
    if (allowed != hipSuccess) return allowed;
    const int cus = device_cus();
    const int turn = c.n_seqs == 1 && g.splits == 1 && cus % c.hkv == 0 && g.items >= 2 * cus ? cus / c.hkv : 1 << 29;
    kv_attn_wide_kernel<D, FMT, LO><<<(unsigned)(g.items * g.splits), W::kThreads, kLds, stream>>>(c, a, g.splits, turn);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || g.join == 0) return e;
    if (g.few && a.shared > 0) kv_attn_wide_join_few_kernel<D, true><<<(unsigned)g.join, 256, 0, stream>>>(c, a, g.splits);
    else if (g.few) kv_attn_wide_join_few_kernel<D, false><<<(unsigned)g.join, 256, 0, stream>>>(c, a, g.splits);
    else kv_attn_wide_join_kernel<D><<<(unsigned)g.join, 256, 0, stream>>>(c, a, g.splits);
    return hipGetLastError();
}

template <int D>
static hipError_t wide_dim(const KvView &c, int fmt, const AttnArgs &a, hipStream_t stream) {
    if (fmt == MGQ_KV_I8)
        return a.out_f16 ? wide_run<D, kFmtI8, false>(c, a, stream) : wide_run<D, kFmtI8, true>(c, a, stream);
    return a.out_f16 ? wide_run<D, kFmtE4M3, false>(c, a, stream) : wide_run<D, kFmtE4M3, true>(c, a, stream);
}

hipError_t kv_attn_wide_launch(const KvView &c, int dim, int fmt, const AttnArgs &a, hipStream_t stream) {
    switch (dim) {
    case 64: return wide_dim<64>(c, fmt, a, stream);
    case 96: return wide_dim<96>(c, fmt, a, stream);
    case 128: return wide_dim<128>(c, fmt, a, stream);
    default: return wide_dim<256>(c, fmt, a, stream);
    }
}

// Of 4 wavefronts two a CU, of 8 one: kPerSimd of both.
template <int D, int FMT, bool LO>
constexpr int prefix_slots() {
    return 256 * 4 * WideShape<D, FMT, LO>::kPerSimd / WideShape<D, FMT, LO>::NW;
}
template <int D>
static int prefix_slots_of(int fmt, bool out_f16) {
    if (fmt == MGQ_KV_I8) return out_f16 ? prefix_slots<D, kFmtI8, false>() : prefix_slots<D, kFmtI8, true>();
    return out_f16 ? prefix_slots<D, kFmtE4M3, false>() : prefix_slots<D, kFmtE4M3, true>();
}
int kv_attn_prefix_slots(int dim, int fmt, bool out_f16) {
    switch (dim) {
    case 64: return prefix_slots_of<64>(fmt, out_f16);
    case 96: return prefix_slots_of<96>(fmt, out_f16);
    case 128: return prefix_slots_of<128>(fmt, out_f16);
    default: return prefix_slots_of<256>(fmt, out_f16);
    }
}

template <int D, int FMT, bool LO>
static hipError_t prefix_run(const KvView &c, const AttnArgs &a, hipStream_t stream) {
    typedef WideShape<D, FMT, LO> W;
    const hipError_t allowed = wide_allow<D, FMT, LO, true>();
    if (allowed != hipSuccess) return allowed;
    kv_attn_prefix_kernel<D, FMT, LO><<<(unsigned)(prefix_runs(a) * c.hkv), W::kThreads, W::template lds_bytes<true>(),
                                        stream>>>(c, a);
    return hipGetLastError();
}

template <int D>
static hipError_t prefix_dim(const KvView &c, int fmt, const AttnArgs &a, hipStream_t stream) {
    if (fmt == MGQ_KV_I8)
        return a.out_f16 ? prefix_run<D, kFmtI8, false>(c, a, stream) : prefix_run<D, kFmtI8, true>(c, a, stream);
    return a.out_f16 ? prefix_run<D, kFmtE4M3, false>(c, a, stream) : prefix_run<D, kFmtE4M3, true>(c, a, stream);
}

hipError_t kv_attn_prefix_launch(const KvView &c, int dim, int fmt, const AttnArgs &a, hipStream_t stream) {
    switch (dim) {
    case 64: return prefix_dim<64>(c, fmt, a, stream);
    case 96: return prefix_dim<96>(c, fmt, a, stream);
    case 128: return prefix_dim<128>(c, fmt, a, stream);
    default: return prefix_dim<256>(c, fmt, a, stream);
    }
}

}  // namespace mgq
