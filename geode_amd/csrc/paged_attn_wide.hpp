// paged_attn_wide.hpp - the paged attention of many columns (drafts x query heads of a KV head), head_dim above 64.
//
// The few-column kernel (paged_attn.hpp) holds a column tile's whole O^T (dims x 16 columns) in each wave's registers; with
// three tiles of 256 dims that is 192 registers, and with a workgroup a tile the keys and values are read once a tile
// (three tiles: 57 us where one reading takes 22, the L2's bandwidth). Here a round of 64 positions is the workgroup's:
//   * wave w makes S^T of positions 16 w .. + 15 for all CT column tiles (its keys in registers, as there);
//   * the weights go through LDS (16-bit parts, 2 KB a column tile and round), in the layout the second product takes them in;
//   * each wave then makes O^T of 64 of the dims for all columns: values of those dims alone, CT x 16 registers of sums.
//     head_dim 256: four waves of 64 dims, all 64 positions each; head_dim 128: two by two, 32 positions each, added at the end.
// So keys and values are read once for CT x 16 columns, by registers' worth of 16 positions or 64 dims.
// The columns' maximum over the round has to be known to all four waves before the weights are made: it goes through LDS
// too, a round ahead of its use. A round between two barriers: O^T of the round before; the weights of this round; S^T and
// the maxima of the next - one barrier a round, the weights and maxima in two buffers.
// 32 sequences of up to 4,096 positions and 5 rows, 16 heads of 256 on 2, fp16 (108 MB) 36 us, in which CT tiles are worked also
// where a sequence has columns for one; one of 32,001 positions and 17 rows, int8: 45 us, of which a SIMD spends 18.7 on the
// vector instructions (the softmax of every column, int8 codes made fp16) and 7.5 on products. The rest are waits: keys and
// values are asked for one round ahead, each round ends in a barrier, and the LDS (74 KB) leaves room for two workgroups a CU.
#pragma once

#include "paged_attn.hpp"

namespace gv {

template <int NT, int CT, int QP, int PP>
constexpr int attn_wide_lds() {
    return CT * QP * (NT / 2) * 1024 + 2 * 2 * CT * PP * 1024;
}

// Values that are not finite and that only some columns see (a sequence's own rows; v: an operand, rows: its rows that
// are such rows, two to a word as there). In the product they would reach every column (0 x inf is no number), so they are
// taken out of it, and the columns that see one (seen: their ones, as the weights' operand) have the dim's sum made NaN.
template <bool BF>
__device__ inline uint32_t not_finite(uint32_t w) {
    constexpr uint32_t e = BF ? 0x7F80u : 0x7C00u;
    return ((w & e) == e ? 0xFFFFu : 0u) | ((w >> 16 & e) == e ? 0xFFFF0000u : 0u);
}
template <bool BF, int CT, int PP>
__device__ inline void guarded_product(au4 v, const uint32_t (&rows)[4], const au4 (&weight)[CT][PP], const au4 (&seen)[CT],
                                       af4 (&acc)[CT]) {
    au4 flag;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bad = not_finite<BF>(v[i]) & rows[i];
        v[i] &= ~bad;
        flag[i] = bad & (BF ? 0x3F803F80u : 0x3C003C00u);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
        for (int q = 0; q < PP; ++q) acc[ct] = mfma<BF>(v, weight[ct][q], acc[ct]);
        const af4 hit = mfma<BF>(flag, seen[ct], af4{0, 0, 0, 0});
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[ct][r] = hit[r] > 0.0f ? __builtin_nanf("") : acc[ct][r];
    }
}
// the bits of 8 positions as an operand's words: masks, or ones of its type
__device__ inline void bit_pairs(uint32_t bits, uint32_t word, uint32_t (&out)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = word & ((bits >> (2 * i) & 1 ? 0xFFFFu : 0u) | (bits >> (2 * i + 1) & 1 ? 0xFFFF0000u : 0u));
}

template <int KV, int QP, int PP, int NT, bool EX, int CT>
__device__ inline void attn_many_columns(const AttnArgs &a, const AttnUnit &u) {
    constexpr bool BF = KV == GV_BF16, I8 = KV == GV_I8;
    constexpr int ES = I8 ? 1 : 2;
    constexpr int NCH = NT / 2, KL = I8 ? NCH / 2 : NCH;
    constexpr int DW = NT / 4;             // waves that share the dims (64 each)
    constexpr int KS = 2 / (4 / DW);       // 32-position products a wave makes of a round's values
    constexpr int VW = ES;                 // words a lane a value row: four dims
    constexpr int kRound = 64;
    extern __shared__ au4 lds_q[];         // [CT][QP][NCH][64], then the weights [2][2][CT][PP][64]
    au4 *lds_p = lds_q + CT * QP * NCH * 64;
    __shared__ float lds_amax[CT * 16], lds_max[2][kAttnWaves][CT * 16], lds_wmax[I8 ? 2 : 1][kAttnWaves][CT * 16];
    const int lane = threadIdx.x & 63, i16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int dq = wave % DW, pg = wave / DW;   // which 64 dims, which of the round's products
    const Seq &s = u.s;
    const int p0 = u.p0, p1 = u.p1, ctx = u.ctx;
    const auto qu = load_queries<I8, QP, NCH, EX, CT>(a, u);
    // every tile of the chunk a lane (chunks of at most 1,024)
    const AttnTiles at = attn_tiles(a, u, p0 + 16 * lane, 16 * lane < a.chunk);

    const uint32_t klane = (static_cast<uint32_t>(i16) * static_cast<uint32_t>(a.kv.pos_stride) + g4 * (I8 ? 16 : 8)) * ES;
    const int vdim = dq * 64 + i16 * 4;
    const uint32_t vlane = (static_cast<uint32_t>(4 * g4) * static_cast<uint32_t>(a.kv.pos_stride) + vdim) * ES;
    const uint32_t vrow = static_cast<uint32_t>(a.kv.pos_stride) * ES;
    au4 kf[KL];
    float ksc[4], vsc_next[4];
    const auto load_k = [&](int t) {   // this wave's tile of round t
        const auto kb = place(a.kv.k + lane64(at.off, 4 * t + wave) * ES);
#pragma unroll
        for (int c = 0; c < KL; ++c) {
            constexpr uint32_t per = I8 ? 64 : 32 * ES;
            if constexpr (EX) {
                kf[c] = load16(kb, klane + c * per, 0);
            } else {
                const int d = I8 ? c * 64 + g4 * 16 : c * 32 + g4 * 8;
                kf[c] = load16(kb, d < a.kv.hd ? klane + c * per : kNowhere, 0);
            }
        }
        if constexpr (I8) {
            const int64_t so = lane64(at.scale_off, 4 * t + wave);
            const float4 x = load4f(a.kv.ks + so, 16 * g4), y = load4f(a.kv.vs + so, 16 * g4);
            ksc[0] = x.x, ksc[1] = x.y, ksc[2] = x.z, ksc[3] = x.w;
            vsc_next[0] = y.x, vsc_next[1] = y.y, vsc_next[2] = y.z, vsc_next[3] = y.w;
        }
    };
    uint32_t vr[KS][8][VW];
    const auto load_v = [&](int t) {   // 64 dims of its 32 or 64 positions
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const auto vb = place(a.kv.v + lane64(at.off, 4 * t + 2 * (pg * KS + k) + h) * ES);
                const uint32_t lo = EX || vdim < a.kv.hd ? vlane : kNowhere;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (VW == 2) {
                        const au2 x = load8b(vb, lo, r * vrow);
                        vr[k][4 * h + r][0] = x[0], vr[k][4 * h + r][1] = x[1];
                    } else {
                        vr[k][4 * h + r][0] = load4b(vb, lo, r * vrow);
                    }
                }
            }
    };
    const int rounds = (p1 - p0 + kRound - 1) / kRound;
    load_k(0);   // (on its way while the queries are made ready)
    const QueryScale qs = stage_queries<BF, I8, QP, NCH, CT>(a, qu, lds_q, lds_amax);

    float sc[CT], m[CT], l[CT], most[CT], up[CT];   // (as there)
    uint32_t bits[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        sc[ct] = a.scale * qs.undo(ct) * (I8 ? kI8Unit : 1.0f);
        m[ct] = most[ct] = -INFINITY, l[ct] = 0.0f, up[ct] = I8 ? weight_factor(-INFINITY) : 16384.0f;
        bits[ct] = seen_rows(a, u, u.q0 + ct * 16 + i16);
    }
    af4 acc[4][CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n][ct] = af4{0, 0, 0, 0};

    // ---- S^T of round t (scores in sv, masked; the value scales with them), its maxima to LDS
    af4 sv[CT];
    float vsc[4];
    const auto scores = [&](int t) {
        int ql = lane;   // (pinned: the queries are read from LDS in every round, not kept in registers)
        asm volatile("" : "+v"(ql));
        af4 part[CT][QP];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int q = 0; q < QP; ++q) part[ct][q] = af4{0, 0, 0, 0};
        // (a chunk's queries are read while the chunk before is in the products; the barriers keep the compiler from reading
        // further ahead, for which there are no registers)
        au4 qb[2][CT][QP];
        const auto read_q = [&](int c) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int q = 0; q < QP; ++q) qb[c & 1][ct][q] = lds_q[((ct * QP + q) * NCH + c) * 64 + ql];
        };
        read_q(0);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            if (c + 1 < NCH) read_q(c + 1);
            au4 kk;
            if constexpr (I8) {
                const uint32_t w0 = kf[c / 2][2 * (c & 1)] ^ 0x80808080u, w1 = kf[c / 2][2 * (c & 1) + 1] ^ 0x80808080u;
                kk = au4{i8_pair(0, w0, 0x0C010C00u), i8_pair(0, w0, 0x0C030C02u), i8_pair(0, w1, 0x0C010C00u), i8_pair(0, w1, 0x0C030C02u)};
            } else {
                kk = kf[c];
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int q = 0; q < QP; ++q) part[ct][q] = mfma<BF>(kk, qb[c & 1][ct][q], part[ct][q]);
            __builtin_amdgcn_sched_barrier(0);
        }
        const int p = p0 + kRound * t + 16 * wave;
        const bool use = at.usable >> (4 * t + wave) & 1, tail = p + 16 > ctx || !use;   // (uniform)
        float f[4], vlog[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            f[r] = I8 ? ksc[r] : 1.0f;
            if constexpr (I8) vsc[r] = vsc_next[r], vlog[r] = __builtin_amdgcn_logf(fabsf(vsc[r]));
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            af4 x = part[ct][0];
#pragma unroll
            for (int q = 1; q < QP; ++q) x += part[ct][q];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[r] *= I8 ? sc[ct] * f[r] : sc[ct];
                if (tail) {
                    const int pos = p + 4 * g4 + r;
                    const bool seen = use && pos < p1 && (pos < ctx || (bits[ct] >> ((pos - ctx) & 31) & 1));
                    x[r] = seen ? x[r] : -INFINITY;
                }
            }
            sv[ct] = x;
            const float top = rows_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
            float wtop = -INFINITY;   // log2 of the largest weight x scale, relative to `top`
            if constexpr (I8) {
                const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (int r = 0; r < 4; ++r) wtop = fmaxf(wtop, __builtin_fmaf(x[r] - base, kLog2e, vlog[r]));
                wtop = rows_max(wtop);
            }
            if (lane < 16) {
                lds_max[t & 1][wave][ct * 16 + lane] = top;
                if constexpr (I8) lds_wmax[t & 1][wave][ct * 16 + lane] = wtop;
            }
        }
    };
    // ---- the columns' maxima with round t's, the sums brought to them; round t's weights to LDS
    const auto weights = [&](int t) {
        const bool tail = p0 + kRound * t + 16 * wave + 16 > ctx || !(at.usable >> (4 * t + wave) & 1);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float mn = m[ct], theirs[kAttnWaves];
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) theirs[w] = lds_max[t & 1][w][ct * 16 + i16], mn = fmaxf(mn, theirs[w]);
            const float down = mn == m[ct] ? 0.0f : (m[ct] - mn) * kLog2e;
            float wn = most[ct] + down;
            if constexpr (I8)
#pragma unroll
                for (int w = 0; w < kAttnWaves; ++w)   // (of a wave that saw nothing: -inf, or no number, which is passed over)
                    wn = fmaxf(wn, __builtin_fmaf(theirs[w] - mn, kLog2e, lds_wmax[t & 1][w][ct * 16 + i16]));
            if (__any(mn > m[ct] || wn > most[ct])) {
                float f = __builtin_amdgcn_exp2f(down);
                l[ct] *= f;
                if constexpr (I8) {
                    const float now = weight_factor(wn);
                    f = __builtin_amdgcn_exp2f(down + log2_ratio(now, up[ct]));
                    most[ct] = wn, up[ct] = now;
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) acc[n][ct] *= f;
                m[ct] = mn;
            }
            const float base = mn == -INFINITY ? 0.0f : mn;
            float x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[r] = __builtin_amdgcn_exp2f((sv[ct][r] - base) * kLog2e);
                l[ct] += x[r];
                if constexpr (I8) {
                    const float w = x[r] * vsc[r] * up[ct];
                    x[r] = tail && sv[ct][r] == -INFINITY ? 0.0f : w;   // (a scale that is not seen may be anything)
                } else if constexpr (!BF) {
                    x[r] *= up[ct];
                }
            }
            uint2 part[PP];
            split4<BF, PP>(x, part);
#pragma unroll
            for (int q = 0; q < PP; ++q)   // [product wave / 2][column tile][part][lane]: the tile's four positions of the lane's eight
                reinterpret_cast<uint2 *>(lds_p + ((((t & 1) * 2 + wave / 2) * CT + ct) * PP + q) * 64 + lane)[wave & 1] = part[q];
        }
    };
    // ---- O^T of round t
    const auto v_tile = [&](int k, int n) {
        au4 v;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            if constexpr (I8) {
                const uint32_t lo = vr[k][2 * jj][0] ^ 0x80808080u, hi = vr[k][2 * jj + 1][0] ^ 0x80808080u;
                v[jj] = i8_pair(hi, lo, 0x0C000C00u | static_cast<uint32_t>(n) | static_cast<uint32_t>(4 + n) << 16);
            } else {
                v[jj] = perm(vr[k][2 * jj + 1][n / 2], vr[k][2 * jj][n / 2], n & 1 ? 0x07060302u : 0x05040100u);
            }
        }
        return v;
    };
    const auto products = [&](int t) {
        const au4 *pt = lds_p + ((t & 1) * 2 + pg * KS) * CT * PP * 64 + lane;
        const bool tail = p0 + kRound * (t + 1) > ctx || at.lost;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            au4 pb[CT][PP];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int q = 0; q < PP; ++q) pb[ct][q] = pt[((k * CT + ct) * PP + q) * 64];
            if constexpr (!I8) {   // (int8: a hole's weights are 0 and its codes finite)
                if (tail) {
                    const int p = p0 + kRound * t + 32 * (pg * KS + k), bit = 4 * t + 2 * (pg * KS + k);
                    uint32_t own = 0;   // (bit j: the lane's position j is one of the sequence's rows)
                    bool wild = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int pos = p + 16 * (j / 4) + 4 * g4 + j % 4;
                        const bool hole = pos >= p1 || !(at.usable >> (bit + j / 4) & 1);
#pragma unroll
                        for (int i = 0; i < VW; ++i) vr[k][j][i] = hole ? 0u : vr[k][j][i];
                        if (pos >= ctx) own |= 1u << j;
                        wild |= pos >= ctx && any_not_finite<BF, VW>(vr[k][j]);
                    }
                    if (__any(wild)) {
                        uint32_t rows[4];
                        bit_pairs(own, 0xFFFFFFFFu, rows);
                        au4 seen[CT];
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct) {
                            uint32_t see = 0, w[4];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const int row = p + 16 * (j / 4) + 4 * g4 + j % 4 - ctx;
                                if (row >= 0 && row < 32 && (bits[ct] >> row & 1)) see |= 1u << j;
                            }
                            bit_pairs(see, BF ? 0x3F803F80u : 0x3C003C00u, w);
                            seen[ct] = au4{w[0], w[1], w[2], w[3]};
                        }
                        // (the rows pinned: their transposition would else be made, and kept, for both ways on)
#pragma unroll
                        for (int r = 0; r < 8; ++r)
#pragma unroll
                            for (int i = 0; i < VW; ++i) asm volatile("" : "+v"(vr[k][r][i]));
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            guarded_product<BF, CT, PP>(v_tile(k, n), rows, pb, seen, acc[n]);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        continue;
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const au4 v = v_tile(k, n);
#pragma unroll
                for (int q = 0; q < PP; ++q)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) acc[n][ct] = mfma<BF>(v, pb[ct][q], acc[n][ct]);
            }
        }
    };

    // (each part of a round once in the code: the first time round makes the first scores alone)
    for (int t = -1;; ++t) {
        if (t >= 0) weights(t);
        if (t + 1 < rounds) {
            scores(t + 1);
            if (t + 2 < rounds) load_k(t + 2);
        }
        __syncthreads();
        if (t >= 0) products(t);
        if (t + 1 == rounds) break;
        load_v(t + 1);
    }
    __syncthreads();   // (the queries' place is used again)

    // ---- the sums of weights over the waves; two waves of the same dims added; then out
    float *lds_l = reinterpret_cast<float *>(lds_q);   // [wave][CT * 16] (the queries are done with), then the sums
    af4 *lds_o = reinterpret_cast<af4 *>(lds_q + kAttnWaves * CT * 4);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        l[ct] = rows_sum(l[ct]);
        if (lane < 16) lds_l[wave * CT * 16 + ct * 16 + lane] = l[ct];
    }
    if constexpr (DW == 2) {
        if (pg == 1)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int n = 0; n < 4; ++n) lds_o[((dq * CT + ct) * 4 + n) * 64 + lane] = acc[n][ct];
    }
    __syncthreads();
    if (DW == 2 && pg == 1) return;
    const bool whole = s.len <= a.chunk;
    const int qes = a.type == GV_F32 ? 4 : 2;
    int el = lane;   // (pinned: the rows' places are worked out here, not kept through the rounds)
    asm volatile("" : "+v"(el));
    const int c16 = el & 15, e4 = el >> 4;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int x = u.q0 + ct * 16 + c16;
        if (x >= u.nq) continue;
        if constexpr (DW == 2)
#pragma unroll
            for (int n = 0; n < 4; ++n) acc[n][ct] += lds_o[((dq * CT + ct) * 4 + n) * 64 + lane];
        float ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) ll += lds_l[w * CT * 16 + ct * 16 + c16];
        const int xr = row_of(a, x), row = s.first + xr, hq = u.head * a.group + x - xr * a.group;
        const float unit_v = BF ? 1.0f : I8 ? kI8Unit / up[ct] : 1.0f / 16384.0f;
        const bool some = ll > 0.0f || ll != ll;
        const int64_t to = (static_cast<int64_t>(u.chunk) * a.b.n_rows + row) * a.nh + hq;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = dq * 64 + (4 * e4 + r) * 4;
            if (!EX && d >= a.kv.hd) continue;
            float4 v = float4{acc[0][ct][r] * unit_v, acc[1][ct][r] * unit_v, acc[2][ct][r] * unit_v, acc[3][ct][r] * unit_v};
            if (!whole) {
                store4<GV_F32>(reinterpret_cast<char *>(a.parts + to * a.kv.hd + d), v);
                continue;
            }
            v = some ? float4{v.x / ll, v.y / ll, v.z / ll, v.w / ll} : float4{0, 0, 0, 0};
            char *dst = a.out + (row * a.out_row + static_cast<int64_t>(hq) * a.kv.hd + d) * qes;
            if (a.type == GV_F32) store4<GV_F32>(dst, v);
            else if (a.type == GV_F16) store4<GV_F16>(dst, v);
            else store4<GV_BF16>(dst, v);
        }
        if (dq == 0 && e4 == 0) {
            if (!whole) *reinterpret_cast<float2 *>(a.ml + to * 2) = float2{joined_max(m[ct], ll), ll};
            else if (a.lse) a.lse[static_cast<int64_t>(row) * a.nh + hq] = some ? m[ct] + logf(ll) : -INFINITY;
        }
    }
}

// (two workgroups a CU, where the LDS has room for them and the registers for the compiler)
template <int KV, int QP, int PP, int NT, bool EX, int CT>
__global__ __launch_bounds__(kAttnThreads, (NT == 16 && (QP > 2 || (!EX && QP > 1)) ? 1 : 2)) void paged_attn_wide_kernel(const AttnArgs a) {
    touch_args(a);
    AttnUnit u;
    if (attn_unit<CT, false>(a, blockIdx.x, u) > 0) attn_many_columns<KV, QP, PP, NT, EX, CT>(a, u);
}

template <int KV, int QP, int PP, int NT, bool EX>
int launch_attn_wide(const AttnArgs &a, unsigned grid, hipStream_t st) {
    constexpr int CT = kWideTiles, lds = attn_wide_lds<NT, CT, QP, PP>();
    static int granted = 0;
    if (lds_grant(reinterpret_cast<const void *>(&paged_attn_wide_kernel<KV, QP, PP, NT, EX, CT>), lds, granted) != 0) return -1;
    hipLaunchKernelGGL((paged_attn_wide_kernel<KV, QP, PP, NT, EX, CT>), dim3(grid), dim3(kAttnThreads), lds, st, a);
    GV_CHECK_HIP(hipGetLastError());
    return 0;
}

// ---------------------------------------------------------------- the kernel of a call
template <int KV, int QP, int PP, int NT, bool EX>
int launch_attn_ct(const AttnArgs &a, int ct, unsigned grid, hipStream_t st) {
    if (ct == 1) return launch_attn_few<KV, QP, PP, NT, EX, 1>(a, grid, st);
    if constexpr (NT == 4) return launch_attn_few<KV, QP, PP, NT, EX, kWideTiles>(a, grid, st);
    else return launch_attn_wide<KV, QP, PP, NT, EX>(a, grid, st);
}
template <int KV, int QP, int PP>
int launch_attn_nt(const AttnArgs &a, int ct, unsigned grid, hipStream_t st) {
    switch (a.kv.hd) {
    case 64: return launch_attn_ct<KV, QP, PP, 4, true>(a, ct, grid, st);
    case 128: return launch_attn_ct<KV, QP, PP, 8, true>(a, ct, grid, st);
    case 256: return launch_attn_ct<KV, QP, PP, 16, true>(a, ct, grid, st);
    }
    return a.kv.hd < 64 ? launch_attn_ct<KV, QP, PP, 4, false>(a, ct, grid, st)
           : a.kv.hd < 128 ? launch_attn_ct<KV, QP, PP, 8, false>(a, ct, grid, st)
                           : launch_attn_ct<KV, QP, PP, 16, false>(a, ct, grid, st);
}

}  // namespace gv
