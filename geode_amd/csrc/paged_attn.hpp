// paged_attn.hpp - attention of a few rows a sequence over a paged cache, on the matrix cores. The kernels' template;
// paged_attn_f16.hip, paged_attn_bf16.hip and paged_attn_i8.hip build it for a cache type each.
//
// For a sequence and a KV head, the rows x the query heads that share the head are the columns of S^T = K Q^T (positions
// x queries) and O^T = V^T P^T (dims x queries). A wave takes 32 positions a step (two tiles of 16, each within a page):
//   * K tile [16 positions][hd]: a lane's 16-byte loads are MFMA operands as they are (lane: position lane % 16, dims
//     8 (lane / 16) ..).
//   * S^T comes out with lane (query lane % 16, positions 4 (lane / 16) .. + 3 of each tile), which is the layout the
//     second product takes P^T in, when its 8 values a lane are positions {4 g .. 4 g + 3} of the first tile, then of
//     the second: the weights never leave the registers.
//   * V rows of those 8 positions: a lane loads NT consecutive dims of each (coalesced over lane % 16) and transposes
//     the 8 x NT values among its own registers (v_perm_b32, 16-bit pairs): the operand of dim tile n holds dims
//     {i NT + n}, so no LDS is touched and nothing is stored transposed in the cache.
// Running maximum and sum a query (fp32); the accumulators are multiplied only in steps where some maximum rose.
// The four waves of a workgroup take steps in turn over a chunk of positions and are joined in LDS; a sequence of one
// chunk is finished there, else the chunk's sums go to the workspace and paged_join_kernel (paged_attn.hip) joins them.
//
// Rounding: queries and weights go to the matrix cores as PARTS 16-bit parts (fp16: 11 bits each, bf16: 8), keys and
// values exactly (int8: as fp16 (code) / 512); products are summed in fp32. A query exact in the cache's type is one
// part, an fp32 one two of fp16 (truncated: 2^-21 at most, down to 2^-35 of its row's largest) or three of bf16 (exact); the
// weights are two parts (bf16: off by 2^-16 at most, for results of 8 bits; fp16: truncated, by 2^-21) or, for fp32 results
// over bf16, three (exact). fp16 parts are taken of values scaled by powers of two (queries by their row's
// largest value, weights by 2^14, an int8 cache's weights x value scales by their largest's: weight_factor), so that neither
// overflows nor, where it counts, falls below fp16's range.
// The weights' exponential takes the difference to the maximum: exp2((s - m) log2 e), accurate whatever the scores' size.
//
// Bound by the bytes of keys and values where there are many (131,073 positions, 2 KV heads of 256, fp16, 268 MB: 51 us; 64
// sequences of up to 8,192, 8 KV heads of 128, bf16, 702 MB: 135 us; 5.2 TB/s), by its chain of loads (lengths, pages,
// then keys, values and queries) where there are few (one sequence of 1,003 positions: 10.3 us).
#pragma once

#include <type_traits>

#include "paged.hpp"

namespace gv {

typedef _Float16 ah8 __attribute__((ext_vector_type(8)));
typedef _Float16 ah2 __attribute__((ext_vector_type(2)));
typedef __bf16 ab8 __attribute__((ext_vector_type(8)));
typedef float af4 __attribute__((ext_vector_type(4)));
typedef uint32_t au4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
    KvView kv;
    BatchView b;
    const char *q;
    char *out;
    float *lse;
    const uint32_t *visible;
    float *parts, *ml;   // [chunk][row][head][hd] sums, [chunk][row][head][2] (maximum, sum of weights)
    int64_t q_row, out_row;
    int nh, group;       // query heads, and those of a KV head
    float group_inv;     // 1 / group
    int type;            // of q and out
    int chunk, n_chunks; // positions a workgroup takes; chunks of max_len
    int col_groups;      // groups of CT x 16 columns that max_rows x group take
    int inner_heads;     // KV heads whose workgroups follow each other: 1 or all of them
    float scale;
    int *faults;
};

constexpr int kAttnThreads = 256, kAttnWaves = 4, kAttnStep = 32;
constexpr int kAttnMaxRows = 32;

// a kernel's LDS: the queries' operands, then (in the same place) the waves' sums of one column tile
template <int NT, int CT, int QP>
constexpr int attn_lds() {
    constexpr int q = CT * QP * (NT / 2) * 64 * 16;
    constexpr int o = kAttnWaves * 16 * (NT * 16 + 4) * 4;
    return q > o ? q : o;
}

// waves a SIMD a kernel's registers leave room for (asked of the compiler: more, and it spills)
template <int NT, int CT, bool COUNTED>
constexpr int attn_waves() {
    if (CT > 1) return COUNTED ? 1 : 2;
    if (COUNTED) return NT == 16 ? 1 : 3;   // (the loop over the units takes a few more)
    return NT == 4 ? 4 : NT == 8 ? 3 : 2;
}

__device__ inline uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }

// the maximum / sum over the four 16-lane rows, in every lane (each lane keeps its column)
__device__ inline void rows_pair(float v, int step16, float &a, float &b) {   // v of the two 16-lane rows (halves) of a pair
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = step16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t x = r[0], y = r[1];   // (a vector's element itself is not what a bit cast reads)
    a = __builtin_bit_cast(float, x), b = __builtin_bit_cast(float, y);
}
__device__ inline float rows_max(float v) {
    float a, b;
    rows_pair(v, 1, a, b);
    rows_pair(fmaxf(a, b), 0, a, b);
    return fmaxf(a, b);
}
__device__ inline float rows_sum(float v) {
    float a, b;
    rows_pair(v, 1, a, b);
    rows_pair(a + b, 0, a, b);
    return a + b;
}

// N parts of K floats in the operand's type, two to a word: each part the leading bits of what the parts before left
// (truncated, so that the rest is exact; the last of bf16 parts rounded to nearest, the same one instruction)
template <bool BF, int N, int K, typename Part>
__device__ inline void split_parts(const float (&x)[K], Part &&put) {
    float r[K];
#pragma unroll
    for (int j = 0; j < K; ++j) r[j] = x[j];
#pragma unroll
    for (int p = 0; p < N; ++p) {
#pragma unroll
        for (int j = 0; j < K; j += 2) {
            if constexpr (BF) {
                if (p + 1 == N) {
                    put(p, j / 2, pack_bf16(r[j], r[j + 1]));
                } else {
                    const uint32_t a = __builtin_bit_cast(uint32_t, r[j]), b = __builtin_bit_cast(uint32_t, r[j + 1]);
                    put(p, j / 2, perm(b, a, 0x07060302u));
                    r[j] -= __builtin_bit_cast(float, a & 0xFFFF0000u);
                    r[j + 1] -= __builtin_bit_cast(float, b & 0xFFFF0000u);
                }
            } else {
                const auto h = __builtin_amdgcn_cvt_pkrtz(r[j], r[j + 1]);
                put(p, j / 2, __builtin_bit_cast(uint32_t, h));
                if (p + 1 < N) {
                    r[j] -= static_cast<float>(h[0]);
                    r[j + 1] -= static_cast<float>(h[1]);
                }
            }
        }
    }
}
template <bool BF, int N>
__device__ inline void split8(const float (&x)[8], au4 (&part)[N]) {
    split_parts<BF, N>(x, [&](int p, int j, uint32_t w) { part[p][j] = w; });
}
template <bool BF, int N>
__device__ inline void split4(const float (&x)[4], uint2 (&part)[N]) {
    split_parts<BF, N>(x, [&](int p, int j, uint32_t w) { (j ? part[p].y : part[p].x) = w; });
}

template <bool BF>
__device__ inline af4 mfma(au4 a, au4 b, af4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ab8, a), __builtin_bit_cast(ab8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ah8, a), __builtin_bit_cast(ah8, b), c, 0, 0, 0);
}

// bytes (a, b) of two words, each + 128 (their sign bits turned before), as the fp16 pair (a / 512, b / 512): the byte
// is an fp16 subnormal b 2^-24, times 2^15, minus 128 / 512 (exact)
__device__ inline uint32_t i8_pair(uint32_t hi, uint32_t lo, uint32_t sel) {
    const ah2 b = __builtin_bit_cast(ah2, perm(hi, lo, sel));
    const ah2 v = __builtin_elementwise_fma(b, ah2{static_cast<_Float16>(32768.0f), static_cast<_Float16>(32768.0f)},
                                            ah2{static_cast<_Float16>(-0.25f), static_cast<_Float16>(-0.25f)});
    return __builtin_bit_cast(uint32_t, v);
}
constexpr float kI8Unit = 512.0f;   // a code's operand x this is the code

// An int8 cache's weights take the value scales with them, times a power of two that brings a column's largest weight x scale
// to 2^13 .. 2^14 (of all scales, whatever their weight, it would push the weights that count below fp16's range). most: log2 of
// the largest weight x scale so far, relative to the largest score (differences of scores alone, so that the scores' size costs
// it nothing); -inf: nothing seen yet. The factor is held between 2^-114 and 2^126 (weights x scales below 2^-113 lose bits).
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMostFactor = 126;
__device__ inline float weight_factor(float most) {
    const float e = fminf(fmaxf(floorf(most), 13.0f - kMostFactor), 127.0f);
    return __builtin_amdgcn_ldexpf(1.0f, 13 - static_cast<int>(e));
}
// log2 of one power of two over another
__device__ inline float log2_ratio(float a, float b) {
    return static_cast<float>((__float_as_int(a) - __float_as_int(b)) >> 23);
}

// ---------------------------------------------------------------- what both kernels begin with
// A workgroup's unit: a chunk of a sequence's positions, a KV head, CT column tiles.
struct AttnUnit {
    Seq s;
    int seq, head, chunk, p0, p1, ctx, nq, q0;   // positions [p0, p1) of len; ctx: those before its own rows; columns, first
};
// The index-th unit (false: there is none, or nothing in it to do). Column groups of a (sequence, chunk, KV head) follow
// each other on one XCD (workgroups go round the eight), where the second finds the first's keys and values in the L2; so do the
// KV heads where their rows share cache lines (inner_heads). The units are those of max_len, a chunk of every sequence after
// the other, and the ones past a sequence's end are empty; or (COUNTED) every wave counts the chunks that the lengths
// make, 64 sequences at a time, and takes the index-th of those.
template <int CT, bool COUNTED>
__device__ inline int attn_unit(const AttnArgs &a, unsigned index, AttnUnit &u) {   // 1: a unit, 0: an empty one, -1: past the last
    const unsigned xcd = index & 7, idx = index >> 3, groups = static_cast<unsigned>(a.col_groups);
    const unsigned inner = groups * static_cast<unsigned>(a.inner_heads), in = idx % inner;
    const unsigned cg = in % groups, outer_heads = static_cast<unsigned>(a.kv.nkv / a.inner_heads);
    unsigned unit = idx / inner * 8 + xcd, outer;
    const int lane = threadIdx.x & 63;
    if constexpr (COUNTED) {
        int base = 0;
        for (;; base += 64) {
            if (base >= a.b.n_seqs) return -1;
            const int i = min(base + lane, a.b.n_seqs - 1);
            const int first = a.b.row_start[i], last = a.b.row_start[i + 1], len = a.b.lens[i];
            const Seq s = make_seq(a.b, first, last, len);
            const bool mine = base + lane < a.b.n_seqs;
            if (mine && !s.fits) queue_fault(a.faults, kFaultRows);
            const int n = mine && s.fits && s.rows > 0 ? (s.len + a.chunk - 1) / a.chunk * static_cast<int>(outer_heads) : 0;
            const int incl = wave_incl_scan(n);
            const unsigned all = static_cast<unsigned>(__builtin_amdgcn_readlane(incl, 63));
            if (unit < all) {
                const int at = __popcll(__ballot(static_cast<unsigned>(incl) <= unit));
                u.seq = base + at;
                u.s = make_seq(a.b, __builtin_amdgcn_readlane(first, at), __builtin_amdgcn_readlane(last, at), __builtin_amdgcn_readlane(len, at));
                unit -= static_cast<unsigned>(__builtin_amdgcn_readlane(incl - n, at));
                break;
            }
            unit -= all;
        }
        u.chunk = static_cast<int>(unit / outer_heads), outer = unit % outer_heads;
    } else {
        const unsigned items = static_cast<unsigned>(a.b.n_seqs) * outer_heads;
        u.chunk = static_cast<int>(unit / items);
        if (u.chunk >= a.n_chunks) return -1;
        // (a chunk's items start three further on than the chunk before's: else each XCD would have the same sequences' chunks
        // all along, and the XCD of the longest ones would end last)
        const unsigned item = (unit % items + 3u * static_cast<unsigned>(u.chunk)) % items;
        u.seq = static_cast<int>(item / outer_heads), outer = item % outer_heads;
        u.s = seq_load(a.b, u.seq);
        if (!u.s.fits) {
            if (threadIdx.x == 0) queue_fault(a.faults, kFaultRows);
            return 0;
        }
    }
    u.head = static_cast<int>(outer) * a.inner_heads + static_cast<int>(in / groups);
    u.p0 = u.chunk * a.chunk;
    u.nq = u.s.rows * a.group, u.q0 = static_cast<int>(cg) * CT * 16;
    u.ctx = u.s.len - u.s.rows, u.p1 = min(u.p0 + a.chunk, u.s.len);
    return u.q0 < u.nq && u.p0 < u.s.len;
}

// A tile of 16 positions a lane: where its keys and values lie. One that is not wanted, lies past the chunk or names a page
// outside the pool reads the pool's first page (lost: the last was met; usable: the lanes' tiles that count).
struct AttnTiles {
    int64_t off, scale_off;   // elements
    uint64_t usable;
    bool lost;
};
__device__ inline AttnTiles attn_tiles(const AttnArgs &a, const AttnUnit &u, int tile, bool wanted) {
    const int entry = min(tile, a.b.max_len - 1) / a.kv.page;   // (within the table's row whatever the length)
    const int page = a.b.pages[u.seq * a.b.ld_pages + entry];
    const bool own = wanted && tile < u.p1, good = page >= 0 && page < a.kv.n_pages;
    if (own && !good) queue_fault(a.faults, kFaultPage);
    AttnTiles t;
    t.lost = __any(own && !good);
    t.usable = __ballot(own && good);
    const int64_t pg = own && good ? page : 0;
    const int slot = tile % a.kv.page;
    t.off = pg * a.kv.page_stride + u.head * a.kv.head_stride + slot * a.kv.pos_stride;
    t.scale_off = (pg * a.kv.nkv + u.head) * a.kv.page + slot;
    return t;
}
__device__ inline int64_t lane64(int64_t v, int l) {   // lane l's value, uniform
    const uint64_t u = static_cast<uint64_t>(v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(u)), l);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(u >> 32)), l);
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// Loads from a uniform place plus a lane's 32-bit byte offset and a uniform one: buffer instructions, whose addresses take
// no vector registers (a 64-bit address a lane and load took up to 40).
typedef uint32_t au2 __attribute__((ext_vector_type(2)));
// a lane's offset past the buffer's 2^31 - 1 bytes, for dims past head_dim: the load gives zeros and asks no memory (24 heads of
// 80: 27.0 -> 25.8 us; 16 heads of 192: 19.2 -> 17.5, with selects in its place before)
constexpr uint32_t kNowhere = 0x80000000u;
__device__ inline __amdgpu_buffer_rsrc_t place(const void *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), static_cast<short>(0), 0x7FFFFFFF, 0x00020000);
}
__device__ inline au4 load16(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint32_t off) {
    return __builtin_amdgcn_raw_buffer_load_b128(r, lane_off, off, 0);
}
__device__ inline au2 load8b(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint32_t off) {
    return __builtin_amdgcn_raw_buffer_load_b64(r, lane_off, off, 0);
}
__device__ inline uint32_t load4b(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint32_t off) {
    return __builtin_amdgcn_raw_buffer_load_b32(r, lane_off, off, 0);
}
__device__ inline float4 load4f(const float *p, uint32_t lane_off) { return __builtin_bit_cast(float4, load16(place(p), lane_off, 0)); }

// x / group of a column x < 32 group (group at most 4,096): the quotient's distance to a whole number, at least 0.5 / group,
// is far above the error of 32 x 2^-22
__device__ inline int row_of(const AttnArgs &a, int x) { return static_cast<int>((static_cast<float>(x) + 0.5f) * a.group_inv); }

// The columns' powers of two (fp16 products of other types' queries): a column's largest value to 2^10 .. 2^11 (0 and not
// finite: left). A lane's column is 16 ct + lane % 16.
struct QueryScale {
    const float *amax;
    bool scaled;
    __device__ int exponent(int ct) const {
        const int e = static_cast<int>(__float_as_uint(amax[ct * 16 + (threadIdx.x & 15)]) >> 23);
        return scaled && e > 0 && e < 255 ? min(max(137 - e, -126), 126) : 0;
    }
    __device__ float undo(int ct) const { return __uint_as_float(static_cast<uint32_t>(127 - exponent(ct)) << 23); }
};
// The queries as a thread has them on their way: eight values of each of QU columns and 32-dim chunks (QP > 1: fp32, else
// one 16-bit type's), which of them count. Asked for before the pages are: what is asked for later arrives later.
template <int QP, int NCH, int CT>
struct Queries {
    static constexpr int QU = (CT * NCH + kAttnWaves - 1) / kAttnWaves;
    au4 raw[QU][QP > 1 ? 2 : 1];
    uint32_t in = 0;
};
template <bool I8, int QP, int NCH, bool EX, int CT>
__device__ inline Queries<QP, NCH, CT> load_queries(const AttnArgs &a, const AttnUnit &u) {
    constexpr bool F32 = QP > 1;
    const int lane = threadIdx.x & 63, i16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    Queries<QP, NCH, CT> qu;
#pragma unroll
    for (int k = 0; k < qu.QU; ++k) {
        const int c = (k * kAttnWaves + wave) % NCH, ct = (k * kAttnWaves + wave) / NCH;
        const int x = u.q0 + ct * 16 + i16;
        const int d = I8 ? (c >> 1) * 64 + g4 * 16 + (c & 1) * 8 : c * 32 + g4 * 8;
        const bool ok = ct < CT && x < u.nq && (EX || d < a.kv.hd);
        const int xc = ok ? x : 0, r = row_of(a, xc);
        const au4 *from = reinterpret_cast<const au4 *>(
            a.q + ((u.s.first + r) * a.q_row + static_cast<int64_t>(u.head * a.group + xc - r * a.group) * a.kv.hd + (ok ? d : 0)) * (F32 ? 4 : 2));
        qu.raw[k][0] = from[0];
        if constexpr (F32) qu.raw[k][1] = from[1];
        if (ok) qu.in |= 1u << k;
    }
    return qu;
}
// The queries' operands to LDS in the order the products take them, [column tile][part][chunk][lane], by the whole
// workgroup; ends with a barrier.
template <bool BF, bool I8, int QP, int NCH, int CT>
__device__ inline QueryScale stage_queries(const AttnArgs &a, const Queries<QP, NCH, CT> &qu, au4 *lds_q, float *lds_amax) {
    constexpr bool F32 = QP > 1;
    constexpr int QU = Queries<QP, NCH, CT>::QU;
    const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const QueryScale qs{lds_amax, F32 ? !BF : I8 && a.type != GV_F16};
    if (qs.scaled) {
        if (tid < CT * 16) lds_amax[tid] = 0.0f;
        __syncthreads();
    }
    float qv[QU][8];
#pragma unroll
    for (int k = 0; k < QU; ++k) {
        const bool ok = qu.in >> k & 1;
        const int ct = (k * kAttnWaves + wave) / NCH;
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t w = ok ? qu.raw[k][F32 ? j / 4 : 0][F32 ? j % 4 : j / 2] : 0u;
            if constexpr (F32) qv[k][j] = __uint_as_float(w);
            else if (BF || (I8 && a.type == GV_BF16)) qv[k][j] = j & 1 ? bf16_hi(w) : bf16_lo(w);
            else qv[k][j] = j & 1 ? half_hi(w) : half_lo(w);
            m = fmaxf(m, fabsf(qv[k][j]));
        }
        if (qs.scaled) {   // (positive floats order as their bits)
            m = rows_max(m);
            if (lane < 16 && ct < CT) atomicMax(reinterpret_cast<unsigned *>(lds_amax) + ct * 16 + i16, __float_as_uint(m));
        }
    }
    if (qs.scaled) __syncthreads();
#pragma unroll
    for (int k = 0; k < QU; ++k) {
        const int c = (k * kAttnWaves + wave) % NCH, ct = (k * kAttnWaves + wave) / NCH;
        if (ct >= CT) continue;
        if (qs.scaled) {
            const float f = __uint_as_float(static_cast<uint32_t>(127 + qs.exponent(ct)) << 23);
#pragma unroll
            for (int j = 0; j < 8; ++j) qv[k][j] *= f;
        }
        au4 part[QP];
        split8<BF, QP>(qv[k], part);
#pragma unroll
        for (int p = 0; p < QP; ++p) lds_q[((ct * QP + p) * NCH + c) * 64 + lane] = part[p];
    }
    __syncthreads();
    return qs;
}
// a chunk's maximum for the join, which passes over chunks that have none (a sum that is no number is one to be joined)
__device__ inline float joined_max(float m, float l) { return l != l && m == -INFINITY ? 0.0f : m; }
// which of its sequence's rows column x sees
__device__ inline uint32_t seen_rows(const AttnArgs &a, const AttnUnit &u, int x) {
    const int r = row_of(a, x);
    return x >= u.nq ? 0u : a.visible ? a.visible[u.s.first + r] : 0xFFFFFFFFu >> (31 - r);
}

// whether one of 2 N 16-bit values is not finite (their magnitudes' largest, two to a word)
template <bool BF, int N>
__device__ inline bool any_not_finite(const uint32_t (&w)[N]) {
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
    us2 top = __builtin_bit_cast(us2, w[0] & 0x7FFF7FFFu);
#pragma unroll
    for (int k = 1; k < N; ++k) top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, w[k] & 0x7FFF7FFFu));
    const uint32_t t = __builtin_bit_cast(uint32_t, top);
    return max(t & 0xFFFFu, t >> 16) >= (BF ? 0x7F80u : 0x7C00u);
}

// ---------------------------------------------------------------- few columns
// KV: the cache's type. QP, PP: the parts of the queries and of the weights. NT: dim tiles of 16 (head_dim at most
// 16 NT; EX: exactly). CT: column tiles of 16 queries a workgroup takes.
template <int KV, int QP, int PP, int NT, bool EX, int CT>
__device__ inline void attn_few_columns(const AttnArgs &a, const AttnUnit &u) {
    constexpr bool BF = KV == GV_BF16, I8 = KV == GV_I8;
    constexpr int ES = I8 ? 1 : 2;         // bytes a cached element
    constexpr int NCH = NT / 2;            // 32-dim chunks of S^T's products
    constexpr int KL = I8 ? NCH / 2 : NCH; // 16-byte loads a lane a K tile
    constexpr int VW = NT * ES / 4;        // words a lane a V row
    extern __shared__ au4 lds_q[];         // [CT][QP][NCH][64]
    __shared__ float lds_amax[CT * 16];
    __shared__ float lds_m[kAttnWaves][CT * 16], lds_l[kAttnWaves][CT * 16];
    const int lane = threadIdx.x & 63, i16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));   // (uniform: its branches are)

    const Seq &s = u.s;
    const int p0 = u.p0, p1 = u.p1, ctx = u.ctx, nq = u.nq, q0 = u.q0, head = u.head;
    const auto qu = load_queries<I8, QP, NCH, EX, CT>(a, u);
    // the pages of this wave's tiles (lane t: step t / 2, tile t % 2)
    const int tile = p0 + kAttnStep * (wave + kAttnWaves * (lane >> 1)) + 16 * (lane & 1);
    const AttnTiles at = attn_tiles(a, u, tile, (lane >> 1) * kAttnWaves * kAttnStep < a.chunk);
    const int64_t toff = at.off, soff = at.scale_off;
    const uint64_t usable = at.usable;
    const bool lost = at.lost;

    const uint32_t klane = (static_cast<uint32_t>(i16) * static_cast<uint32_t>(a.kv.pos_stride) + g4 * (I8 ? 16 : 8)) * ES;
    const uint32_t vlane = (static_cast<uint32_t>(4 * g4) * static_cast<uint32_t>(a.kv.pos_stride) + i16 * NT) * ES;
    const uint32_t vrow = static_cast<uint32_t>(a.kv.pos_stride) * ES;

    // ---- one step's operands: keys (with their scales) and values; a tile that is not used reads the pool's first page
    au4 kf[2][KL];
    uint32_t vr[8][VW];
    float ksc[2][4], vsc[2][4];
    const auto load_k = [&](int st) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const auto kb = place(a.kv.k + lane64(toff, 2 * st + h) * ES);
#pragma unroll
            for (int c = 0; c < KL; ++c) {
                constexpr uint32_t per = I8 ? 64 : 32 * ES;   // bytes between a lane's loads
                if constexpr (EX) {
                    kf[h][c] = load16(kb, klane + c * per, 0);
                } else {
                    const int d = I8 ? c * 64 + g4 * 16 : c * 32 + g4 * 8;
                    kf[h][c] = load16(kb, d < a.kv.hd ? klane + c * per : kNowhere, 0);
                }
            }
            if constexpr (I8) {
                const float4 x = load4f(a.kv.ks + lane64(soff, 2 * st + h), 16 * g4);
                ksc[h][0] = x.x, ksc[h][1] = x.y, ksc[h][2] = x.z, ksc[h][3] = x.w;
            }
        }
    };
    const auto load_v = [&](int st) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const auto vb = place(a.kv.v + lane64(toff, 2 * st + h) * ES);
            const uint32_t lo = EX || i16 * NT < a.kv.hd ? vlane : kNowhere;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t(&w)[VW] = vr[4 * h + r];
                if constexpr (VW >= 4) {
#pragma unroll
                    for (int k = 0; k < VW / 4; ++k) {
                        const au4 x = load16(vb, lo + 16 * k, r * vrow);
                        w[4 * k] = x[0], w[4 * k + 1] = x[1], w[4 * k + 2] = x[2], w[4 * k + 3] = x[3];
                    }
                } else if constexpr (VW == 2) {
                    const au2 x = load8b(vb, lo, r * vrow);
                    w[0] = x[0], w[1] = x[1];
                } else {
                    w[0] = load4b(vb, lo, r * vrow);
                }
            }
            if constexpr (I8) {
                const float4 y = load4f(a.kv.vs + lane64(soff, 2 * st + h), 16 * g4);
                vsc[h][0] = y.x, vsc[h][1] = y.y, vsc[h][2] = y.z, vsc[h][3] = y.w;
            }
        }
    };

    const int mine = p1 - p0 - kAttnStep * wave, open = ctx - p0 - kAttnStep * (wave + 1);
    constexpr int kRound = kAttnStep * kAttnWaves;
    const int steps = mine > 0 ? (mine + kRound - 1) / kRound : 0;
    const int free_steps = lost || open < 0 ? 0 : min(steps, open / kRound + 1);
    if (steps > 0) {   // (the first step's keys and values on their way while the queries are made ready)
        load_k(0);
        load_v(0);
    }

    const QueryScale qs = stage_queries<BF, I8, QP, NCH, CT>(a, qu, lds_q, lds_amax);
    const int qes = a.type == GV_F32 ? 4 : 2;

    float sc[CT], m[CT], l[CT];           // a column's score factor, maximum, sum
    float most[CT], up[CT];               // int8: log2 of the largest weight x scale; its weights' factor for the products
    uint32_t bits[CT];                    // which of the sequence's rows it sees
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        sc[ct] = a.scale * qs.undo(ct) * (I8 ? kI8Unit : 1.0f);
        m[ct] = most[ct] = -INFINITY, l[ct] = 0.0f, up[ct] = I8 ? weight_factor(-INFINITY) : 16384.0f;
        bits[ct] = seen_rows(a, u, q0 + ct * 16 + i16);
    }
    af4 acc[CT][NT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[ct][n] = af4{0, 0, 0, 0};

    // One step: the next step's keys are asked for once this one's are in the products, its values likewise. `tail`: a
    // step with positions that some query does not see (the sequence's own rows, its end, a lost page).
    const auto step = [&](auto tail_c, int st, bool more) {
        constexpr bool tail = decltype(tail_c)::value;
        const int p = p0 + kAttnStep * (wave + kAttnWaves * st);
        int ql = lane;   // (pinned: the queries are read from LDS in every step, not kept in registers)
        if constexpr (CT * NT * QP >= 16) asm volatile("" : "+v"(ql));
        // ---- scores
        af4 sv[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) sv[ct][0] = sv[ct][1] = af4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            au4 kk[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (I8) {
                    const uint32_t w0 = kf[h][c / 2][2 * (c & 1)] ^ 0x80808080u, w1 = kf[h][c / 2][2 * (c & 1) + 1] ^ 0x80808080u;
                    kk[h] = au4{i8_pair(0, w0, 0x0C010C00u), i8_pair(0, w0, 0x0C030C02u), i8_pair(0, w1, 0x0C010C00u),
                                i8_pair(0, w1, 0x0C030C02u)};
                } else {
                    kk[h] = kf[h][c];
                }
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int q = 0; q < QP; ++q) {
                    const au4 b = lds_q[((ct * QP + q) * NCH + c) * 64 + ql];
                    sv[ct][0] = mfma<BF>(kk[0], b, sv[ct][0]);
                    sv[ct][1] = mfma<BF>(kk[1], b, sv[ct][1]);
                }
        }
        float kk_sc[8];
        if constexpr (I8)
#pragma unroll
            for (int j = 0; j < 8; ++j) kk_sc[j] = ksc[j / 4][j % 4];
        if constexpr (!tail)
            if (more) load_k(st + 1);
        const bool use0 = usable >> (2 * st) & 1, use1 = usable >> (2 * st + 1) & 1;
        uint32_t hole = 0;   // (bit j: the lane's position j is not there at all)
        if constexpr (tail) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int pos = p + 16 * (j / 4) + 4 * g4 + j % 4;
                if (pos >= p1 || !(j < 4 ? use0 : use1)) hole |= 1u << j;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int k = 0; k < VW; ++k) vr[j][k] = hole >> j & 1 ? 0u : vr[j][k];
        }
        uint32_t see[CT];   // (bit j: the lane's column sees its position j)
        au4 pb[CT][PP];
        float vlog[8];
        if constexpr (I8)
#pragma unroll
            for (int j = 0; j < 8; ++j) vlog[j] = __builtin_amdgcn_logf(fabsf(vsc[j / 4][j % 4]));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float x[8], vs[8];
            see[ct] = 0xFFu;
            if constexpr (tail) {
                see[ct] = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int pos = p + 16 * (j / 4) + 4 * g4 + j % 4;
                    const bool seen = pos < ctx || (bits[ct] >> ((pos - ctx) & 31) & 1);
                    if (seen && !(hole >> j & 1)) see[ct] |= 1u << j;
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float f = sc[ct];
                if constexpr (I8) f *= kk_sc[j], vs[j] = vsc[j / 4][j % 4];
                x[j] = sv[ct][j / 4][j % 4] * f;
                if constexpr (tail) {
                    x[j] = see[ct] >> j & 1 ? x[j] : -INFINITY;
                    if constexpr (I8) vs[j] = see[ct] >> j & 1 ? vs[j] : 0.0f;
                }
                top = fmaxf(top, x[j]);
            }
            const float mn = fmaxf(m[ct], rows_max(top));
            const float base = mn == -INFINITY ? 0.0f : mn;
            float wn = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = (x[j] - base) * kLog2e;
                if constexpr (I8) wn = fmaxf(wn, x[j] + vlog[j]);
            }
            const float down = mn == m[ct] ? 0.0f : (m[ct] - mn) * kLog2e;
            if constexpr (I8) wn = fmaxf(rows_max(wn), most[ct] + down);
            if (__any(mn > m[ct] || wn > most[ct])) {
                float f = __builtin_amdgcn_exp2f(down);
                l[ct] *= f;
                if constexpr (I8) {   // (at most about 2, whatever its two parts are)
                    const float now = weight_factor(wn);
                    f = __builtin_amdgcn_exp2f(down + log2_ratio(now, up[ct]));
                    most[ct] = wn, up[ct] = now;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[ct][n] *= f;
                m[ct] = mn;
            }
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = __builtin_amdgcn_exp2f(x[j]);
                sum += x[j];
                if constexpr (I8) {   // (weight x scale first: the scale alone may be far above the largest of them)
                    x[j] = x[j] * vs[j] * up[ct];
                    if constexpr (tail) x[j] = see[ct] >> j & 1 ? x[j] : 0.0f;
                } else if constexpr (!BF) {
                    x[j] *= up[ct];
                }
            }
            l[ct] += sum;
            split8<BF, PP>(x, pb[ct]);
        }

        // ---- values: dim tile n's operand from the 8 rows
        const auto v_tile = [&](int n) {
            au4 v;
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                if constexpr (I8) {
                    const uint32_t lo = vr[2 * jj][n / 4] ^ 0x80808080u, hi = vr[2 * jj + 1][n / 4] ^ 0x80808080u;
                    const uint32_t k = n & 3;
                    v[jj] = i8_pair(hi, lo, 0x0C000C00u | k | (4 + k) << 16);
                } else {
                    v[jj] = perm(vr[2 * jj + 1][n / 2], vr[2 * jj][n / 2], n & 1 ? 0x07060302u : 0x05040100u);
                }
            }
            return v;
        };
        if constexpr (!tail || I8) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const au4 v = v_tile(n);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int q = 0; q < PP; ++q) acc[ct][n] = mfma<BF>(v, pb[ct][q], acc[ct][n]);
            }
            if (tail && more) load_k(st + 1);
            if (more) load_v(st + 1);
            return;
        }
        // 16-bit values of the sequence's own rows that are not finite reach only the columns that see them: left out of
        // the step's product (0 x inf would be NaN), then added position by position to those columns
        uint32_t wild = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int pos = p + 16 * (j / 4) + 4 * g4 + j % 4;
            const bool w = any_not_finite<BF, VW>(vr[j]);
            if (w && pos >= ctx) wild |= 1u << j;
        }
        if (__any(wild != 0))   // wild for every lane if it is for one of the 16 that hold the position's dims
            for (int o = 1; o < 16; o <<= 1) wild |= __shfl_xor(wild, o, 64);
        for (int pp = -1; pp < kAttnStep; ++pp) {   // position pp of the step: lane row pp % 16 / 4, its j
            const int j = pp < 0 ? 0 : pp / 16 * 4 + pp % 4, g = pp < 0 ? 0 : pp % 16 / 4;
            if (pp >= 0 && !(__builtin_amdgcn_readlane(static_cast<int>(wild), 16 * g) >> j & 1)) continue;
            const uint32_t in = pp < 0 ? ~wild : g4 == g ? 1u << j : 0u;
            uint32_t keep[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) keep[k] = (in >> (2 * k) & 1 ? 0xFFFFu : 0u) | (in >> (2 * k + 1) & 1 ? 0xFFFF0000u : 0u);
            // (the rows pinned each time round: their transposition would else be kept for all dim tiles at once)
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int k = 0; k < VW; ++k) asm volatile("" : "+v"(vr[r][k]));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                au4 v = v_tile(n);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] &= keep[k];
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    af4 d = af4{0, 0, 0, 0};
#pragma unroll
                    for (int q = 0; q < PP; ++q) d = mfma<BF>(v, pb[ct][q], d);
                    const bool sees = pp < 0 || (__shfl(see[ct], 16 * g + i16, 64) >> j & 1);
                    if (sees) acc[ct][n] += d;
                }
            }
            if (!__any(wild != 0)) break;
        }
        if (more) {
            load_k(st + 1);
            load_v(st + 1);
        }
    };
    int st = 0;
    for (; st < free_steps; ++st) step(std::false_type{}, st, st + 1 < steps);
    for (; st < steps; ++st) step(std::true_type{}, st, st + 1 < steps);

    // ---- the four waves joined, a column tile after the other
    constexpr int OLD = NT * 16 + 4;   // floats a column in LDS
    float *lds_o = reinterpret_cast<float *>(lds_q);
    __syncthreads();                   // (the queries are done with)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        l[ct] = rows_sum(l[ct]);
        if (lane < 16) lds_m[wave][ct * 16 + lane] = m[ct], lds_l[wave][ct * 16 + lane] = l[ct];
    }
    __syncthreads();
    const bool whole = s.len <= a.chunk;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        if (q0 + ct * 16 >= nq) break;
        const int col = ct * 16 + i16;
        float mt = lds_m[0][col];
#pragma unroll
        for (int w = 1; w < kAttnWaves; ++w) mt = fmaxf(mt, lds_m[w][col]);
        // (int8: each wave's own factor taken out, so that the sums are the values')
        const float out_log = I8 ? log2_ratio(kI8Unit, up[ct]) : 0.0f;
        const float f = m[ct] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[ct] - mt) * kLog2e + out_log);
        float *o = lds_o + (wave * 16 + i16) * OLD;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < NT; n += 4)
                *reinterpret_cast<float4 *>(o + (4 * g4 + r) * NT + n) =
                    float4{acc[ct][n][r] * f, acc[ct][n + 1][r] * f, acc[ct][n + 2][r] * f, acc[ct][n + 3][r] * f};
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * NT * 4; e += kAttnThreads) {
            const int c = e / (NT * 4), d = e % (NT * 4) * 4;
            const int x = q0 + ct * 16 + c;
            if (x >= nq || (!EX && d >= a.kv.hd)) continue;
            float mm = lds_m[0][ct * 16 + c];
#pragma unroll
            for (int w = 1; w < kAttnWaves; ++w) mm = fmaxf(mm, lds_m[w][ct * 16 + c]);
            float ll = 0.0f;
            float4 v = float4{0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) {
                const float mw = lds_m[w][ct * 16 + c];
                const float lw = lds_l[w][ct * 16 + c];
                if (mw != -INFINITY || lw != lw) ll += lw * __builtin_amdgcn_exp2f((mw - mm) * kLog2e);
                const float4 y = *reinterpret_cast<const float4 *>(lds_o + (w * 16 + c) * OLD + d);
                v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
            }
            const int r = row_of(a, x), row = s.first + r, hq = head * a.group + x - r * a.group;
            const float unit_v = BF || I8 ? 1.0f : 1.0f / 16384.0f;
            v.x *= unit_v, v.y *= unit_v, v.z *= unit_v, v.w *= unit_v;
            if (whole) {
                if (ll > 0.0f || ll != ll) v = float4{v.x / ll, v.y / ll, v.z / ll, v.w / ll};
                else v = float4{0, 0, 0, 0};
                char *dst = a.out + (row * a.out_row + static_cast<int64_t>(hq) * a.kv.hd + d) * qes;
                if (a.type == GV_F32) store4<GV_F32>(dst, v);
                else if (a.type == GV_F16) store4<GV_F16>(dst, v);
                else store4<GV_BF16>(dst, v);
                if (a.lse && d == 0) a.lse[static_cast<int64_t>(row) * a.nh + hq] = ll > 0.0f || ll != ll ? mm + logf(ll) : -INFINITY;
            } else {
                const int64_t to = (static_cast<int64_t>(u.chunk) * a.b.n_rows + row) * a.nh + hq;
                store4<GV_F32>(reinterpret_cast<char *>(a.parts + to * a.kv.hd + d), v);
                if (d == 0) *reinterpret_cast<float2 *>(a.ml + to * 2) = float2{joined_max(mm, ll), ll};
            }
        }
        __syncthreads();
    }
}

// COUNTED: a workgroup takes one unit after the other of those that the lengths make (attn_unit)
template <int KV, int QP, int PP, int NT, bool EX, int CT, bool COUNTED>
__global__ __launch_bounds__(kAttnThreads, (attn_waves<NT, CT, COUNTED>())) void paged_attn_kernel(const AttnArgs a) {
    touch_args(a);
    AttnUnit u;
    if constexpr (!COUNTED) {
        if (attn_unit<CT, false>(a, blockIdx.x, u) > 0) attn_few_columns<KV, QP, PP, NT, EX, CT>(a, u);
        return;
    }
    for (unsigned i = blockIdx.x;; i += gridDim.x) {
        const int is = attn_unit<CT, true>(a, i, u);
        if (is < 0) return;
        if (is > 0) attn_few_columns<KV, QP, PP, NT, EX, CT>(a, u);
        __syncthreads();
    }
}

// the column tiles a workgroup takes where there is more than one
constexpr int kWideTiles = 3;
// the kernels of one cache type, by parts (16-bit or fp32 rows), dims and column tiles (paged_attn_<type>.hip)
int launch_attn_f16(const AttnArgs &a, int ct, unsigned grid, hipStream_t st);
int launch_attn_bf16(const AttnArgs &a, int ct, unsigned grid, hipStream_t st);
int launch_attn_i8(const AttnArgs &a, int ct, unsigned grid, hipStream_t st);

template <int KV, int QP, int PP, int NT, bool EX, int CT, bool COUNTED>
int launch_attn_one(const AttnArgs &a, unsigned grid, hipStream_t st) {
    constexpr int lds = attn_lds<NT, CT, QP>();
    static int granted = 0;
    if (lds_grant(reinterpret_cast<const void *>(&paged_attn_kernel<KV, QP, PP, NT, EX, CT, COUNTED>), lds, granted) != 0) return -1;
    hipLaunchKernelGGL((paged_attn_kernel<KV, QP, PP, NT, EX, CT, COUNTED>), dim3(grid), dim3(kAttnThreads), lds, st, a);
    GV_CHECK_HIP(hipGetLastError());
    return 0;
}
// The units by max_len, or COUNTED in as many workgroups as are there at once: where there are more than 32 units a CU. An
// empty workgroup keeps its place for a microsecond, so that a batch with one long sequence spends its time on them: one
// of 65,537 positions among thirty short ones (24 heads of 80, bf16; 16,000 units, most of them empty) 45 us by max_len,
// 24 counted; 64 full sequences of 8,192 (8,192 units) 137 and 139. With heads of 256 (fp16), where the counted form has one
// wave a SIMD and the other two: one of 131,072 among 63 short ones 113 and 86, 32 full ones of 131,072 (16,384 units) 1,593
// and 1,615. Each unit scans the lengths, so only up to kCountSeqs sequences.
constexpr int kCountUnits = 32 * 256, kCountSeqs = 256;
template <int KV, int QP, int PP, int NT, bool EX, int CT>
int launch_attn_few(const AttnArgs &a, unsigned grid, hipStream_t st) {
    if (grid > kCountUnits && a.b.n_seqs <= kCountSeqs)
        return launch_attn_one<KV, QP, PP, NT, EX, CT, true>(a, 256 * attn_waves<NT, CT, true>(), st);
    return launch_attn_one<KV, QP, PP, NT, EX, CT, false>(a, grid, st);
}
}  // namespace gv
