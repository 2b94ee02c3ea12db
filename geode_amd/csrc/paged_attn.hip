// paged_attn.hip - gv_paged_attention: its launches, its workspace, and the joining of a sequence's chunks.
#include <algorithm>
#include <string>

#include "paged_attn.hpp"

namespace gv {

// A workgroup a (row, query head, 64 dims): the chunks' sums times exp(their maximum - the largest), over the sum of
// weights. 4 or 16 groups of 16 lanes (four dims a lane) take chunks in turn, one to eight in flight each, with a running maximum,
// and are joined in LDS. Bound by latency (the row's sequence, then the sums, which were just written and lie in the
// caches): one pass, nothing waits for the overall maximum.
constexpr int kJoinLanes = 16, kJoinDims = 4 * kJoinLanes;
struct JoinArgs {
    BatchView b;
    const float *parts, *ml;
    char *out;
    float *lse;
    int64_t out_row;
    int nh, hd, type, chunk;
};

template <int GROUPS>
__global__ __launch_bounds__(GROUPS * kJoinLanes) void paged_join_kernel(const JoinArgs a) {
    __shared__ float4 lds_o[GROUPS][kJoinLanes];
    __shared__ float2 lds_ml[GROUPS];
    touch_args(a);
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    const int grp = tid / kJoinLanes, l16 = tid % kJoinLanes, d = blockIdx.z * kJoinDims + 4 * l16;
    Seq s;
    bool misfit;   // (told by the first launch)
    if (seq_of_row(a.b, row, s, misfit) >= a.b.n_seqs) return;
    if (!s.fits || row < s.first || row >= s.first + s.rows || s.len <= a.chunk) return;
    const int nc = (s.len + a.chunk - 1) / a.chunk;
    const int64_t step = static_cast<int64_t>(a.b.n_rows) * a.nh, at = static_cast<int64_t>(row) * a.nh + head;
    const float2 *ml = reinterpret_cast<const float2 *>(a.ml) + at;
    const float *src = a.parts + at * a.hd + min(d, a.hd - 4);
    float m = -INFINITY, l = 0.0f;
    float4 o = float4{0, 0, 0, 0};
    const auto take = [&](auto in_flight) {
        constexpr int U = decltype(in_flight)::value;
        for (int c0 = grp; c0 < nc; c0 += U * GROUPS) {
            float2 x[U];
            float4 y[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int64_t c = min(c0 + k * GROUPS, nc - 1);
                x[k] = ml[c * step];
                y[k] = *reinterpret_cast<const float4 *>(src + c * step * a.hd);
            }
            float mn = m;
#pragma unroll
            for (int k = 0; k < U; ++k) mn = fmaxf(mn, x[k].x);   // (the last chunk again past the end: no harm)
            if (mn == -INFINITY) continue;
            const float f = __builtin_amdgcn_exp2f((m - mn) * kLog2e);
            l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f, m = mn;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (c0 + k * GROUPS >= nc || x[k].x == -INFINITY) continue;
                const float w = __builtin_amdgcn_exp2f((x[k].x - m) * kLog2e);
                l += x[k].y * w;
                o.x += y[k].x * w, o.y += y[k].y * w, o.z += y[k].z * w, o.w += y[k].w * w;
            }
        }
    };
    if (nc <= GROUPS) take(std::integral_constant<int, 1>{});
    else if (nc <= 4 * GROUPS) take(std::integral_constant<int, 4>{});
    else take(std::integral_constant<int, 8>{});
    lds_o[grp][l16] = o;
    if (l16 == 0) lds_ml[grp] = float2{m, l};
    __syncthreads();
    if (tid >= kJoinLanes || d >= a.hd) return;
    m = lds_ml[0].x;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) m = fmaxf(m, lds_ml[g].x);
    l = 0.0f, o = float4{0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const float2 x = lds_ml[g];
        const float w = x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((x.x - m) * kLog2e);
        const float4 y = lds_o[g][l16];
        l += x.y * w;
        o.x += y.x * w, o.y += y.y * w, o.z += y.z * w, o.w += y.w * w;
    }
    const bool some = l > 0.0f || l != l;
    if (some) o = float4{o.x / l, o.y / l, o.z / l, o.w / l};
    else o = float4{0, 0, 0, 0};
    char *dst = a.out + (row * a.out_row + static_cast<int64_t>(head) * a.hd + d) * (a.type == GV_F32 ? 4 : 2);
    if (a.type == GV_F32) store4<GV_F32>(dst, o);
    else if (a.type == GV_F16) store4<GV_F16>(dst, o);
    else store4<GV_BF16>(dst, o);
    if (a.lse && d == 0) a.lse[at] = some ? m + logf(l) : -INFINITY;
}

// How a call is cut: column tiles a workgroup takes, groups of them, and positions a chunk.
struct AttnPlan {
    int ct, col_groups, chunk, n_chunks, inner_heads;
};
static AttnPlan attn_plan(const gv_paged_kv &kv, const gv_paged_batch &b, int n_heads) {
    AttnPlan p;
    const int cols = b.max_rows * (n_heads / kv.n_kv_heads);
    p.ct = cols <= 16 ? 1 : kWideTiles;
    p.col_groups = (cols + 16 * p.ct - 1) / (16 * p.ct);
    const bool wide = p.ct > 1 && kv.head_dim > 64;
    const int64_t items = static_cast<int64_t>(b.n_seqs) * kv.n_kv_heads * p.col_groups;
    // The chunk whose workgroups end first, by what a workgroup takes: some rounds' time to begin and end, and its chunk's rounds.
    double best = 0.0;
    if (wide) {
        // Rounds of 64 positions, seven to begin and end; the lengths of several sequences taken as three fifths of the longest
        // (a guess at their spread).
        // Two workgroups share a CU's units where their LDS and registers leave room (one alone takes 0.82 of the time it takes
        // beside another). Measured, chunks of 256 / 320 / 384 / 512: 32 sequences of up to 4,096 positions and 5 rows (16 heads
        // of 256, fp16) 41 / 36 / 38 / 44 us; one of 32,001 positions and 17 rows (int8) 56 / 61 / 45 / 51; chunks of 128 / 256 /
        // 512: two of 4,406 positions and 22 rows (fp16 queries) 30 / 23 / 27.
        const bool shared = kv.head_dim == 256 || kv.head_dim <= 128;
        const int64_t rounds = (static_cast<int64_t>(b.max_len + 63) / 64 * (b.n_seqs > 1 ? 3 : 5) + 4) / 5;
        for (int r = 2; r <= 8; ++r) {
            const int64_t a_cu = (items * ((rounds + r - 1) / r) + 255) / 256;
            const double t = (shared ? a_cu == 1 ? 0.82 : 0.5 * static_cast<double>(a_cu) : static_cast<double>(a_cu)) *
                                 (std::min<int64_t>(r, rounds) + 7) + (b.max_len > 64 * r ? 1.5 : 0.0);
            if (r == 2 || t < best) best = t, p.chunk = 64 * r;
        }
    } else {
        // Microseconds: rounds of 128 positions (32 a wave), what it takes to begin and end, and the second launch where chunks
        // are to be joined; workgroups at once as the kernels' registers allow. Measured, chunks of 128 / 256 / 512: one sequence
        // of 1,003 positions (16 heads of 256) 10.3 / 12.7 / 16.5 us and 4 for the join; 33 of 2,701 (16 heads of 192, one KV head,
        // fp32 queries) 21 + 6 / 19 + 4 / 17 + 5. A longer chunk leaves a ragged batch's CUs idle.
        const int hd = kv.head_dim;
        const int at_once = 256 * (p.ct > 1 ? 2 : hd <= 64 ? 4 : hd <= 128 ? 3 : 2);
        for (int chunk = 128; chunk <= 512; chunk *= 2) {
            const int64_t turns = (items * ((b.max_len + chunk - 1) / chunk) + at_once - 1) / at_once;
            const int rounds = (std::min(chunk, b.max_len) + 127) / 128;
            const double t = static_cast<double>(turns) * (rounds * (0.4 + 0.0064 * hd) + 4 + 0.019 * hd) + (b.max_len > chunk ? 4.8 : 0.0);
            if (chunk == 128 || t < best) best = t, p.chunk = chunk;
        }
    }
    p.n_chunks = (b.max_len + p.chunk - 1) / p.chunk;
    // (heads inside positions: a head's row of a position shares its cache lines with the next head's)
    p.inner_heads = kv.head_stride < kv.pos_stride && static_cast<int64_t>(b.n_seqs) * p.n_chunks >= 64 ? kv.n_kv_heads : 1;
    return p;
}
static size_t attn_ws_bytes(const AttnPlan &p, const gv_paged_kv &kv, const gv_paged_batch &b, int n_heads) {
    if (p.n_chunks == 1) return 0;
    return static_cast<size_t>(p.n_chunks) * static_cast<size_t>(b.n_rows) * static_cast<size_t>(n_heads) *
           (static_cast<size_t>(kv.head_dim) + 2) * 4;
}

static int64_t attn_grid(const AttnPlan &p, const gv_paged_kv &kv, const gv_paged_batch &b) {
    const int64_t units = static_cast<int64_t>(b.n_seqs) * (kv.n_kv_heads / p.inner_heads) * p.n_chunks;
    return (units + 7) / 8 * 8 * p.col_groups * p.inner_heads;
}

static int check_attention(const gv_paged_kv *kv, const gv_paged_batch *batch, int n_heads, const char *call) {
    if (check_kv(kv, call) != 0 || check_batch(batch, kv, call) != 0) return -1;
    GV_CHECK_ARG(batch->max_rows <= kAttnMaxRows, "at most 32 rows a sequence");
    GV_CHECK_ARG(n_heads >= 1 && n_heads <= 4096 && n_heads % kv->n_kv_heads == 0, "n_heads: a multiple of n_kv_heads, at most 4096");
    // (a launch's threads along an axis are counted in 32 bits; the partial results' size in 64, far from their end)
    const AttnPlan p = attn_plan(*kv, *batch, n_heads);
    GV_CHECK_ARG(attn_grid(p, *kv, *batch) < 1 << 24 &&
                     static_cast<int64_t>(p.n_chunks) * batch->n_rows < (int64_t{1} << 46) / (n_heads * int64_t{kv->head_dim + 2} * 4),
                 "too many sequences, rows, heads and positions for one call");
    return 0;
}

}  // namespace gv

using namespace gv;

extern "C" {

size_t gv_paged_attention_workspace_bytes(const gv_paged_kv *kv, const gv_paged_batch *batch, int n_heads) {
    if (check_attention(kv, batch, n_heads, "gv_paged_attention_workspace_bytes") != 0) return 0;
    return attn_ws_bytes(attn_plan(*kv, *batch, n_heads), *kv, *batch, n_heads);
}

int gv_paged_attention(const gv_paged_kv *kv, const gv_paged_batch *batch, const gv_attention_rows *r, void *ws,
                       size_t ws_bytes) {
    const char *call = "gv_paged_attention";
    GV_CHECK_ARG(r, "no rows");
    if (check_attention(kv, batch, r->n_heads, call) != 0) return -1;
    GV_CHECK_ARG(float_type(r->type) && (r->type == GV_F32 || r->type == kv->type || kv->type == GV_I8),
                 "q and out are GV_F32 or the cache's type (GV_I8: any floating type)");
    const int64_t width = static_cast<int64_t>(r->n_heads) * kv->head_dim, most = int64_t{1} << 36;
    GV_CHECK_ARG(r->q && r->out && aligned(r->q, 16) && aligned(r->out, 16) && r->q_row >= width && r->out_row >= width &&
                     r->q_row % 8 == 0 && r->out_row % 8 == 0 && r->q_row < most && r->out_row < most,
                 "q and out: 16-byte aligned, rows of at least n_heads * head_dim elements, a multiple of 8");
    GV_CHECK_ARG(r->q != r->out, "out is not q");
    GV_CHECK_ARG(r->scale == r->scale, "scale is not a number");
    const AttnPlan p = attn_plan(*kv, *batch, r->n_heads);
    const size_t need = attn_ws_bytes(p, *kv, *batch, r->n_heads);
    GV_CHECK_ARG(need == 0 || (ws && aligned(ws, 16) && ws_bytes >= need),
                 "a 16-byte aligned workspace of gv_paged_attention_workspace_bytes");
    if (ensure_init() != 0) return -1;
    OnDevice dev;
    int *faults = queued_faults();
    if (!dev.ok || !faults) return -1;
    AttnArgs a{};
    a.kv = kv_view(*kv), a.b = batch_view(*batch);
    a.q = static_cast<const char *>(r->q), a.out = static_cast<char *>(r->out);
    a.lse = r->lse, a.visible = r->visible;
    a.parts = static_cast<float *>(ws);
    a.ml = need ? a.parts + static_cast<size_t>(p.n_chunks) * batch->n_rows * r->n_heads * kv->head_dim : nullptr;
    a.q_row = r->q_row, a.out_row = r->out_row;
    a.nh = r->n_heads, a.group = r->n_heads / kv->n_kv_heads, a.type = r->type;
    a.group_inv = 1.0f / static_cast<float>(a.group);
    a.chunk = p.chunk, a.n_chunks = p.n_chunks, a.col_groups = p.col_groups, a.inner_heads = p.inner_heads;
    a.scale = r->scale, a.faults = faults;
    const unsigned g = static_cast<unsigned>(attn_grid(p, *kv, *batch));
    const int rc = kv->type == GV_F16    ? launch_attn_f16(a, p.ct, g, stream())
                   : kv->type == GV_BF16 ? launch_attn_bf16(a, p.ct, g, stream())
                                         : launch_attn_i8(a, p.ct, g, stream());
    if (rc != 0 || p.n_chunks == 1) return rc;
    JoinArgs j{};
    j.b = a.b, j.parts = a.parts, j.ml = a.ml, j.out = a.out, j.lse = a.lse, j.out_row = a.out_row;
    j.nh = a.nh, j.hd = kv->head_dim, j.type = a.type, j.chunk = p.chunk;
    // (few chunks: a wave a workgroup. 109 rows of 16 heads of 256 with up to 13 chunks 5.9 us where four waves take 10.6)
    const dim3 grid_j(static_cast<unsigned>(batch->n_rows), static_cast<unsigned>(r->n_heads),
                      static_cast<unsigned>((kv->head_dim + kJoinDims - 1) / kJoinDims));
    if (p.n_chunks <= 16) hipLaunchKernelGGL(paged_join_kernel<4>, grid_j, dim3(4 * kJoinLanes), 0, stream(), j);
    else hipLaunchKernelGGL(paged_join_kernel<16>, grid_j, dim3(16 * kJoinLanes), 0, stream(), j);
    GV_CHECK_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
