// paged.hip - the paged cache of several conversations: new rows' keys and values appended to it (gv_paged_append),
// and what the paged calls share on the host.
#include <string>

#include "paged.hpp"

namespace gv {

namespace {

const char *kFaultText[kFaultCount] = {
    "a sequence's row starts or length do not fit the batch (rows ascending within n_rows, at most max_rows of them, "
    "at most lens[i]; lens[i] at most max_len)",
    "a page outside the pool",
    "a rotary position outside the tables",
    "a token range, bias range or mask outside its array",
};

int *g_fault_host = nullptr, *g_fault_dev = nullptr;

}  // namespace

int *queued_faults() {
    if (g_fault_dev) return g_fault_dev;
    void *h = nullptr, *d = nullptr;
    // (portable: any of the process's GPUs may write it; kept until the process ends)
    if (hipHostMalloc(&h, 64, hipHostMallocMapped | hipHostMallocPortable) != hipSuccess ||
        hipHostGetDevicePointer(&d, h, 0) != hipSuccess) {
        (void)hipGetLastError();
        if (h) (void)hipHostFree(h);
        set_error("no pinned memory for the queued calls' faults");
        return nullptr;
    }
    g_fault_host = static_cast<int *>(h);
    for (int i = 0; i < kFaultCount; ++i) g_fault_host[i] = 0;
    g_fault_dev = static_cast<int *>(d);
    return g_fault_dev;
}

int take_queued_faults() {
    if (!g_fault_host) return 0;
    std::string msg;
    for (int i = 0; i < kFaultCount; ++i) {
        volatile int *w = g_fault_host + i;
        if (!*w) continue;
        *w = 0;
        msg += (msg.empty() ? "a queued call met: " : "; ") + std::string(kFaultText[i]);
    }
    GV_REQUIRE(msg.empty(), msg);
    return 0;
}

OnDevice::OnDevice() {
    const int want = device();
    if (hipGetDevice(&before) != hipSuccess || before != want) ok = hipSetDevice(want) == hipSuccess;
    if (!ok) set_error("the library's GPU cannot be made current");
    if (before == want) before = -1;
}
OnDevice::~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
}

int check_kv(const gv_paged_kv *c, const char *call) {
    GV_CHECK_ARG(c, "no cache");
    GV_CHECK_ARG(c->type == GV_F16 || c->type == GV_BF16 || c->type == GV_I8, "a cache is GV_F16, GV_BF16 or GV_I8");
    GV_CHECK_ARG(c->n_kv_heads >= 1 && c->n_kv_heads <= 4096, "KV heads: 1 to 4096");
    GV_CHECK_ARG(c->head_dim >= 16 && c->head_dim <= 256 && c->head_dim % 16 == 0,
                 "head_dim: a multiple of 16, at most 256");
    GV_CHECK_ARG(c->page_size >= 16 && c->page_size % 16 == 0 && c->page_size <= 65536,
                 "page_size: a multiple of 16, at most 65536");
    GV_CHECK_ARG(c->n_pages >= 1, "no pages");
    GV_CHECK_ARG(c->k && c->v && aligned(c->k, 16) && aligned(c->v, 16), "k and v: 16-byte aligned device memory");
    GV_CHECK_ARG(c->type != GV_I8 || (c->k_scale && c->v_scale && aligned(c->k_scale, 16) && aligned(c->v_scale, 16)),
                 "k_scale and v_scale: 16-byte aligned device memory for GV_I8");
    const int64_t small = int64_t{1} << 24;
    GV_CHECK_ARG(c->pos_stride >= 16 && c->pos_stride % 16 == 0 && c->pos_stride < small && c->head_stride >= 16 &&
                     c->head_stride % 16 == 0 && c->head_stride < small && c->page_stride >= 16 &&
                     c->page_stride % 16 == 0 && c->page_stride < int64_t{1} << 40,
                 "strides: positive multiples of 16, head_stride and pos_stride below 2^24, page_stride below 2^40");
    return 0;
}

int check_batch(const gv_paged_batch *b, const gv_paged_kv *c, const char *call) {
    GV_CHECK_ARG(b, "no batch");
    GV_CHECK_ARG(b->n_seqs >= 1 && b->n_seqs <= 1 << 20, "n_seqs: 1 to 2^20");
    GV_CHECK_ARG(b->n_rows >= 1 && b->n_rows <= 1 << 24, "n_rows: 1 to 2^24");
    GV_CHECK_ARG(b->max_rows >= 1, "max_rows: at least 1");
    GV_CHECK_ARG(b->row_start && b->lens && b->pages, "row_start, lens and pages are needed");
    GV_CHECK_ARG(b->ld_pages >= 1 && b->ld_pages <= INT32_MAX, "ld_pages: at least 1");
    GV_CHECK_ARG(b->max_len >= 1 && b->max_len <= 1 << 30 && b->max_len <= b->ld_pages * c->page_size,
                 "max_len: at most ld_pages * page_size and 2^30");
    return 0;
}

// ---------------------------------------------------------------- append
// Row t, head u (query heads, then key heads, then value heads): y = x / sqrt(mean x^2 + eps) * (1 + w) where the head
// has a norm weight, its first 2 * half values turned by the row's angles, then rounded once: queries to q_out, keys and
// values to the row's place in the cache. Sums of squares in 64 bits; every other operation one fp32 operation of the
// model's own order (qk_rope_kernel, model.hip), so a row gives the model's bits.
//
// A group of LG lanes a head, four values a lane: norm and amax are lane sums, and a whole head is read by one wave
// before anything of it is written (q_out may be q). The value a value turns with is read from memory again (a cache
// hit) instead of exchanged between lanes, so that every load of a head is issued before the first use.
// Bound by latency for a step's few rows (the row's sequence, then its page entry, then the stores) and by the rows'
// bytes for prompts.
struct AppendArgs {
    KvView kv;
    BatchView b;
    const char *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    const float *q_norm, *k_norm;
    float eps;
    int half, interleaved;
    const float *cos_t, *sin_t;
    int n_positions;
    const int *positions;
    int nh, q_type;
    char *q_out;
    int64_t q_out_row;
    int *faults;
    int units, lg;   // heads in all; lanes a head takes
};

__device__ inline double group_sum(double v, int lg) {
    for (int o = lg / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ inline float group_max(float v, int lg) {
    for (int o = lg / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

template <int TIN, int TKV>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
    const int t = blockIdx.x, hd = a.kv.hd, nkv = a.kv.nkv;
    const int l = threadIdx.x & (a.lg - 1), i0 = 4 * l;
    const int u = blockIdx.y * (256 / a.lg) + static_cast<int>(threadIdx.x) / a.lg;
    const bool live = u < a.units && i0 < hd;
    const int uc = min(u, a.units - 1), ic = min(i0, hd - 4);
    const int kind = uc < a.nh ? 0 : uc < a.nh + nkv ? 1 : 2;
    const int h = kind == 0 ? uc : kind == 1 ? uc - a.nh : uc - a.nh - nkv;
    const char *src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const int64_t at = kind == 0 ? t * a.q_row + h * a.q_head : kind == 1 ? t * a.k_row + h * a.k_head : t * a.v_row + h * a.v_head;
    constexpr int64_t es = TIN == GV_F32 ? 4 : 2;
    const int rot = kind == 2 ? 0 : 2 * a.half;
    // the values this lane's turn with (half pairs: four values half a rotation away; interleaved: its own)
    const bool turns = i0 < rot, first = i0 < a.half;
    const int ip = turns && !a.interleaved ? (first ? i0 + a.half : i0 - a.half) : ic;
    float4 x = load4<TIN>(src + (at + ic) * es);
    float4 xp = load4<TIN>(src + (at + ip) * es);
    const float *nw = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    float4 w = float4{0, 0, 0, 0}, wp = w;
    if (nw) {
        w = float4{nw[ic], nw[ic + 1], nw[ic + 2], nw[ic + 3]};
        wp = float4{nw[ip], nw[ip + 1], nw[ip + 2], nw[ip + 3]};
    }

    const int i = seq_of_row(a.b, t);
    if (i >= a.b.n_seqs) return;   // a row behind the last sequence
    const Seq s = seq_load(a.b, i);
    const int j = t - s.first;
    if (j < 0 && i == 0) return;   // a row before the first sequence
    if (!s.fits || j < 0 || j >= s.rows) {
        if (threadIdx.x == 0) queue_fault(a.faults, kFaultRows);
        return;
    }
    const int pos = s.len - s.rows + j;
    const int page = a.b.pages[i * a.b.ld_pages + pos / a.kv.page];
    const int rp = a.positions ? a.positions[t] : pos;
    if (page < 0 || page >= a.kv.n_pages) {
        if (threadIdx.x == 0) queue_fault(a.faults, kFaultPage);
        return;
    }
    if (a.half > 0 && (rp < 0 || rp >= a.n_positions)) {
        if (threadIdx.x == 0) queue_fault(a.faults, kFaultPosition);
        return;
    }
    float4 c = float4{1, 1, 1, 1}, sn = float4{0, 0, 0, 0};
    if (turns) {
        const int64_t ang = static_cast<int64_t>(rp) * a.half;
        if (a.interleaved) {
            const int f = i0 / 2;
            c = float4{a.cos_t[ang + f], a.cos_t[ang + f], a.cos_t[ang + f + 1], a.cos_t[ang + f + 1]};
            sn = float4{a.sin_t[ang + f], a.sin_t[ang + f], a.sin_t[ang + f + 1], a.sin_t[ang + f + 1]};
        } else {
            const int f = first ? i0 : i0 - a.half;
            c = *reinterpret_cast<const float4 *>(a.cos_t + ang + f);
            sn = *reinterpret_cast<const float4 *>(a.sin_t + ang + f);
        }
    }

    if (nw) {
        const auto sq = [](float v) { return static_cast<double>(v) * static_cast<double>(v); };
        const double ss = group_sum(live ? (sq(x.x) + sq(x.y)) + (sq(x.z) + sq(x.w)) : 0.0, a.lg);
        const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(static_cast<float>(ss / static_cast<double>(hd)), a.eps)));
        const auto nrm = [inv](float v, float g) { return __fmul_rn(__fmul_rn(v, inv), __fadd_rn(1.0f, g)); };
        x = float4{nrm(x.x, w.x), nrm(x.y, w.y), nrm(x.z, w.z), nrm(x.w, w.w)};
        xp = float4{nrm(xp.x, wp.x), nrm(xp.y, wp.y), nrm(xp.z, wp.z), nrm(xp.w, wp.w)};
    }
    float4 y = x;
    if (turns) {
        if (a.interleaved) {
            y = float4{__fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(x.y, sn.x)), __fadd_rn(__fmul_rn(x.y, c.y), __fmul_rn(x.x, sn.y)),
                       __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(x.w, sn.z)), __fadd_rn(__fmul_rn(x.w, c.w), __fmul_rn(x.z, sn.w))};
        } else {   // (x c - b s in the first half, x c + a s in the second: the sign bit of the product turned)
            const uint32_t neg = first ? 0x80000000u : 0u;
            const auto turn = [neg](float v, float p, float cc, float ssn) {
                const float m = __fmul_rn(p, ssn);
                return __fadd_rn(__fmul_rn(v, cc), __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, m) ^ neg));
            };
            y = float4{turn(x.x, xp.x, c.x, sn.x), turn(x.y, xp.y, c.y, sn.y), turn(x.z, xp.z, c.z, sn.z), turn(x.w, xp.w, c.w, sn.w)};
        }
    }
    if (kind == 0) {
        if (!live) return;
        char *o = a.q_out + (t * a.q_out_row + static_cast<int64_t>(h) * hd + i0) * (a.q_type == GV_F32 ? 4 : 2);
        if (a.q_type == GV_F32) store4<GV_F32>(o, y);
        else if (a.q_type == GV_F16) store4<GV_F16>(o, y);
        else store4<GV_BF16>(o, y);
        return;
    }
    const int slot = pos % a.kv.page;
    char *pool = kind == 1 ? a.kv.k : a.kv.v;
    const int64_t to = page * a.kv.page_stride + h * a.kv.head_stride + slot * a.kv.pos_stride + i0;
    if constexpr (TKV == GV_I8) {   // the row's largest value at 127 steps (quant_kv_row, engine/src/model.cpp:3766-3774)
        const float m = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
        const float amax = group_max(live ? m : 0.0f, a.lg);
        const float inv = amax > 0.0f ? __fdiv_rn(127.0f, amax) : 0.0f;
        const auto q8 = [inv](float v) {
            return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(rintf(__fmul_rn(v, inv)), -127.0f), 127.0f))) & 0xFFu;
        };
        if (!live) return;
        *reinterpret_cast<uint32_t *>(pool + to) = q8(y.x) | q8(y.y) << 8 | q8(y.z) << 16 | q8(y.w) << 24;
        if (l == 0)
            (kind == 1 ? a.kv.ks : a.kv.vs)[(static_cast<int64_t>(page) * nkv + h) * a.kv.page + slot] = __fdiv_rn(amax, 127.0f);
    } else if (live) {
        store4<TKV>(pool + to * 2, y);
    }
}

template <int TIN>
void launch_append(const AppendArgs &a, int kv_type, dim3 grid, hipStream_t st) {
    if (kv_type == GV_F16) hipLaunchKernelGGL((paged_append_kernel<TIN, GV_F16>), grid, dim3(256), 0, st, a);
    else if (kv_type == GV_BF16) hipLaunchKernelGGL((paged_append_kernel<TIN, GV_BF16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<TIN, GV_I8>), grid, dim3(256), 0, st, a);
}

}  // namespace gv

using namespace gv;

extern "C" int gv_paged_append(const gv_paged_kv *kv, const gv_paged_batch *batch, const gv_append_rows *r) {
    const char *call = "gv_paged_append";
    if (check_kv(kv, call) != 0 || check_batch(batch, kv, call) != 0) return -1;
    GV_CHECK_ARG(r, "no rows");
    GV_CHECK_ARG(float_type(r->type), "rows are GV_F32, GV_F16 or GV_BF16");
    GV_CHECK_ARG(r->n_heads >= 0 && r->n_heads <= 4096, "n_heads: 0 to 4096");
    const size_t al = 4 * static_cast<size_t>(type_bytes(r->type));
    const auto part = [al](const void *p, int64_t row, int64_t head) {
        const int64_t most = int64_t{1} << 36;
        return p && aligned(p, al) && row >= 0 && row < most && row % 4 == 0 && head >= 0 && head < most && head % 4 == 0;
    };
    GV_CHECK_ARG(part(r->k, r->k_row, r->k_head) && part(r->v, r->v_row, r->v_head),
                 "k and v: four elements aligned, strides multiples of 4");
    GV_CHECK_ARG(r->rope_dim >= 0 && r->rope_dim % 8 == 0 && r->rope_dim <= kv->head_dim,
                 "rope_dim: a multiple of 8, at most head_dim");
    GV_CHECK_ARG(r->rope_dim == 0 || (r->cos && r->sin && aligned(r->cos, 16) && aligned(r->sin, 16) && r->n_positions >= 1),
                 "cos and sin: 16-byte aligned tables for a rotation");
    if (r->n_heads > 0) {
        GV_CHECK_ARG(part(r->q, r->q_row, r->q_head), "q: four elements aligned, strides multiples of 4");
        GV_CHECK_ARG(float_type(r->q_type), "q_out is GV_F32, GV_F16 or GV_BF16");
        GV_CHECK_ARG(r->q_out && aligned(r->q_out, 4 * static_cast<size_t>(type_bytes(r->q_type))) && r->q_out_row % 4 == 0 &&
                         r->q_out_row >= static_cast<int64_t>(r->n_heads) * kv->head_dim && r->q_out_row < int64_t{1} << 36,
                     "q_out: four elements aligned, rows of at least n_heads * head_dim, a multiple of 4");
        GV_CHECK_ARG(r->q_out != r->q || (r->q_type == r->type && r->q_out_row == r->q_row && r->q_head == kv->head_dim),
                     "q_out is q only with q's type and layout");
    }
    if (ensure_init() != 0) return -1;
    OnDevice dev;
    int *faults = queued_faults();
    if (!dev.ok || !faults) return -1;
    AppendArgs a{};
    a.kv = kv_view(*kv);
    a.b = batch_view(*batch);
    a.q = static_cast<const char *>(r->q), a.k = static_cast<const char *>(r->k), a.v = static_cast<const char *>(r->v);
    a.q_row = r->q_row, a.q_head = r->q_head, a.k_row = r->k_row, a.k_head = r->k_head, a.v_row = r->v_row, a.v_head = r->v_head;
    a.q_norm = r->q_norm, a.k_norm = r->k_norm, a.eps = r->eps;
    a.half = r->rope_dim / 2, a.interleaved = r->interleaved != 0;
    a.cos_t = r->cos, a.sin_t = r->sin, a.n_positions = r->n_positions, a.positions = r->positions;
    a.nh = r->n_heads, a.q_type = r->q_type, a.q_out = static_cast<char *>(r->q_out), a.q_out_row = r->q_out_row;
    a.faults = faults;
    a.units = r->n_heads + 2 * kv->n_kv_heads;
    a.lg = 4;
    while (a.lg * 4 < kv->head_dim) a.lg *= 2;
    const int per = 256 / a.lg;
    const dim3 grid(static_cast<unsigned>(batch->n_rows), static_cast<unsigned>((a.units + per - 1) / per));
    if (r->type == GV_F32) launch_append<GV_F32>(a, kv->type, grid, stream());
    else if (r->type == GV_F16) launch_append<GV_F16>(a, kv->type, grid, stream());
    else launch_append<GV_BF16>(a, kv->type, grid, stream());
    GV_CHECK_HIP(hipGetLastError());
    return 0;
}
