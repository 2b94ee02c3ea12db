// paged.hip - the paged cache of several conversations: new rows' keys and values appended to it (gv_paged_append),
// and what the paged calls share on the host.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>
#include <vector>

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

constexpr int kFaultLine = 16;    // words a host thread's take: a line of 64 bytes
constexpr int kFaultLines = 64;   // lines allocated at a time (kept until the process ends)

struct FaultLine {
    volatile int *host = nullptr;
    int *dev = nullptr;
    uint64_t ended = 0;   // how many threads had ended when its own had, itself among them
};
struct FaultLines {
    std::mutex use;
    std::vector<FaultLine> idle, ended;   // of no thread; of threads that have ended with calls that may still run
    std::atomic<uint64_t> ends{0};
    std::atomic<int> n_ended{0};
};
FaultLines &fault_lines() {
    static FaultLines *lines = new FaultLines;   // (never destroyed: a thread may end after main has)
    return *lines;
}

// the calling thread's line, from its first queued call to its end
struct ThreadLine {
    FaultLine line;
    ~ThreadLine() {
        if (!line.dev) return;
        FaultLines &all = fault_lines();
        const std::lock_guard<std::mutex> lock(all.use);
        line.ended = all.ends.fetch_add(1) + 1;
        all.ended.push_back(line);
        all.n_ended.fetch_add(1);
    }
};
thread_local ThreadLine t_line;

int more_lines(FaultLines &all) {
    constexpr size_t bytes = size_t{kFaultLines} * kFaultLine * sizeof(int);
    void *h = nullptr, *d = nullptr;
    // (portable: any of the process's GPUs may write it)
    if (hipHostMalloc(&h, bytes, hipHostMallocMapped | hipHostMallocPortable) != hipSuccess ||
        hipHostGetDevicePointer(&d, h, 0) != hipSuccess) {
        (void)hipGetLastError();
        if (h) (void)hipHostFree(h);
        set_error("no pinned memory for the queued calls' faults");
        return -1;
    }
    memset(h, 0, bytes);
    for (int i = kFaultLines - 1; i >= 0; --i) {
        FaultLine l;
        l.host = static_cast<int *>(h) + i * kFaultLine, l.dev = static_cast<int *>(d) + i * kFaultLine;
        all.idle.push_back(l);
    }
    return 0;
}

unsigned taken(const FaultLine &l) {   // the kinds met (a bit each), the words cleared
    unsigned kinds = 0;
    for (int i = 0; i < kFaultCount; ++i)
        if (l.host[i]) kinds |= 1u << i, l.host[i] = 0;
    return kinds;
}

}  // namespace

int *queued_faults() {
    if (t_line.line.dev) return t_line.line.dev;
    FaultLines &all = fault_lines();
    const std::lock_guard<std::mutex> lock(all.use);
    if (all.idle.empty() && more_lines(all) != 0) return nullptr;
    t_line.line = all.idle.back();
    all.idle.pop_back();
    return t_line.line.dev;
}

FaultWait::FaultWait() : ends(fault_lines().ends.load()) {}

int FaultWait::told() const {
    unsigned kinds = t_line.line.dev ? taken(t_line.line) : 0u;
    FaultLines &all = fault_lines();
    if (all.n_ended.load() > 0) {
        const std::lock_guard<std::mutex> lock(all.use);
        for (size_t i = 0; i < all.ended.size();) {
            if (all.ended[i].ended > ends) {   // (it ended after this wait had begun: its calls may not be done)
                ++i;
                continue;
            }
            kinds |= taken(all.ended[i]);
            all.idle.push_back(all.ended[i]);
            all.ended[i] = all.ended.back();
            all.ended.pop_back();
            all.n_ended.fetch_sub(1);
        }
    }
    std::string msg;
    for (int i = 0; i < kFaultCount; ++i)
        if (kinds >> i & 1) msg += (msg.empty() ? "a queued call met: " : "; ") + std::string(kFaultText[i]);
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
                     c->page_stride % 16 == 0 && c->page_stride < int64_t{1} << 40 &&
                     c->n_kv_heads * c->head_stride < int64_t{1} << 28,
                 "strides: positive multiples of 16, head_stride and pos_stride below 2^24, page_stride below 2^40, "
                 "n_kv_heads * head_stride below 2^28");
    return 0;
}

int check_batch(const gv_paged_batch *b, const gv_paged_kv *c, const char *call) {
    GV_CHECK_ARG(b, "no batch");
    GV_CHECK_ARG(b->n_seqs >= 1 && b->n_seqs <= 1 << 20, "n_seqs: 1 to 2^20");
    // (a launch's threads along an axis are counted in 32 bits)
    GV_CHECK_ARG(b->n_rows >= 1 && b->n_rows < 1 << 24, "n_rows: 1 to 2^24 - 1");
    GV_CHECK_ARG(b->max_rows >= 1, "max_rows: at least 1");
    GV_CHECK_ARG(b->row_start && b->lens && b->pages, "row_start, lens and pages are needed");
    GV_CHECK_ARG(b->ld_pages >= 1 && b->ld_pages <= INT32_MAX, "ld_pages: at least 1");
    GV_CHECK_ARG(b->max_len >= 1 && b->max_len <= 1 << 30 && b->max_len <= b->ld_pages * c->page_size,
                 "max_len: at most ld_pages * page_size and 2^30");
    return 0;
}

// ---------------------------------------------------------------- append
// Row t's heads (query heads, then key heads, then value heads): y = x / sqrt(mean x^2 + eps) * (1 + w) where the kind
// has a norm weight, the first 2 * half values turned by the row's angles, then rounded once: queries to q_out, keys and
// values to the row's place in the cache. Sums of squares in 64 bits; every other operation one fp32 operation of the
// model's own order (qk_rope_kernel, model.hip), so a row gives the model's bits.
//
// A wave takes rounds of 64 / lg heads of one kind, lg lanes a head, four values a lane: norm, amax and the value that a
// value turns with are exchanges between lanes, and a whole head is read by one wave before anything of it is written
// (q_out may be q). A round's loads are issued before the round before is worked
// on, the first's before the row's sequence is looked for.
// Bound by its chain of loads (row starts, the sequence's, the page entry, the angles: about 4 us from launch to stores) for
// a step's rows, and by the rows' bytes for prompts, where a wave goes on to further rounds behind one such chain.
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
    int lg;          // lanes a head takes
    int q_rounds, kv_rounds, rounds;   // waves' rounds of 64 / lg heads: of the queries, of the keys (or values), in all
};

__device__ inline double group_sum(double v, int lg) {
    for (int o = lg / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// the largest size of the group's values: of their bits without the sign, which order as the sizes do, a NaN above infinity
__device__ inline uint32_t size_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ inline float group_size(uint32_t v, int lg) {
    for (int o = lg / 2; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o, 64)));
    return __uint_as_float(v);
}

template <int TIN>
struct Raw4 {   // four values as they lie in memory
    using type = uint2;
};
template <>
struct Raw4<GV_F32> {
    using type = float4;
};
template <int TIN>
__device__ inline float4 raw_floats(typename Raw4<TIN>::type r) {
    if constexpr (TIN == GV_F32) return r;
    else if constexpr (TIN == GV_F16) return float4{half_lo(r.x), half_hi(r.x), half_lo(r.y), half_hi(r.y)};
    else return float4{bf16_lo(r.x), bf16_hi(r.x), bf16_lo(r.y), bf16_hi(r.y)};
}

// D: heads a lane group takes in a round (their control flow once)
template <int TIN, int TKV, int D>
__device__ inline void append_row(const AppendArgs &a, int t, int wave) {
    const int hd = a.kv.hd, nkv = a.kv.nkv, lane = threadIdx.x & 63;
    const int l = lane & (a.lg - 1), i0 = 4 * l, hw = 64 / a.lg, in_round = lane / a.lg;
    const int ic = min(i0, hd - 4);
    constexpr int es = TIN == GV_F32 ? 4 : 2;
    typename Raw4<TIN>::type raw[D];
    const auto load = [&](int r) {   // a round's values
        const bool is_q = r < a.q_rounds, is_k = !is_q && r < a.q_rounds + a.kv_rounds;
        const int h = (r - (is_q ? 0 : is_k ? a.q_rounds : a.q_rounds + a.kv_rounds)) * (D * hw) + in_round, last = (is_q ? a.nh : nkv) - 1;
        const char *row = (is_q ? a.q : is_k ? a.k : a.v) + t * (is_q ? a.q_row : is_k ? a.k_row : a.v_row) * es;
        const uint32_t step = static_cast<uint32_t>(is_q ? a.q_head : is_k ? a.k_head : a.v_head);
#pragma unroll
        for (int d = 0; d < D; ++d)
            raw[d] = *reinterpret_cast<const typename Raw4<TIN>::type *>(row + (static_cast<uint32_t>(min(h + d * hw, last)) * step + ic) * es);
    };
    int r = blockIdx.y * 4 + wave;
    if (r >= a.rounds) return;
    load(r);
    float4 wq = float4{0, 0, 0, 0}, wk = wq;   // the lane's norm weights, every head's alike
    if (a.q_norm) wq = *reinterpret_cast<const float4 *>(a.q_norm + ic);
    if (a.k_norm) wk = *reinterpret_cast<const float4 *>(a.k_norm + ic);

    Seq s;
    bool misfit;
    const int i = seq_of_row(a.b, t, s, misfit);
    if (misfit && lane == 0) queue_fault(a.faults, kFaultRows);   // (whichever rows it has, and also none)
    if (i >= a.b.n_seqs) return;   // a row behind the last sequence
    if (t < s.first && i == 0) return;   // a row before the first sequence
    if (!s.fits || t < s.first || t >= s.first + s.rows) {
        if (lane == 0) queue_fault(a.faults, kFaultRows);
        return;
    }
    const int pos = s.len - s.rows + t - s.first;
    const int page = a.b.pages[i * a.b.ld_pages + pos / a.kv.page], slot = pos % a.kv.page;
    const int rp = a.positions ? a.positions[t] : pos;
    if (a.half > 0 && (rp < 0 || rp >= a.n_positions)) {
        if (lane == 0) queue_fault(a.faults, kFaultPosition);
        return;
    }
    // the lane's angles, likewise
    const bool turns = i0 < 2 * a.half, first = i0 < a.half;
    float4 c = float4{1, 1, 1, 1}, sn = float4{0, 0, 0, 0};
    if (turns) {
        const int64_t ang = static_cast<int64_t>(rp) * a.half;
        const float *ct = a.cos_t + ang, *st = a.sin_t + ang;
        if (a.interleaved) {
            const int f = i0 / 2;
            c = float4{ct[f], ct[f], ct[f + 1], ct[f + 1]};
            sn = float4{st[f], st[f], st[f + 1], st[f + 1]};
        } else {
            const int f = first ? i0 : i0 - a.half;
            c = *reinterpret_cast<const float4 *>(ct + f);
            sn = *reinterpret_cast<const float4 *>(st + f);
        }
    }
    if (page < 0 || page >= a.kv.n_pages) {
        if (lane == 0) queue_fault(a.faults, kFaultPage);
        return;
    }
    const int partner = turns ? (first ? lane + a.half / 4 : lane - a.half / 4) : lane;   // (half pairs)
    const int64_t place = page * a.kv.page_stride + slot * a.kv.pos_stride;

    bool more;
    do {
        float4 x[D];
#pragma unroll
        for (int d = 0; d < D; ++d) x[d] = raw_floats<TIN>(raw[d]);
        const int now = r;
        r += gridDim.y * 4;
        more = r < a.rounds;
        if (more) load(r);
        const int kind = now < a.q_rounds ? 0 : now < a.q_rounds + a.kv_rounds ? 1 : 2;
        const int h = (now - (kind == 0 ? 0 : kind == 1 ? a.q_rounds : a.q_rounds + a.kv_rounds)) * (D * hw) + in_round;
        const int n = i0 < hd ? (kind == 0 ? a.nh : nkv) : 0;   // (heads below it are this lane's to write)
        if (kind == 0 ? a.q_norm != nullptr : kind == 1 && a.k_norm != nullptr) {
            const float4 w = kind == 0 ? wq : wk;
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const auto sq = [](float v) { return static_cast<double>(v) * static_cast<double>(v); };
                const double ss = group_sum(i0 < hd ? (sq(x[d].x) + sq(x[d].y)) + (sq(x[d].z) + sq(x[d].w)) : 0.0, a.lg);
                const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(static_cast<float>(ss / static_cast<double>(hd)), a.eps)));
                const auto nrm = [inv](float v, float g) { return __fmul_rn(__fmul_rn(v, inv), __fadd_rn(1.0f, g)); };
                x[d] = float4{nrm(x[d].x, w.x), nrm(x[d].y, w.y), nrm(x[d].z, w.z), nrm(x[d].w, w.w)};
            }
        }
        if (kind != 2 && a.half > 0) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const float4 v = x[d];
                float4 y;
                if (a.interleaved) {
                    y = float4{__fsub_rn(__fmul_rn(v.x, c.x), __fmul_rn(v.y, sn.x)), __fadd_rn(__fmul_rn(v.y, c.y), __fmul_rn(v.x, sn.y)),
                               __fsub_rn(__fmul_rn(v.z, c.z), __fmul_rn(v.w, sn.z)), __fadd_rn(__fmul_rn(v.w, c.w), __fmul_rn(v.z, sn.w))};
                } else {   // (x c - b s in the first half, x c + a s in the second: the sign bit of the product turned)
                    const uint32_t neg = first ? 0x80000000u : 0u;
                    const auto turn = [neg](float v, float o, float cc, float ssn) {
                        const float m = __fmul_rn(o, ssn);
                        return __fadd_rn(__fmul_rn(v, cc), __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, m) ^ neg));
                    };
                    const float4 o = float4{__shfl(v.x, partner, 64), __shfl(v.y, partner, 64), __shfl(v.z, partner, 64), __shfl(v.w, partner, 64)};
                    y = float4{turn(v.x, o.x, c.x, sn.x), turn(v.y, o.y, c.y, sn.y), turn(v.z, o.z, c.z, sn.z), turn(v.w, o.w, c.w, sn.w)};
                }
                if (turns) x[d] = y;
            }
        }
        if (kind == 0) {
            const uint32_t to = static_cast<uint32_t>(h) * hd + i0, step = hw * hd;
            const int64_t row = t * a.q_out_row;
            const auto put = [&](auto type) {
                constexpr int T = decltype(type)::value, ts = T == GV_F32 ? 4 : 2;
                char *o = a.q_out + row * ts;
#pragma unroll
                for (int d = 0; d < D; ++d)
                    if (h + d * hw < n) store4<T>(o + (to + d * step) * ts, x[d]);
            };
            if (a.q_type == GV_F32) put(std::integral_constant<int, GV_F32>{});
            else if (a.q_type == GV_F16) put(std::integral_constant<int, GV_F16>{});
            else put(std::integral_constant<int, GV_BF16>{});
            continue;
        }
        char *pool = (kind == 1 ? a.kv.k : a.kv.v) + place * (TKV == GV_I8 ? 1 : 2);
        const uint32_t to = static_cast<uint32_t>(h) * static_cast<uint32_t>(a.kv.head_stride) + i0;
        const uint32_t step = static_cast<uint32_t>(hw) * static_cast<uint32_t>(a.kv.head_stride);
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const float4 y = x[d];
            const bool live = h + d * hw < n;
            if constexpr (TKV == GV_I8) {
                // the row's largest value at 127 steps (quant_kv_row, engine/src/model.cpp:3766-3774), but a NaN, which that passes
                // over, is the largest: the scale is then no number, and the row not one that looks in order
                const uint32_t m = max(max(size_bits(y.x), size_bits(y.y)), max(size_bits(y.z), size_bits(y.w)));
                const float amax = group_size(i0 < hd ? m : 0u, a.lg);
                const float inv = amax > 0.0f ? __fdiv_rn(127.0f, amax) : 0.0f;
                const auto q8 = [inv](float v) {
                    return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(rintf(__fmul_rn(v, inv)), -127.0f), 127.0f))) & 0xFFu;
                };
                if (live) *reinterpret_cast<uint32_t *>(pool + to + d * step) = q8(y.x) | q8(y.y) << 8 | q8(y.z) << 16 | q8(y.w) << 24;
                if (live && l == 0)
                    (kind == 1 ? a.kv.ks : a.kv.vs)[(static_cast<int64_t>(page) * nkv + h + d * hw) * a.kv.page + slot] = __fdiv_rn(amax, 127.0f);
            } else if (live) {
                store4<TKV>(pool + (to + d * step) * 2, y);
            }
        }
    } while (more);
}

template <int TIN, int TKV, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
    touch_args(a);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    append_row<TIN, TKV, D>(a, static_cast<int>(blockIdx.x), wave);
    if (a.b.n_seqs > 64 && blockIdx.y == 0 && wave == 0) check_sequences(a.b, static_cast<int>(blockIdx.x), a.faults);
}

template <int TIN, int D>
void launch_append(const AppendArgs &a, int kv_type, dim3 grid, hipStream_t st) {
    if (kv_type == GV_F16) hipLaunchKernelGGL((paged_append_kernel<TIN, GV_F16, D>), grid, dim3(256), 0, st, a);
    else if (kv_type == GV_BF16) hipLaunchKernelGGL((paged_append_kernel<TIN, GV_BF16, D>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<TIN, GV_I8, D>), grid, dim3(256), 0, st, a);
}
template <int TIN>
void launch_append_rows(AppendArgs &a, int kv_type, int n_rows, hipStream_t st) {
    const int hw = 64 / a.lg;
    const auto rounds = [&](int d) {   // with d heads a lane group; the workgroups that take one round a wave
        a.q_rounds = (a.nh + d * hw - 1) / (d * hw), a.kv_rounds = (a.kv.nkv + d * hw - 1) / (d * hw);
        a.rounds = a.q_rounds + 2 * a.kv_rounds;
        return (a.rounds + 3) / 4;
    };
    // A head a lane group and a round a wave while the call has at most 4,096 workgroups (its time is the chain of loads);
    // beyond, four heads and every round of a row in one workgroup. Measured: one row of 16 + 2 + 2 heads of 256 4.2 us as
    // the first, 8.7 as the second; 9,981 bf16 rows of 32 + 8 + 8 heads of 128 (250 MB) 145 us as the first, 68, 51 and 50
    // with one, two and four heads in one workgroup (5.0 TB/s, a copy's rate; the rounds' scalar control was the bound).
    const int many = rounds(1);
    if (static_cast<int64_t>(n_rows) * many <= 4096) {
        launch_append<TIN, 1>(a, kv_type, dim3(static_cast<unsigned>(n_rows), static_cast<unsigned>(many)), st);
    } else {
        rounds(4);
        launch_append<TIN, 4>(a, kv_type, dim3(static_cast<unsigned>(n_rows)), st);
    }
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
    const auto part = [al](const void *p, int64_t row, int64_t head, int n) {
        const int64_t most = int64_t{1} << 36;   // (a row's heads within 2^28 elements: 32-bit offsets in a row)
        return p && aligned(p, al) && row >= 0 && row < most && row % 4 == 0 && head >= 0 && head % 4 == 0 && head < int64_t{1} << 28 &&
               head * n < int64_t{1} << 28;
    };
    GV_CHECK_ARG(part(r->k, r->k_row, r->k_head, kv->n_kv_heads) && part(r->v, r->v_row, r->v_head, kv->n_kv_heads),
                 "k and v: four elements aligned, strides multiples of 4, a row's heads within 2^28 elements");
    GV_CHECK_ARG(aligned(r->q_norm, 16) && aligned(r->k_norm, 16), "q_norm and k_norm: 16-byte aligned");
    GV_CHECK_ARG(r->rope_dim >= 0 && r->rope_dim % 8 == 0 && r->rope_dim <= kv->head_dim,
                 "rope_dim: a multiple of 8, at most head_dim");
    GV_CHECK_ARG(r->rope_dim == 0 || (r->cos && r->sin && aligned(r->cos, 16) && aligned(r->sin, 16) && r->n_positions >= 1),
                 "cos and sin: 16-byte aligned tables for a rotation");
    if (r->n_heads > 0) {
        GV_CHECK_ARG(part(r->q, r->q_row, r->q_head, r->n_heads), "q: four elements aligned, strides multiples of 4, a row's heads within 2^28 elements");
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
    a.lg = 4;
    while (a.lg * 4 < kv->head_dim) a.lg *= 2;
    if (r->type == GV_F32) launch_append_rows<GV_F32>(a, kv->type, batch->n_rows, stream());
    else if (r->type == GV_F16) launch_append_rows<GV_F16>(a, kv->type, batch->n_rows, stream());
    else launch_append_rows<GV_BF16>(a, kv->type, batch->n_rows, stream());
    GV_CHECK_HIP(hipGetLastError());
    return 0;
}
