// logits.hip - the rules of each row's request on its logits before a token is sampled (gv_process_logits): penalties
// for tokens of the row's history, biases, grammar masks.
#include <algorithm>
#include <string>

#include "paged.hpp"

namespace gv {

// A workgroup a (row, slice of the vocabulary). The row's history is counted into the slice's LDS words first (bit 31:
// in the history; below: times generated; integer adds, so any order gives the same counts), its biases are summed
// there in the list's order, then the slice's logits are read, changed and written once.
// Bound by the logits read and written for many rows. A slice reads the whole history (from L2 after the first): a
// longer slice reads it fewer times, a shorter one gives few rows more workgroups (rules_slice).
constexpr int kRuleThreads = 512;
constexpr int kRuleMin = 2048, kRuleMax = 16384;   // tokens a slice: 512 threads of four
constexpr int kRuleTags = 1024;

struct RuleArgs {
    gv_logits_rules r;
    const char *logits;
    int64_t ld, ldo;
    float *out;
    int V, slice, n_slices;
    int in_place;
    int *faults;
};

// The row's biases of tokens [v0, v0 + n) added up in the list's order, by one wave: 64 of the list at a time, at once
// where no two share a tag (then no two share a token), else one after the other.
__device__ inline void sum_biases(const RuleArgs &a, int begin, int end, int v0, int n, float *bias, int *tag) {
    const int lane = threadIdx.x & 63;
    for (int i0 = begin; i0 < end; i0 += 64) {
        const int i = i0 + lane;
        const bool in = i < end;
        const int v = in ? a.r.bias_token[i] - v0 : -1;
        const float b = in ? a.r.bias_value[i] : 0.0f;
        const bool mine = v >= 0 && v < n;
        uint64_t todo = __ballot(mine);
        if (todo == 0) continue;
        volatile int *tg = tag + (v & (kRuleTags - 1));
        volatile float *bs = bias;
        if (mine) *tg = lane;
        const bool alone = !mine || *tg == lane;
        if (__all(alone)) {
            if (mine) bs[v] = bs[v] + b;
            continue;
        }
        for (; todo; todo &= todo - 1)
            if (lane == __builtin_ctzll(todo)) bs[v] = bs[v] + b;
    }
}

template <int TYPE, bool VEC>
__device__ inline float4 load_logits(const char *row, int v, int n) {   // VEC: v .. v + 3 (n of them); else v alone
    constexpr int es = TYPE == GV_F32 ? 4 : 2;
    const char *p = row + static_cast<int64_t>(v) * es;
    if (VEC && n >= 4) return load4<TYPE>(p);
    const auto one = [p](int k) {
        if constexpr (TYPE == GV_F32) return *reinterpret_cast<const float *>(p + 4 * k);
        const uint32_t w = *reinterpret_cast<const uint16_t *>(p + 2 * k);
        if constexpr (TYPE == GV_F16) return half_lo(w);
        return bf16_lo(w);
    };
    float4 x = float4{one(0), 0, 0, 0};
    if (VEC) {
        if (n > 1) x.y = one(1);
        if (n > 2) x.z = one(2);
    }
    return x;
}

template <int TYPE, bool VEC>
__global__ __launch_bounds__(kRuleThreads) void logits_rules_kernel(const RuleArgs a) {
    extern __shared__ uint32_t lds[];
    const int row = blockIdx.x / a.n_slices, v0 = (blockIdx.x % a.n_slices) * a.slice;
    const int n = min(a.slice, a.V - v0), tid = threadIdx.x;
    // the row's ranges and numbers
    const bool penal = a.r.tokens != nullptr;
    int begin = 0, end = 0, gen = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (penal) {
        begin = a.r.begin[row], end = a.r.end[row];
        gen = a.r.generated ? a.r.generated[row] : begin;
        if (a.r.repetition) rep = a.r.repetition[row];
        if (a.r.frequency) freq = a.r.frequency[row];
        if (a.r.presence) pres = a.r.presence[row];
        if (begin < 0 || end < begin || end > a.r.n_tokens) {
            if (tid == 0) queue_fault(a.faults, kFaultRange);
            begin = end = 0;
        }
        if (rep == 1.0f && freq == 0.0f && pres == 0.0f) end = begin;
    }
    int bb = 0, be = 0;
    if (a.r.bias_token) {
        bb = a.r.bias_begin[row], be = a.r.bias_end[row];
        if (bb < 0 || be < bb || be > a.r.n_biases) {
            if (tid == 0) queue_fault(a.faults, kFaultRange);
            bb = be = 0;
        }
    }
    const uint32_t *mask = nullptr;
    if (a.r.masks) {
        const int m = a.r.mask_of[row];
        if (m >= a.r.n_masks) {
            if (tid == 0) queue_fault(a.faults, kFaultRange);
        } else if (m >= 0) {
            mask = a.r.masks + m * a.r.ld_mask + v0 / 32;
        }
    }
    const bool counted = end > begin, biased = be > bb;   // (uniform over the workgroup)
    uint32_t *word = lds;
    float *bias = reinterpret_cast<float *>(lds + a.slice);
    int *tag = reinterpret_cast<int *>(lds + 2 * a.slice);
    if (counted || biased) {
        for (int i = 4 * tid; i < a.slice; i += 4 * kRuleThreads) {
            if (counted) *reinterpret_cast<uint4 *>(word + i) = uint4{0, 0, 0, 0};
            if (biased) *reinterpret_cast<float4 *>(bias + i) = float4{0, 0, 0, 0};
        }
        __syncthreads();
        if (counted) {
            constexpr int U = 4;   // tokens a thread has in flight
            for (int64_t i0 = begin; i0 < end; i0 += U * kRuleThreads) {
                int v[U];
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const int64_t i = i0 + k * kRuleThreads + tid;
                    v[k] = i < end ? a.r.tokens[i] - v0 : -1;
                }
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const int64_t i = i0 + k * kRuleThreads + tid;
                    if (v[k] >= 0 && v[k] < n) {
                        if (i >= gen) atomicAdd(word + v[k], 1u);
                        else atomicOr(word + v[k], 0x80000000u);
                    }
                }
            }
        }
        if (biased && tid < 64) sum_biases(a, bb, be, v0, n, bias, tag);
        __syncthreads();
    }
    const char *src = a.logits + (row * a.ld + v0) * (TYPE == GV_F32 ? 4 : 2);
    float *dst = a.out + row * a.ldo + v0;
    const auto apply = [&](float x, int v) {
        if (counted) {
            const uint32_t w = word[v];
            if (w) {
                x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
                const uint32_t c = w & 0x7FFFFFFFu;
                if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(c))), pres);
            }
        }
        if (biased) x = __fadd_rn(x, bias[v]);
        return x;
    };
    constexpr int W = VEC ? 4 : 1;
    for (int v = W * tid; v < n; v += W * kRuleThreads) {
        uint32_t keep = 0xFu;
        if (mask) keep = mask[v / 32] >> (v % 32);
        const int m = VEC ? min(4, n - v) : 1;
        if (a.in_place) {
            uint32_t touched = 0;
            for (int k = 0; k < m; ++k) touched |= (counted ? word[v + k] : 0u) | (biased ? __float_as_uint(bias[v + k]) : 0u);
            if (touched == 0 && (keep & (VEC ? 0xFu >> (4 - m) : 1u)) == (VEC ? 0xFu >> (4 - m) : 1u)) continue;
        }
        float4 x = load_logits<TYPE, VEC>(src, v, m);
        x.x = keep & 1u ? apply(x.x, v) : -INFINITY;
        if constexpr (VEC) {
            if (m >= 4) {
                x.y = keep & 2u ? apply(x.y, v + 1) : -INFINITY;
                x.z = keep & 4u ? apply(x.z, v + 2) : -INFINITY;
                x.w = keep & 8u ? apply(x.w, v + 3) : -INFINITY;
                *reinterpret_cast<float4 *>(dst + v) = x;
                continue;
            }
            if (m > 1) dst[v + 1] = keep & 2u ? apply(x.y, v + 1) : -INFINITY;
            if (m > 2) dst[v + 2] = keep & 4u ? apply(x.z, v + 2) : -INFINITY;
        }
        dst[v] = x.x;
    }
}

// The slice: as long as 1,024 workgroups are there with it (four a CU), at least kRuleMin, at most kRuleMax, or half of
// it where the biases' sums lie beside the counts.
static int rules_slice(int rows, int V, bool biases) {
    int s = biases ? kRuleMax / 2 : kRuleMax;
    while (s > kRuleMin && static_cast<int64_t>(rows) * ((V + s - 1) / s) < 1024) s /= 2;
    return s;
}

template <int TYPE>
int launch_rules(const RuleArgs &a, int rows, bool vec, size_t lds, hipStream_t st) {
    static int granted[2] = {0, 0};
    const dim3 grid(static_cast<unsigned>(rows) * static_cast<unsigned>(a.n_slices));
    const void *kernel = vec ? reinterpret_cast<const void *>(&logits_rules_kernel<TYPE, true>)
                             : reinterpret_cast<const void *>(&logits_rules_kernel<TYPE, false>);
    if (lds_grant(kernel, lds, granted[vec]) != 0) return -1;
    if (vec) hipLaunchKernelGGL((logits_rules_kernel<TYPE, true>), grid, dim3(kRuleThreads), lds, st, a);
    else hipLaunchKernelGGL((logits_rules_kernel<TYPE, false>), grid, dim3(kRuleThreads), lds, st, a);
    GV_CHECK_HIP(hipGetLastError());
    return 0;
}

}  // namespace gv

using namespace gv;

extern "C" int gv_process_logits(const gv_logits_rules *rules, const void *logits, int type, int64_t ld, int rows,
                                 int V, float *out, int64_t ldo) {
    const char *call = "gv_process_logits";
    GV_CHECK_ARG(rules, "no rules");
    GV_CHECK_ARG(float_type(type), "logits are GV_F32, GV_F16 or GV_BF16");
    GV_CHECK_ARG(rows >= 1 && rows <= 65536 && V >= 1 && V <= 1 << 24, "rows: 1 to 65536, V: 1 to 2^24");
    GV_CHECK_ARG(logits && out && aligned(logits, static_cast<size_t>(type_bytes(type))) && aligned(out, 4),
                 "logits and out: device memory");
    GV_CHECK_ARG(ld >= V && ldo >= V && ld < int64_t{1} << 36 && ldo < int64_t{1} << 36, "ld and ldo: at least V");
    GV_CHECK_ARG(logits != out || (type == GV_F32 && ld == ldo), "out is logits only with GV_F32 and ldo = ld");
    GV_CHECK_ARG(!rules->tokens || (rules->begin && rules->end && rules->n_tokens >= 0),
                 "tokens need begin, end and n_tokens");
    GV_CHECK_ARG(rules->tokens || !(rules->repetition || rules->frequency || rules->presence), "penalties need tokens");
    GV_CHECK_ARG(!rules->bias_token || (rules->bias_value && rules->bias_begin && rules->bias_end && rules->n_biases >= 0),
                 "biases need bias_value, bias_begin, bias_end and n_biases");
    GV_CHECK_ARG(!rules->masks || (rules->mask_of && rules->n_masks >= 1 && rules->ld_mask >= (V + 31) / 32),
                 "masks need mask_of, n_masks and ld_mask of at least ceil(V / 32)");
    if (ensure_init() != 0) return -1;
    OnDevice dev;
    int *faults = queued_faults();
    if (!dev.ok || !faults) return -1;
    RuleArgs a{};
    a.r = *rules;
    a.logits = static_cast<const char *>(logits), a.out = out;
    a.ld = ld, a.ldo = ldo;
    a.V = V, a.slice = rules_slice(rows, V, rules->bias_token != nullptr), a.n_slices = (V + a.slice - 1) / a.slice;
    a.in_place = logits == static_cast<const void *>(out);
    a.faults = faults;
    const bool vec = ld % 4 == 0 && ldo % 4 == 0 && aligned(out, 16) && aligned(logits, 4 * static_cast<size_t>(type_bytes(type)));
    const size_t lds = 4 * static_cast<size_t>(a.slice) * (rules->bias_token ? 2 : 1) + (rules->bias_token ? 4 * kRuleTags : 0);
    if (type == GV_F32) return launch_rules<GV_F32>(a, rows, vec, lds, stream());
    if (type == GV_F16) return launch_rules<GV_F16>(a, rows, vec, lds, stream());
    return launch_rules<GV_BF16>(a, rows, vec, lds, stream());
}
