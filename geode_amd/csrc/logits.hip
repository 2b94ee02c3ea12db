// logits.hip - the rules of each row's request on its logits before a token is sampled (gv_process_logits): penalties
// for tokens of the row's history, biases, grammar masks.
#include <algorithm>
#include <string>

#include "paged.hpp"

namespace gv {

// A workgroup a (row, slice of the vocabulary). Its logits are asked for first; while they come the row's history is
// counted into the slice's LDS words (bit 31: in the history; bit 30: has a bias; below: times generated; integer
// operations, so any order gives the same words); then the logits are changed and written once. A logit with biases goes
// through its word: one wave adds them there in the list's order. In place, only what a rule changes is read and written.
// Bound by the logits read and written for many rows, by its chain of loads for few. A slice reads the whole history
// (from L2 after the first): a longer slice reads it fewer times, a shorter one gives few rows more workgroups
// (rules_quads).
constexpr int kRuleThreads = 256;
constexpr int kRuleQuad = 4 * kRuleThreads;   // tokens a workgroup takes at a time: four a thread
constexpr int kRuleTags = 256;
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kTimes = 0x3FFFFFFFu;

struct RuleArgs {
    gv_logits_rules r;
    const char *logits;
    int64_t ld, ldo;
    float *out;
    int V, n_slices;
    int *faults;
};

struct Bias {
    int token;
    float value;
};
__device__ inline Bias bias_at(const RuleArgs &a, int64_t i, int end) {
    return i < end ? Bias{a.r.bias_token[i], a.r.bias_value[i]} : Bias{-1, 0.0f};
}

// The row's biases of tokens [v0, v0 + n) added to their logits in LDS in the list's order, by one wave: 64 of the list
// at a time (the first are in hand), at once where no two share a tag (then no two share a token), else one after the
// other.
__device__ inline void add_biases(const RuleArgs &a, Bias first, int begin, int end, int v0, int n, volatile float *x, volatile int *tag) {
    const int lane = threadIdx.x & 63;
    for (int64_t i0 = begin; i0 < end; i0 += 64) {
        const Bias e = i0 == begin ? first : bias_at(a, i0 + lane, end);
        const int v = e.token;
        const float b = e.value;
        const int at = v - v0;
        const bool mine = v >= v0 && at < n;
        uint64_t todo = __ballot(mine);
        if (todo == 0) continue;
        if (mine) tag[at & (kRuleTags - 1)] = lane;
        const bool alone = !mine || tag[at & (kRuleTags - 1)] == lane;
        if (__all(alone)) {
            if (mine) x[at] = __fadd_rn(x[at], b);
            continue;
        }
        for (; todo; todo &= todo - 1)
            if (lane == __builtin_ctzll(todo)) x[at] = __fadd_rn(x[at], b);
    }
}

// four logits from an address of their own alignment (the wide load takes it), or the m < 4 that a row ends in
template <int TYPE>
__device__ inline float4 load_logits(const char *p, int m) {
    struct __attribute__((packed, aligned(4))) F4 { float x, y, z, w; };
    struct __attribute__((packed, aligned(2))) H4 { uint32_t lo, hi; };
    if (m >= 4) {
        if constexpr (TYPE == GV_F32) {
            const F4 v = *reinterpret_cast<const F4 *>(p);
            return float4{v.x, v.y, v.z, v.w};
        } else {
            const H4 w = *reinterpret_cast<const H4 *>(p);
            if constexpr (TYPE == GV_F16) return float4{half_lo(w.lo), half_hi(w.lo), half_lo(w.hi), half_hi(w.hi)};
            return float4{bf16_lo(w.lo), bf16_hi(w.lo), bf16_lo(w.hi), bf16_hi(w.hi)};
        }
    }
    const auto one = [p](int k) {
        if constexpr (TYPE == GV_F32) return *reinterpret_cast<const float *>(p + 4 * k);
        const uint32_t w = *reinterpret_cast<const uint16_t *>(p + 2 * k);
        if constexpr (TYPE == GV_F16) return half_lo(w);
        return bf16_lo(w);
    };
    return float4{m > 0 ? one(0) : 0.0f, m > 1 ? one(1) : 0.0f, m > 2 ? one(2) : 0.0f, 0.0f};
}
__device__ inline void store_logits(float *p, float4 x, int m) {
    struct __attribute__((packed, aligned(4))) F4 { float x, y, z, w; };
    if (m >= 4) *reinterpret_cast<F4 *>(p) = F4{x.x, x.y, x.z, x.w};
    else {
        if (m > 0) p[0] = x.x;
        if (m > 1) p[1] = x.y;
        if (m > 2) p[2] = x.z;
    }
}

// Q: quads a thread takes (the slice: Q x 1,024 tokens)
template <int TYPE, int Q, bool IN_PLACE>
__global__ __launch_bounds__(kRuleThreads) void logits_rules_kernel(const RuleArgs a) {
    constexpr int S = Q * kRuleQuad;
    __shared__ __align__(16) uint32_t word[S];
    touch_args(a);
    const int row = blockIdx.x / a.n_slices, v0 = (blockIdx.x % a.n_slices) * S;
    const int n = min(S, a.V - v0), tid = threadIdx.x;
    const char *src = a.logits + (row * a.ld + v0) * (TYPE == GV_F32 ? 4 : 2);
    float *dst = a.out + row * a.ldo + v0;
    float4 x[Q];
    if constexpr (!IN_PLACE)
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const int v = 4 * tid + k * kRuleQuad;
            x[k] = load_logits<TYPE>(src + static_cast<int64_t>(v) * (TYPE == GV_F32 ? 4 : 2), n - v);
        }
    // the row's ranges and numbers, all asked for at once (an array that is not given: some other word, not used)
    const bool penal = a.r.tokens != nullptr, has_bias = a.r.bias_token != nullptr, has_mask = a.r.masks != nullptr;
    const auto word_of = [&](const void *p) { return static_cast<const int *>(p ? p : a.out)[row]; };
    int begin = word_of(a.r.begin), end = word_of(a.r.end), gen = word_of(a.r.generated);
    float rep = __int_as_float(word_of(a.r.repetition)), freq = __int_as_float(word_of(a.r.frequency));
    float pres = __int_as_float(word_of(a.r.presence));
    int bb = word_of(a.r.bias_begin), be = word_of(a.r.bias_end), of = word_of(a.r.mask_of);
    if (!a.r.generated) gen = begin;
    if (!a.r.repetition) rep = 1.0f;
    if (!a.r.frequency) freq = 0.0f;
    if (!a.r.presence) pres = 0.0f;
    const bool bad_tokens = penal && (begin < 0 || end < begin || end > a.r.n_tokens);
    const bool bad_biases = has_bias && (bb < 0 || be < bb || be > a.r.n_biases), bad_mask = has_mask && of >= a.r.n_masks;
    if ((bad_tokens || bad_biases || bad_mask) && tid == 0) queue_fault(a.faults, kFaultRange);
    if (!penal || bad_tokens || (rep == 1.0f && freq == 0.0f && pres == 0.0f)) begin = end = 0;
    if (!has_bias || bad_biases) bb = be = 0;
    // then what they point to: the quads' mask bits, the first tokens, the first biases
    uint32_t keep[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) keep[k] = 0xFu;
    if (has_mask && of >= 0 && !bad_mask) {
        const uint32_t *mask = a.r.masks + of * a.r.ld_mask + v0 / 32;
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const int v = 4 * tid + k * kRuleQuad;
            keep[k] = mask[min(v, n - 1) / 32] >> (v % 32);   // (a quad lies within a word; past the end: not used)
        }
    }
    const bool counted = end > begin, biased = be > bb;   // (uniform over the workgroup)
    constexpr int U = 8;   // tokens a thread has in flight
    int tok[U];
    const auto tokens_from = [&](int64_t i0) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int64_t i = i0 + k * kRuleThreads + tid;
            tok[k] = i < end ? a.r.tokens[i] : -1;
        }
    };
    if (counted) tokens_from(begin);
    Bias first{-1, 0.0f};
    if (biased) first = bias_at(a, static_cast<int64_t>(bb) + tid, be);
    if (counted || biased) {
#pragma unroll
        for (int k = 0; k < Q; ++k) *reinterpret_cast<uint4 *>(word + 4 * tid + k * kRuleQuad) = uint4{0, 0, 0, 0};
        __syncthreads();
        for (int64_t i0 = begin; i0 < end; i0 += U * kRuleThreads) {
            if (i0 > begin) tokens_from(i0);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int64_t i = i0 + k * kRuleThreads + tid;
                const int at = tok[k] - v0;
                if (tok[k] >= v0 && at < n) {
                    if (i >= gen) atomicAdd(word + at, 1u);
                    else atomicOr(word + at, kSeen);
                }
            }
        }
        for (int64_t i0 = bb; i0 < be; i0 += kRuleThreads) {
            const int v = i0 == bb ? first.token : bias_at(a, i0 + tid, be).token, at = v - v0;
            if (v >= v0 && at < n) atomicOr(word + at, kBiased);
        }
        __syncthreads();
    }
    const auto rule = [&](float y, uint32_t w) {
        if (w & ~kBiased) {
            y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
            const uint32_t c = w & kTimes;
            if (c) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(c))), pres);
        }
        return y;
    };
    uint32_t through = 0, still = 0;   // (bit 4 k + e: the logit has biases; in place: the quad stays as it is)
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int v = 4 * tid + k * kRuleQuad, m = min(4, n - v);
        uint4 w = uint4{0, 0, 0, 0};
        if (counted || biased) w = *reinterpret_cast<const uint4 *>(word + v);
        if constexpr (IN_PLACE) {
            const uint32_t all = m > 0 ? 0xFu >> (4 - m) : 0u;
            if ((w.x | w.y | w.z | w.w) == 0 && (keep[k] & all) == all) {
                still |= 1u << k;
                continue;
            }
            x[k] = load_logits<TYPE>(src + static_cast<int64_t>(v) * 4, m);
        }
        x[k] = float4{rule(x[k].x, w.x), rule(x[k].y, w.y), rule(x[k].z, w.z), rule(x[k].w, w.w)};
        if (biased) {
            float *y = reinterpret_cast<float *>(word + v);
            if (w.x & kBiased) through |= 1u << (4 * k), y[0] = x[k].x;
            if (w.y & kBiased) through |= 2u << (4 * k), y[1] = x[k].y;
            if (w.z & kBiased) through |= 4u << (4 * k), y[2] = x[k].z;
            if (w.w & kBiased) through |= 8u << (4 * k), y[3] = x[k].w;
        }
    }
    if (biased) {
        __shared__ int tag[kRuleTags];
        __syncthreads();
        if (tid < 64) add_biases(a, first, bb, be, v0, n, reinterpret_cast<float *>(word), tag);
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int v = 4 * tid + k * kRuleQuad;
        if (IN_PLACE && (still >> k & 1)) continue;
        if (biased) {
            const float *y = reinterpret_cast<const float *>(word + v);
            const uint32_t t = through >> (4 * k);
            if (t & 1u) x[k].x = y[0];
            if (t & 2u) x[k].y = y[1];
            if (t & 4u) x[k].z = y[2];
            if (t & 8u) x[k].w = y[3];
        }
        store_logits(dst + v, float4{keep[k] & 1u ? x[k].x : -INFINITY, keep[k] & 2u ? x[k].y : -INFINITY,
                                     keep[k] & 4u ? x[k].z : -INFINITY, keep[k] & 8u ? x[k].w : -INFINITY}, n - v);
    }
}

// The slice's quads a thread: 4 where that leaves 1,024 workgroups (four a CU), else 2 or 1. Measured, quads 1 / 2 / 4: one
// row of 151,936 logits with 300 tokens 3.8 / 4.3 / 5.0 us; 160 rows of 248,320 with up to 8,192 tokens 121 / 82 / 70 (4.5
// TB/s of logits; 8 quads: 77); 64 bf16 rows of 151,936 with masks, biases and up to 2,048 tokens 24.9 / 18.5 / 18.5 (12.4
// as a plain copy: masks, tokens and biases add their chains of loads, 2 to 3 us each).
static int rules_quads(int rows, int V) {
    int q = 4;
    while (q > 1 && static_cast<int64_t>(rows) * ((V + q * kRuleQuad - 1) / (q * kRuleQuad)) < 1024) q /= 2;
    return q;
}

template <int TYPE, int Q, bool IN_PLACE>
int launch_rules(const RuleArgs &a, int rows, hipStream_t st) {
    hipLaunchKernelGGL((logits_rules_kernel<TYPE, Q, IN_PLACE>), dim3(static_cast<unsigned>(rows) * static_cast<unsigned>(a.n_slices)),
                       dim3(kRuleThreads), 0, st, a);
    GV_CHECK_HIP(hipGetLastError());
    return 0;
}
template <int TYPE, bool IN_PLACE = false>
int launch_rules_q(const RuleArgs &a, int rows, int q, hipStream_t st) {
    switch (q) {
    case 1: return launch_rules<TYPE, 1, IN_PLACE>(a, rows, st);
    case 2: return launch_rules<TYPE, 2, IN_PLACE>(a, rows, st);
    }
    return launch_rules<TYPE, 4, IN_PLACE>(a, rows, st);
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
    GV_CHECK_ARG(!rules->tokens || (rules->begin && rules->end && rules->n_tokens >= 0 && rules->n_tokens < 1 << 30),
                 "tokens need begin, end and n_tokens (below 2^30)");
    GV_CHECK_ARG(rules->tokens || !(rules->repetition || rules->frequency || rules->presence), "penalties need tokens");
    GV_CHECK_ARG(!rules->bias_token || (rules->bias_value && rules->bias_begin && rules->bias_end && rules->n_biases >= 0),
                 "biases need bias_value, bias_begin, bias_end and n_biases");
    GV_CHECK_ARG(!rules->masks || (rules->mask_of && rules->n_masks >= 1 && rules->ld_mask >= (V + 31) / 32),
                 "masks need mask_of, n_masks and ld_mask of at least ceil(V / 32)");
    const int q = rules_quads(rows, V), n_slices = (V + q * kRuleQuad - 1) / (q * kRuleQuad);
    GV_CHECK_ARG(static_cast<int64_t>(rows) * n_slices < 1 << 24, "too many logits for one call (2^36)");
    if (ensure_init() != 0) return -1;
    OnDevice dev;
    int *faults = queued_faults();
    if (!dev.ok || !faults) return -1;
    RuleArgs a{};
    a.r = *rules;
    a.logits = static_cast<const char *>(logits), a.out = out;
    a.ld = ld, a.ldo = ldo;
    a.V = V, a.n_slices = n_slices;
    a.faults = faults;
    if (logits == static_cast<const void *>(out)) return launch_rules_q<GV_F32, true>(a, rows, q, stream());
    if (type == GV_F32) return launch_rules_q<GV_F32>(a, rows, q, stream());
    if (type == GV_F16) return launch_rules_q<GV_F16>(a, rows, q, stream());
    return launch_rules_q<GV_BF16>(a, rows, q, stream());
}
