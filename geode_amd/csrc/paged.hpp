// paged.hpp - what the calls over several conversations share: the paged cache and the batch as the kernels take them,
// the checks of the host's arguments, the device's own of what lies in device memory, and the faults it reports.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/geode_verify.h"
#include "common.hpp"
#include "kernels.hpp"

namespace gv {

// ---------------------------------------------------------------- faults met in device memory
// A kernel that meets one sets its word in pinned host memory (every writer writes 1, past the caches: a volatile store). The
// words are the host thread's whose call it is. The calls that wait and hand out results (gv_synchronize, gv_memcpy_d2h, the
// sampling and acceptance calls) read the calling thread's behind their wait, and those of threads that ended before it,
// clear them and fail.
enum QueuedFault { kFaultRows = 0, kFaultPage = 1, kFaultPosition = 2, kFaultRange = 3, kFaultCount = 4 };
int *queued_faults();   // the calling thread's words as the device addresses them (null: no memory, the error set)
struct FaultWait {      // made before the wait for the library's stream
    uint64_t ends;      // threads that had ended by then
    FaultWait();
    int told() const;   // behind the wait: 0, or -1 and a message, the words cleared
};
__device__ inline void queue_fault(int *words, int kind) {
    *reinterpret_cast<volatile int *>(words + kind) = 1;
}

// The library's GPU current for the calling thread while a call runs, whatever the thread's own choice.
struct OnDevice {
    int before = -1;
    bool ok = true;
    OnDevice();
    ~OnDevice();
};

struct KvView {
    char *k, *v;
    float *ks, *vs;
    int64_t page_stride, head_stride, pos_stride;   // elements
    int nkv, hd, page, n_pages;
};
struct BatchView {
    const int *row_start, *lens, *pages;
    int64_t ld_pages;
    int n_seqs, n_rows, max_rows, max_len;
};
inline KvView kv_view(const gv_paged_kv &c) {
    return KvView{static_cast<char *>(c.k), static_cast<char *>(c.v), c.k_scale, c.v_scale, c.page_stride, c.head_stride,
                  c.pos_stride, c.n_kv_heads, c.head_dim, c.page_size, c.n_pages};
}
inline BatchView batch_view(const gv_paged_batch &b) {
    return BatchView{b.row_start, b.lens, b.pages, b.ld_pages, b.n_seqs, b.n_rows, b.max_rows, b.max_len};
}

inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline int64_t type_bytes(int type) { return type == GV_F32 ? 4 : type == GV_I8 ? 1 : 2; }
inline bool float_type(int type) { return type == GV_F32 || type == GV_F16 || type == GV_BF16; }

// a refused argument: the call's name (a `call` in scope) before the reason
#define GV_CHECK_ARG(cond, what) GV_REQUIRE(cond, std::string(call) + ": " + (what))
// 0, or -1 and the reason
int check_kv(const gv_paged_kv *c, const char *call);
int check_batch(const gv_paged_batch *b, const gv_paged_kv *c, const char *call);

#ifdef __HIPCC__
// A kernel's argument struct, one word of each of its 64-byte lines asked for at once: the compiler asks for a field
// where it is first used, and the lines' first touches (the arguments lie in host memory) then wait one after the other
// (one appended row 5.0 -> 4.2 us).
template <typename T>
__device__ inline void touch_args(const T &a) {
    static_assert(sizeof(T) % 4 == 0 && sizeof(T) <= 512, "argument struct");
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&a);
    uint32_t v[(sizeof(T) + 63) / 64];
#pragma unroll
    for (unsigned i = 0; i < (sizeof(T) + 63) / 64; ++i) v[i] = w[i * 16];
#pragma unroll
    for (unsigned i = 0; i < (sizeof(T) + 63) / 64; ++i) asm volatile("" ::"s"(v[i]));
}

// a sequence's rows and positions as the batch gives them, and whether they fit it
struct Seq {
    int first, rows, len;   // row_start, rows, positions in the cache
    bool fits;
};
__device__ inline Seq make_seq(const BatchView &b, int a, int e, int len) {
    const int n = static_cast<int>(static_cast<unsigned>(e) - static_cast<unsigned>(a));   // (used where it fits)
    return Seq{a, n, len, a >= 0 && e >= a && e <= b.n_rows && n <= b.max_rows && len >= n && len <= b.max_len};
}
__device__ inline Seq seq_load(const BatchView &b, int i) { return make_seq(b, b.row_start[i], b.row_start[i + 1], b.lens[i]); }

// The sequence of row t, the first whose rows end behind t (n_seqs: none), and what the batch says of it. A 64-way search
// by a whole wave, one round of loads up to 64 sequences, two up to 4,096; the last round's lanes hold their sequences'
// starts and lengths too (misfit: one of those does not fit). Row starts that descend give some sequence of the batch.
__device__ inline int seq_of_row(const BatchView &b, int t, Seq &s, bool &misfit) {
    const int lane = threadIdx.x & 63;
    const int *end = b.row_start + 1;
    int lo = 0, hi = b.n_seqs;
    while (hi - lo > 64) {
        const int step = (hi - lo + 63) / 64;
        const int i = min(lo + (lane + 1) * step, hi) - 1;
        const int full = __popcll(__ballot(end[i] <= t));
        lo = min(lo + full * step, hi);
        hi = min(lo + step, hi);
    }
    const int i = lo + lane, ic = min(i, b.n_seqs - 1);
    const int first = b.row_start[ic], last = end[ic], len = b.lens[ic];
    misfit = __any(!make_seq(b, first, last, len).fits);   // (lanes past the last sequence: the last again)
    const int at = __popcll(__ballot(i < hi && last <= t));   // (64: behind all of them)
    const int src = min(at, 63);
    s = make_seq(b, __builtin_amdgcn_readlane(first, src), __builtin_amdgcn_readlane(last, src), __builtin_amdgcn_readlane(len, src));
    return lo + at < hi ? lo + at : b.n_seqs;
}

// A wave's share of the check of every sequence, row t's: of more than a row's search looks at
__device__ inline void check_sequences(const BatchView &b, int t, int *faults) {
    for (int64_t i0 = int64_t{64} * t; i0 < b.n_seqs; i0 += int64_t{64} * b.n_rows) {
        const int64_t i = i0 + (threadIdx.x & 63);
        if (i < b.n_seqs && !seq_load(b, static_cast<int>(i)).fits) queue_fault(faults, kFaultRows);
    }
}

// 32-bit floats to the 16-bit types, rounded to nearest even
__device__ inline uint32_t pack_f16(float lo, float hi) {
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, f16_of(lo))) |
           static_cast<uint32_t>(__builtin_bit_cast(uint16_t, f16_of(hi))) << 16;
}
__device__ inline uint32_t pack_bf16(float lo, float hi) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ inline float half_lo(uint32_t w) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w))); }
__device__ inline float half_hi(uint32_t w) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w >> 16))); }
__device__ inline float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ inline float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xFFFF0000u); }

// four floats stored as a type (16 or 8 bytes, aligned)
template <int TYPE>
__device__ inline void store4(char *p, float4 x) {
    if constexpr (TYPE == GV_F32) *reinterpret_cast<float4 *>(p) = x;
    else if constexpr (TYPE == GV_F16) *reinterpret_cast<uint2 *>(p) = uint2{pack_f16(x.x, x.y), pack_f16(x.z, x.w)};
    else *reinterpret_cast<uint2 *>(p) = uint2{pack_bf16(x.x, x.y), pack_bf16(x.z, x.w)};
}
#endif

}  // namespace gv
