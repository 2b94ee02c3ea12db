// paged_attn_bf16.hip - the paged attention's kernels over a bf16 cache.
#include "paged_attn_wide.hpp"

namespace gv {

int launch_attn_bf16(const AttnArgs &a, int ct, unsigned grid, hipStream_t st) {
    return a.type == GV_F32 ? launch_attn_nt<GV_BF16, 3, 3>(a, ct, grid, st) : launch_attn_nt<GV_BF16, 1, 2>(a, ct, grid, st);
}

}  // namespace gv
