// paged_attn_f16.hip - the paged attention's kernels over an fp16 cache.
#include "paged_attn_wide.hpp"

namespace gv {

int launch_attn_f16(const AttnArgs &a, int ct, unsigned grid, hipStream_t st) {
    return a.type == GV_F32 ? launch_attn_nt<GV_F16, 2, 2>(a, ct, grid, st) : launch_attn_nt<GV_F16, 1, 2>(a, ct, grid, st);
}

}  // namespace gv
