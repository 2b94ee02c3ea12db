// paged_attn_i8.hip - the paged attention's kernels over an int8 cache.
#include "paged_attn_wide.hpp"

namespace gv {

int launch_attn_i8(const AttnArgs &a, int ct, unsigned grid, hipStream_t st) {
    return a.type == GV_F32 ? launch_attn_nt<GV_I8, 2, 2>(a, ct, grid, st) : launch_attn_nt<GV_I8, 1, 2>(a, ct, grid, st);
}

}  // namespace gv
