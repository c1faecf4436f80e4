// The instances of hq4_paged_tc.cuh for f16 (a file to a type: they compile side by side).
#include "hq4_paged_tc.cuh"

namespace hq4 {

int paged_tc_f16(const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st) { return launch_pt_dim<__half>(p, pl, st); }

}  // namespace hq4
