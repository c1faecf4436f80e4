// The instances of hq4_paged_rows.cuh for bf16 caches (a file to a type: they compile side by side).
#include "hq4_paged_rows.cuh"

namespace hq4 {

int paged_rows_bf16(bool f32, const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st) {
    return f32 ? launch_pa_dim<float, __nv_bfloat16>(p, pl, st) : launch_pa_dim<__nv_bfloat16, __nv_bfloat16>(p, pl, st);
}

}  // namespace hq4
