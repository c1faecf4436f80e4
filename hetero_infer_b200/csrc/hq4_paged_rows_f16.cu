// The instances of hq4_paged_rows.cuh for f16 caches (a file to a type: they compile side by side).
#include "hq4_paged_rows.cuh"

namespace hq4 {

int paged_rows_f16(bool f32, const PagedAttnParams& p, const PaPlan& pl, cudaStream_t st) {
    return f32 ? launch_pa_dim<float, __half>(p, pl, st) : launch_pa_dim<__half, __half>(p, pl, st);
}

}  // namespace hq4
