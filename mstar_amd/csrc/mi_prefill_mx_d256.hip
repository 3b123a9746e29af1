// Prefill tiles over microscaled caches at head_dim 256 (mi_prefill_rs.h).
#include "mi_prefill_rs.h"

namespace mi {

template <typename MT>
static int launch(const PrefillParams& pp, int kvt, int grid, hipStream_t stream) {
  const dim3 block(512);
  switch (kvt) {
    case kKvMx8: hipLaunchKernelGGL((prefill_rs_kernel<MT, kKvMx8, 256, false>), dim3(grid), block, 0, stream, pp); break;
    case kKvMx4: hipLaunchKernelGGL((prefill_rs_kernel<MT, kKvMx4, 256, false>), dim3(grid), block, 0, stream, pp); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

int prefill_mx_d256_launch(const PrefillParams& pp, bool f16, int kvt, int grid, hipStream_t stream) {
  return f16 ? launch<F16>(pp, kvt, grid, stream) : launch<BF16>(pp, kvt, grid, stream);
}

}  // namespace mi
