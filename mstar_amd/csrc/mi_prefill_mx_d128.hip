// Prefill tiles over microscaled caches at head_dim 128 (mi_prefill_kernel.h).
// Built with the scheduler of mi_prefill_d128.hip.
#include "mi_prefill_kernel.h"

namespace mi {

template <typename MT>
static int launch(const PrefillParams& pp, int kvt, int grid, hipStream_t stream) {
  const dim3 block(64 * pf_waves(128));
  switch (kvt) {
    case kKvMx8: hipLaunchKernelGGL((prefill_kernel<MT, kKvMx8, 128, false>), dim3(grid), block, 0, stream, pp); break;
    case kKvMx4: hipLaunchKernelGGL((prefill_kernel<MT, kKvMx4, 128, false>), dim3(grid), block, 0, stream, pp); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

int prefill_mx_d128_launch(const PrefillParams& pp, bool f16, int kvt, int grid, hipStream_t stream) {
  return f16 ? launch<F16>(pp, kvt, grid, stream) : launch<BF16>(pp, kvt, grid, stream);
}

}  // namespace mi
