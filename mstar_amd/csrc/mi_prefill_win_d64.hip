// Windowed prefill tiles at head_dim 64, over every KV format (mi_prefill_kernel.h).
#include "mi_prefill_kernel.h"

namespace mi {

template <typename MT>
static int launch(const PrefillParams& pp, int kvt, int grid, hipStream_t stream) {
  const dim3 block(64 * pf_waves(64));
  switch (kvt) {
    case kKv16: hipLaunchKernelGGL((prefill_kernel<MT, kKv16, 64, true>), dim3(grid), block, 0, stream, pp); break;
    case kKvFp8: hipLaunchKernelGGL((prefill_kernel<MT, kKvFp8, 64, true>), dim3(grid), block, 0, stream, pp); break;
    case kKvMx8: hipLaunchKernelGGL((prefill_kernel<MT, kKvMx8, 64, true>), dim3(grid), block, 0, stream, pp); break;
    case kKvMx4: hipLaunchKernelGGL((prefill_kernel<MT, kKvMx4, 64, true>), dim3(grid), block, 0, stream, pp); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

int prefill_win_d64_launch(const PrefillParams& pp, bool f16, int kvt, int grid, hipStream_t stream) {
  return f16 ? launch<F16>(pp, kvt, grid, stream) : launch<BF16>(pp, kvt, grid, stream);
}

}  // namespace mi
