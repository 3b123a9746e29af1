// Accumulated attention weights over fp8 and microscaled caches: instantiations (mi_weights.hip).
#include "mi_weights_kernel.h"

namespace mi {

template <typename MT>
static int launch_scaled(const WeightsParams& p, int kvt, int head_dim, int which, dim3 grid, hipStream_t s) {
  switch (kvt) {
    case kKvFp8: return launch_weights_kvt<MT, kKvFp8>(p, head_dim, which, grid, s);
    case kKvMx8: return launch_weights_kvt<MT, kKvMx8>(p, head_dim, which, grid, s);
    case kKvMx4: return launch_weights_kvt<MT, kKvMx4>(p, head_dim, which, grid, s);
    default: return MI_ERR_UNSUPPORTED;
  }
}

int weights_launch_scaled(const WeightsParams& p, int q_dtype, int kvt, int head_dim, int which, dim3 grid, hipStream_t s) {
  return q_dtype == MI_BF16 ? launch_scaled<BF16>(p, kvt, head_dim, which, grid, s)
                            : launch_scaled<F16>(p, kvt, head_dim, which, grid, s);
}

}  // namespace mi
