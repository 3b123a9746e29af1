// Decode over microscaled caches: the attend kernels of mi_decode_kernel.h (the
// plan and the merge are those of the other formats).
#include "mi_decode_kernel.h"

namespace mi {

int decode_mx_launch(const DecodeParams& dp, int q_dtype, int kvt, int head_dim, int grid, hipStream_t stream) {
  if (q_dtype == MI_BF16)
    return kvt == kKvMx8 ? launch_decode_kernel<BF16, kKvMx8, false>(dp, head_dim, grid, stream)
                         : launch_decode_kernel<BF16, kKvMx4, false>(dp, head_dim, grid, stream);
  return kvt == kKvMx8 ? launch_decode_kernel<F16, kKvMx8, false>(dp, head_dim, grid, stream)
                       : launch_decode_kernel<F16, kKvMx4, false>(dp, head_dim, grid, stream);
}

}  // namespace mi
