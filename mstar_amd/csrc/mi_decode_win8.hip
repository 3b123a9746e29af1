// Windowed decode by workgroups of eight wavefronts (mi_decode_kernel.h, NW = 8).
#include "mi_decode_kernel.h"

namespace mi {

template <typename MT>
static int launch(const DecodeParams& dp, int kvt, int head_dim, int grid, hipStream_t stream) {
  switch (kvt) {
    case kKv16: return launch_decode_kernel<MT, kKv16, true, 8>(dp, head_dim, grid, stream);
    case kKvFp8: return launch_decode_kernel<MT, kKvFp8, true, 8>(dp, head_dim, grid, stream);
    case kKvMx8: return launch_decode_kernel<MT, kKvMx8, true, 8>(dp, head_dim, grid, stream);
    case kKvMx4: return launch_decode_kernel<MT, kKvMx4, true, 8>(dp, head_dim, grid, stream);
    default: return MI_ERR_UNSUPPORTED;
  }
}

bool decode_win8_serves(int kvt, int head_dim) { return decode_waves(kvt, head_dim, true) == 2; }

int decode_win8_launch(const DecodeParams& dp, int q_dtype, int kvt, int head_dim, int grid, hipStream_t stream) {
  return q_dtype == MI_BF16 ? launch<BF16>(dp, kvt, head_dim, grid, stream) : launch<F16>(dp, kvt, head_dim, grid, stream);
}

}  // namespace mi
