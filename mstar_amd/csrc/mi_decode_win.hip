// Windowed decode: the attend kernels with a sliding window and sinks over every
// KV format, and the merge of their items (mi_decode_kernel.h, mi_merge.h).
#include "mi_decode_kernel.h"
#include "mi_merge.h"

namespace mi {

template <typename MT>
static int launch_win(const DecodeParams& dp, int kvt, int head_dim, int grid, hipStream_t stream) {
  switch (kvt) {
    case kKv16: return launch_decode_kernel<MT, kKv16, true>(dp, head_dim, grid, stream);
    case kKvFp8: return launch_decode_kernel<MT, kKvFp8, true>(dp, head_dim, grid, stream);
    case kKvMx8: return launch_decode_kernel<MT, kKvMx8, true>(dp, head_dim, grid, stream);
    case kKvMx4: return launch_decode_kernel<MT, kKvMx4, true>(dp, head_dim, grid, stream);
    default: return MI_ERR_UNSUPPORTED;
  }
}

int decode_win_launch(const DecodeParams& dp, int q_dtype, int kvt, int head_dim, int grid, hipStream_t stream) {
  return q_dtype == MI_BF16 ? launch_win<BF16>(dp, kvt, head_dim, grid, stream)
                            : launch_win<F16>(dp, kvt, head_dim, grid, stream);
}

template <typename MT, int D, int RUN>
__global__ __launch_bounds__(256) void merge_win_kernel(DecodeParams p) {
  merge_body<MT, D, RUN, false, true>(p, p.batch, (int)blockIdx.x);
}

template <typename MT, int D>
static void launch_merge_win(const DecodeParams& dp, bool bytes, hipStream_t stream) {
  const dim3 grid(dp.batch * dp.num_kv_heads);
  if (bytes) hipLaunchKernelGGL((merge_win_kernel<MT, D, lane_run(D, 1)>), grid, dim3(256), 0, stream, dp);
  else hipLaunchKernelGGL((merge_win_kernel<MT, D, lane_run(D, 2)>), grid, dim3(256), 0, stream, dp);
}

template <typename MT>
static int launch_merge_d(const DecodeParams& dp, bool bytes, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: launch_merge_win<MT, 64>(dp, bytes, stream); break;
    case 128: launch_merge_win<MT, 128>(dp, bytes, stream); break;
    case 256: launch_merge_win<MT, 256>(dp, bytes, stream); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

int decode_win_merge_launch(const DecodeParams& dp, int q_dtype, int kvt, int head_dim, hipStream_t stream) {
  const bool bytes = kvt != kKv16;
  return q_dtype == MI_BF16 ? launch_merge_d<BF16>(dp, bytes, head_dim, stream)
                            : launch_merge_d<F16>(dp, bytes, head_dim, stream);
}

}  // namespace mi
