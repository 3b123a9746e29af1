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

int decode_win_launch(const DecodeParams& dp, int q_dtype, int kvt, int head_dim, bool pair, int grid, hipStream_t stream) {
  if (pair) {  // 16-bit caches only
    if (q_dtype == MI_BF16) hipLaunchKernelGGL((decode_kernel<BF16, kKv16, 256, true, true>), dim3(grid), dim3(256), 0, stream, dp);
    else hipLaunchKernelGGL((decode_kernel<F16, kKv16, 256, true, true>), dim3(grid), dim3(256), 0, stream, dp);
    return MI_OK;
  }
  return q_dtype == MI_BF16 ? launch_win<BF16>(dp, kvt, head_dim, grid, stream)
                            : launch_win<F16>(dp, kvt, head_dim, grid, stream);
}

template <typename MT, int D, int RUN, bool PAIR = false>
__global__ __launch_bounds__(256) void merge_win_kernel(DecodeParams p, int32_t batch) {
  merge_body<MT, D, RUN, PAIR, true>(p, batch, (int)blockIdx.x);
}

template <typename MT, int D>
static void launch_merge_win(const DecodeParams& dp, bool bytes, dim3 grid, int batch, hipStream_t stream) {
  if (bytes) hipLaunchKernelGGL((merge_win_kernel<MT, D, lane_run(D, 1)>), grid, dim3(256), 0, stream, dp, batch);
  else hipLaunchKernelGGL((merge_win_kernel<MT, D, lane_run(D, 2)>), grid, dim3(256), 0, stream, dp, batch);
}

template <typename MT>
static int launch_merge_d(const DecodeParams& dp, bool bytes, int head_dim, bool pair, int batch, hipStream_t stream) {
  const dim3 grid(batch * dp.num_kv_heads);
  if (pair) {
    hipLaunchKernelGGL((merge_win_kernel<MT, 256, lane_run(256, 2), true>), grid, dim3(256), 0, stream, dp, batch);
    return MI_OK;
  }
  switch (head_dim) {
    case 64: launch_merge_win<MT, 64>(dp, bytes, grid, batch, stream); break;
    case 128: launch_merge_win<MT, 128>(dp, bytes, grid, batch, stream); break;
    case 256: launch_merge_win<MT, 256>(dp, bytes, grid, batch, stream); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

int decode_win_merge_launch(const DecodeParams& dp, int q_dtype, int kvt, int head_dim, bool pair, int batch,
                            hipStream_t stream) {
  const bool bytes = kvt != kKv16;
  return q_dtype == MI_BF16 ? launch_merge_d<BF16>(dp, bytes, head_dim, pair, batch, stream)
                            : launch_merge_d<F16>(dp, bytes, head_dim, pair, batch, stream);
}

}  // namespace mi
