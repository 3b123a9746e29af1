// Split-KV paged GQA decode for MI355X (gfx950).
//
// Replaces FlashInfer's BatchDecodeWithPagedKVCacheWrapper plan/run as used by
// FlashInferDecodeWrapper (mstar/utils/flashinfer_utils.py:369-465), and the
// short-query part of the prefill wrapper (requests whose
// qo_len * group <= 16).
//
// Work decomposition
//   plan  : one 1024-thread workgroup splits every request's page list into
//           items of at most `item_pages` pages (chosen on the GPU from the
//           batch's total page count so the machine gets ~8K wavefronts) and
//           writes the item list into the caller's workspace.
//   decode: one workgroup per (item, kv-head); its 4 wavefronts take
//           contiguous quarters of the item's 16-token tiles.  A wavefront's
//           16 MFMA columns are the (query token, q-head-in-group) rows that
//           share the kv-head, so K/V are read from HBM once per GQA group.
//           Per tile:
//             S^T[16 tok x 16 rows] = K[16 x D] . Q^T      (v_mfma 16x16x32)
//             online softmax on S (fp32, exp2 domain)
//             O^T[D x 16 rows]     += V^T[D x 16 tok] . P^T (v_mfma 16x16x16)
//           K and V rows are read as whole head_dim rows (16 lanes x 128 bits
//           per row for D=128; every load instruction covers 256 contiguous
//           bytes of a row, see dim_of) with non-temporal loads, two tiles
//           ahead of the MFMA work.  The MFMA A operand wants one token per lane%16, which
//           a register-only layout can only feed with 64-byte row segments
//           (measured ~15% slower to stream from HBM), so K passes through a
//           small per-wave LDS buffer: ds_write of the rows, ds_read of the
//           fragments.  V is transposed in registers (v_perm_b32): output
//           row i of output tile m is the dim lane i loaded as its element m
//           (dim_of), which turns the transpose into a 4x(D/16) shuffle
//           inside each lane.
//           The 4 wavefronts' softmax states are merged in LDS; an item that
//           covers its whole request writes the final output, otherwise a
//           partial (o, lse).  Partial stores are HBM writes interleaved with
//           a read-saturated stream and cost far more than their bytes
//           (measured: ~33 MB of partials added ~14% to the kernel), which
//           is why an item spans 4 wavefronts' worth of pages.
//   merge : log-sum-exp merge of the item partials of split requests, in the
//           same register-order layout (whole-cache-line loads and stores).
#include "mi_common.h"
#include "mi_internal.h"
#include "mi_plan.h"
#include "mi_decode_kernel.h"
#include "mi_merge.h"

namespace mi {

constexpr int kMinChunkTokens = 1024;  // never split a request finer than this (4 waves x 256)
// ... except in small jobs, down to this, while the items fit one round of
// resident workgroups (decode_plan_body)
constexpr int kSmallChunkTokens = 256;

// Target number of wavefronts for one plan: ~4K (item, kv-head, quarter)
// wave units fill 256 CUs x 2 resident workgroups about twice; with the
// longest-first work order the drain tail stays short while few requests
// need partials (measured on c3: 4096 -> 545 us, 8192 -> 558 us,
// 16384 -> 586 us; 2048 and 1024 units: 538-540 and 609 us).
constexpr int32_t kDecodeTargetUnits = 4096;
// head_dim 256: one resident workgroup per CU and twice the bytes per token,
// so fewer and longer items: c3's contexts at 16 q / 2 kv heads 536 -> 507 us
// (1536 units: 524 us); smaller batches, whose items kMinChunkTokens bounds
// (Pi0.5's 8 q / 1 kv), are unchanged.
constexpr int32_t kDecodeTargetUnitsWide = 1024;

SplitLayout split_layout(int32_t batch, int32_t nkv, int32_t head_dim, int64_t ws_avail, bool pair) {
  SplitLayout L;
  // a paired plan is a head_dim 256 plan over half the kv-heads
  const int32_t tnkv = pair ? nkv / 2 : nkv, thd = pair ? 2 * head_dim : head_dim;
  const int32_t units = thd > 128 ? kDecodeTargetUnitsWide : kDecodeTargetUnits;
  int32_t target = units / (4 * (tnkv > 0 ? tnkv : 1));  // 4 waves per item
  if (target < 16) target = 16;
  int64_t max_chunks = (int64_t)target + batch;
  if (ws_avail >= 0) {  // fewer, longer chunks when the caller's workspace is smaller
    const int64_t fixed = 256 + mi_align_up(4LL * (batch + 1), 256) + 3 * 256;
    const int64_t per_chunk = 16 + 4LL * nkv * kRows + 4LL * nkv * kRows * head_dim;
    const int64_t fit = (ws_avail - fixed) / per_chunk;
    if (fit < max_chunks) max_chunks = fit;
  }
  L.max_chunks = (int32_t)max_chunks;
  int64_t off = 0;
  L.hdr = off;
  off += 256;
  L.chunk_indptr = off;
  off = mi_align_up(off + 4LL * (batch + 1), 256);
  L.work = off;
  off = mi_align_up(off + 16LL * L.max_chunks, 256);
  L.lse = off;
  off = mi_align_up(off + 4LL * L.max_chunks * nkv * kRows, 256);
  L.opart = off;
  off = mi_align_up(off + 4LL * L.max_chunks * nkv * kRows * head_dim, 256);
  L.total = off;
  return L;
}

__global__ __launch_bounds__(1024) void decode_plan_kernel(PlanParams p) { decode_plan_body(p); }

// The index arrays in the argument: they are in LDS for the plan, so its
// chain of reads does not wait for memory either.
__global__ __launch_bounds__(1024) void decode_plan_host_kernel(PlanParams p, HostIndices m) {
  __shared__ int32_t s_idx[MI_PLAN_HOST_ARGS];
  host_indices_copy(m, s_idx, true);
  p.kv_indptr = s_idx;
  p.kv_indices = s_idx + m.end[0];
  p.last_page_len = s_idx + m.end[1];
  decode_plan_body(p);
}

// The index arrays in pinned host memory: workgroup 0 reads the per-request
// ones over the bus into LDS, plans from there and writes their device copies,
// the others copy the page list.  One launch for a host-to-device copy, three
// device copies into a graph's static buffers and the plan: 64 requests of up
// to 4096 tokens, a captured pass of three layers 216.5 -> 204.5 us (this
// kernel 6.7 us, the plan kernel over device arrays 5-6).
struct PinnedIndices {
  const int32_t* src;  // [kv_indptr | last_page_len | kv_indices]
  int32_t num_indices;
  int32_t *kv_indptr, *kv_indices, *last_page_len;
};
__global__ __launch_bounds__(1024) void decode_plan_pinned_kernel(PlanParams p, PinnedIndices m) {
  __shared__ int32_t s_idx[2 * MI_PLAN_PINNED_BATCH + 1];
  const int b = p.batch;
  const int32_t* idx = m.src + 2 * b + 1;
  if (blockIdx.x > 0) {
    for (int i = ((int)blockIdx.x - 1) * 1024 + (int)threadIdx.x; i < m.num_indices; i += ((int)gridDim.x - 1) * 1024)
      m.kv_indices[i] = idx[i];
    return;
  }
  for (int i = (int)threadIdx.x; i < 2 * b + 1; i += 1024) {
    const int32_t v = m.src[i];
    s_idx[i] = v;
    if (i <= b) m.kv_indptr[i] = v; else m.last_page_len[i - b - 1] = v;
  }
  __syncthreads();
  p.kv_indptr = s_idx;
  p.last_page_len = s_idx + b + 1;
  p.kv_indices = idx;  // each request's last page, for the write locations
  decode_plan_body(p);
}

// ----------------------------------------------------------------- merge
template <typename MT, int D, int RUN, bool PAIR = false>
__global__ __launch_bounds__(256) void merge_kernel(DecodeParams p, int32_t batch) {
  merge_body<MT, D, RUN, PAIR>(p, batch, (int)blockIdx.x);
}

// ------------------------------------------------------------ host side
static bool supported_head_dim(int d) { return d == 64 || d == 128 || d == 256; }

int decode_plan_params(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                       const int32_t* last_page_len, int32_t batch, int32_t page_size,
                       int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                       int64_t* kv_locations, void* workspace, int64_t workspace_bytes,
                       int64_t ws_offset, PlanParams* out, bool ragged_pair) {
  if (batch < 0 || !kv_indptr || !last_page_len || !workspace) return MI_ERR_INVALID;
  if (batch > 0 && !kv_indices) return MI_ERR_INVALID;
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads) return MI_ERR_INVALID;
  if (num_qo_heads / num_kv_heads > kRows) return MI_ERR_UNSUPPORTED;
  if (page_size <= 0) return MI_ERR_INVALID;
  if (page_size % 16) return MI_ERR_UNSUPPORTED;
  if (!supported_head_dim(head_dim)) return MI_ERR_UNSUPPORTED;
  const bool pair = pair_heads(qo_indptr, batch, num_kv_heads, num_qo_heads / num_kv_heads, head_dim, ragged_pair);
  const SplitLayout L = split_layout(batch, num_kv_heads, head_dim, workspace_bytes - ws_offset, pair);
  if (L.max_chunks <= batch || workspace_bytes < ws_offset + L.total) return MI_ERR_WORKSPACE;
  uint8_t* ws = (uint8_t*)workspace + ws_offset;
  PlanParams& pp = *out;
  pp.short_rows = pair_short_rows(pair);
  pp.qo_indptr = qo_indptr;
  pp.kv_indptr = kv_indptr;
  pp.num_pages = nullptr;
  pp.kv_indices = kv_indices;
  pp.last_page_len = last_page_len;
  pp.batch = batch;
  pp.target = L.max_chunks - batch;
  pp.min_chunk_pages = (kMinChunkTokens + page_size - 1) / page_size;
  pp.max_chunks = L.max_chunks;
  // resident workgroups per kv-head (or pair): two per CU at head_dim <= 128,
  // one for the head_dim 256 kernels
  const int heads = pair ? num_kv_heads / 2 : num_kv_heads;
  const int per_cu = (pair || head_dim > 128) ? 1 : 2;
  const int slots = device_cu_count() * per_cu / heads;
  pp.slots = slots < 1 ? 1 : (slots < L.max_chunks ? slots : L.max_chunks);
  pp.floor_pages = (kSmallChunkTokens + page_size - 1) / page_size;
  pp.group = num_qo_heads / num_kv_heads;
  pp.hdr = (int32_t*)(ws + L.hdr);
  pp.chunk_indptr = (int32_t*)(ws + L.chunk_indptr);
  pp.work = (int4*)(ws + L.work);
  pp.kv_locations = kv_locations;
  return MI_OK;
}

int decode_plan_impl(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                     const int32_t* last_page_len, int32_t batch, int32_t page_size,
                     int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                     int64_t* kv_locations, void* workspace, int64_t workspace_bytes,
                     int64_t ws_offset, hipStream_t stream) {
  PlanParams pp{};
  const int st = decode_plan_params(qo_indptr, kv_indptr, kv_indices, last_page_len, batch, page_size, num_qo_heads,
                                    num_kv_heads, head_dim, kv_locations, workspace, workspace_bytes, ws_offset, &pp);
  if (st != MI_OK) return st;
  hipLaunchKernelGGL(decode_plan_kernel, dim3(1), dim3(1024), 0, stream, pp);
  MI_CHECK_LAUNCH();
  return MI_OK;
}

static int decode_plan_host_impl(const int32_t* const* src, int32_t num_indices, int32_t* const* dst, int32_t batch,
                                 int32_t page_size, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                 int64_t* kv_locations, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  PlanParams pp{};
  int st = decode_plan_params(nullptr, dst[0], dst[1], dst[2], batch, page_size, num_qo_heads, num_kv_heads, head_dim,
                              kv_locations, workspace, workspace_bytes, 0, &pp);
  if (st != MI_OK) return st;
  const int32_t len[3] = {batch + 1, num_indices, batch};
  HostIndices m;
  st = host_indices(src, len, dst, 3, &m);
  if (st != MI_OK) return st;
  if (src[0][batch] > num_indices) return MI_ERR_INVALID;  // pages past the argument's
  hipLaunchKernelGGL(decode_plan_host_kernel, dim3(1), dim3(1024), 0, stream, pp, m);
  MI_CHECK_LAUNCH();
  return MI_OK;
}

template <typename MT, bool FP8, int D>
static void launch_decode(const DecodeParams& dp, int grid, int batch, int phases, hipStream_t stream) {
  if (phases & kPhaseAttend)
    hipLaunchKernelGGL((decode_kernel<MT, FP8, D>), dim3(grid), dim3(256), 0, stream, dp);
  if ((phases & kPhaseMerge) && batch > 0)
    hipLaunchKernelGGL((merge_kernel<MT, D, lane_run(D, FP8 ? 1 : 2)>), dim3(batch * dp.num_kv_heads),
                       dim3(256), 0, stream, dp, batch);
}

// Paired kv-heads (dp.num_kv_heads counts pairs): the head_dim 256 kernels.
template <typename MT, bool FP8>
static void launch_decode_pair(const DecodeParams& dp, int grid, int batch, int phases, hipStream_t stream) {
  if (phases & kPhaseAttend)
    hipLaunchKernelGGL((decode_kernel<MT, FP8, 256, true>), dim3(grid), dim3(256), 0, stream, dp);
  if ((phases & kPhaseMerge) && batch > 0)
    hipLaunchKernelGGL((merge_kernel<MT, 256, lane_run(256, FP8 ? 1 : 2), true>),
                       dim3(batch * dp.num_kv_heads), dim3(256), 0, stream, dp, batch);
}

template <int D>
static void launch_merge_f32(const DecodeParams& dp, int batch, hipStream_t stream) {
  hipLaunchKernelGGL((merge_kernel<F32Out, D, lane_run(D, 4)>), dim3(batch * dp.num_kv_heads), dim3(256),
                     0, stream, dp, batch);
}

int merge_launch(const DecodeParams& dp, int head_dim, int out_dtype, int batch, hipStream_t stream) {
  if (out_dtype != MI_F32) return MI_ERR_UNSUPPORTED;
  if (batch <= 0) return MI_OK;
  switch (head_dim) {
    case 64: launch_merge_f32<64>(dp, batch, stream); break;
    case 128: launch_merge_f32<128>(dp, batch, stream); break;
    case 256: launch_merge_f32<256>(dp, batch, stream); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

template <typename MT, bool FP8>
static int dispatch_d(const DecodeParams& dp, int head_dim, int grid, int batch, int phases, hipStream_t stream) {
  switch (head_dim) {
    case 64: launch_decode<MT, FP8, 64>(dp, grid, batch, phases, stream); break;
    case 128: launch_decode<MT, FP8, 128>(dp, grid, batch, phases, stream); break;
    case 256: launch_decode<MT, FP8, 256>(dp, grid, batch, phases, stream); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

constexpr int32_t kPageTokensMax = 1 << 24;

// Windows and sink counts are clamped here: beyond any context, and sums with a length stay in 32 bits.
constexpr int32_t kWinMax = 1 << 30;

// Items of a windowed run: a request's share of the resident workgroups, at most
// win_items_max of its tiles, within the workspace's partials.  One request of 1028
// keys at 4 kv heads: one item a head 13.1 us, 2 8.6, 3 7.3, 4 and more 6.5; of 32k
// keys: 16 items 25 us + 4.5 for the merge, 32 16 + 7; 96 requests of 4100 keys at 2
// kv heads, 4 bits: one 58 us, 2 45 + 4.  With more (request, kv-head) pairs than workgroups
// no cut paid (256 requests of up to 8256 keys at 4 kv heads, one item 384 us, two to
// four 384-394 + 4); taking the longest first did (455 -> 384 us), as uncut requests
// are as uneven as their lengths.
// n is a floor: one pair more than half of the places, or all of them, has about half the
// wavefronts (windows of 1028 keys at head_dim 128: 256 pairs 26.7 us, 260 to 264 37;
// 512 48, 516 to 520 60 to 71), and with one item a request those stand on CUs as they come.
static void win_items(DecodeParams& dp, int heads, int slots, int max_chunks) {
  int64_t n = slots / ((int64_t)dp.batch * heads);
  const int most = win_items_max(win_tiles_max(dp));
  if (n > most) n = most;
  if (n > max_chunks / dp.batch) n = max_chunks / dp.batch;
  dp.splits = n < 1 ? 1 : (int)n;
  dp.sorted = dp.batch <= kSortedMax && (int64_t)dp.batch * heads * dp.splits > slots;
}

// Whether requests that win_items cuts go whole to a workgroup of eight wavefronts:
// without partials and merge.  Cut in two they had as many wavefronts (us, cut -> whole:
// 60 requests at 4 kv heads x 128, windows of 250 11.7 -> 8.4, 1024 26.9 -> 22.8, 4090
// 87 -> 83; 96 at 2 x 256 in 4 bits, 4090 47.3 -> 43.1); cut in more, short windows
// still gain (one request, 250 keys 7.9 -> 6.2, 500 8.8 -> 7.6) and longer ones lose
// (1024 keys 9.0 -> 9.6 at 4 x 128, 11.4 -> 15.1 at 2 x 256 in 4 bits).  The rule goes by
// the window, as the requests' lengths are on the device: short requests behind a long
// window are cut.  Not measured: eight wavefronts where a request has one item anyway.
constexpr int kWinEightTiles = 40;
static bool win_by_eight(const DecodeParams& dp) {
  return dp.splits == 2 || (dp.splits > 2 && win_tiles_max(dp) <= kWinEightTiles);
}

int decode_run_impl(const void* q, int32_t q_dtype, int64_t q_stride_token, int64_t q_stride_head,
                    const mi_paged_kv* kv, const int32_t* qo_indptr, const int32_t* kv_indptr,
                    const int32_t* kv_indices, const int32_t* last_page_len, int32_t batch,
                    int32_t num_qo_heads, int32_t causal, float sm_scale, void* workspace,
                    int64_t workspace_bytes, int64_t ws_offset, void* out,
                    int64_t out_stride_token, int64_t out_stride_head, int phases, hipStream_t stream,
                    bool ragged_pair, DecodeParams* merge_args, int32_t window_left, int32_t sinks) {
  if (!kv || batch < 0 || !workspace) return MI_ERR_INVALID;
  if (batch == 0) return MI_OK;
  if (!q || !out || !kv->data || !kv_indptr || !kv_indices || !last_page_len) return MI_ERR_INVALID;
  const int nkv = kv->num_kv_heads, D = kv->head_dim;
  if (nkv <= 0 || num_qo_heads <= 0 || num_qo_heads % nkv) return MI_ERR_INVALID;
  if (num_qo_heads / nkv > kRows) return MI_ERR_UNSUPPORTED;
  if (kv->page_size <= 0) return MI_ERR_INVALID;
  if (kv->page_size % 16 || !supported_head_dim(D)) return MI_ERR_UNSUPPORTED;
  const bool fp8 = kv->dtype == MI_FP8_E4M3, mx = kv_is_mx(kv->dtype), win = window_left >= 0;
  if (q_dtype != MI_BF16 && q_dtype != MI_F16 && q_dtype != MI_F32) return MI_ERR_UNSUPPORTED;
  if (!fp8 && !mx && kv->dtype != q_dtype) return MI_ERR_UNSUPPORTED;
  if ((fp8 || mx || win) && q_dtype == MI_F32) return MI_ERR_UNSUPPORTED;
  if (!kv_scales_ok(kv)) return MI_ERR_INVALID;
  const int qesz = q_dtype == MI_F32 ? 4 : 2;
  if (!rows_aligned16(q, q_stride_token, q_stride_head, qesz) ||
      !rows_aligned16(out, out_stride_token, out_stride_head, qesz) || !kv_aligned16(kv))
    return MI_ERR_INVALID;
  // decode_kernel keeps a slot's offset within a page in 32 bits, the fp32 kernel one within
  // 16 tokens, and both the tokens of 64 pages
  const int64_t offsets = q_dtype == MI_F32 ? 16 : kv->page_size;
  if (kv->token_stride < 0 || kv->token_stride >= (1LL << 32) || kv->page_size > kPageTokensMax ||
      offsets * kv->token_stride * kv_elem_bytes(kv->dtype) >= (1LL << 32))
    return MI_ERR_UNSUPPORTED;
  // the same pairing decision as the plan's (shapes only), so the layouts agree
  const bool pair = pair_heads(qo_indptr, batch, nkv, num_qo_heads / nkv, D, ragged_pair);
  const SplitLayout L = split_layout(batch, nkv, D, workspace_bytes - ws_offset, pair);
  if (L.max_chunks <= batch || workspace_bytes < ws_offset + L.total) return MI_ERR_WORKSPACE;
  uint8_t* ws = (uint8_t*)workspace + ws_offset;
  // the paired kernels: 16-bit caches whose pairs' two 128-element rows are
  // adjacent (NHD pools); fp8, fp32 and other layouts run the per-head
  // kernels on the same plan
  const bool pair_kernel = pair && !fp8 && !mx && q_dtype != MI_F32 && kv->head_stride == D;

  DecodeParams dp{};
  dp.q = q;
  dp.q_stride_tok = q_stride_token;
  dp.q_stride_head = q_stride_head;
  dp.kv = kv->data;
  dp.page_stride = kv->page_stride;
  dp.kv_stride = kv->kv_stride;
  dp.token_stride = kv->token_stride;
  dp.head_stride = kv->head_stride;
  dp.k_scale = kv->k_scale;
  dp.v_scale = kv->v_scale;
  dp.qo_indptr = qo_indptr;
  dp.kv_indptr = kv_indptr;
  dp.kv_indices = kv_indices;
  dp.last_page_len = last_page_len;
  dp.hdr = (const int32_t*)(ws + L.hdr);
  dp.work = (const int4*)(ws + L.work);
  dp.chunk_indptr = (const int32_t*)(ws + L.chunk_indptr);
  dp.lse_part = (float*)(ws + L.lse);
  dp.o_part = (float*)(ws + L.opart);
  dp.out = out;
  dp.out_stride_tok = out_stride_token;
  dp.out_stride_head = out_stride_head;
  dp.num_kv_heads = nkv;
  dp.group = num_qo_heads / nkv;
  dp.page_size = kv->page_size;
  dp.causal = causal ? 1 : 0;
  dp.scale_log2 = sm_scale * 1.4426950408889634f;
  dp.short_rows = pair_short_rows(pair);
  const int grid = (int)((L.max_chunks + 7) / 8 * 8 * (int64_t)nkv);
  int st;
  if (win) {
    dp.window_left = window_left < kWinMax ? window_left : kWinMax;
    dp.sinks = sinks < kWinMax ? sinks : kWinMax;
    dp.batch = batch;
    const int heads = pair_kernel ? nkv / 2 : nkv;
    const int kvt = kv_format(kv->dtype);
    win_items(dp, heads, device_cu_count() * decode_waves(kvt, pair_kernel ? 256 : D, true), L.max_chunks);
    if (pair_kernel) {
      dp.num_kv_heads = heads;
      dp.head_stride = 2 * kv->head_stride;
    }
    const bool eight = !pair_kernel && win_by_eight(dp) && decode_win8_serves(kvt, D);
    if (eight) dp.splits = 1;
    st = MI_OK;
    if (phases & kPhaseAttend) {
      const int wgrid = (int)(((int64_t)batch * dp.splits + 7) / 8 * 8 * heads);
      st = eight ? decode_win8_launch(dp, q_dtype, kvt, D, wgrid, stream)
                 : decode_win_launch(dp, q_dtype, kvt, D, pair_kernel, wgrid, stream);
    }
    if (st == MI_OK && (phases & kPhaseMerge) && dp.splits > 1)
      st = decode_win_merge_launch(dp, q_dtype, kvt, D, pair_kernel, batch, stream);
    if (st != MI_OK) return st;
    MI_CHECK_LAUNCH();
    return MI_OK;
  }
  if (merge_args) *merge_args = dp;
  if (pair_kernel) {
    dp.num_kv_heads = nkv / 2;
    dp.head_stride = 2 * kv->head_stride;
    const int pgrid = (int)((L.max_chunks + 7) / 8 * 8 * (int64_t)(nkv / 2));
    if (q_dtype == MI_BF16)
      fp8 ? launch_decode_pair<BF16, true>(dp, pgrid, batch, phases, stream)
          : launch_decode_pair<BF16, false>(dp, pgrid, batch, phases, stream);
    else
      fp8 ? launch_decode_pair<F16, true>(dp, pgrid, batch, phases, stream)
          : launch_decode_pair<F16, false>(dp, pgrid, batch, phases, stream);
    MI_CHECK_LAUNCH();
    return MI_OK;
  }
  if (q_dtype == MI_F32) {  // fp32 q, cache and output
    st = MI_OK;
    if (phases & kPhaseAttend) st = f32_attend_launch(dp, D, grid, stream);
    if (st == MI_OK && (phases & kPhaseMerge)) st = merge_launch(dp, D, MI_F32, batch, stream);
    if (st != MI_OK) return st;
    MI_CHECK_LAUNCH();
    return MI_OK;
  }
  if (mx && (phases & kPhaseAttend)) {
    st = decode_mx_launch(dp, q_dtype, kv_format(kv->dtype), D, grid, stream);
    if (st != MI_OK) return st;
    phases &= ~kPhaseAttend;  // the merge is that of fp8 caches: a lane holds the same elements
  }
  const bool bytes = fp8 || mx;
  if (q_dtype == MI_BF16)
    st = bytes ? dispatch_d<BF16, true>(dp, D, grid, batch, phases, stream)
               : dispatch_d<BF16, false>(dp, D, grid, batch, phases, stream);
  else
    st = bytes ? dispatch_d<F16, true>(dp, D, grid, batch, phases, stream)
               : dispatch_d<F16, false>(dp, D, grid, batch, phases, stream);
  if (st != MI_OK) return st;
  MI_CHECK_LAUNCH();
  return MI_OK;
}

int64_t decode_workspace_bytes_impl(int32_t batch, int32_t num_kv_heads, int32_t head_dim) {
  if (batch < 0 || num_kv_heads <= 0 || head_dim <= 0) return MI_ERR_INVALID;
  return split_layout(batch, num_kv_heads, head_dim, -1).total;
}

}  // namespace mi

extern "C" {

int64_t mi_decode_workspace_bytes(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                  int32_t head_dim) {
  if (num_qo_heads <= 0) return MI_ERR_INVALID;
  return mi::decode_workspace_bytes_impl(batch, num_kv_heads, head_dim);
}

int mi_decode_plan(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                   const int32_t* last_page_len, int32_t batch, int32_t page_size,
                   int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                   int64_t* kv_locations, void* workspace, int64_t workspace_bytes, void* stream) {
  return mi::decode_plan_impl(qo_indptr, kv_indptr, kv_indices, last_page_len, batch, page_size,
                              num_qo_heads, num_kv_heads, head_dim, kv_locations, workspace,
                              workspace_bytes, 0, (hipStream_t)stream);
}

int mi_decode_plan_host(const int32_t* kv_indptr_host, const int32_t* kv_indices_host,
                        const int32_t* last_page_len_host, int32_t num_indices, int32_t* kv_indptr,
                        int32_t* kv_indices, int32_t* last_page_len, int32_t batch, int32_t page_size,
                        int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, int64_t* kv_locations,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  const int32_t* const src[3] = {kv_indptr_host, kv_indices_host, last_page_len_host};
  int32_t* const dst[3] = {kv_indptr, kv_indices, last_page_len};
  return mi::decode_plan_host_impl(src, num_indices, dst, batch, page_size, num_qo_heads, num_kv_heads, head_dim,
                                   kv_locations, workspace, workspace_bytes, (hipStream_t)stream);
}

int mi_decode_plan_pinned(const int32_t* indices_pinned, int32_t num_indices, int32_t* kv_indptr,
                          int32_t* kv_indices, int32_t* last_page_len, int32_t batch, int32_t page_size,
                          int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, int64_t* kv_locations,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace mi;
  PlanParams pp{};
  const int st = decode_plan_params(nullptr, kv_indptr, kv_indices, last_page_len, batch, page_size, num_qo_heads,
                                    num_kv_heads, head_dim, kv_locations, workspace, workspace_bytes, 0, &pp);
  if (st != MI_OK) return st;
  if (batch > MI_PLAN_PINNED_BATCH) return MI_ERR_UNSUPPORTED;
  if (num_indices < 0 || (num_indices > 0 && !kv_indices)) return MI_ERR_INVALID;  // copied also without requests
  if (!indices_pinned || !device_reachable(indices_pinned)) return MI_ERR_INVALID;
  const PinnedIndices m{indices_pinned, num_indices, kv_indptr, kv_indices, last_page_len};
  const int copies = num_indices < 64 * 1024 ? (num_indices + 1023) / 1024 : 64;
  hipLaunchKernelGGL(decode_plan_pinned_kernel, dim3(1 + copies), dim3(1024), 0, (hipStream_t)stream, pp, m);
  MI_CHECK_LAUNCH();
  return MI_OK;
}

#define MI_DECODE_ARGS                                                                           \
  const void *q, int32_t q_dtype, int64_t q_stride_token, int64_t q_stride_head,                 \
      const mi_paged_kv *kv, const int32_t *qo_indptr, const int32_t *kv_indptr,                 \
      const int32_t *kv_indices, const int32_t *last_page_len, int32_t batch, int32_t num_qo_heads, \
      int32_t causal, float sm_scale, void *workspace, int64_t workspace_bytes, void *out,       \
      int64_t out_stride_token, int64_t out_stride_head, void *stream
#define MI_DECODE_FWD(phases)                                                                      \
  mi::decode_run_impl(q, q_dtype, q_stride_token, q_stride_head, kv, qo_indptr, kv_indptr,         \
                      kv_indices, last_page_len, batch, num_qo_heads, causal, sm_scale, workspace, \
                      workspace_bytes, 0, out, out_stride_token, out_stride_head, phases,          \
                      (hipStream_t)stream)

int mi_decode_run(MI_DECODE_ARGS) { return MI_DECODE_FWD(mi::kPhaseAttend | mi::kPhaseMerge); }
int mi_decode_attend(MI_DECODE_ARGS) { return MI_DECODE_FWD(mi::kPhaseAttend); }
int mi_decode_merge(MI_DECODE_ARGS) { return MI_DECODE_FWD(mi::kPhaseMerge); }

int mi_decode_run_window(const void* q, int32_t q_dtype, int64_t q_stride_token, int64_t q_stride_head,
                         const mi_paged_kv* kv, const int32_t* qo_indptr, const int32_t* kv_indptr,
                         const int32_t* kv_indices, const int32_t* last_page_len, int32_t batch, int32_t num_qo_heads,
                         int32_t causal, float sm_scale, int32_t window_left, int32_t sink_tokens, void* workspace,
                         int64_t workspace_bytes, void* out, int64_t out_stride_token, int64_t out_stride_head,
                         void* stream) {
  if (sink_tokens < 0) return MI_ERR_INVALID;
  return mi::decode_run_impl(q, q_dtype, q_stride_token, q_stride_head, kv, qo_indptr, kv_indptr, kv_indices,
                             last_page_len, batch, num_qo_heads, causal, sm_scale, workspace, workspace_bytes, 0, out,
                             out_stride_token, out_stride_head, mi::kPhaseAttend | mi::kPhaseMerge, (hipStream_t)stream,
                             false, nullptr, window_left, sink_tokens);
}

}  // extern "C"
