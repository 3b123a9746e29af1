// Eviction from a paged cache by weights of its tokens (mi_kv_evict).
//
// For each (layer, request, kv head) with more than `keep` tokens the first `sinks`, the
// last `recent` and the keep - sinks - recent heaviest of the tokens between stay (ties to the lowest
// index).  K, V, a microscaled layer's scale bytes and the weights of those that stay move to the
// request's first `keep` slots, in their order.
//
// Two launches.  evict_select_kernel finds, a workgroup for each (layer, request, kv head), the
// weight of the last token that stays by a radix select over the weights' order-preserving bits
// and lists the places that stay.  evict_move_kernel goes through that list in tiles: a tile's rows are
// all in registers before the first of them is written.  Places ascend, so a tile's
// sources lie at or behind its own first destination, and what it writes lies before every later tile's
// sources: one barrier a tile keeps the move in place, and no second copy of the cache is needed.  Tiles
// of one row are in turn, so rows are split over workgroups by head, K and V, and by pieces of the
// row where that leaves places of the chip empty.
#include "mi_internal.h"

namespace mi {

struct EvictParams {
  uint8_t* cache;
  int64_t layer_stride, page_stride, kv_stride, token_stride, head_stride, max_pages;  // bytes
  uint8_t* scales;  // microscaled: [page][K, V][kv head][block][slot]
  int64_t scale_layer_stride;
  const float* weights;
  float* out_weights;
  int64_t weights_layer_stride;
  const int32_t *kv_indptr, *kv_indices, *last_page_len;
  int32_t* kept;
  int32_t batch, num_indices, num_kv_heads, page_size, keep, recent, sinks;
  int32_t row_pieces, splits, blocks;  // 16-byte pieces of a row, workgroups that share them; blocks of a row with a scale
};

MI_DEVICE int evict_len(const EvictParams& p, int b, int& first, int& pages) {
  first = p.kv_indptr[b];
  pages = min(p.kv_indptr[b + 1], p.num_indices) - first;
  return pages > 0 ? max(0, (pages - 1) * p.page_size + min(p.last_page_len[b], p.page_size)) : 0;
}

// Bits that order as the weights do, from 1: NaN is 0, below every number, and -0 is 0.
MI_DEVICE uint32_t weight_bits(float w) {
  const uint32_t u = bitcast<uint32_t>(w + 0.f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024, kSelBins = 2048;

// Weights of four adjacent tokens t .. t + 3 (t a multiple of four: they lie in one page).
MI_DEVICE void load_bits4(const EvictParams& p, const float* weights, int first, int h, int t, int len, uint32_t (&u)[4]) {
  float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
  bool ok = t < len;
  if (ok) {
    const int e = (int)((unsigned)t / (unsigned)p.page_size), s = t - e * p.page_size;
    const int64_t page = p.kv_indices[first + e];
    ok = page >= 0 && page < p.max_pages;
    if (ok) w = *(const float4*)(weights + (page * p.num_kv_heads + h) * p.page_size + s);
  }
  u[0] = ok ? weight_bits(w.x) : 0u;
  u[1] = ok ? weight_bits(w.y) : 0u;
  u[2] = ok ? weight_bits(w.z) : 0u;
  u[3] = ok ? weight_bits(w.w) : 0u;
}

// Inclusive sum over the workgroup's 1024 threads of two counts of at most 2^31 in one 64-bit word each.
__device__ __forceinline__ void select_scan(int a, int b, int& before_a, int& before_b, int* smem) {
  int ta, tb;
  before_a = block_exclusive_scan_1024(a, ta, smem);
  before_b = block_exclusive_scan_1024(b, tb, smem);
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictParams p) {
  __shared__ int s_hist[kSelBins];
  __shared__ int s_scan[32];
  __shared__ int s_digit, s_left;
  const int tid = (int)threadIdx.x;
  const int h = uniform((int)(blockIdx.x % p.num_kv_heads)), rest = uniform((int)(blockIdx.x / p.num_kv_heads));
  const int b = uniform(rest % p.batch), layer = uniform(rest / p.batch);
  int first, pages;
  const int len = evict_len(p, b, first, pages);
  int32_t* out = p.kept + (((int64_t)layer * p.batch + b) * p.num_kv_heads + h) * p.keep;
  if (len <= p.keep) {
    for (int j = tid; j < p.keep; j += kSelThreads) out[j] = j < len ? j : -1;
    return;
  }
  const float* weights = p.weights + (int64_t)layer * p.weights_layer_stride;
  const int lo = p.sinks, hi = len - p.recent;
  int left = p.keep - p.sinks - p.recent;  // to take of [lo, hi), at least one fewer than there are
  uint32_t prefix = 0, done = 0;           // digits found of the last taken weight, and their mask
  if (left > 0) {
    for (int shift = 21; shift >= -1; shift -= 11) {  // bits 21-31, 10-20, then the last ten
      const int sh = shift < 0 ? 0 : shift;
      const uint32_t digit = shift < 0 ? 0x3ffu : 0x7ffu;
      for (int i = tid; i < kSelBins; i += kSelThreads) s_hist[i] = 0;
      __syncthreads();
      for (int t = 4 * tid; t < len; t += 4 * kSelThreads) {
        uint32_t u[4];
        load_bits4(p, weights, first, h, t, len, u);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i >= lo && t + i < hi && (u[i] & done) == prefix) atomicAdd(&s_hist[(u[i] >> sh) & digit], 1);
      }
      __syncthreads();
      // the digit at which the count of heavier weights reaches `left`: thread i holds bins 2047 - 2i and below
      const int n0 = s_hist[kSelBins - 1 - 2 * tid], n1 = s_hist[kSelBins - 2 - 2 * tid];
      int total;
      const int before = block_exclusive_scan_1024(n0 + n1, total, s_scan);
      if (before < left && before + n0 >= left) {
        s_digit = kSelBins - 1 - 2 * tid;
        s_left = left - before;
      } else if (before + n0 < left && before + n0 + n1 >= left) {
        s_digit = kSelBins - 2 - 2 * tid;
        s_left = left - before - n0;
      }
      __syncthreads();
      prefix |= (uint32_t)s_digit << sh;
      done |= digit << sh;
      left = s_left;
      __syncthreads();
    }
  }
  // `left` of the tokens whose bits equal prefix stay, the first ones; none where nothing is taken by weight
  const bool take = p.keep - p.sinks - p.recent > 0;
  const int per_thread = 4 * ((len + 4 * kSelThreads - 1) / (4 * kSelThreads));
  const int t0 = min(tid * per_thread, len), t1 = min(t0 + per_thread, len);
  int heavy = 0, equal = 0;
  for (int t = t0; t < t1; t += 4) {
    uint32_t u[4];
    load_bits4(p, weights, first, h, t, len, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = t + i;
      if (at >= t1) continue;
      const bool mid = at >= lo && at < hi;
      heavy += !mid || (take && u[i] > prefix);
      equal += mid && take && u[i] == prefix;
    }
  }
  int heavy_before, equal_before;
  select_scan(heavy, equal, heavy_before, equal_before, s_scan);
  for (int t = t0; t < t1; t += 4) {
    uint32_t u[4];
    load_bits4(p, weights, first, h, t, len, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = t + i;
      if (at >= t1) continue;
      const bool mid = at >= lo && at < hi;
      const bool is_heavy = !mid || (take && u[i] > prefix), is_equal = mid && take && u[i] == prefix;
      if (is_heavy || (is_equal && equal_before < left)) {
        const int to = heavy_before + min(equal_before, left);
        if (to < p.keep) out[to] = at;  // always, where the weights do not change under the call
      }
      heavy_before += is_heavy;
      equal_before += is_equal;
    }
  }
}

constexpr int kMoveThreads = 256, kMoveRows = 8;  // 16-byte pieces a thread has in flight

// Where token t of a request lies: page id and slot, false where the id is out of range.
MI_DEVICE bool evict_place(const EvictParams& p, int first, int pages, int t, int64_t& page, int& slot) {
  const int e = (int)((unsigned)t / (unsigned)p.page_size);
  slot = t - e * p.page_size;
  page = e < pages ? p.kv_indices[first + e] : -1;
  return page >= 0 && page < p.max_pages;
}

// Workgroups: (layer, request, kv head) x parts; part 0 .. 2 splits - 1: a share of the pieces of the
// K, then of the V rows; the last: weights and scale bytes.
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictParams p) {
  const int tid = (int)threadIdx.x, parts = 2 * p.splits + 1;
  const int part = uniform((int)(blockIdx.x % parts)), unit = uniform((int)(blockIdx.x / parts));
  const int h = uniform(unit % p.num_kv_heads), rest = uniform(unit / p.num_kv_heads);
  const int b = uniform(rest % p.batch), layer = uniform(rest / p.batch);
  int first, pages;
  const int len = evict_len(p, b, first, pages);
  const int32_t* kept = p.kept + (int64_t)unit * p.keep;
  const bool cut = len > p.keep;
  const int n = min(len, p.keep);
  if (part < 2 * p.splits) {
    if (!cut) return;
    const int v = part >= p.splits, share = part - v * p.splits;
    const int per = p.row_pieces / p.splits;  // pieces of a row, a power of two
    const int row = tid / per, piece = share * per + tid % per, rows = kMoveThreads / per;
    uint8_t* base = p.cache + layer * p.layer_stride + v * p.kv_stride + h * p.head_stride + 16 * piece;
    for (int j0 = 0; j0 < n; j0 += rows * kMoveRows) {
      uint4 x[kMoveRows];
      int64_t from[kMoveRows], to[kMoveRows];
#pragma unroll
      for (int i = 0; i < kMoveRows; ++i) {
        const int j = j0 + i * rows + row, src = j < n ? kept[j] : -1;
        int64_t page, page_to;
        int slot, slot_to;
        const bool move = src > j && evict_place(p, first, pages, src, page, slot) &&  // not there already
                          evict_place(p, first, pages, j, page_to, slot_to);
        from[i] = move ? page * p.page_stride + slot * p.token_stride : -1;
        to[i] = move ? page_to * p.page_stride + slot_to * p.token_stride : -1;
      }
#pragma unroll
      for (int i = 0; i < kMoveRows; ++i) x[i] = from[i] >= 0 ? *(const uint4*)(base + from[i]) : make_uint4(0, 0, 0, 0);
      __syncthreads();  // the tile's rows are in registers
#pragma unroll
      for (int i = 0; i < kMoveRows; ++i)
        if (to[i] >= 0) *(uint4*)(base + to[i]) = x[i];
    }
    return;
  }
  // weights (copied for every request, moved in place or not), then scale bytes
  const float* weights = p.weights + (int64_t)layer * p.weights_layer_stride;
  float* out_weights = p.out_weights + (int64_t)layer * p.weights_layer_stride;
  if (cut || p.weights != p.out_weights) {
    for (int j0 = 0; j0 < n; j0 += kMoveThreads * kMoveRows) {
      float x[kMoveRows];
      float* to[kMoveRows];
#pragma unroll
      for (int i = 0; i < kMoveRows; ++i) {
        const int j = j0 + i * kMoveThreads + tid, src = j < n ? kept[j] : -1;
        int64_t page, page_to;
        int slot, slot_to;
        const bool move = src >= 0 && evict_place(p, first, pages, src, page, slot) && evict_place(p, first, pages, j, page_to, slot_to);
        x[i] = move ? weights[(page * p.num_kv_heads + h) * p.page_size + slot] : 0.f;
        to[i] = move ? out_weights + (page_to * p.num_kv_heads + h) * p.page_size + slot_to : nullptr;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMoveRows; ++i)
        if (to[i]) *to[i] = x[i];
    }
  }
  if (!cut || !p.scales) return;
  uint8_t* scales = p.scales + (int64_t)layer * p.scale_layer_stride;
  for (int row = 0; row < 2 * p.blocks; ++row) {  // K's blocks, then V's
    const int v = row >= p.blocks, blk = row - v * p.blocks;
    for (int j0 = 0; j0 < n; j0 += kMoveThreads * kMoveRows) {
      uint8_t x[kMoveRows];
      uint8_t* to[kMoveRows];
#pragma unroll
      for (int i = 0; i < kMoveRows; ++i) {
        const int j = j0 + i * kMoveThreads + tid, src = j < n ? kept[j] : -1;
        int64_t page, page_to;
        int slot, slot_to;
        const bool move = src > j && evict_place(p, first, pages, src, page, slot) && evict_place(p, first, pages, j, page_to, slot_to);
        const int64_t line = (int64_t)(v * p.num_kv_heads + h) * p.blocks + blk, lines = 2LL * p.num_kv_heads * p.blocks;
        x[i] = move ? scales[(page * lines + line) * p.page_size + slot] : 0;
        to[i] = move ? scales + (page_to * lines + line) * p.page_size + slot_to : nullptr;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMoveRows; ++i)
        if (to[i]) *to[i] = x[i];
    }
  }
}

}  // namespace mi

extern "C" int mi_kv_evict(const mi_paged_kv* kv, int32_t num_layers, int64_t layer_stride, int64_t scale_layer_stride,
                           const float* weights, float* out_weights, int64_t weights_layer_stride, const int32_t* kv_indptr,
                           const int32_t* kv_indices, const int32_t* last_page_len, int32_t batch, int32_t num_indices, int32_t keep,
                           int32_t recent, int32_t sinks, int32_t* kept, void* stream) {
  using namespace mi;
  if (!kv || num_layers < 0 || batch < 0 || num_indices < 0) return MI_ERR_INVALID;
  if (keep <= 0 || recent < 0 || sinks < 0 || recent > keep - sinks) return MI_ERR_INVALID;
  if (num_layers == 0 || batch == 0) return MI_OK;
  if (!kv->data || !weights || !out_weights || !kv_indptr || !kv_indices || !last_page_len || !kept) return MI_ERR_INVALID;
  if (kv->num_kv_heads <= 0 || kv->head_dim <= 0 || kv->page_size <= 0 || kv->max_pages < 0) return MI_ERR_INVALID;
  // places in the page list are counted in 32 bits
  if (kv->page_size % 4 || kv->page_size > (1 << 24) || (int64_t)num_indices * kv->page_size > INT32_MAX - (1 << 25))
    return MI_ERR_UNSUPPORTED;
  const bool mx = kv_is_mx(kv->dtype);
  if (!mx && kv->dtype != MI_BF16 && kv->dtype != MI_F16 && kv->dtype != MI_F32 && kv->dtype != MI_FP8_E4M3) return MI_ERR_UNSUPPORTED;
  if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return MI_ERR_UNSUPPORTED;
  const int esz = kv_elem_bytes(kv->dtype);
  if (!kv_aligned16(kv) || (layer_stride * esz) % 16) return MI_ERR_INVALID;
  if (((uintptr_t)weights | (uintptr_t)out_weights) % 16 || weights_layer_stride % 4) return MI_ERR_INVALID;
  if (mx && (!kv_scales_ok(kv) || kv->head_dim % kMxBlock)) return MI_ERR_INVALID;
  EvictParams p{};
  p.cache = (uint8_t*)kv->data;
  p.layer_stride = layer_stride * esz;
  p.page_stride = kv->page_stride * esz;
  p.kv_stride = kv->kv_stride * esz;
  p.token_stride = kv->token_stride * esz;
  p.head_stride = kv->head_stride * esz;
  p.max_pages = kv->max_pages;
  p.blocks = kv->head_dim / kMxBlock;
  if (mx) {
    // one array: V's bytes follow K's within a page
    if ((const uint8_t*)kv->v_scale - (const uint8_t*)kv->k_scale != (int64_t)kv->num_kv_heads * p.blocks * kv->page_size)
      return MI_ERR_INVALID;
    p.scales = (uint8_t*)kv->k_scale;
    p.scale_layer_stride = scale_layer_stride;
  }
  p.weights = weights;
  p.out_weights = out_weights;
  p.weights_layer_stride = weights_layer_stride;
  p.kv_indptr = kv_indptr;
  p.kv_indices = kv_indices;
  p.last_page_len = last_page_len;
  p.kept = kept;
  p.batch = batch;
  p.num_indices = num_indices;
  p.num_kv_heads = kv->num_kv_heads;
  p.page_size = kv->page_size;
  p.keep = keep;
  p.recent = recent;
  p.sinks = sinks;
  p.row_pieces = (kv->dtype == MI_MXFP4 ? kv->head_dim / 2 : kv->head_dim * esz) / 16;
  const int64_t units = (int64_t)num_layers * batch * kv->num_kv_heads;
  p.splits = 1;
  while (p.splits * 4 < p.row_pieces && 2 * units * p.splits < 4LL * device_cu_count()) p.splits *= 2;
  if (units * (2 * p.splits + 1) > INT32_MAX) return MI_ERR_UNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(evict_select_kernel, dim3((uint32_t)units), dim3(kSelThreads), 0, s, p);
  hipLaunchKernelGGL(evict_move_kernel, dim3((uint32_t)(units * (2 * p.splits + 1))), dim3(kMoveThreads), 0, s, p);
  MI_CHECK_LAUNCH();
  return MI_OK;
}
