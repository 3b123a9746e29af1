// Eviction from a paged cache by weights of its tokens (mi_kv_evict).
//
// For each (layer, request, kv head) with more than `keep` tokens the first `sinks`, the
// last `recent` and the keep - sinks - recent heaviest of the tokens between stay (ties to the lowest
// index).  K, V, a microscaled layer's scale bytes and the weights of those that stay move to the
// request's first `keep` slots, in their order.
//
// Two launches.  evict_select_kernel finds, a workgroup for each (layer, request, kv head), the
// weight of the last token that stays by a radix select over the weights' order-preserving bits,
// held in registers, and lists the places that stay.  evict_move_kernel goes through that list in tiles.  Places
// ascend, so a tile's sources lie at or behind its own first destination, and what it writes lies before every
// later tile's sources: a tile is written once its rows are all in registers, while the next one's are loaded, one
// barrier a tile keeps the move in place, and no second copy of the cache is needed.  Tiles of one row are
// in turn, so rows are split over workgroups by head, K and V, and by pieces of 128 bytes of the row where that
// leaves places of the chip empty (pieces of 64 bytes: 123 -> 147 us for one request in 28 layers, none: 140).
// Where little is kept, and there is a compute unit for each (layer, request, kv head), one launch does both
// (evict_small_kernel: 8 requests x 2 heads, 256 of 300 to 700 tokens stay, 11 us against 15; with 4096 units of 256 KiB
// it took 545 against 370).
//
// HBM bound: 256 requests of 512 to 32768 tokens, 4 heads x 128, bf16, 2048 stay: selecting 40 us, moving 1.38 GB (in and
// out) 327 us, 4.2 TB/s in pieces of 256 bytes, of the 5.0 that a copy in order reaches.
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
  int32_t batch, num_indices, num_kv_heads, page_size, page_shift, keep, recent, sinks;
  int32_t row_pieces, splits, blocks, parts;  // 16-byte pieces of a row, workgroups that share them; blocks with a scale
};

MI_DEVICE int evict_len(const EvictParams& p, int b, int& first, int& pages) {
  first = p.kv_indptr[b];
  pages = min(p.kv_indptr[b + 1], p.num_indices) - first;
  return pages > 0 ? max(0, (pages - 1) * p.page_size + min(p.last_page_len[b], p.page_size)) : 0;
}

// Bits that order as the tokens do: 0 for none, 1 for a NaN and a page out of range, then the numbers (-0 as 0), and above
// all of those the first and last tokens, which stay whatever they weigh.
constexpr uint32_t kNanBits = 0x7fc00000u;
MI_DEVICE uint32_t token_bits(const EvictParams& p, uint32_t weight, int t, int len) {
  const uint32_t u = bitcast<uint32_t>(bitcast<float>(weight) + 0.f);
  uint32_t bits = (u & 0x7fffffffu) > 0x7f800000u ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u;
  if (t < p.sinks || t >= len - p.recent) bits = 0xffffffffu;
  return t < len ? bits : 0u;
}

constexpr int kSelBins = 2048;
constexpr int kSelRegs = 8;  // of a thread, each the weights of four tokens; what is past them is read again

struct SelectShared {
  int hist[2][kSelBins];  // in turn: one is cleared while the other is in use
  int sum[16], digit, left, count, heavy[16], equal[16];
};

MI_DEVICE bool evict_page_ok(const EvictParams& p, int page) { return page >= 0 && page < p.max_pages; }
MI_DEVICE const uint4* weights_at(const EvictParams& p, const float* weights, int64_t page, int h, int slot) {
  return (const uint4*)(weights + (page * p.num_kv_heads + h) * p.page_size + slot);
}

// Entry of a request's page list that holds token t.
MI_DEVICE int entry_of(const EvictParams& p, int t) {
  return p.page_shift >= 0 ? t >> p.page_shift : (int)((unsigned)t / (unsigned)p.page_size);
}
// Exclusive sum over a workgroup of NT threads (smem: NT / 64 ints, free again after the caller's next barrier).
template <int NT>
MI_DEVICE int before_mine(int v, int* smem) {
  const int lane = lane_id(), w = uniform((int)threadIdx.x >> 6), x = wave_inclusive_sum(v);
  if (lane == 63) smem[w] = x;
  __syncthreads();
  const int t = wave_inclusive_sum(lane < NT / kWave ? smem[lane] : 0);
  return (w ? __builtin_amdgcn_readlane(t, w - 1) : 0) + x - v;
}

// Bits of four adjacent tokens t .. t + 3 (t a multiple of four: they lie in one page).
MI_DEVICE void load_bits4(const EvictParams& p, const float* weights, int first, int h, int t, int len, uint32_t (&u)[4]) {
  uint4 w = make_uint4(kNanBits, kNanBits, kNanBits, kNanBits);
  if (t < len) {
    const int e = entry_of(p, t), page = p.kv_indices[first + e];
    if (evict_page_ok(p, page)) w = *weights_at(p, weights, page, h, t - e * p.page_size);
  }
  u[0] = token_bits(p, w.x, t, len), u[1] = token_bits(p, w.y, t + 1, len);
  u[2] = token_bits(p, w.z, t + 2, len), u[3] = token_bits(p, w.w, t + 3, len);
}

MI_DEVICE int lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The places that stay of a (layer, request, kv head), to out, and to list where it is not null (in LDS); len > keep.
// Wavefront w has the tokens of run w, four to a lane, 256 at a time.
template <int NT>
__device__ __forceinline__ void evict_select(const EvictParams& p, SelectShared& s, const float* weights, int first, int h, int len,
                                             int32_t* out, int32_t* list) {
  const int tid = (int)threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6);
  const int rounds = (len + 4 * NT - 1) / (4 * NT), base = wave * rounds * 256;
  const int mine = uniform(min(rounds, (len - base + 255) >> 8));  // rounds with tokens; none where it is not positive
  uint32_t u[kSelRegs][4];
  {
    int page[kSelRegs];
#pragma unroll
    for (int i = 0; i < kSelRegs; ++i) {
      const int t = base + 256 * i + 4 * lane;
      page[i] = i < mine && t < len ? p.kv_indices[first + entry_of(p, t)] : -1;
    }
    for (int i = tid; i < 2 * kSelBins / 4; i += NT) ((int4*)s.hist)[i] = make_int4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kSelRegs; ++i) {
      uint4 w = make_uint4(kNanBits, kNanBits, kNanBits, kNanBits);
      const int t = base + 256 * i + 4 * lane;
      if (evict_page_ok(p, page[i])) w = *weights_at(p, weights, page[i], h, t - entry_of(p, t) * p.page_size);
      u[i][0] = w.x, u[i][1] = w.y, u[i][2] = w.z, u[i][3] = w.w;
    }
#pragma unroll
    for (int i = 0; i < kSelRegs; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) u[i][j] = token_bits(p, u[i][j], base + 256 * i + 4 * lane + j, len);
  }
  auto visit = [&](auto&& f) {  // four tokens at a time, ascending
#pragma unroll
    for (int i = 0; i < kSelRegs; ++i)
      if (i < mine) f(base + 256 * i, u[i]);
    for (int i = kSelRegs; i < mine; ++i) {
      uint32_t x[4];
      load_bits4(p, weights, first, h, base + 256 * i + 4 * lane, len, x);
      f(base + 256 * i, x);
    }
  };
  int left = p.keep, count = 0;   // to take, fewer than there are; tokens that share the digits found
  uint32_t prefix = 0, done = 0;  // digits found of the last taken token, and their mask
  __syncthreads();
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {  // bits 21-31, 10-20, then the last ten
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit = pass == 2 ? 0x3ffu : 0x7ffu;
    int* hist = s.hist[pass & 1];
    visit([&](int, const uint32_t (&x)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((x[j] & done) == prefix) atomicAdd(&hist[(x[j] >> shift) & digit], 1);
    });
    __syncthreads();
    // the digit at which the count of heavier tokens reaches `left`: thread i holds bins BINS (NT - 1 - i) and on
    constexpr int BINS = kSelBins / NT;
    const int* bins = hist + BINS * (NT - 1 - tid);
    int n[BINS], sum = 0;
#pragma unroll
    for (int i = 0; i < BINS; ++i) sum += n[i] = bins[i];
    int before = before_mine<NT>(sum, s.sum);
    if (before < left && before + sum >= left) {
#pragma unroll
      for (int i = BINS - 1; i >= 0; --i) {
        if (before < left && before + n[i] >= left) {
          s.digit = BINS * (NT - 1 - tid) + i;
          s.left = left - before;
          s.count = n[i];
        }
        before += n[i];
      }
    }
    if (pass == 0) {  // the third digit's
      // every thread is past its reading of the first's: before_mine has a barrier behind it
      for (int i = tid; i < kSelBins / 4; i += NT) ((int4*)s.hist[0])[i] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    prefix |= (uint32_t)s.digit << shift;
    done |= digit << shift;
    left = s.left;
    count = s.count;
    if (count == left) break;  // all that share these digits stay
    __syncthreads();
  }
  auto put = [&](int to, int t) {
    if (to >= p.keep) return;  // never, where the weights do not change under the call
    out[to] = t;
    if (list) list[to] = t;
  };
  if (count == left) {  // what stays: its digits reach those found
    int stay = 0;
    visit([&](int, const uint32_t (&x)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) stay += __popcll(__builtin_amdgcn_ballot_w64((x[j] & done) >= prefix));
    });
    if (lane == 0) s.heavy[wave] = stay;
    __syncthreads();
    stay = 0;
    for (int i = 0; i < wave; ++i) stay += s.heavy[i];
    visit([&](int t, const uint32_t (&x)[4]) {
      int to = stay;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t m = __builtin_amdgcn_ballot_w64((x[j] & done) >= prefix);
        to += lanes_before(m);
        stay += __popcll(m);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((x[j] & done) >= prefix) put(to++, t + 4 * lane + j);
    });
    return;
  }
  // ties: the heavier ones, and the first `left` of those that weigh the same
  int heavy = 0, equal = 0;
  visit([&](int, const uint32_t (&x)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      heavy += __popcll(__builtin_amdgcn_ballot_w64(x[j] > prefix));
      equal += __popcll(__builtin_amdgcn_ballot_w64(x[j] == prefix));
    }
  });
  if (lane == 0) {
    s.heavy[wave] = heavy;
    s.equal[wave] = equal;
  }
  __syncthreads();
  heavy = equal = 0;
  for (int i = 0; i < wave; ++i) heavy += s.heavy[i], equal += s.equal[i];
  visit([&](int t, const uint32_t (&x)[4]) {
    int h0 = heavy, e0 = equal;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t a = __builtin_amdgcn_ballot_w64(x[j] > prefix), b = __builtin_amdgcn_ballot_w64(x[j] == prefix);
      h0 += lanes_before(a);
      e0 += lanes_before(b);
      heavy += __popcll(a);
      equal += __popcll(b);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool a = x[j] > prefix, b = x[j] == prefix;
      if (a || (b && e0 < left)) put(h0 + min(e0, left), t + 4 * lane + j);
      h0 += a;
      e0 += b;
    }
  });
}

template <int NT>
__global__ __launch_bounds__(NT, NT == 256 ? 6 : 8) void evict_select_kernel(EvictParams p) {
  __shared__ __attribute__((aligned(16))) SelectShared s;
  const int h = uniform((int)(blockIdx.x % p.num_kv_heads)), rest = uniform((int)(blockIdx.x / p.num_kv_heads));
  const int b = uniform(rest % p.batch), layer = uniform(rest / p.batch);
  int first, pages;
  const int len = evict_len(p, b, first, pages);
  int32_t* out = p.kept + (((int64_t)layer * p.batch + b) * p.num_kv_heads + h) * p.keep;
  if (len <= p.keep) {
    for (int j = (int)threadIdx.x; j < p.keep; j += NT) out[j] = j < len ? j : -1;
    return;
  }
  evict_select<NT>(p, s, p.weights + (int64_t)layer * p.weights_layer_stride, first, h, len, out, nullptr);
}

constexpr int kSelFew = 4096;  // tokens of a request, on average, up to which 256 threads select
constexpr int kMoveThreads = 256, kMoveRows = 8;  // 16-byte pieces a thread has in flight, of a tile
constexpr int kMovePlaces = 256;                  // rows of a tile, at most

// Where token t of a request lies: page id and slot, false where the id is out of range.
MI_DEVICE bool evict_place(const EvictParams& p, int first, int pages, int t, int64_t& page, int& slot) {
  const int e = t >= 0 ? entry_of(p, t) : pages;
  slot = t - e * p.page_size;
  page = e < pages ? p.kv_indices[first + e] : -1;
  return page >= 0 && page < p.max_pages;
}

// One value of type T a token, THREADS threads: src(page, slot) -> dst(page, slot) of the kept ones; `still`: those that stay
// where they are as well.
template <typename T, int THREADS, typename Src, typename Dst>
__device__ __forceinline__ void evict_values(const EvictParams& p, int first, int pages, const int32_t* kept, int n, bool still,
                                             Src src, Dst dst) {
  for (int j0 = 0; j0 < n; j0 += THREADS * kMoveRows) {
    T x[kMoveRows];
    T* to[kMoveRows];
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i) {
      const int j = j0 + i * THREADS + (int)threadIdx.x, t = j < n ? kept[j] : -1;
      int64_t page, page_to;
      int slot, slot_to;
      const bool move = t >= 0 && (still || t > j) && evict_place(p, first, pages, t, page, slot) &&
                        evict_place(p, first, pages, j, page_to, slot_to);
      x[i] = move ? *src(page, slot) : T(0);
      to[i] = move ? dst(page_to, slot_to) : nullptr;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i)
      if (to[i]) *to[i] = x[i];
  }
}
template <int THREADS>
__device__ __forceinline__ void evict_weights(const EvictParams& p, int layer, int h, int first, int pages, const int32_t* kept, int n) {
  const bool still = p.weights != p.out_weights;
  auto at = [=](int64_t page, int slot) {
    return layer * p.weights_layer_stride + (page * p.num_kv_heads + h) * p.page_size + slot;
  };
  evict_values<float, THREADS>(p, first, pages, kept, n, still, [&](int64_t page, int slot) { return p.weights + at(page, slot); },
                               [&](int64_t page, int slot) { return p.out_weights + at(page, slot); });
}
// line: a block of K's rows, then of V's
template <int THREADS>
__device__ __forceinline__ void evict_scales(const EvictParams& p, int layer, int h, int first, int pages, const int32_t* kept, int n, int line) {
  const int v = line >= p.blocks, blk = line - v * p.blocks;
  uint8_t* base = p.scales + (int64_t)layer * p.scale_layer_stride;
  const int64_t row = (int64_t)(v * p.num_kv_heads + h) * p.blocks + blk, rows = 2LL * p.num_kv_heads * p.blocks;
  auto at = [&](int64_t page, int slot) { return base + (page * rows + row) * p.page_size + slot; };
  evict_values<uint8_t, THREADS>(p, first, pages, kept, n, false, at, at);
}

// Workgroups: (layer, request, kv head) x parts; part 0 .. 2 splits - 1: a share of the pieces of the
// K, then of the V rows; then the weights, and the lines of scale bytes.
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictParams p) {
  __shared__ int64_t s_from[4][kMovePlaces], s_to[4][kMovePlaces];
  const int tid = (int)threadIdx.x;
  const int part = uniform((int)(blockIdx.x % p.parts)), unit = uniform((int)(blockIdx.x / p.parts));
  const int h = uniform(unit % p.num_kv_heads), rest = uniform(unit / p.num_kv_heads);
  const int b = uniform(rest % p.batch), layer = uniform(rest / p.batch);
  int first, pages;
  const int len = evict_len(p, b, first, pages);
  const int32_t* kept = p.kept + (int64_t)unit * p.keep;
  const bool cut = len > p.keep;
  const int n = min(len, p.keep);
  if (part == 2 * p.splits) {
    if (cut || p.weights != p.out_weights) evict_weights<kMoveThreads>(p, layer, h, first, pages, kept, n);
    return;
  }
  if (!cut) return;
  if (part > 2 * p.splits) {
    evict_scales<kMoveThreads>(p, layer, h, first, pages, kept, n, part - 2 * p.splits - 1);
    return;
  }
  const int v = part >= p.splits, share = part - v * p.splits;
  const int per = p.row_pieces / p.splits;  // pieces of a row, a power of two
  const int row = tid / per, piece = share * per + tid % per, rows = kMoveThreads / per;
  const int steps = min(kMoveRows, kMovePlaces / rows), tile = rows * steps;
  uint8_t* base = p.cache + layer * p.layer_stride + v * p.kv_stride + h * p.head_stride + 16 * piece;
  const int tiles = (n + tile - 1) / tile;
  auto places = [&](int i) {  // of tile i's rows
    if (i >= tiles) return;
    for (int k = tid; k < tile; k += kMoveThreads) {
      const int j = i * tile + k, t = j < n ? kept[j] : -1;
      int64_t page, page_to;
      int slot, slot_to;
      const bool move = t > j && evict_place(p, first, pages, t, page, slot) &&  // not there already
                        evict_place(p, first, pages, j, page_to, slot_to);
      s_from[i & 3][k] = move ? page * p.page_stride + slot * p.token_stride : -1;
      s_to[i & 3][k] = move ? page_to * p.page_stride + slot_to * p.token_stride : -1;
    }
  };
  auto load = [&](int i, u32x4_t (&x)[kMoveRows]) {
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      const int64_t from = k < steps && i < tiles ? s_from[i & 3][k * rows + row] : -1;
      // what is read is not read again (one request of 32k tokens in 28 layers 123 -> 108 us; such stores as well: 125)
      x[k] = from >= 0 ? __builtin_nontemporal_load((const u32x4_t*)(base + from)) : u32x4_t{0u, 0u, 0u, 0u};
    }
  };
  auto store = [&](int i, const u32x4_t (&x)[kMoveRows]) {
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      const int64_t to = k < steps ? s_to[i & 3][k * rows + row] : -1;
      if (to >= 0) *(u32x4_t*)(base + to) = x[k];
    }
  };
  u32x4_t x[kMoveRows], y[kMoveRows];
  places(0);
  places(1);
  __syncthreads();
  load(0, x);
  for (int i = 0; i < tiles; i += 2) {
    places(i + 2);
    __syncthreads();  // tile i is in registers
    load(i + 1, y);
    store(i, x);
    if (i + 1 >= tiles) break;
    places(i + 3);
    __syncthreads();
    load(i + 2, x);
    store(i + 1, y);
  }
}

// Both in one launch, a workgroup for each (layer, request, kv head): K and V rows of a tile side by side, and the
// weights with the first.  It waits far more than it moves: 512 threads 11.0 us for 8 requests x 2 heads, 1024 12.1, 256 16.1.
constexpr int kSmallThreads = 512, kSmallKeep = 4096, kSmallPages = 1024, kSmallPlaces = 512;
static_assert(kSmallPlaces <= kSmallThreads, "a thread finds one place of a tile");
constexpr int64_t kSmallBytes = 256 << 10;  // of K and V that stay: four tiles
__global__ __launch_bounds__(kSmallThreads) void evict_small_kernel(EvictParams p) {
  __shared__ __attribute__((aligned(16))) SelectShared s;
  __shared__ int32_t s_kept[kSmallKeep], s_page[kSmallPages];
  __shared__ int64_t s_from[kSmallPlaces], s_to[kSmallPlaces];
  const int tid = (int)threadIdx.x;
  const int unit = (int)blockIdx.x, h = uniform(unit % p.num_kv_heads), rest = uniform(unit / p.num_kv_heads);
  const int b = uniform(rest % p.batch), layer = uniform(rest / p.batch);
  int first, pages;
  const int len = evict_len(p, b, first, pages), n = min(len, p.keep);
  const bool cut = len > p.keep;
  int32_t* out = p.kept + (int64_t)unit * p.keep;
  const float* weights = p.weights + (int64_t)layer * p.weights_layer_stride;
  float* out_weights = p.out_weights + (int64_t)layer * p.weights_layer_stride;
  for (int i = tid; i < min(pages, kSmallPages); i += kSmallThreads) s_page[i] = p.kv_indices[first + i];
  if (cut) {
    evict_select<kSmallThreads>(p, s, weights, first, h, len, out, s_kept);
  } else {
    for (int j = tid; j < p.keep; j += kSmallThreads) {
      s_kept[j] = j;
      out[j] = j < len ? j : -1;
    }
    if (p.weights == p.out_weights) return;
  }
  __syncthreads();
  auto place = [&](int t, int64_t& page, int& slot) {  // as evict_place
    const int e = t >= 0 ? entry_of(p, t) : pages;
    slot = t - e * p.page_size;
    page = e >= pages ? -1 : e < kSmallPages ? s_page[e] : p.kv_indices[first + e];
    return page >= 0 && page < p.max_pages;
  };
  constexpr int kNW = kSmallKeep / kSmallThreads;
  float w[kNW];
  int64_t w_to[kNW];
#pragma unroll
  for (int i = 0; i < kNW; ++i) {
    const int j = tid + i * kSmallThreads;
    int64_t page, page_to;
    int slot, slot_to;
    const bool move = j < n && place(s_kept[j], page, slot) && place(j, page_to, slot_to);
    w[i] = move ? weights[(page * p.num_kv_heads + h) * p.page_size + slot] : 0.f;
    w_to[i] = move ? (page_to * p.num_kv_heads + h) * p.page_size + slot_to : -1;
  }
  auto put_weights = [&]() {
#pragma unroll
    for (int i = 0; i < kNW; ++i)
      if (w_to[i] >= 0) out_weights[w_to[i]] = w[i];
  };
  if (!cut) {
    put_weights();
    return;
  }
  const int per = 2 * p.row_pieces, row = tid / per, rows = kSmallThreads / per;
  const int steps = min(kMoveRows, kSmallPlaces / rows), tile = rows * steps;
  const int v = tid % per >= p.row_pieces, piece = tid % per - v * p.row_pieces;
  uint8_t* base = p.cache + layer * p.layer_stride + v * p.kv_stride + h * p.head_stride + 16 * piece;
  for (int j0 = 0; j0 < n; j0 += tile) {
    if (tid < tile) {  // at most kSmallPlaces, as many as there are threads
      const int j = j0 + tid, src = j < n ? s_kept[j] : -1;
      int64_t page, page_to;
      int slot, slot_to;
      const bool move = src > j && place(src, page, slot) && place(j, page_to, slot_to);
      s_from[tid] = move ? page * p.page_stride + slot * p.token_stride : -1;
      s_to[tid] = move ? page_to * p.page_stride + slot_to * p.token_stride : -1;
    }
    __syncthreads();
    u32x4_t x[kMoveRows];
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      const int64_t from = k < steps ? s_from[k * rows + row] : -1;
      x[k] = from >= 0 ? *(const u32x4_t*)(base + from) : u32x4_t{0u, 0u, 0u, 0u};
    }
    __syncthreads();  // the tile's rows are in registers, and all weights
    if (j0 == 0) put_weights();
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      const int64_t to = k < steps ? s_to[k * rows + row] : -1;
      if (to >= 0) *(u32x4_t*)(base + to) = x[k];
    }
    __syncthreads();
  }
  if (p.scales)
    for (int line = 0; line < 2 * p.blocks; ++line) evict_scales<kSmallThreads>(p, layer, h, first, pages, s_kept, n, line);
}

}  // namespace mi

extern "C" int mi_kv_evict_block(const mi_kv_evict_args* args) {
  using namespace mi;
  if (!args) return MI_ERR_INVALID;
  const mi_kv_evict_args& a = *args;
  if (!a.kv || a.num_layers < 0 || a.batch < 0 || a.num_indices < 0) return MI_ERR_INVALID;
  if (a.keep <= 0 || a.recent < 0 || a.sinks < 0 || a.recent > a.keep - a.sinks) return MI_ERR_INVALID;
  if (a.num_layers == 0 || a.batch == 0) return MI_OK;
  if (!a.kv->data || !a.weights || !a.out_weights || !a.kv_indptr || !a.kv_indices || !a.last_page_len || !a.kept) return MI_ERR_INVALID;
  if (a.kv->num_kv_heads <= 0 || a.kv->head_dim <= 0 || a.kv->page_size <= 0 || a.kv->max_pages < 0) return MI_ERR_INVALID;
  // places in the page list are counted in 32 bits
  if (a.kv->page_size % 4 || a.kv->page_size > (1 << 24) || (int64_t)a.num_indices * a.kv->page_size > INT32_MAX - (1 << 25))
    return MI_ERR_UNSUPPORTED;
  const bool mx = kv_is_mx(a.kv->dtype);
  if (!mx && a.kv->dtype != MI_BF16 && a.kv->dtype != MI_F16 && a.kv->dtype != MI_F32 && a.kv->dtype != MI_FP8_E4M3) return MI_ERR_UNSUPPORTED;
  if (a.kv->head_dim != 64 && a.kv->head_dim != 128 && a.kv->head_dim != 256) return MI_ERR_UNSUPPORTED;
  const int esz = kv_elem_bytes(a.kv->dtype);
  if (!kv_aligned16(a.kv) || (a.layer_stride * esz) % 16) return MI_ERR_INVALID;
  if (((uintptr_t)a.weights | (uintptr_t)a.out_weights) % 16 || a.weights_layer_stride % 4) return MI_ERR_INVALID;
  if (mx && (!kv_scales_ok(a.kv) || a.kv->head_dim % kMxBlock)) return MI_ERR_INVALID;
  EvictParams p{};
  p.cache = (uint8_t*)a.kv->data;
  p.layer_stride = a.layer_stride * esz;
  p.page_stride = a.kv->page_stride * esz;
  p.kv_stride = a.kv->kv_stride * esz;
  p.token_stride = a.kv->token_stride * esz;
  p.head_stride = a.kv->head_stride * esz;
  p.max_pages = a.kv->max_pages;
  p.blocks = a.kv->head_dim / kMxBlock;
  if (mx) {
    // one array: V's bytes follow K's within a page
    if ((const uint8_t*)a.kv->v_scale - (const uint8_t*)a.kv->k_scale != (int64_t)a.kv->num_kv_heads * p.blocks * a.kv->page_size)
      return MI_ERR_INVALID;
    p.scales = (uint8_t*)a.kv->k_scale;
    p.scale_layer_stride = a.scale_layer_stride;
  }
  p.weights = a.weights;
  p.out_weights = a.out_weights;
  p.weights_layer_stride = a.weights_layer_stride;
  p.kv_indptr = a.kv_indptr;
  p.kv_indices = a.kv_indices;
  p.last_page_len = a.last_page_len;
  p.kept = a.kept;
  p.batch = a.batch;
  p.num_indices = a.num_indices;
  p.num_kv_heads = a.kv->num_kv_heads;
  p.page_size = a.kv->page_size;
  p.page_shift = (a.kv->page_size & (a.kv->page_size - 1)) == 0 ? __builtin_ctz((unsigned)a.kv->page_size) : -1;
  p.keep = a.keep;
  p.recent = a.recent;
  p.sinks = a.sinks;
  p.row_pieces = (a.kv->dtype == MI_MXFP4 ? a.kv->head_dim / 2 : a.kv->head_dim * esz) / 16;
  const int64_t units = (int64_t)a.num_layers * a.batch * a.kv->num_kv_heads;
  p.splits = 1;
  while (p.row_pieces / p.splits >= 16 && 2 * units * p.splits < 2LL * device_cu_count()) p.splits *= 2;
  p.parts = 2 * p.splits + 1 + (mx ? 2 * p.blocks : 0);
  if (units * p.parts > INT32_MAX) return MI_ERR_UNSUPPORTED;
  hipStream_t s = (hipStream_t)a.stream;
  if (units <= device_cu_count() && a.keep <= kSmallKeep && 32LL * p.row_pieces * a.keep <= kSmallBytes) {
    hipLaunchKernelGGL(evict_small_kernel, dim3((uint32_t)units), dim3(kSmallThreads), 0, s, p);
  } else {
    // a workgroup of 256 holds 8192 tokens, and more of them share a compute unit: waiting, not bytes, is what selecting few
    // tokens costs (4096 units of 500 to 4000 tokens: 41 us against 80 with 1024 threads)
    if ((int64_t)a.num_indices * p.page_size / a.batch <= kSelFew)
      hipLaunchKernelGGL(evict_select_kernel<256>, dim3((uint32_t)units), dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL(evict_select_kernel<1024>, dim3((uint32_t)units), dim3(1024), 0, s, p);
    hipLaunchKernelGGL(evict_move_kernel, dim3((uint32_t)(units * p.parts)), dim3(kMoveThreads), 0, s, p);
  }
  MI_CHECK_LAUNCH();
  return MI_OK;
}

extern "C" int mi_kv_evict(const mi_paged_kv* kv, int32_t num_layers, int64_t layer_stride, int64_t scale_layer_stride,
                           const float* weights, float* out_weights, int64_t weights_layer_stride, const int32_t* kv_indptr,
                           const int32_t* kv_indices, const int32_t* last_page_len, int32_t batch, int32_t num_indices, int32_t keep,
                           int32_t recent, int32_t sinks, int32_t* kept, void* stream) {
  const mi_kv_evict_args args = {kv, weights, out_weights, kv_indptr, kv_indices, last_page_len, kept, stream, layer_stride, scale_layer_stride, weights_layer_stride, num_layers, batch, num_indices, keep, recent, sinks};
  return mi_kv_evict_block(&args);
}
