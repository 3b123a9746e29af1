// Accumulated attention weights of cached tokens: the kernels (mi_weights.hip describes them
// and launches them; mi_weights_*.hip hold the instantiations).
#pragma once

#include "mi_internal.h"

namespace mi {

// fp32 queries and caches: a step is 16 elements of a row, four to a lane, on the fp32 MFMA.
struct F32 {
  static constexpr int kDtype = MI_F32;
  MI_DEVICE static f32x4 mma_16x16x32(const uint4& a, const uint4& b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(bitcast<float>(a.x), bitcast<float>(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(bitcast<float>(a.y), bitcast<float>(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(bitcast<float>(a.z), bitcast<float>(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(bitcast<float>(a.w), bitcast<float>(b.w), c, 0, 0, 0);
  }
};

struct WeightsParams {
  const void* q;
  int64_t q_stride_tok, q_stride_head;
  const uint8_t* k;
  int64_t page_stride, token_stride, head_stride, max_pages;  // elements (bytes of codes: microscaled)
  const void* k_scale;
  const int32_t *qo_indptr, *kv_indptr, *kv_indices, *last_page_len;
  float* weights;  // [max_pages][kv head][slot]
  float *scores, *unit_lse;  // short queries: [16-token tile of the page list][kv head][row][16], [unit][kv head][16]
  float *row_lse, *sums;     // long ones: [split][kv head][row], [split][kv head][place in the page list]
  int64_t total_rows, places;
  int32_t batch, num_kv_heads, group, page_size, causal, max_tokens, num_indices;
  int32_t unit_pages, finish_pages, score_rows;  // of the short path
  int32_t key_splits, row_splits, key_pages;  // of the long one; key_pages: of a block of keys
  float scale_log2;
};

constexpr int kWRows = 16;       // rows of a short-query request
constexpr int kRowBlock = 128;   // rows of a workgroup of the fp32 long path's first pass
constexpr int kKeyBlock = 128;   // keys of a workgroup of its second
typedef __attribute__((ext_vector_type(16))) float f32x16;

// The request of a unit, where request r's units begin at indptr[r] * mul / div + r: at least as many places
// as it needs, and found from the index array alone.  -1: before the first.
MI_DEVICE int unit_request(const int32_t* indptr, int mul, int div, int batch, int unit) {
  int lo = 0, n = batch;  // the last r of [lo, lo + n) with begin(r) <= unit
  const int lane = lane_id();
  while (n > 0) {
    const int step = (n + 63) / 64, r = lo + lane * step;
    const bool in = lane * step < n && (int)((int64_t)indptr[r] * mul / div) + r <= unit;
    const int count = __popcll(__builtin_amdgcn_ballot_w64(in));  // begins ascend
    if (count == 0) return -1;
    const int next = lo + (count - 1) * step;
    if (step == 1) return next;
    n = min(step, lo + n - next);
    lo = next;
  }
  return -1;
}
MI_DEVICE int unit_begin(const int32_t* indptr, int mul, int div, int r) { return (int)((int64_t)indptr[r] * mul / div) + r; }

// A request, held to the sizes that the call's scratch was made for.
struct WRequest {
  int first, pages, len, qo_start, qo_len, rows;
};
MI_DEVICE WRequest w_request(const WeightsParams& p, int r) {
  WRequest q;
  q.first = p.kv_indptr[r];
  q.pages = min(p.kv_indptr[r + 1], p.num_indices) - q.first;
  q.len = q.pages > 0 ? max(0, (q.pages - 1) * p.page_size + min(p.last_page_len[r], p.page_size)) : 0;
  q.qo_start = p.qo_indptr ? p.qo_indptr[r] : r;
  q.qo_len = p.qo_indptr ? min(p.qo_indptr[r + 1], p.max_tokens) - q.qo_start : 1;
  q.rows = q.qo_len * p.group;
  return q;
}

// How a lane holds a row of the cache: runs of RUN consecutive elements, 16 bytes each where
// the row is long enough, run c at element c * 4 * RUN + grp * RUN (grp: which 16 lanes).  Any one order of
// the elements serves a product, as long as q is held in the same.
template <typename MT, int KVT, int D>
struct KeyTile {
  static constexpr bool F = MT::kDtype == MI_F32, MX = KVT == kKvMx8 || KVT == kKvMx4;
  static constexpr int BITS = F ? 32 : KVT == kKv16 ? 16 : KVT == kKvMx4 ? 4 : 8;
  static constexpr int RUN = D / 4 < 128 / BITS ? D / 4 : 128 / BITS;
  static constexpr int NC = D / (4 * RUN), WORDS = RUN * BITS / 32;
  static constexpr int STEP = F ? 4 : 8;                    // elements of a lane in a step
  static constexpr int STEPS = D / (4 * STEP), PER = RUN / STEP;  // steps, and of a run
  static constexpr int ESZ = F ? 4 : KVT == kKv16 ? 2 : 1;  // of the strides
  static constexpr int NBLK = D / kMxBlock;
  uint32_t w[NC][WORDS];
  uint8_t s[MX ? NC : 1];

  // The lane's row `row` of the 16 tokens at (page, slot0) of kv head h.
  MI_DEVICE void load(const WeightsParams& p, int64_t page, int slot, int h, int grp) {
    const uint8_t* src = p.k + (page * p.page_stride + slot * p.token_stride + h * p.head_stride) * ESZ + grp * (RUN * BITS / 8);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if constexpr (WORDS == 4) {
        const u32x4_t u = *(const u32x4_t*)(src + c * (4 * RUN * BITS / 8));
        w[c][0] = u.x, w[c][1] = u.y, w[c][2] = u.z, w[c][3] = u.w;
      } else {
        const uint2 u = *(const uint2*)(src + c * (4 * RUN * BITS / 8));
        w[c][0] = u.x, w[c][1] = u.y;
      }
    }
    if constexpr (MX) {
      const uint8_t* sc = (const uint8_t*)p.k_scale + (page * 2 * p.num_kv_heads + h) * NBLK * p.page_size + slot;
#pragma unroll
      for (int c = 0; c < NC; ++c) s[c] = sc[(int64_t)((c * 4 * RUN + grp * RUN) / kMxBlock) * p.page_size];
    }
  }
  // The same from 16 rows in LDS, PITCH bytes apart.
  template <int PITCH>
  MI_DEVICE void read(const uint8_t* rows, int row, int grp) {
    const uint8_t* src = rows + row * PITCH + grp * (RUN * BITS / 8);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if constexpr (WORDS == 4) {
        const u32x4_t u = *(const u32x4_t*)(src + c * (4 * RUN * BITS / 8));
        w[c][0] = u.x, w[c][1] = u.y, w[c][2] = u.z, w[c][3] = u.w;
      } else {
        const u32x2_t u = *(const u32x2_t*)(src + c * (4 * RUN * BITS / 8));
        w[c][0] = u.x, w[c][1] = u.y;
      }
    }
  }
  MI_DEVICE void fragments(uint4 (&f)[STEPS]) const {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if constexpr (KVT == kKv16) {
        f[c] = make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
      } else {
        uint32_t o[4 * PER];
        if constexpr (KVT == kKvFp8) {
#pragma unroll
          for (int i = 0; i < 2 * PER; ++i) {
            o[2 * i] = fp8x2_to_mt<MT>(w[c][i], false);
            o[2 * i + 1] = fp8x2_to_mt<MT>(w[c][i], true);
          }
        } else {
          mx_to_mt<MT, KVT>(w[c], bitcast<float>((uint32_t)s[c] << 23), o);
          if constexpr (MT::kDtype == MI_F16)
            if (mx_past_f16<KVT>(s[c])) f16_saturate(o);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) f[c * PER + i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
    }
  }
  // A row of q in the same order.
  MI_DEVICE static void query(const WeightsParams& p, int64_t tok, int head, int grp, uint4 (&f)[STEPS]) {
    const uint8_t* src = (const uint8_t*)p.q + (tok * p.q_stride_tok + head * p.q_stride_head) * (F ? 4 : 2);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < PER; ++i) f[c * PER + i] = *(const uint4*)(src + (c * 4 * RUN + grp * RUN + i * STEP) * (F ? 4 : 2));
  }
};

// Sixteen rows as they are loaded: a lane has 16 bytes of every 1024, so an instruction covers
// whole rows, and whole cache lines of them.  (Each lane loading what the MFMA wants of it, 64 bytes of a row an
// instruction, streams K slower: 495 -> 440 us over 1.95 GB.)  They pass through LDS.
template <typename MT, int KVT, int D>
struct RawTile {
  using Tile = KeyTile<MT, KVT, D>;
  static constexpr int ROW = D * Tile::BITS / 8, PITCH = ROW + 16, N = (16 * ROW + 1023) / 1024;
  static constexpr bool ALL = 16 * ROW % 1024 == 0;
  u32x4_t r[N];
  uint8_t s[Tile::MX ? Tile::NC : 1];

  MI_DEVICE void load(const WeightsParams& p, int64_t page, int slot, int h, int lane) {
    const uint8_t* src = p.k + (page * p.page_stride + slot * p.token_stride + h * p.head_stride) * Tile::ESZ;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int at = 16 * lane + 1024 * j, row = at / ROW;
      if (!ALL && at >= 16 * ROW) continue;
      const u32x4_t* from = (const u32x4_t*)(src + (int64_t)row * p.token_stride * Tile::ESZ + at % ROW);
      if constexpr (ROW >= 128) r[j] = __builtin_nontemporal_load(from);
      else r[j] = *from;  // the rest of the line is another head's
    }
    if constexpr (Tile::MX) {
      const int col = lane & 15, grp = lane >> 4;
      const uint8_t* sc = (const uint8_t*)p.k_scale + (page * 2 * p.num_kv_heads + h) * Tile::NBLK * p.page_size + slot + col;
#pragma unroll
      for (int c = 0; c < Tile::NC; ++c) s[c] = sc[(int64_t)((c * 4 * Tile::RUN + grp * Tile::RUN) / kMxBlock) * p.page_size];
    }
  }
  // Through the wavefront's part of LDS into the MFMA's order.
  MI_DEVICE void order(uint8_t* lds, int lane, Tile& t) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int at = 16 * lane + 1024 * j;
      if (!ALL && at >= 16 * ROW) continue;
      *(u32x4_t*)(lds + at / ROW * PITCH + at % ROW) = r[j];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    t.template read<PITCH>(lds, lane & 15, lane >> 4);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if constexpr (Tile::MX)
#pragma unroll
      for (int c = 0; c < Tile::NC; ++c) t.s[c] = s[c];
  }
};

// Page of entry e of the page list, page 0 for ids out of range (whose tokens' weights are not written).
MI_DEVICE int64_t safe_page(const WeightsParams& p, int e) {
  const int64_t page = p.kv_indices[e];
  return page >= 0 && page < p.max_pages ? page : 0;
}

constexpr float kWInf = __builtin_inff();

// The log2 of a row's sum, from its running maximum and sum; +inf where it saw nothing, which
// makes every exp2(s - lse) zero; NaN where a score was NaN or +inf.
MI_DEVICE float w_lse(float m, float l) { return l > 0.f ? m + fast_log2(l) : l == 0.f ? kWInf : __builtin_nanf(""); }

// ------------------------------------------------------------ short queries
// Requests of at most 16 (query, q head) rows: HBM bound, K is read once.  A workgroup takes a unit
// (unit_pages pages of a request, one kv head); each wavefront's tiles of 16 keys give S^T = K Q^T, whose
// scores (log2 domain) go to scratch, and the unit's log-sum-exp of each row.
template <typename MT, int KVT, int D>
__global__ __launch_bounds__(256) void weights_scores_kernel(WeightsParams p) {
  using Tile = KeyTile<MT, KVT, D>;
  using Raw = RawTile<MT, KVT, D>;
  __shared__ __attribute__((aligned(16))) uint8_t s_rows[4][16 * Raw::PITCH];
  __shared__ float s_m[4][kWRows], s_l[4][kWRows];
  const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6), nkv = p.num_kv_heads;
  const int h = uniform((int)(blockIdx.x % nkv)), unit = uniform((int)(blockIdx.x / nkv));
  const int r = uniform(unit_request(p.kv_indptr, 1, p.unit_pages, p.batch, unit));
  if (r < 0) return;
  const WRequest q = w_request(p, r);
  if (q.rows <= 0 || q.rows > kWRows) return;
  const int tok0 = (unit - unit_begin(p.kv_indptr, 1, p.unit_pages, r)) * p.unit_pages * p.page_size;
  const int tok1 = min(tok0 + p.unit_pages * p.page_size, q.len);
  if (tok0 >= tok1) return;
  const int tiles = (tok1 - tok0 + 15) >> 4, share = tiles / 4, extra = tiles % 4;
  const int t0 = wave * share + min(wave, extra), t1 = t0 + share + (wave < extra ? 1 : 0);

  const int col = lane & 15, grp = lane >> 4;
  const int qtok = col / p.group, g = col - qtok * p.group;
  const bool valid = col < q.rows;
  const int lim = p.causal ? q.len - q.qo_len + qtok : q.len - 1;
  uint4 qf[Tile::STEPS] = {};
  if (valid) Tile::query(p, q.qo_start + qtok, h * p.group + g, grp, qf);
  const float sl2 = KVT == kKvFp8 ? p.scale_log2 * ((const float*)p.k_scale)[h] : p.scale_log2;

  float m = -kWInf, l = 0.f;
  // Pages and slots of 64 tiles, one a lane: a page id loaded behind a tile's K would wait for that K.
  int ids = 0, slots = 0, ids_first = t0 - 64;
  auto load = [&](Raw& t, int i) {
    if (i >= ids_first + 64) {
      ids_first = i;
      const int tok = tok0 + 16 * min(i + lane, t1 - 1), e = (int)((unsigned)tok / (unsigned)p.page_size);
      ids = (int)safe_page(p, q.first + e);
      slots = tok - e * p.page_size;
    }
    t.load(p, __builtin_amdgcn_readlane(ids, i - ids_first), __builtin_amdgcn_readlane(slots, i - ids_first), h, lane);
  };
  auto compute = [&](const Raw& raw, int i) {
    const int tok = tok0 + 16 * i;
    Tile t;
    raw.order(s_rows[wave], lane, t);
    uint4 kf[Tile::STEPS];
    t.fragments(kf);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < Tile::STEPS; ++st) acc = MT::mma_16x16x32(kf[st], qf[st], acc);
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j] = acc[j] * sl2;
      if (tok + 4 * grp + j > lim) s[j] = -kWInf;
    }
    if (valid) {
      const int64_t tile = ((int64_t)q.first * p.page_size + tok) >> 4;
      *(float4*)(p.scores + ((tile * nkv + h) * p.score_rows + col) * 16 + 4 * grp) = make_float4(s[0], s[1], s[2], s[3]);
    }
    const float mn = fmaxf(m, fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
    const float mu = mn == -kWInf ? 0.f : mn;
    l = l * fast_exp2(m - mu) + ((fast_exp2(s[0] - mu) + fast_exp2(s[1] - mu)) + (fast_exp2(s[2] - mu) + fast_exp2(s[3] - mu)));
    m = mn;
  };
  Raw a, b;
  if (t0 < t1) load(a, t0);
  for (int i = t0; i < t1; i += 2) {
    if (i + 1 < t1) load(b, i + 1);
    compute(a, i);
    if (i + 2 < t1) load(a, i + 2);
    if (i + 1 < t1) compute(b, i + 1);
  }
  // the four groups of lanes, then the four wavefronts
  const float mg = rows4_max(m), mgu = mg == -kWInf ? 0.f : mg;
  l = rows4_sum(l * fast_exp2(m - mgu));
  if (grp == 0) {
    s_m[wave][col] = mg;
    s_l[wave][col] = l;
  }
  __syncthreads();
  if (threadIdx.x < kWRows) {
    float M = -kWInf, L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w][col]);
    const float Mu = M == -kWInf ? 0.f : M;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += s_l[w][col] * fast_exp2(s_m[w][col] - Mu);
    p.unit_lse[((int64_t)unit * nkv + h) * kWRows + col] = w_lse(M, L);
  }
}

// All of it in one launch, a workgroup for each request and kv head, where the batch's scores of a head fit its
// LDS: tiles in turn over 16 wavefronts, scores to LDS, and behind one barrier the sums.
constexpr int kOneScores = 32768;                      // floats
// Half the wavefronts where a row of K and of q are 64 registers each.
template <typename MT>
constexpr int one_threads(int d) { return MT::kDtype == MI_F32 && d == 256 ? 512 : 1024; }
constexpr int kOnePad = 20;                            // of a row of scores: up to 15 tokens, and 16 rows in different banks
template <typename MT, int KVT, int D>
__global__ __launch_bounds__(one_threads<MT>(D)) void weights_one_kernel(WeightsParams p) {
  using Tile = KeyTile<MT, KVT, D>;
  constexpr int NT = one_threads<MT>(D), NW = NT / kWave;
  __shared__ __attribute__((aligned(16))) float s_scores[kOneScores];
  __shared__ float s_m[NW][kWRows], s_l[NW][kWRows], s_lse[kWRows];
  const int tid = (int)threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6), nkv = p.num_kv_heads;
  const int h = uniform((int)(blockIdx.x % nkv)), r = uniform((int)(blockIdx.x / nkv));
  const WRequest q = w_request(p, r);
  if (q.rows <= 0 || q.rows > kWRows || q.len <= 0) return;
  const int tiles = (q.len + 15) >> 4, pitch = (q.len & ~15) + kOnePad, off = q.len - q.qo_len;
  const int col = lane & 15, grp = lane >> 4;
  const int qtok = col / p.group, g = col - qtok * p.group;
  const bool valid = col < q.rows;
  const int lim = p.causal ? off + qtok : q.len - 1;
  uint4 qf[Tile::STEPS] = {};
  if (valid) Tile::query(p, q.qo_start + qtok, h * p.group + g, grp, qf);
  const float sl2 = KVT == kKvFp8 ? p.scale_log2 * ((const float*)p.k_scale)[h] : p.scale_log2;
  float m = -kWInf, l = 0.f;
  int ids = 0, slots = 0, round = -64;  // of 64 of the wavefront's tiles, one a lane
  auto load = [&](Tile& t, int k) {     // its k-th tile
    if (k >= round + 64) {
      round = k;
      const int tok = 16 * min(wave + NW * (k + lane), tiles - 1), e = (int)((unsigned)tok / (unsigned)p.page_size);
      ids = (int)safe_page(p, q.first + e);
      slots = tok - e * p.page_size;
    }
    t.load(p, __builtin_amdgcn_readlane(ids, k - round), __builtin_amdgcn_readlane(slots, k - round) + col, h, grp);
  };
  auto compute = [&](const Tile& t, int k) {
    const int tok = 16 * (wave + NW * k);
    uint4 kf[Tile::STEPS];
    t.fragments(kf);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < Tile::STEPS; ++st) acc = MT::mma_16x16x32(kf[st], qf[st], acc);
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j] = acc[j] * sl2;
      if (tok + 4 * grp + j > lim) s[j] = -kWInf;
    }
    if (valid) *(float4*)(s_scores + col * pitch + tok + 4 * grp) = make_float4(s[0], s[1], s[2], s[3]);
    const float mn = fmaxf(m, fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
    const float mu = mn == -kWInf ? 0.f : mn;
    l = l * fast_exp2(m - mu) + ((fast_exp2(s[0] - mu) + fast_exp2(s[1] - mu)) + (fast_exp2(s[2] - mu) + fast_exp2(s[3] - mu)));
    m = mn;
  };
  const int mine = wave < tiles ? (tiles - wave + NW - 1) / NW : 0;
  Tile a, b;
  if (mine > 0) load(a, 0);
  for (int k = 0; k < mine; k += 2) {
    if (k + 1 < mine) load(b, k + 1);
    compute(a, k);
    if (k + 2 < mine) load(a, k + 2);
    if (k + 1 < mine) compute(b, k + 1);
  }
  // the thread's first token's weight, while the wavefronts meet
  auto weight_at = [&](int t) -> float* {
    const int e = (int)((unsigned)t / (unsigned)p.page_size);
    const int64_t page = p.kv_indices[q.first + e];
    return page >= 0 && page < p.max_pages ? p.weights + (page * nkv + h) * p.page_size + t - e * p.page_size : nullptr;
  };
  float* at = tid < q.len ? weight_at(tid) : nullptr;
  float old = at && tid < off ? *at : 0.f;
  const float mg = rows4_max(m), mgu = mg == -kWInf ? 0.f : mg;
  l = rows4_sum(l * fast_exp2(m - mgu));
  if (grp == 0) {
    s_m[wave][col] = mg;
    s_l[wave][col] = l;
  }
  __syncthreads();
  if (tid < kWRows) {
    float M = -kWInf, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w][tid]);
    const float Mu = M == -kWInf ? 0.f : M;
#pragma unroll
    for (int w = 0; w < NW; ++w) L += s_l[w][tid] * fast_exp2(s_m[w][tid] - Mu);
    s_lse[tid] = w_lse(M, L);
  }
  __syncthreads();
  for (int t = tid; t < q.len; t += NT) {
    if (t != tid) {
      at = weight_at(t);
      old = at && t < off ? *at : 0.f;
    }
    float sum = 0.f;
    // from the first row that sees the token on: the others add nothing, also where their log-sum-exp is NaN
    for (int row = p.causal ? max(0, t - off) * p.group : 0; row < q.rows; ++row)
      sum += fast_exp2(s_scores[row * pitch + t] - s_lse[row]);
    if (at) *at = old + sum;
  }
}

// Adds a key's sum to its weight, or leaves it to weights_sum_kernel where other workgroups have the other rows.
MI_DEVICE void w_add(const WeightsParams& p, const WRequest& q, int h, int split, int key, int off, float total) {
  if (p.row_splits > 1) {
    p.sums[((int64_t)split * p.num_kv_heads + h) * p.places + (int64_t)q.first * p.page_size + key] = total;
    return;
  }
  const int e = (int)((unsigned)key / (unsigned)p.page_size);
  const int64_t page = p.kv_indices[q.first + e];
  if (page < 0 || page >= p.max_pages) return;
  float* w = p.weights + (page * p.num_kv_heads + h) * p.page_size + key - e * p.page_size;
  *w = key >= off ? total : *w + total;
}

// ------------------------------------------------------------ long queries
// Both passes hold one side of the product in registers and stream the other through LDS in tiles
// of 32, on the 32x32x16 MFMA: a tile's fragment serves all of a wavefront's columns.  An exponential
// is 16 cycles of a wavefront, as long as its share of the products at head_dim 128, and each pass has one a
// score beside an FMA and an addition.  The two take turns (MFMA busy 35-37 % of the cycles, VALU 65-67 %), so no one unit bounds them: of a
// first pass over 4 chunks and 22k keys that took 212 us (203 now) 27 went without the exponentials, 66 without seven eighths of the
// products, 43 without the loads.
template <typename MT>
MI_DEVICE f32x16 mma_32x32x16(const uint4& a, const uint4& b, f32x16 c) {
  if constexpr (MT::kDtype == MI_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bitcast<bf16x8>(a), bitcast<bf16x8>(b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(bitcast<f16x8>(a), bitcast<f16x8>(b), c, 0, 0, 0);
}
// Sum and maximum of the two lanes that hold a column's rows.
MI_DEVICE float both_sum(float x) {
  const uint32_t u = bitcast<uint32_t>(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return bitcast<float>((uint32_t)a[0]) + bitcast<float>((uint32_t)a[1]);
}
MI_DEVICE float both_max(float x) {
  const uint32_t u = bitcast<uint32_t>(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(bitcast<float>((uint32_t)a[0]), bitcast<float>((uint32_t)a[1]));
}

constexpr int kTile = 32;                                        // rows of a streamed tile
constexpr int stationary(int d) { return d <= 128 ? 2 : 1; }     // columns / 32 that a wavefront holds
constexpr int mma_block(int d) { return 4 * kTile * stationary(d); }

// A tile in LDS: rows of D 16-bit elements, 16-byte pieces swapped about so that the 16 rows that a
// read takes at once lie in different banks.
template <int D>
MI_DEVICE int tile_at(int row, int piece) {
  return row * (2 * D) + 16 * (piece ^ (D == 64 ? (row >> 1) & 7 : row & 15));
}
template <int D>
MI_DEVICE uint4 tile_fragment(const uint8_t* tile, int row, int step, int hi) {
  return *(const uint4*)(tile + tile_at<D>(row, 2 * step + hi));
}

// Eight elements of a cached row from element 8 * piece on, in the MFMA type.
template <typename MT, int KVT, int D>
MI_DEVICE uint4 key_piece(const WeightsParams& p, int64_t page, int slot, int h, int piece) {
  constexpr int BITS = KVT == kKv16 ? 16 : KVT == kKvMx4 ? 4 : 8, ESZ = KVT == kKv16 ? 2 : 1;
  const uint8_t* src = p.k + (page * p.page_stride + slot * p.token_stride + h * p.head_stride) * ESZ + piece * BITS;
  if constexpr (KVT == kKv16) {
    return *(const uint4*)src;
  } else {
    uint32_t w[KVT == kKvMx4 ? 1 : 2], o[4];
    if constexpr (KVT == kKvMx4) {
      w[0] = *(const uint32_t*)src;
    } else {
      const uint2 u = *(const uint2*)src;
      w[0] = u.x, w[1] = u.y;
    }
    if constexpr (KVT == kKvFp8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        o[2 * i] = fp8x2_to_mt<MT>(w[i], false);
        o[2 * i + 1] = fp8x2_to_mt<MT>(w[i], true);
      }
    } else {
      constexpr int NBLK = D / kMxBlock;
      const uint8_t s = ((const uint8_t*)p.k_scale)[((page * 2 * p.num_kv_heads + h) * NBLK + piece / 4) * (int64_t)p.page_size + slot];
      mx_to_mt<MT, KVT>(w, bitcast<float>((uint32_t)s << 23), o);
      if constexpr (MT::kDtype == MI_F16)
        if (mx_past_f16<KVT>(s)) f16_saturate(o);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// The keys of a request as a stream of tiles: what a thread loads of each, and where in the cache that lies.
// A wavefront's rows of a unit are 16 or fewer that begin at a multiple of their number, so they lie in one
// page: the page's address is scalar, and a thread's offset in it is the same for every tile.  (With both
// computed by each thread, that was half of the loop's instructions.)
template <typename MT, int KVT, int D>
struct KeyStream {
  static constexpr int UNIT = KVT == kKv16 ? 8 : 16;  // elements a thread loads at once
  static constexpr int PER_ROW = D / UNIT, NU = (kTile * PER_ROW + 255) / 256;
  static constexpr int WROWS = kWave / PER_ROW;  // rows of a wavefront's unit
  static constexpr bool MX = KVT == kKvMx8 || KVT == kKvMx4;
  static_assert(WROWS >= 1 && WROWS <= 16, "a unit lies in one page");
  struct Tile {
    u32x4_t w[NU];  // mx4: two words
    uint8_t s[NU];
  };
  int entry[NU], slot[NU];
  int64_t page[NU];
  uint32_t at, scale_at;  // the thread's bytes from its unit's first row

  MI_DEVICE static int unit(int u) { return (int)threadIdx.x + 256 * u; }
  MI_DEVICE static bool active(int u) { return kTile * PER_ROW % 256 == 0 || unit(u) < kTile * PER_ROW; }
  MI_DEVICE void begin(const WeightsParams& p, const WRequest& q, int tile) {
    constexpr int ESZ = KVT == kKv16 ? 2 : 1;
    const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6), part = lane % PER_ROW, row = lane / PER_ROW;
    at = (uint32_t)row * (uint32_t)(p.token_stride * ESZ) + part * (KVT == kKvMx4 ? 8 : 16);
    scale_at = (uint32_t)(part / 2) * (uint32_t)p.page_size + row;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int tok = kTile * tile + WROWS * (wave + 4 * u);
      entry[u] = (int)((unsigned)tok / (unsigned)p.page_size);
      slot[u] = tok - entry[u] * p.page_size;
      page[u] = safe_page(p, q.first + min(entry[u], q.pages - 1));
    }
  }
  // Loads the tile that `page` is of, and the pages of the next; past a request's last, any keys of its last page.
  MI_DEVICE void load(const WeightsParams& p, const WRequest& q, int h, Tile& t) {
    constexpr int ESZ = KVT == kKv16 ? 2 : 1;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if (active(u)) {
        const uint8_t* src = p.k + (page[u] * p.page_stride + slot[u] * p.token_stride + h * p.head_stride) * ESZ;
        if constexpr (KVT == kKvMx4) {
          const uint2 x = *(const uint2*)(src + at);
          t.w[u] = u32x4_t{x.x, x.y, 0u, 0u};
        } else {
          t.w[u] = *(const u32x4_t*)(src + at);
        }
        if constexpr (MX) {
          const uint8_t* sc = (const uint8_t*)p.k_scale + (page[u] * 2 * p.num_kv_heads + h) * (D / kMxBlock) * (int64_t)p.page_size + slot[u];
          t.s[u] = sc[scale_at];
        }
      }
      slot[u] += kTile;
      while (slot[u] >= p.page_size) slot[u] -= p.page_size, ++entry[u];
      page[u] = safe_page(p, q.first + min(entry[u], q.pages - 1));
    }
  }
  MI_DEVICE static void store(const Tile& t, uint8_t* tile) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if (!active(u)) continue;
      const int row = unit(u) / PER_ROW, part = unit(u) % PER_ROW;
      if constexpr (KVT == kKv16) {
        *(u32x4_t*)(tile + tile_at<D>(row, part)) = t.w[u];
      } else {
        uint32_t o[8];
        if constexpr (KVT == kKvFp8) {
          const uint32_t x[4] = {t.w[u].x, t.w[u].y, t.w[u].z, t.w[u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[2 * i] = fp8x2_to_mt<MT>(x[i], false);
            o[2 * i + 1] = fp8x2_to_mt<MT>(x[i], true);
          }
        } else {
          const float scale = bitcast<float>((uint32_t)t.s[u] << 23);
          if constexpr (KVT == kKvMx8) {
            const uint32_t x[4] = {t.w[u].x, t.w[u].y, t.w[u].z, t.w[u].w};
            mx_to_mt<MT, KVT>(x, scale, o);
          } else {
            const uint32_t x[2] = {t.w[u].x, t.w[u].y};
            mx_to_mt<MT, KVT>(x, scale, o);
          }
          if constexpr (MT::kDtype == MI_F16)
            if (mx_past_f16<KVT>(t.s[u])) f16_saturate(o);
        }
        *(uint4*)(tile + tile_at<D>(row, 2 * part)) = make_uint4(o[0], o[1], o[2], o[3]);
        *(uint4*)(tile + tile_at<D>(row, 2 * part + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
  }
};

// First pass: the log-sum-exp of every (query, q head) row.  A workgroup takes 128 or 256 rows of a
// request and kv head and a share of the keys: S^T = K Q^T, a lane's scores all of one row.
template <typename MT, int KVT, int D>
__global__ __launch_bounds__(256, 2) void weights_rows_kernel(WeightsParams p) {
  constexpr int NS = stationary(D), STEPS = D / 16, BLOCK = mma_block(D);
  __shared__ __attribute__((aligned(16))) uint8_t s_tile[2][kTile * 2 * D];
  const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6), nkv = p.num_kv_heads;
  const int h = uniform((int)(blockIdx.x % nkv)), rest = uniform((int)(blockIdx.x / nkv));
  const int split = uniform(rest % p.key_splits), unit = uniform(rest / p.key_splits);
  const int r = uniform(unit_request(p.qo_indptr, p.group, BLOCK, p.batch, unit));
  if (r < 0) return;
  const WRequest q = w_request(p, r);
  if (q.rows <= kWRows || q.len <= 0) return;
  const int row0 = (unit - unit_begin(p.qo_indptr, p.group, BLOCK, r)) * BLOCK;
  if (row0 >= q.rows) return;
  const int off = q.len - q.qo_len, last_row = min(row0 + BLOCK, q.rows) - 1;
  const int keys = p.causal ? min(q.len, off + last_row / p.group + 1) : q.len;  // seen by some row
  const int tiles = keys > 0 ? (keys + kTile - 1) / kTile : 0;
  const int t0 = share_begin(split, p.key_splits, tiles), t1 = share_begin(split + 1, p.key_splits, tiles);
  const int col = lane & 31, hi = lane >> 5;
  float sl2 = KVT == kKvFp8 ? p.scale_log2 * ((const float*)p.k_scale)[h] : p.scale_log2;
  const uint32_t flip = sl2 < 0.f ? 0x80008000u : 0u;  // the maximum is taken of unscaled scores: the scale's sign goes to q
  sl2 = fabsf(sl2);
  // Hidden scores are -inf before the scale, which zero would make NaN: then the products are scaled first, in every tile.
  const bool zero = sl2 == 0.f;
  if (zero) sl2 = 1.f;
  uint4 qf[NS][STEPS];
  int lim[NS], row[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    row[n] = row0 + kTile * (NS * wave + n) + col;
    const int at = min(row[n], q.rows - 1), tok = at / p.group;
    const uint16_t* src = (const uint16_t*)p.q + (int64_t)(q.qo_start + tok) * p.q_stride_tok + (int64_t)(h * p.group + at - tok * p.group) * p.q_stride_head;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      uint4 u = *(const uint4*)(src + 16 * st + 8 * hi);
      u.x ^= flip, u.y ^= flip, u.z ^= flip, u.w ^= flip;
      qf[n][st] = u;
    }
    lim[n] = p.causal ? off + tok : q.len - 1;
  }
  float m[NS], l[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) m[n] = -kWInf, l[n] = 0.f;
  const int clear = zero ? -1 : p.causal ? off + row0 / p.group : q.len - 1;  // keys up to here are seen by every row
  // One tile a barrier: with two, the registers of both leave room for two wavefronts instead of three (205 -> 232 us).
  using Keys = KeyStream<MT, KVT, D>;
  Keys keys_in;
  typename Keys::Tile next;
  if (t0 < t1) {
    keys_in.begin(p, q, t0);
    keys_in.load(p, q, h, next);
    Keys::store(next, s_tile[0]);
    if (t0 + 1 < t1) keys_in.load(p, q, h, next);
  }
  __syncthreads();
  for (int i = t0; i < t1; ++i) {
    const uint8_t* tile = s_tile[(i - t0) & 1];
    if (i + 1 < t1) Keys::store(next, s_tile[(i - t0 + 1) & 1]);
    if (i + 2 < t1) keys_in.load(p, q, h, next);
    f32x16 acc[NS] = {};
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const uint4 a = tile_fragment<D>(tile, col, st, hi);
#pragma unroll
      for (int n = 0; n < NS; ++n) acc[n] = mma_32x32x16<MT>(a, qf[n][st], acc[n]);
    }
    const int tok = kTile * i;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      if (tok + kTile - 1 > clear) {
        if (zero)
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[n][j] *= 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (tok + (j & 3) + 8 * (j >> 2) + 4 * hi > lim[n]) acc[n][j] = -kWInf;
      }
      float top = fmaxf(acc[n][0], acc[n][1]);
#pragma unroll
      for (int j = 2; j < 16; j += 2) top = fmaxf(top, fmaxf(acc[n][j], acc[n][j + 1]));
      top *= sl2;
      if (__builtin_amdgcn_ballot_w64(top > m[n] + 8.f)) {  // raised only past 2^8: harmless in an fp32 sum, and rare
        const float mn = fmaxf(m[n], top);
        l[n] *= mn == -kWInf ? 0.f : fast_exp2(m[n] - mn);
        m[n] = mn;
      }
      const float mu = m[n] == -kWInf ? 0.f : m[n];
      float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j & 3] += fast_exp2(fmaf(acc[n][j], sl2, -mu));
      l[n] += (x[0] + x[1]) + (x[2] + x[3]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const float mg = both_max(m[n]), mgu = mg == -kWInf ? 0.f : mg;
    const float lg = both_sum(l[n] * fast_exp2(m[n] - mgu));
    if (hi == 0 && row[n] < q.rows)
      p.row_lse[((int64_t)split * nkv + h) * p.total_rows + (int64_t)q.qo_start * p.group + row[n]] = w_lse(mg, lg);
  }
}

// Second pass: each key's sum of exp2(s - lse) over the rows that see it.  A workgroup takes 128 or 256
// keys of a request and kv head and a share of the rows: S = Q K^T, a lane's scores all of one key.
template <typename MT, int KVT, int D>
__global__ __launch_bounds__(256, 2) void weights_cols_kernel(WeightsParams p) {
  constexpr int NS = stationary(D), STEPS = D / 16, BLOCK = mma_block(D), PIECES = D / 8, NU = kTile * PIECES / 256;
  __shared__ __attribute__((aligned(16))) uint8_t s_tile[4][kTile * 2 * D];
  __shared__ __attribute__((aligned(16))) float s_lse[4][kTile];
  const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6), nkv = p.num_kv_heads, tid = (int)threadIdx.x;
  const int h = uniform((int)(blockIdx.x % nkv)), rest = uniform((int)(blockIdx.x / nkv));
  const int split = uniform(rest % p.row_splits), unit = uniform(rest / p.row_splits);
  const int r = uniform(unit_request(p.kv_indptr, 1, p.key_pages, p.batch, unit));
  if (r < 0) return;
  const WRequest q = w_request(p, r);
  if (q.rows <= kWRows) return;
  // the unit's pages in blocks: one, but for pages that hold more keys
  const int tok0 = (unit - unit_begin(p.kv_indptr, 1, p.key_pages, r)) * p.key_pages * p.page_size;
  const int tok1 = min(tok0 + p.key_pages * p.page_size, q.len);
  const int off = q.len - q.qo_len, G = p.group, step_tok = kTile / G, step_g = kTile % G;
  const int col = lane & 31, hi = lane >> 5;
  const float sl2 = KVT == kKvFp8 ? p.scale_log2 * ((const float*)p.k_scale)[h] : p.scale_log2;
  const float* lse = p.row_lse + (int64_t)h * p.total_rows + (int64_t)q.qo_start * G;
  for (int base = tok0; base < tok1; base += BLOCK) {
    // rows from the first that sees the block's first key on
    const int first = p.causal ? (max(0, base - off) * G) / kTile : 0, tiles = max(0, (q.rows + kTile - 1) / kTile - first);
    const int clear = p.causal ? max(0, min(base + BLOCK, q.len) - 1 - off) * G : 0;  // rows from here on see every key
    const int t0 = first + share_begin(split, p.row_splits, tiles), t1 = first + share_begin(split + 1, p.row_splits, tiles);
    // the stream of q rows: pieces of 16 bytes, and the tile's log-sum-exps
    struct Rows {
      u32x4_t w[NU];
      float e;
    };
    int tok[NU], g[NU];
    const uint16_t* src[NU];  // of row (tok, g): 32 rows on, and a token on with a group's heads back, are fixed steps
    const int64_t step = step_tok * p.q_stride_tok + step_g * p.q_stride_head, wrap = p.q_stride_tok - G * p.q_stride_head;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int at = kTile * t0 + (tid + 256 * u) / PIECES;
      tok[u] = at / G;
      g[u] = at - tok[u] * G;
      src[u] = (const uint16_t*)p.q + (int64_t)(q.qo_start + tok[u]) * p.q_stride_tok + (int64_t)(h * G + g[u]) * p.q_stride_head +
               8 * ((tid + 256 * u) % PIECES);
    }
    int lse_row = kTile * t0 + tid;
    // rows past the last are read as the last token's, which sees every key (a NaN of it is one of theirs), with an lse of infinity
    const uint16_t* const none = (const uint16_t*)p.q + (int64_t)(q.qo_start + q.qo_len - 1) * p.q_stride_tok + (int64_t)h * G * p.q_stride_head;
    const int end = min(q.rows, kTile * t1);
    auto load = [&](Rows& t) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        t.w[u] = *(const u32x4_t*)(tok[u] < q.qo_len ? src[u] : none);
        tok[u] += step_tok;
        g[u] += step_g;
        src[u] += step;
        if (g[u] >= G) {
          g[u] -= G;
          ++tok[u];
          src[u] += wrap;
        }
      }
      t.e = lse[min(lse_row, q.rows - 1)];
      if (lse_row >= end) t.e = kWInf;
      lse_row += kTile;
    };
    auto store = [&](const Rows& t, int b) {
#pragma unroll
      for (int u = 0; u < NU; ++u) *(u32x4_t*)(s_tile[b] + tile_at<D>((tid + 256 * u) / PIECES, (tid + 256 * u) % PIECES)) = t.w[u];
      if (tid < kTile) s_lse[b][tid] = t.e;
    };
    Rows ra, rb;
    if (t0 < t1) {
      load(ra);
      load(rb);
    }
    uint4 kf[NS][STEPS];
    int key[NS], from[NS];  // the key, and the first row that sees it
    float sum[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      key[n] = base + kTile * (NS * wave + n) + col;
      from[n] = p.causal ? max(0, key[n] - off) * G : 0;
      sum[n] = 0.f;
      const int at = min(key[n], tok1 - 1), en = (int)((unsigned)at / (unsigned)p.page_size);
      const int64_t page = safe_page(p, q.first + en);
#pragma unroll
      for (int st = 0; st < STEPS; ++st) kf[n][st] = key_piece<MT, KVT, D>(p, page, at - en * p.page_size, h, 2 * st + hi);
    }
    auto tile_of = [&](int b, int i) {
      f32x16 acc[NS] = {};
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const uint4 a = tile_fragment<D>(s_tile[b], col, st, hi);
#pragma unroll
        for (int n = 0; n < NS; ++n) acc[n] = mma_32x32x16<MT>(a, kf[n][st], acc[n]);
      }
      float le[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 v = *(const float4*)(&s_lse[b][8 * j + 4 * hi]);
        le[4 * j] = v.x, le[4 * j + 1] = v.y, le[4 * j + 2] = v.z, le[4 * j + 3] = v.w;
      }
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (kTile * i < clear) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float v = fast_exp2(fmaf(acc[n][j], sl2, -le[j]));
            x[j & 3] += kTile * i + (j & 3) + 8 * (j >> 2) + 4 * hi < from[n] ? 0.f : v;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j & 3] += fast_exp2(fmaf(acc[n][j], sl2, -le[j]));
        }
        sum[n] += (x[0] + x[1]) + (x[2] + x[3]);
      }
    };
    if (t0 < t1) {
      store(ra, 0);
      store(rb, 1);
      load(ra);
      load(rb);
    }
    __syncthreads();
    // Two tiles a barrier, the next two on their way into LDS and two more into registers (211 -> 197 us).
    for (int i = t0, b = 0; i < t1; i += 2, b ^= 2) {
      store(ra, b ^ 2);
      store(rb, (b ^ 2) + 1);
      load(ra);
      load(rb);
      tile_of(b, i);
      tile_of(b + 1, i + 1);
      __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const float total = both_sum(sum[n]);
      if (hi != 0 || key[n] >= tok1) continue;
      w_add(p, q, h, split, key[n], off, total);
    }
  }
}

// ------------------------------------------------------------ long queries, fp32
// First pass: the log-sum-exp of every (query, q head) row.  A workgroup takes 128 rows of a
// request and kv head, 32 to a wavefront, and a share of the keys: S^T = K Q^T with the rows' q in
// registers, a lane's four scores all of one row.
template <int D>
__global__ __launch_bounds__(256) void weights_rows_f32_kernel(WeightsParams p) {
  using MT = F32;
  using Tile = KeyTile<MT, kKv16, D>;
  constexpr int NB = 2;
  const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6), nkv = p.num_kv_heads;
  const int h = uniform((int)(blockIdx.x % nkv)), rest = uniform((int)(blockIdx.x / nkv));
  const int split = uniform(rest % p.key_splits), unit = uniform(rest / p.key_splits);
  const int r = uniform(unit_request(p.qo_indptr, p.group, kRowBlock, p.batch, unit));
  if (r < 0) return;
  const WRequest q = w_request(p, r);
  if (q.rows <= kWRows || q.len <= 0) return;
  const int row0 = (unit - unit_begin(p.qo_indptr, p.group, kRowBlock, r)) * kRowBlock;
  if (row0 >= q.rows) return;
  const int off = q.len - q.qo_len, last_row = min(row0 + kRowBlock, q.rows) - 1;
  const int keys = p.causal ? min(q.len, off + last_row / p.group + 1) : q.len;  // seen by some row
  const int tiles = keys > 0 ? (keys + 15) >> 4 : 0;
  const int t0 = share_begin(split, p.key_splits, tiles), t1 = share_begin(split + 1, p.key_splits, tiles);
  const int col = lane & 15, grp = lane >> 4;
  const float sl2 = p.scale_log2;
  uint4 qf[NB][Tile::STEPS];
  int lim[NB], row[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    row[n] = row0 + 32 * wave + 16 * n + col;
    const int at = min(row[n], q.rows - 1), tok = at / p.group;
    Tile::query(p, q.qo_start + tok, h * p.group + at - tok * p.group, grp, qf[n]);
    lim[n] = p.causal ? off + tok : q.len - 1;
  }
  float m[NB], l[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) m[n] = -kWInf, l[n] = 0.f;
  const int clear = p.causal ? off + row0 / p.group : q.len - 1;  // keys up to here are seen by every row
  auto load = [&](Tile& t, int i) {
    const int tok = 16 * i, e = (int)((unsigned)tok / (unsigned)p.page_size);
    t.load(p, safe_page(p, q.first + e), tok - e * p.page_size + col, h, grp);
  };
  auto compute = [&](const Tile& t, int i) {
    const int tok = 16 * i;
    uint4 kf[Tile::STEPS];
    t.fragments(kf);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < Tile::STEPS; ++st) acc = MT::mma_16x16x32(kf[st], qf[n][st], acc);
      float s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = acc[j] * sl2;
      if (tok + 15 > clear)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (tok + 4 * grp + j > lim[n]) s[j] = -kWInf;
      const float mn = fmaxf(m[n], fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
      const float mu = mn == -kWInf ? 0.f : mn;
      l[n] = l[n] * fast_exp2(m[n] - mu) +
             ((fast_exp2(s[0] - mu) + fast_exp2(s[1] - mu)) + (fast_exp2(s[2] - mu) + fast_exp2(s[3] - mu)));
      m[n] = mn;
    }
  };
  Tile a, b;
  if (t0 < t1) load(a, t0);
  for (int i = t0; i < t1; i += 2) {
    if (i + 1 < t1) load(b, i + 1);
    compute(a, i);
    if (i + 2 < t1) load(a, i + 2);
    if (i + 1 < t1) compute(b, i + 1);
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const float mg = rows4_max(m[n]), mgu = mg == -kWInf ? 0.f : mg;
    const float lg = rows4_sum(l[n] * fast_exp2(m[n] - mgu));
    if (grp == 0 && row[n] < q.rows)
      p.row_lse[((int64_t)split * nkv + h) * p.total_rows + (int64_t)q.qo_start * p.group + row[n]] = w_lse(mg, lg);
  }
}

// Second pass: each key's sum of exp2(s - lse) over the rows that see it.  A workgroup takes 128
// keys of a request and kv head, 32 to a wavefront, in registers, and a share of the rows: S = Q K^T, a
// lane's four scores all of one key.
template <int D>
__global__ __launch_bounds__(256) void weights_cols_f32_kernel(WeightsParams p) {
  using MT = F32;
  using Tile = KeyTile<MT, kKv16, D>;
  constexpr int NB = 2;
  const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6), nkv = p.num_kv_heads;
  const int h = uniform((int)(blockIdx.x % nkv)), rest = uniform((int)(blockIdx.x / nkv));
  const int split = uniform(rest % p.row_splits), unit = uniform(rest / p.row_splits);
  const int r = uniform(unit_request(p.kv_indptr, 1, p.key_pages, p.batch, unit));
  if (r < 0) return;
  const WRequest q = w_request(p, r);
  if (q.rows <= kWRows) return;
  // the unit's pages in blocks of 128 keys: one, but for pages that hold more
  const int tok0 = (unit - unit_begin(p.kv_indptr, 1, p.key_pages, r)) * p.key_pages * p.page_size;
  const int tok1 = min(tok0 + p.key_pages * p.page_size, q.len);
  const int off = q.len - q.qo_len, G = p.group;
  const int col = lane & 15, grp = lane >> 4;
  const float sl2 = p.scale_log2;
  const float* lse = p.row_lse + (int64_t)h * p.total_rows + (int64_t)q.qo_start * G;
  for (int base = tok0; base < tok1; base += kKeyBlock) {
    uint4 kf[NB][Tile::STEPS];
    int key[NB], from[NB];  // the key, and the first row that sees it
    float sum[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int t16 = base + 32 * wave + 16 * n;
      key[n] = t16 + col;
      from[n] = p.causal ? max(0, key[n] - off) * G : 0;
      sum[n] = 0.f;
      const int at = min(t16, tok1 - 1) & ~15, e = (int)((unsigned)at / (unsigned)p.page_size);
      Tile t;
      t.load(p, safe_page(p, q.first + e), at - e * p.page_size + col, h, grp);
      t.fragments(kf[n]);
    }
    // rows from the first that sees the block's first key, in tiles of 16
    const int first = p.causal ? (max(0, base - off) * G) >> 4 : 0, tiles = ((q.rows + 15) >> 4) - first;
    const int clear = p.causal ? max(0, min(base + kKeyBlock, q.len) - 1 - off) * G : 0;  // rows from here on see every key
    const int t0 = first + share_begin(split, p.row_splits, max(0, tiles));
    const int t1 = first + share_begin(split + 1, p.row_splits, max(0, tiles));
    auto load = [&](uint4 (&qf)[Tile::STEPS], float (&e)[4], int i) {
      const int at = min(16 * i + col, q.rows - 1), tok = at / G;
      Tile::query(p, q.qo_start + tok, h * G + at - tok * G, grp, qf);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 16 * i + 4 * grp + j;
        e[j] = row < q.rows ? lse[row] : kWInf;
      }
    };
    auto compute = [&](const uint4 (&qf)[Tile::STEPS], const float (&e)[4], int i) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < Tile::STEPS; ++st) acc = MT::mma_16x16x32(qf[st], kf[n][st], acc);
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fast_exp2(acc[j] * sl2 - e[j]);
        if (16 * i < clear)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (16 * i + 4 * grp + j < from[n]) x[j] = 0.f;
        sum[n] += (x[0] + x[1]) + (x[2] + x[3]);
      }
    };
    uint4 qa[Tile::STEPS], qb[Tile::STEPS];
    float ea[4], eb[4];
    if (t0 < t1) load(qa, ea, t0);
    for (int i = t0; i < t1; i += 2) {
      if (i + 1 < t1) load(qb, eb, i + 1);
      compute(qa, ea, i);
      if (i + 2 < t1) load(qa, ea, i + 2);
      if (i + 1 < t1) compute(qb, eb, i + 1);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float total = rows4_sum(sum[n]);
      if (grp != 0 || key[n] >= tok1) continue;
      w_add(p, q, h, split, key[n], off, total);
    }
  }
}

enum : int { kWScores = 0, kWRowsPass = 1, kWColsPass = 2, kWOne = 3 };

template <typename MT, int KVT, int D>
static void launch_weights_d(const WeightsParams& p, int which, dim3 grid, hipStream_t s) {
  if (which == kWOne) hipLaunchKernelGGL((weights_one_kernel<MT, KVT, D>), grid, dim3(one_threads<MT>(D)), 0, s, p);
  else if (which == kWScores) hipLaunchKernelGGL((weights_scores_kernel<MT, KVT, D>), grid, dim3(256), 0, s, p);
  else if constexpr (MT::kDtype == MI_F32) {
    if (which == kWRowsPass) hipLaunchKernelGGL((weights_rows_f32_kernel<D>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((weights_cols_f32_kernel<D>), grid, dim3(256), 0, s, p);
  } else {
    if (which == kWRowsPass) hipLaunchKernelGGL((weights_rows_kernel<MT, KVT, D>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((weights_cols_kernel<MT, KVT, D>), grid, dim3(256), 0, s, p);
  }
}

template <typename MT, int KVT>
static int launch_weights_kvt(const WeightsParams& p, int head_dim, int which, dim3 grid, hipStream_t s) {
  switch (head_dim) {
    case 64: launch_weights_d<MT, KVT, 64>(p, which, grid, s); return MI_OK;
    case 128: launch_weights_d<MT, KVT, 128>(p, which, grid, s); return MI_OK;
    case 256: launch_weights_d<MT, KVT, 256>(p, which, grid, s); return MI_OK;
    default: return MI_ERR_UNSUPPORTED;
  }
}

int weights_launch_16(const WeightsParams& p, int q_dtype, int head_dim, int which, dim3 grid, hipStream_t s);
int weights_launch_scaled(const WeightsParams& p, int q_dtype, int kvt, int head_dim, int which, dim3 grid, hipStream_t s);

}  // namespace mi
