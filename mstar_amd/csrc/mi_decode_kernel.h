// The split-KV decode kernel (decode_kernel) and its launch, shared by
// mi_decode.hip (plan, merge, 16-bit and per-head fp8 caches), mi_decode_win.hip
// (windows) and mi_decode_mx.hip (microscaled caches).  The kernel's description
// heads mi_decode.hip.
#pragma once

#include "mi_common.h"
#include "mi_internal.h"
#include "mi_plan.h"

namespace mi {


// Per-lane registers of one 16-token tile.
template <int KVT, int D>
struct TileRegs {
  // words of a lane's D/16 elements of a row: row slices as stored, converted
  // right before use (half a word at 4 bits and head_dim 64)
  static constexpr int N = KVT == kKv16 ? D / 32 : KVT == kKvMx4 ? (D + 127) / 128 : D / 64;
  uint32_t k[4][N];
  uint32_t v[4][N];
};

// Microscaled caches: the scale bytes of the lane's four rows (its elements of
// a row lie in one block of 32), one word each for K and V.
struct TileScales {
  uint32_t k, v;
};

// CACHED: loads that stay in the L2.  A microscaled row is 32 to 128 bytes, less than
// the 128-byte line it lies in or the run of a token's heads: the neighbour's
// workgroup reads the rest of the line soon (streaming loads had it fetched again:
// B=256, 1k-32k contexts, 4 kv heads x 64-byte rows 359 -> 294 us; 64 requests at 8
// kv heads x 128-byte rows 33 -> 31 us).
template <bool CACHED, int N>
MI_DEVICE void load_words(uint32_t (&dst)[N], const uint8_t* src) {
  if constexpr (CACHED && N == 1) {
    dst[0] = *(const uint32_t*)src;
  } else if constexpr (CACHED && N == 2) {
    const uint2 t = *(const uint2*)src;
    dst[0] = t.x;
    dst[1] = t.y;
  } else if constexpr (CACHED) {
    static_assert(N == 4, "a microscaled row slice is at most 16 bytes");
    const uint4 t = *(const uint4*)src;
    dst[0] = t.x;
    dst[1] = t.y;
    dst[2] = t.z;
    dst[3] = t.w;
  } else if constexpr (N == 1) {
    dst[0] = nt_load4(src);
  } else if constexpr (N == 2) {
    const uint2 t = nt_load8(src);
    dst[0] = t.x;
    dst[1] = t.y;
  } else {  // 16-byte chunk k of the lane's elements sits 256*k bytes into the row (see dim_of)
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 t = nt_load16(src + 64 * i);
      dst[i] = t.x;
      dst[i + 1] = t.y;
      dst[i + 2] = t.z;
      dst[i + 3] = t.w;
    }
  }
}

// The request at place `rank` of a windowed batch when its requests are taken by
// classes of tiles, an eighth of the batch's most each, most first: workgroups start
// in order, so the last ones to start are short.  The workgroup's threads class
// 256 requests at a time and count by ballots, from the index arrays alone.
__device__ __forceinline__ int win_item(const DecodeParams& p, int rank) {
  constexpr int kClasses = 8;
  __shared__ int s_count[4][kClasses], s_most[4], s_b;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto tiles_of = [&](int r) {
    const int np = p.kv_indptr[r + 1] - p.kv_indptr[r];
    const int qo_len = p.qo_indptr ? p.qo_indptr[r + 1] - p.qo_indptr[r] : 1;
    if (qo_len <= 0 || qo_len * p.group > p.short_rows) return 0;  // nothing to do here
    return max(0, win_tiles(np > 0 ? (np - 1) * p.page_size + p.last_page_len[r] : 0, qo_len, p).total);
  };
  int mine[kSortedMax / 256], most = 1;
  for (int c = 0; c * 256 < p.batch; ++c) {
    mine[c] = c * 256 + tid < p.batch ? tiles_of(c * 256 + tid) : -1;
    most = max(most, mine[c]);
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) most = max(most, __shfl_xor(most, m, kWave));
  if (lane == 0) s_most[wave] = most;
  __syncthreads();
  const float per_tile = (float)kClasses / (float)max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
  int total[kClasses] = {};  // this wavefront's counts, all chunks of 256
  for (int c = 0; c * 256 < p.batch; ++c) {
    if (mine[c] >= 0) mine[c] = kClasses - 1 - min(kClasses - 1, (int)((float)mine[c] * per_tile));
#pragma unroll
    for (int k = 0; k < kClasses; ++k) total[k] += __popcll(__builtin_amdgcn_ballot_w64(mine[c] == k));
  }
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < kClasses; ++k) s_count[wave][k] = total[k];
  __syncthreads();
  // this wavefront's first place in each class: classes before it, wavefronts before it
  int at[kClasses], sum = 0;
#pragma unroll
  for (int k = 0; k < kClasses; ++k)
    for (int w = 0; w < 4; ++w) {
      if (w == wave) at[k] = sum;
      sum += s_count[w][k];
    }
  for (int c = 0; c * 256 < p.batch; ++c) {
    int place = -1;
#pragma unroll
    for (int k = 0; k < kClasses; ++k) {
      const uint64_t in = __builtin_amdgcn_ballot_w64(mine[c] == k);
      if (mine[c] == k) place = at[k] + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
      at[k] += __popcll(in);
    }
    if (place == rank) s_b = c * 256 + tid;
  }
  __syncthreads();
  return uniform(s_b);
}

// Wavefronts per SIMD the registers are held to.  With two, microscaled kernels
// keep their accumulators out of the AGPRs, so that rescaling them costs no moves
// (4 bits, head_dim 256, 96 windows of 4k: 62.5 -> 60.2 us, and a second workgroup
// a CU); at 8 bits and head_dim 256 that spills.
constexpr int decode_waves(int kvt, int d, bool win) {
  return kvt == kKvMx4 || (kvt == kKvMx8 && d <= 128) || (win && d <= 128) ? 2 : 1;
}

// PAIR (D = 256): two adjacent head_dim 128 kv-heads read as one 256-element
// row; p.num_kv_heads counts the pairs, p.group is the real group size, query
// row col belongs to kv-head 2h + (col >= group) (see pair_heads).
// WIN: the sliding window with its sinks (DecodeParams::window_left, sinks).  A
// request's tiles are then those of its sinks and of its window only
// (win_tiles), in one sequence that its items share evenly.  Which item a
// workgroup takes follows from its place and the lengths (win_item), so a windowed
// run needs no plan of its own and a model may mix windowed and full layers.
// NW: wavefronts of the workgroup.  Eight (WIN, one item a request) where a request
// would have been cut in two workgroups of four, or in few short ones: no partials and
// no merge.
template <typename MT, int KVT, int D, bool PAIR = false, bool WIN = false, int NW = 4>
__global__ __launch_bounds__(64 * NW, decode_waves(KVT, D, WIN)) void decode_kernel(DecodeParams p) {
  static_assert(!PAIR || D == 256, "paired kv-heads form 256-element rows");
  constexpr bool FP8 = KVT == kKvFp8, MX = KVT == kKvMx8 || KVT == kKvMx4, F16_MX = MX && MT::kDtype == MI_F16;
  constexpr int KS = D / 32;  // MFMA k-steps over head_dim for S
  constexpr int VW = D / 16;  // V elements per lane per row == output d-tiles
  constexpr int ESZ = KVT == kKv16 ? 2 : 1;  // of the strides (bytes of codes for microscaled caches)
  constexpr int KRS = D * 2 + 32;  // LDS row stride of the K transpose buffer (8-bank step: conflict-free fragment reads)
  constexpr int RUN = lane_run(D, ESZ);  // consecutive elements per lane (dim_of)
  constexpr int NS = VW / 4;       // float4 groups per lane per output row segment
  constexpr float kNegInf = -__builtin_inff();
  // LDS: during the tile loop, per-wave K staging (rows arrive as whole
  // head_dim rows and leave as MFMA A fragments); after it, the 4 waves'
  // softmax states for the in-workgroup merge.
  constexpr int kStageBytes = NW * 16 * KRS;
  constexpr int kMergeBytes = NW * (4 * NS * 64 * 16);
  __shared__ __attribute__((aligned(16))) uint8_t lds[kStageBytes > kMergeBytes ? kStageBytes : kMergeBytes];
  __shared__ float lds_m[NW][kRows], lds_l[NW][kRows];

  const int lane = lane_id();
  const int wave = uniform((int)threadIdx.x >> 6);
  const int nkv = p.num_kv_heads;
  // workgroup = (item, kv-head); its 4 waves split the item's tiles
  // all kv-heads of an item on one XCD (blocks go to XCDs round-robin), 8 blocks apart
  const int gsz = 8 * nkv;
  const int gi = uniform((int)blockIdx.x / gsz);
  const int gr = (int)blockIdx.x - gi * gsz;
  const int h = uniform(gr >> 3);
  const int item = uniform(gi * 8 + (gr & 7));
  int b, kidx, pg0 = 0, pg1, nitems_b;
  if constexpr (WIN) {
    if (item >= p.batch * p.splits) return;
    kidx = item / p.batch;
    b = item - kidx * p.batch;
    if constexpr (NW == 4)
      if (p.sorted) b = win_item(p, b);
  } else {
    if (item >= p.hdr[kHdrChunks]) return;  // uniform across the workgroup
    const int4 wk = p.work[item];
    b = uniform(wk.x), kidx = uniform(wk.y), pg1 = uniform(wk.z), nitems_b = uniform(wk.w);
    pg0 = kidx * p.hdr[kHdrChunkPages];
  }

  const int ps = p.page_size;
  const int page_base = p.kv_indptr[b];
  const int np = p.kv_indptr[b + 1] - page_base;
  const int kv_len = WIN && np <= 0 ? 0 : (np - 1) * ps + p.last_page_len[b];
  int qo_start = b, qo_len = 1;
  if (p.qo_indptr) {
    qo_start = p.qo_indptr[b];
    qo_len = p.qo_indptr[b + 1] - qo_start;
  }
  const int G = p.group;
  const int rows = min((PAIR ? 2 : 1) * qo_len * G, kRows);
  int item_tok0 = 0, item_tiles, first_tile = 0;
  WinTiles span;
  if constexpr (WIN) {
    if (qo_len <= 0 || qo_len * G > p.short_rows) return;  // no rows, or the prefill kernel's
    span = win_tiles(kv_len, qo_len, p);
    nitems_b = span.items;
    if (kidx >= nitems_b) return;
    pg1 = np;
    first_tile = share_begin(kidx, nitems_b, span.total);
    item_tiles = share_begin(kidx + 1, nitems_b, span.total) - first_tile;
  } else {
    item_tok0 = pg0 * ps;
    const int item_tok1 = min(pg1 * ps, kv_len);
    item_tiles = item_tok1 > item_tok0 ? (item_tok1 - item_tok0 + 15) >> 4 : 0;
  }
  // this wave's contiguous share of the item's tiles
  const int tq = item_tiles / NW, trem = item_tiles % NW;
  const int my_t0 = wave * tq + min(wave, trem);
  const int ntiles = tq + (wave < trem ? 1 : 0);
  const int tok_begin = item_tok0 + 16 * my_t0;

  const int col = lane & 15;  // query row handled in MFMA column `col`
  const int grp = lane >> 4;  // 0..3
  const int half = PAIR && col >= qo_len * G ? 1 : 0;  // PAIR: which head of the pair
  const int rcol = col - half * qo_len * G;
  const int hq = PAIR ? 2 * h + half : h;  // the row's kv-head
  const int qtok = rcol / G;
  const int g = rcol - qtok * G;
  const bool row_valid = col < rows;
  // Keys this row may attend: [0, lim]  (causal: aligned to the end of the KV).
  int lim = p.causal ? (kv_len - qo_len + qtok) : (kv_len - 1);
  lim = min(lim, kv_len - 1);
  // Keys >= mask_from need a per-row check (uniform bound).
  const int mask_from = p.causal ? (kv_len - qo_len + 1) : kv_len;
  // WIN: where the window of the request's first row, of this row and of the last row begins
  const int lo_first = WIN ? kv_len - qo_len - p.window_left : 0, lo_row = lo_first + qtok;
  const int lo_last = lo_first + qo_len - 1;

  // ---- Q as the B operand of S^T = K Q^T: lane holds Q[row col][8*grp + 32*s ...].
  // PAIR: only the row's own 128 elements; both heads' score products use
  // them, and each column keeps the product with its own head's keys.
  constexpr int QS = PAIR ? KS / 2 : KS;
  uint4 qf[QS];
  {
    const uint16_t* qrow = (const uint16_t*)p.q + (int64_t)(qo_start + qtok) * p.q_stride_tok +
                           (int64_t)(hq * G + g) * p.q_stride_head;
#pragma unroll
    for (int s = 0; s < QS; ++s)
      qf[s] = row_valid ? *(const uint4*)(qrow + 32 * s + 8 * grp) : make_uint4(0, 0, 0, 0);
  }
  float kscale = 1.0f, vscale = 1.0f;
  if constexpr (FP8) {
    kscale = p.k_scale[hq];
    vscale = p.v_scale[hq];
  }
  const float sl2 = p.scale_log2 * kscale;

  // Microscaled caches: [page][K, V][kv-head][block][slot] scale bytes
  constexpr int NBLK = D / kMxBlock;
  const int64_t scale_page = 2LL * nkv * NBLK * ps;
  const uint32_t scale_off = MX ? (uint32_t)((h * NBLK + RUN * col / kMxBlock) * ps + 4 * grp) : 0;

  const uint8_t* kv = (const uint8_t*)p.kv;
  const int64_t head_off = (int64_t)h * p.head_stride * ESZ;
  // per-lane byte offset inside a tile: rows 4*grp + r, elements [VW*col, VW*col + VW)
  const uint32_t voff0 = (uint32_t)((4 * grp) * p.token_stride + (KVT == kKvMx4 ? RUN * col / 2 : RUN * col)) * ESZ;
  const uint32_t vrow = (uint32_t)(p.token_stride * ESZ);
  const int64_t kvhalf = p.kv_stride * ESZ;

  // page ids, slots and strides are non-negative: unsigned scalar arithmetic
  // (a signed division and 64-bit multiply per tile cost ~30 scalar ops)
  const uint64_t page_bytes = (uint64_t)p.page_stride * ESZ;
  auto tile_base = [&](int page, int r0) -> const uint8_t* {
    return kv + (uint64_t)(uint32_t)page * page_bytes + (uint32_t)r0 * vrow + head_off;
  };
  auto load_tile = [&](TileRegs<KVT, D>& t, const uint8_t* base) {
    const uint8_t* kb = base + voff0;
    const uint8_t* vb = kb + kvhalf;
    if constexpr (KVT == kKvMx4 && D == 64) {  // four elements of a row: two bytes
#pragma unroll
      for (int r = 0; r < 4; ++r) t.k[r][0] = *(const uint16_t*)(kb + r * vrow);
#pragma unroll
      for (int r = 0; r < 4; ++r) t.v[r][0] = *(const uint16_t*)(vb + r * vrow);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) load_words<MX>(t.k[r], kb + r * vrow);
#pragma unroll
      for (int r = 0; r < 4; ++r) load_words<MX>(t.v[r], vb + r * vrow);
    }
  };
  // The scale words of a tile: the four rows' bytes are adjacent slots of one
  // (head, block), so each is one aligned load.
  auto load_scales = [&](TileScales& t, int page, int r0) {
    if constexpr (MX) {
      const int64_t off = (uint64_t)(uint32_t)page * (uint64_t)scale_page + (uint32_t)r0 + scale_off;
      t.k = *(const uint32_t*)((const uint8_t*)p.k_scale + off);
      t.v = *(const uint32_t*)((const uint8_t*)p.v_scale + off);
    }
  };
  uint8_t* kst = &lds[wave * 16 * KRS];

  f32x4 acc[VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = kNegInf, l_run = 0.f;

  auto compute_tile = [&](TileRegs<KVT, D>& t, TileScales& sc, int tb) {
    const bool past = F16_MX && __builtin_amdgcn_ballot_w64(mx_past_f16<KVT>(sc.k) || mx_past_f16<KVT>(sc.v));
    // ---- K rows -> LDS (row 4*grp + r, elements [VW*col, +VW)) -> A fragments
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      uint32_t w[VW / 2];
      if constexpr (FP8) {
#pragma unroll
        for (int i = 0; i < VW / 4; ++i) {
          w[2 * i] = fp8x2_to_mt<MT>(t.k[r][i], false);
          w[2 * i + 1] = fp8x2_to_mt<MT>(t.k[r][i], true);
        }
      } else if constexpr (MX) {
        mx_to_mt<MT, KVT>(t.k[r], mx_scale(sc.k, r), w);
      } else {
#pragma unroll
        for (int i = 0; i < VW / 2; ++i) w[i] = t.k[r][i];
      }
      uint8_t* dst = kst + (4 * grp + r) * KRS;  // row in natural dim order
      if constexpr (VW == 4) {
        *(uint2*)(dst + 2 * dim_of(RUN, col, 0)) = make_uint2(w[0], w[1]);
      } else {
#pragma unroll
        for (int i = 0; i < VW / 2; i += 4)
          *(uint4*)(dst + 2 * dim_of(RUN, col, 2 * i)) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      }
    }
    if constexpr (F16_MX) {  // a lane corrects the elements that it stored itself
      if (past) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint8_t* row = kst + (4 * grp + r) * KRS;
          if constexpr (VW == 4) {
            uint2* at = (uint2*)(row + 2 * dim_of(RUN, col, 0));
            uint32_t w[2] = {at->x, at->y};
            f16_saturate(w);
            *at = make_uint2(w[0], w[1]);
          } else {
#pragma unroll
            for (int i = 0; i < VW / 2; i += 4) {
              uint4* at = (uint4*)(row + 2 * dim_of(RUN, col, 2 * i));
              uint32_t w[4] = {at->x, at->y, at->z, at->w};
              f16_saturate(w);
              *at = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
    }
    // ---- S^T = K . Q^T  (A fragment: row col, elements 8*grp + 32*st .. +8)
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if constexpr (PAIR) {
      // One accumulator per head of the pair: s takes the keys' k-steps
      // [0, KS/2) (head 2h's elements), s1 the k-steps [KS/2, KS) (head
      // 2h+1's), both against the row's own 128 query elements.  A column
      // keeps the product with its own head's keys (a select, so the other
      // product's values, non-finite ones included, never reach it).
      f32x4 s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < KS / 2; ++st) {
        const uint4 a0 = *(const uint4*)(kst + col * KRS + (8 * grp + 32 * st) * 2);
        const uint4 a1 = *(const uint4*)(kst + col * KRS + (8 * grp + 32 * (st + KS / 2)) * 2);
        s = MT::mma_16x16x32(a0, qf[st], s);
        s1 = MT::mma_16x16x32(a1, qf[st], s1);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = half ? s1[r] : s[r];
    } else {
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        const uint4 a = *(const uint4*)(kst + col * KRS + (8 * grp + 32 * st) * 2);
        s = MT::mma_16x16x32(a, qf[st], s);
      }
    }
    float sv[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) sv[r] = s[r] * sl2;
    const bool need_mask = tb + 16 > mask_from || (WIN && tb < lo_last && tb + 16 > p.sinks);
    if (need_mask) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = tb + 4 * grp + r;
        if (key > lim || (WIN && key < lo_row && key >= p.sinks)) sv[r] = kNegInf;
        // slots past the end hold stale data, those between the sinks and every
        // row's window may: keep NaN/Inf out of P.V
        if (key >= kv_len || (WIN && key < lo_first && key >= p.sinks)) {
#pragma unroll
          for (int i = 0; i < (int)(sizeof(t.v[r]) / 4); ++i) t.v[r][i] = 0u;
          if constexpr (MX) sc.v &= ~(0xffu << (8 * r));  // a NaN scale too
        }
      }
    }
    // ---- online softmax (row = col; the 4 lane groups share a row)
    const float mt = rows4_max(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])));
    // Windowed and microscaled kernels raise the running max only past 2^8, as the
    // prefill kernels do: probabilities stay below 2^8, harmless in fp32 sums and
    // 16-bit P, and the rescale, which a wavefront of 16 rows ran on about 40 % of
    // its first 64 tiles, is rare (4 bits: 368 -> 358 us, 67.3 -> 62.5).
    constexpr bool LAZY = WIN || MX;
    const float m_new = LAZY ? (mt > m_run + 8.f ? mt : m_run) : fmaxf(m_run, mt);
    const float m_use = m_new == kNegInf ? 0.f : m_new;
    const float alpha = fast_exp2(m_run - m_use);
    float pr[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) pr[r] = fast_exp2(sv[r] - m_use);
    l_run = l_run * alpha + ((pr[0] + pr[1]) + (pr[2] + pr[3]));
    if (__builtin_amdgcn_ballot_w64(m_new > m_run)) {
#pragma unroll
      for (int j = 0; j < VW; ++j) acc[j] *= alpha;
    }
    m_run = m_new;
    const uint2 pb = make_uint2(MT::pack2(pr[0], pr[1]), MT::pack2(pr[2], pr[3]));
    // ---- O^T += V^T . P^T, V transposed in registers
    uint32_t vv[4][VW / 2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (FP8) {
#pragma unroll
        for (int i = 0; i < VW / 4; ++i) {
          vv[r][2 * i] = fp8x2_to_mt<MT>(t.v[r][i], false);
          vv[r][2 * i + 1] = fp8x2_to_mt<MT>(t.v[r][i], true);
        }
      } else if constexpr (MX) {
        mx_to_mt<MT, KVT>(t.v[r], mx_scale(sc.v, r), vv[r]);
      } else {
#pragma unroll
        for (int i = 0; i < VW / 2; ++i) vv[r][i] = t.v[r][i];
      }
    }
    if constexpr (F16_MX) {
      if (past) {
#pragma unroll
        for (int r = 0; r < 4; ++r) f16_saturate(vv[r]);
      }
    }
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      uint2 a;
      if (j & 1) {
        a.x = pack_hi16(vv[0][j >> 1], vv[1][j >> 1]);
        a.y = pack_hi16(vv[2][j >> 1], vv[3][j >> 1]);
      } else {
        a.x = pack_lo16(vv[0][j >> 1], vv[1][j >> 1]);
        a.y = pack_lo16(vv[2][j >> 1], vv[3][j >> 1]);
      }
      acc[j] = MT::mma_16x16x16(a, pb, acc[j]);
    }
  };

  // ---- tile loop, in windows of 64 pages.  The window's page ids sit in one
  // VGPR (lane i: page i of the window) and v_readlane hands each tile's page
  // to the scalar unit, so no memory access sits between the loads of
  // consecutive tiles; inside a window the loads run two tiles ahead of the
  // MFMA work (three register buffers).
  auto run_tiles = [&](const int tok_begin, const int ntiles) {
  for (int w0 = 0; w0 < ntiles;) {
    const int wtok = tok_begin + 16 * w0;  // first token of the window
    const int first = (int)((unsigned)wtok / (unsigned)ps);  // its page (request-relative)
    const int wt = min(ntiles - w0, ((first + 64) * ps - wtok) >> 4);
    const int pwin = first + lane < pg1 ? p.kv_indices[page_base + first + lane] : 0;
    auto load = [&](TileRegs<KVT, D>& r, TileScales& sc, int t) {  // t: tile within the window
      const unsigned tok = (unsigned)(wtok + 16 * t);
      const unsigned pg = tok / (unsigned)ps;
      const int page = __builtin_amdgcn_readlane(pwin, (int)pg - first), r0 = (int)(tok - pg * (unsigned)ps);
      load_scales(sc, page, r0);
      load_tile(r, tile_base(page, r0));
    };
    auto compute = [&](TileRegs<KVT, D>& r, TileScales& sc, int t) { compute_tile(r, sc, wtok + 16 * t); };
    TileRegs<KVT, D> A, B, C;
    TileScales sa, sb, sc;
    load(A, sa, 0);
    if (wt > 1) load(B, sb, 1);
    int t = 0;
    // Steady state: every load in the body is in range, so the compiler's
    // vmcnt waits stay exact (two tiles in flight while one is computed).
    for (; t + 4 < wt; t += 3) {
      load(C, sc, t + 2);
      compute(A, sa, t);
      load(A, sa, t + 3);
      compute(B, sb, t + 1);
      load(B, sb, t + 4);
      compute(C, sc, t + 2);
    }
    // Tail: at most four tiles left; A holds tile t, B tile t+1.
    if (t + 2 < wt) load(C, sc, t + 2);
    if (t < wt) compute(A, sa, t);
    if (t + 3 < wt) load(A, sa, t + 3);
    if (t + 1 < wt) compute(B, sb, t + 1);
    if (t + 2 < wt) compute(C, sc, t + 2);
    if (t + 3 < wt) compute(A, sa, t + 3);
    w0 += wt;
  }
  };
  if constexpr (WIN) {  // this wave's tiles of the sinks, then of the window
    const int t0 = first_tile + my_t0, t1 = t0 + ntiles, s1 = min(t1, span.sinks), w1 = max(t0, span.sinks);
    if (s1 > t0) run_tiles(16 * t0, s1 - t0);
    if (t1 > w1) run_tiles(16 * (span.first + w1 - span.sinks), t1 - w1);
  } else {
    run_tiles(tok_begin, ntiles);
  }

  // ---- epilogue: merge the waves' states (m, l, acc) in LDS.  The acc
  // register layout is the same in every wave (lane -> row col, elements
  // d = VW*(4*grp + r) + j), so the merge is lane-local; wave w < 4 finishes
  // the elements with r == w.
  __syncthreads();  // all waves are done with their K staging buffers
  {
    const float l_row = rows4_sum(l_run);
    if (grp == 0) {
      lds_m[wave][col] = m_run;
      lds_l[wave][col] = l_row;
    }
    float4* st = (float4*)lds + (size_t)wave * 4 * NS * 64 + lane;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < VW; j += 4)
        st[(r * NS + j / 4) * 64] = make_float4(acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]);
  }
  __syncthreads();
  if (NW > 4 && wave >= 4) return;
  float M = kNegInf;
#pragma unroll
  for (int w = 0; w < NW; ++w) M = fmaxf(M, lds_m[w][col]);
  const float M_use = M == kNegInf ? 0.f : M;
  float sc[NW], L = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    sc[w] = fast_exp2(lds_m[w][col] - M_use);  // m = -inf -> 0
    L += sc[w] * lds_l[w][col];
  }
  float4 o[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float4* src = (const float4*)lds + (size_t)w * 4 * NS * 64 + (size_t)wave * NS * 64 + lane;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const float4 v = src[i * 64];
      o[i].x += sc[w] * v.x;
      o[i].y += sc[w] * v.y;
      o[i].z += sc[w] * v.z;
      o[i].w += sc[w] * v.w;
    }
  }
  const float inv = L > 0.f ? vscale / L : (L == 0.f ? 0.f : __builtin_nanf(""));  // NaN L: keep the row NaN
  if (!row_valid) return;
  if (nitems_b == 1) {
    // elements j of output row 4*grp + wave: dims dim_of(RUN, 4*grp + wave, j), row col
    uint16_t* dst = (uint16_t*)p.out + (int64_t)(qo_start + qtok) * p.out_stride_tok +
                    (int64_t)(hq * G + g) * p.out_stride_head;
    uint32_t w[VW / 2];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      w[2 * i] = MT::pack2(o[i].x * inv, o[i].y * inv);
      w[2 * i + 1] = MT::pack2(o[i].z * inv, o[i].w * inv);
    }
    if constexpr (VW == 4) {
      *(uint2*)(dst + dim_of(RUN, 4 * grp + wave, 0)) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < VW / 2; i += 4) {
        const int d0 = dim_of(RUN, 4 * grp + wave, 2 * i);  // 8 consecutive elements
        if (PAIR && (d0 >= D / 2) != (half == 1)) continue;  // the other head's half
        *(uint4*)(dst + d0 - (PAIR ? (D / 2) * half : 0)) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      }
    }
  } else {
    // Partial (o, lse) of this item, o in register order: store index
    // i = r*NS + j/4 of every lane is one contiguous 64 x 16-byte block.
    const int64_t unit_idx = (int64_t)((WIN ? b * p.splits : p.chunk_indptr[b]) + kidx) * nkv + h;
    float* ob = p.o_part + unit_idx * kRows * D + 4 * lane;
#pragma unroll
    for (int i = 0; i < NS; ++i)
      *(float4*)(ob + 256 * (wave * NS + i)) = make_float4(o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv);
    // lse: -inf for an empty partial; NaN when the row met a NaN or +inf score,
    // so the merge propagates it as a single softmax over the keys would.
    if (wave == 0 && grp == 0)
      p.lse_part[unit_idx * kRows + col] = L > 0.f ? M + fast_log2(L) : (L == 0.f ? kNegInf : __builtin_nanf(""));
  }
}

// One launch of the kernel (grid: blocks of 8 items x kv-heads).
template <typename MT, int KVT, bool WIN, int NW = 4>
static int launch_decode_kernel(const DecodeParams& dp, int head_dim, int grid, hipStream_t stream) {
  const dim3 g(grid), block(64 * NW);
  switch (head_dim) {
    case 64: hipLaunchKernelGGL((decode_kernel<MT, KVT, 64, false, WIN, NW>), g, block, 0, stream, dp); break;
    case 128: hipLaunchKernelGGL((decode_kernel<MT, KVT, 128, false, WIN, NW>), g, block, 0, stream, dp); break;
    case 256:
      if constexpr (NW == 4 || decode_waves(KVT, 256, WIN) == 2) {
        hipLaunchKernelGGL((decode_kernel<MT, KVT, 256, false, WIN, NW>), g, block, 0, stream, dp);
        break;
      }
      return MI_ERR_UNSUPPORTED;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

}  // namespace mi
