// Norms of q and k head by head, with the rotation and the paged append in the same pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w      over the head_dim elements of a (token, head) row of q or k
//   rotated as mi_rope_apply rotates, by the angle pos * f_i
//   q (and k, if kept) in place; k and v to their cache slots
//
// The row's sum, the norm and the rotation are fp32, and a value is rounded once: to the
// q / k type, and from fp32 to the cache's type.  Angles are formed in turns in 64 bits, pos *
// f_i / (2 pi) less its nearest whole number, which is exact enough at any position (an fp32 angle is off
// by 4e-3 rad at 65k tokens, half a step of bf16 and four of fp16); the f_i are the launch argument.
//
// A row is head_dim / 8 lanes (rounded up to a power of two, 16-byte loads), so a wavefront
// holds 64 / LPR rows of one token; its lanes' (cos, sin) are formed once and serve all the rows that
// it goes through.  The other half of a rotated pair is 16 bytes of another lane of the row.
#include <cmath>

#include "mi_internal.h"
#include "mi_mx.h"

namespace mi {

constexpr int kNormDimMax = 512;

struct NormRopeParams {
  void *q, *k;
  const void* v;
  int64_t q_stride_tok, q_stride_head, k_stride_tok, k_stride_head, v_stride_tok, v_stride_head;
  const void *q_weight, *k_weight, *pos;
  uint8_t* cache;
  int64_t page_stride, kv_stride, token_stride, head_stride, max_pages;  // elements (bytes of codes: microscaled)
  void *k_scale, *v_scale;
  const int64_t *page_idx, *slot_idx;
  int64_t idx_stride;
  const int32_t* num_tokens_device;
  int32_t num_tokens, num_append, num_qo_heads, num_kv_heads, head_dim, page_size, rotary_dim, interleave, pos_is_64;
  int32_t weight_f32, keep_k, rows, steps;  // rows: of a token; steps: that a wavefront goes through
  float eps;
  double turns[kNormDimMax / 2];  // of pair i a position
};

enum : int { kNoCache = -1 };

// Sum over the LPR adjacent lanes of a row, in all of them.
template <int LPR>
MI_DEVICE float row_sum(float x) {
#pragma unroll
  for (int m = 1; m < LPR; m <<= 1) x += __shfl_xor(x, m, kWave);
  return x;
}

template <typename MT, int DST>
MI_DEVICE void norm_cache_store(uint8_t* row, float (&y)[8], const uint4& packed, float inv_scale, uint8_t* scale) {
  if constexpr (DST == MT::kDtype) {
    *(uint4*)row = packed;
  } else if constexpr (DST == MI_F32) {
    ((float4*)row)[0] = make_float4(y[0], y[1], y[2], y[3]);
    ((float4*)row)[1] = make_float4(y[4], y[5], y[6], y[7]);
  } else if constexpr (DST == MI_FP8_E4M3) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float z = y[i] * inv_scale;
      if (z == z) z = fminf(fmaxf(z, -448.f), 448.f);  // NaN stays NaN
      w[i >> 2] |= (uint32_t)f32_to_e4m3fn(z) << (8 * (i & 3));
    }
    *(uint2*)row = make_uint2(w[0], w[1]);
  } else if constexpr (DST == MI_MXFP8 || DST == MI_MXFP4) {
    uint32_t c[2];
    const uint32_t byte = mx_encode8<DST == MI_MXFP8 ? kKvMx8 : kKvMx4>(y, c);
    if constexpr (DST == MI_MXFP8) *(uint2*)row = make_uint2(c[0], c[1]);
    else *(uint32_t*)row = c[0];
    if ((threadIdx.x & 3) == 0) *scale = (uint8_t)byte;
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = DST == MI_BF16 ? f32_to_bf16_rne(y[2 * i]) : f32_to_f16_rne(y[2 * i]);
      const uint32_t hi = DST == MI_BF16 ? f32_to_bf16_rne(y[2 * i + 1]) : f32_to_f16_rne(y[2 * i + 1]);
      w[i] = lo | hi << 16;
    }
    *(uint4*)row = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Rows of a token: q heads, k heads and, with a cache, v heads.
template <typename MT, int DST, int LPR, bool INTERLEAVE>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRopeParams p) {
  constexpr int RPW = kWave / LPR;
  const int lane = lane_id(), sub = lane % LPR, slot_row = lane / LPR;
  const int per_token = (p.rows + RPW * p.steps - 1) / (RPW * p.steps);
  const int64_t unit = (int64_t)blockIdx.x * 4 + uniform((int)threadIdx.x >> 6);
  const int64_t t = unit / per_token;
  if (t >= p.num_tokens) return;
  const int row0 = (int)(unit - t * per_token) * RPW * p.steps;
  const int d0 = 8 * sub, hq = p.num_qo_heads, hkv = p.num_kv_heads;
  const bool in_row = d0 < p.head_dim, rot = d0 < p.rotary_dim;
  const int half = p.rotary_dim >> 1;
  // the lane that holds the other halves of this one's pairs, and whose elements they are
  const int other = INTERLEAVE || !rot ? 0 : d0 < half ? half / 8 : -(half / 8);

  // the token's cache row (K half, head 0)
  int64_t page = -1, slot = 0;
  if (DST != kNoCache && t < p.num_append) {
    const bool real = !p.num_tokens_device || t < *p.num_tokens_device;
    page = p.page_idx[t * p.idx_stride];
    slot = p.slot_idx[t * p.idx_stride];
    if (!real || page >= p.max_pages || slot < 0 || slot >= p.page_size) page = -1;
  }

  float wq[8], wk[8], wqo[8], wko[8];  // weights of this lane's elements and of the other halves
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = in_row ? d0 + e : 0, j = in_row ? d0 + 8 * other + e : 0;
    if (p.weight_f32) {
      wq[e] = ((const float*)p.q_weight)[i], wk[e] = ((const float*)p.k_weight)[i];
      wqo[e] = ((const float*)p.q_weight)[j], wko[e] = ((const float*)p.k_weight)[j];
    } else {
      wq[e] = MT::to_f32(((const uint16_t*)p.q_weight)[i]), wk[e] = MT::to_f32(((const uint16_t*)p.k_weight)[i]);
      wqo[e] = MT::to_f32(((const uint16_t*)p.q_weight)[j]), wko[e] = MT::to_f32(((const uint16_t*)p.k_weight)[j]);
    }
  }
  float c[8], s[8];  // of element e's pair; s with its sign in the element's sum
  {
    const double pos = p.pos_is_64 ? (double)((const int64_t*)p.pos)[t] : (double)((const int32_t*)p.pos)[t];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (INTERLEAVE && (e & 1)) continue;
      const int pair = !rot ? 0 : INTERLEAVE ? (d0 + e) >> 1 : d0 < half ? d0 + e : d0 + e - half;
      const double a = pos * p.turns[pair];
      const float x = (float)(a - rint(a));
      float sn, cs;
      sincospif(2.f * x, &sn, &cs);
      c[e] = cs;
      if constexpr (INTERLEAVE) {
        c[e + 1] = cs;
        s[e] = -sn;
        s[e + 1] = sn;
      } else {
        s[e] = d0 < half ? -sn : sn;
      }
    }
  }
  const float inv_dim = 1.f / (float)p.head_dim;

  for (int st = 0; st < p.steps; ++st) {
    const int r = row0 + st * RPW + slot_row;
    const bool live = r < p.rows && in_row, is_q = r < hq, is_v = r >= hq + hkv;
    const int h = is_q ? r : is_v ? r - hq - hkv : r - hq;
    uint16_t* src = nullptr;
    if (live)
      src = is_q   ? (uint16_t*)p.q + t * p.q_stride_tok + h * p.q_stride_head
            : is_v ? (uint16_t*)p.v + t * p.v_stride_tok + h * p.v_stride_head
                   : (uint16_t*)p.k + t * p.k_stride_tok + h * p.k_stride_head;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (live) u = *(const uint4*)(src + d0);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float y[8], sq = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = MT::to_f32((uint16_t)(w[i] & 0xffffu));
      y[2 * i + 1] = MT::to_f32((uint16_t)(w[i] >> 16));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sq += y[e] * y[e];
    const float rs = rsqrtf(row_sum<LPR>(sq) * inv_dim + p.eps);
    if constexpr (INTERLEAVE) {
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= rs * (is_q ? wq[e] : wk[e]);
        if (rot) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float a = y[e], b = y[e + 1];
            y[e] = a * c[e] + b * s[e];
            y[e + 1] = b * c[e] + a * s[e + 1];
          }
        }
      }
    } else {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = (uint32_t)__shfl((int)w[i], lane + other, kWave);
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint16_t b16 = (uint16_t)(e & 1 ? o[e >> 1] >> 16 : o[e >> 1] & 0xffffu);
          const float a = y[e] * (rs * (is_q ? wq[e] : wk[e])), b = MT::to_f32(b16) * (rs * (is_q ? wqo[e] : wko[e]));
          y[e] = rot ? a * c[e] + b * s[e] : a;
        }
      }
    }
    if (!live) continue;
    uint4 out = u;
    if (!is_v) {
      out = make_uint4(MT::pack2(y[0], y[1]), MT::pack2(y[2], y[3]), MT::pack2(y[4], y[5]), MT::pack2(y[6], y[7]));
      if (is_q || p.keep_k) *(uint4*)(src + d0) = out;
    }
    if constexpr (DST != kNoCache) {
      if (is_q || page < 0) continue;
      constexpr int ESZ = DST == MI_F32 ? 4 : DST == MI_BF16 || DST == MI_F16 ? 2 : 1;
      uint8_t* row = p.cache + (page * p.page_stride + slot * p.token_stride + (is_v ? p.kv_stride : 0) + h * p.head_stride +
                                (DST == MI_MXFP4 ? d0 >> 1 : d0)) * ESZ;
      float inv = 1.f;
      uint8_t* scale = nullptr;
      if constexpr (DST == MI_FP8_E4M3) inv = 1.f / ((const float*)(is_v ? p.v_scale : p.k_scale))[h];
      if constexpr (DST == MI_MXFP8 || DST == MI_MXFP4) {
        const int nblk = p.head_dim / kMxBlock;
        scale = (uint8_t*)(is_v ? p.v_scale : p.k_scale) + page * (2LL * hkv * nblk * p.page_size) +
                (int64_t)(h * nblk + d0 / kMxBlock) * p.page_size + slot;
      }
      norm_cache_store<MT, DST>(row, y, out, inv, scale);
    }
  }
}

template <typename MT, int DST, int LPR>
static void launch_norm_lpr(const NormRopeParams& p, dim3 grid, hipStream_t s) {
  if (p.interleave) hipLaunchKernelGGL((qk_norm_rope_kernel<MT, DST, LPR, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<MT, DST, LPR, false>), grid, dim3(256), 0, s, p);
}

template <typename MT, int DST>
static int launch_norm(NormRopeParams& p, hipStream_t s) {
  const int lanes = p.head_dim / 8, lpr = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
  const int rpw = kWave / lpr, most = (p.rows + rpw - 1) / rpw;
  // wavefronts for every place of the chip first, then more rows to one, which its angles serve
  const int64_t places = 16LL * device_cu_count();
  int64_t steps = (int64_t)p.num_tokens * most / places;
  p.steps = (int)(steps < 1 ? 1 : steps > most ? most : steps);
  const int64_t units = (int64_t)p.num_tokens * ((most + p.steps - 1) / p.steps), blocks = (units + 3) / 4;
  if (blocks > INT32_MAX) return MI_ERR_UNSUPPORTED;
  const dim3 grid((uint32_t)blocks);
  switch (lpr) {
    case 8: launch_norm_lpr<MT, DST, 8>(p, grid, s); break;
    case 16: launch_norm_lpr<MT, DST, 16>(p, grid, s); break;
    case 32: launch_norm_lpr<MT, DST, 32>(p, grid, s); break;
    default: launch_norm_lpr<MT, DST, 64>(p, grid, s); break;
  }
  return MI_OK;
}

template <typename MT>
static int launch_norm_dst(NormRopeParams& p, int dst, hipStream_t s) {
  switch (dst) {
    case kNoCache: return launch_norm<MT, kNoCache>(p, s);
    case MI_BF16: return launch_norm<MT, MI_BF16>(p, s);
    case MI_F16: return launch_norm<MT, MI_F16>(p, s);
    case MI_F32: return launch_norm<MT, MI_F32>(p, s);
    case MI_FP8_E4M3: return launch_norm<MT, MI_FP8_E4M3>(p, s);
    case MI_MXFP8: return launch_norm<MT, MI_MXFP8>(p, s);
    case MI_MXFP4: return launch_norm<MT, MI_MXFP4>(p, s);
    default: return MI_ERR_UNSUPPORTED;
  }
}

// Turns a position of each pair: theta^(-2i / rotary_dim) / scale / (2 pi), by one power and products.
static void norm_turns(NormRopeParams& p, double theta, double scale, bool llama31, double low, double high, double old) {
  const double two_pi = 6.283185307179586476925286766559;
  const double ratio = std::pow(theta, -2.0 / p.rotary_dim);
  double g = 1.0;
  for (int i = 0; i < p.rotary_dim / 2; ++i, g *= ratio) {
    double f = g / scale;
    if (llama31) {
      double smooth = (old * g / two_pi - low) / (high - low);
      smooth = smooth < 0.0 ? 0.0 : smooth > 1.0 ? 1.0 : smooth;
      f = (1.0 - smooth) * f + smooth * g;
    }
    p.turns[i] = f / two_pi;
  }
}

static bool rows_aligned_by8(const void* base, int64_t a, int64_t b) { return (uintptr_t)base % 16 == 0 && a % 8 == 0 && b % 8 == 0; }

}  // namespace mi

extern "C" int mi_qk_norm_rope(void* q, int64_t q_stride_token, int64_t q_stride_head, int32_t num_qo_heads, void* k,
                               int64_t k_stride_token, int64_t k_stride_head, int32_t num_kv_heads, const void* v,
                               int64_t v_stride_token, int64_t v_stride_head, int32_t dtype, int32_t head_dim,
                               const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps, int32_t keep_k,
                               const mi_paged_kv* kv, const int64_t* page_idx, const int64_t* slot_idx, int64_t idx_stride,
                               int32_t num_append_tokens, const int32_t* num_tokens_device, int32_t rotary_dim,
                               const void* pos_ids, int32_t pos_dtype, int32_t num_tokens, int32_t interleave,
                               float rope_scale, float rope_theta, int32_t llama31, float low_freq_factor,
                               float high_freq_factor, float old_context_len, void* stream) {
  using namespace mi;
  if (num_tokens < 0 || num_qo_heads < 0 || num_kv_heads < 0 || num_append_tokens < 0) return MI_ERR_INVALID;
  if (num_tokens == 0 || num_qo_heads + num_kv_heads == 0) return MI_OK;
  if (!pos_ids || (num_qo_heads > 0 && (!q || !q_weight)) || (num_kv_heads > 0 && (!k || !k_weight))) return MI_ERR_INVALID;
  if (dtype != MI_BF16 && dtype != MI_F16) return MI_ERR_UNSUPPORTED;
  if (weight_dtype != dtype && weight_dtype != MI_F32) return MI_ERR_UNSUPPORTED;
  if (pos_dtype != MI_I32 && pos_dtype != MI_I64) return MI_ERR_UNSUPPORTED;
  if (head_dim <= 0 || head_dim % 8 || head_dim > kNormDimMax) return MI_ERR_UNSUPPORTED;
  // a half-split rotation pairs whole 16-byte pieces
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % (interleave ? 8 : 16)) return MI_ERR_UNSUPPORTED;
  if (!(rope_scale > 0.f) || !(rope_theta > 0.f) || !(eps >= 0.f)) return MI_ERR_INVALID;
  if (llama31 && (!(high_freq_factor > low_freq_factor) || !(low_freq_factor > 0.f))) return MI_ERR_INVALID;
  if (num_qo_heads > 0 && !rows_aligned_by8(q, q_stride_token, q_stride_head)) return MI_ERR_INVALID;
  if (num_kv_heads > 0 && !rows_aligned_by8(k, k_stride_token, k_stride_head)) return MI_ERR_INVALID;
  NormRopeParams p{};
  int dst = kNoCache;
  if (kv) {
    dst = kv->dtype;
    if (dst != MI_BF16 && dst != MI_F16 && dst != MI_F32 && !kv_is_scaled(dst)) return MI_ERR_UNSUPPORTED;
    if (!kv->data || !v || !page_idx || !slot_idx || idx_stride <= 0 || kv->page_size <= 0) return MI_ERR_INVALID;
    if (kv->num_kv_heads != num_kv_heads || kv->head_dim != head_dim || num_append_tokens > num_tokens) return MI_ERR_INVALID;
    if (kv_is_mx(dst) && head_dim % kMxBlock) return MI_ERR_UNSUPPORTED;
    if (!rows_aligned_by8(v, v_stride_token, v_stride_head) || !kv_scales_ok(kv)) return MI_ERR_INVALID;
    const int esz = kv_elem_bytes(dst);
    if ((kv->page_stride | kv->kv_stride | kv->token_stride | kv->head_stride) % 8 || (uintptr_t)kv->data % (8 * esz))
      return MI_ERR_INVALID;
    if (kv_is_mx(dst) && !kv_aligned16(kv)) return MI_ERR_INVALID;
    p.cache = (uint8_t*)kv->data;
    p.page_stride = kv->page_stride;
    p.kv_stride = kv->kv_stride;
    p.token_stride = kv->token_stride;
    p.head_stride = kv->head_stride;
    p.max_pages = kv->max_pages;
    p.k_scale = (void*)kv->k_scale;
    p.v_scale = (void*)kv->v_scale;
    p.page_idx = page_idx;
    p.slot_idx = slot_idx;
    p.idx_stride = idx_stride;
    p.num_tokens_device = num_tokens_device;
    p.num_append = num_append_tokens;
    p.page_size = kv->page_size;
  }
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_stride_tok = q_stride_token;
  p.q_stride_head = q_stride_head;
  p.k_stride_tok = k_stride_token;
  p.k_stride_head = k_stride_head;
  p.v_stride_tok = v_stride_token;
  p.v_stride_head = v_stride_head;
  // a side without heads reads the other's weight, and uses none of it
  p.q_weight = num_qo_heads ? q_weight : k_weight;
  p.k_weight = num_kv_heads ? k_weight : q_weight;
  p.pos = pos_ids;
  p.pos_is_64 = pos_dtype == MI_I64;
  p.num_tokens = num_tokens;
  p.num_qo_heads = num_qo_heads;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.rotary_dim = rotary_dim;
  p.interleave = interleave ? 1 : 0;
  p.weight_f32 = weight_dtype == MI_F32;
  p.keep_k = keep_k ? 1 : 0;
  p.rows = num_qo_heads + (kv ? 2 : 1) * num_kv_heads;
  p.eps = eps;
  norm_turns(p, rope_theta, rope_scale, llama31 != 0, low_freq_factor, high_freq_factor, old_context_len);
  hipStream_t s = (hipStream_t)stream;
  const int st = dtype == MI_BF16 ? launch_norm_dst<BF16>(p, dst, s) : launch_norm_dst<F16>(p, dst, s);
  if (st != MI_OK) return st;
  MI_CHECK_LAUNCH();
  return MI_OK;
}
