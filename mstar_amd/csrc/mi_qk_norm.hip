// Norms of q and k head by head, with the rotation and the paged append in the same pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w      over the head_dim elements of a (token, head) row of q or k
//   rotated as mi_rope_apply rotates, by the angle pos * f_i
//   q (and k, if kept) in place; k and v to their cache slots
//
// The row's sum, the norm and the rotation are fp32, and a value is rounded once: to the
// q / k type, and from fp32 to the cache's type.  Angles are formed in turns in 64 bits, pos *
// f_i / (2 pi) less its nearest whole number, which is exact enough at any position (an fp32 angle is off
// by 4e-3 rad at 65k tokens, half a step of bf16 and four of fp16).
//
// A row is head_dim / 8 lanes (rounded up to a power of two, 16-byte loads), so a wavefront
// holds 64 / LPR rows of one token.  Its lanes form each pair's (cos, sin) once, a pair a lane, and share them
// through LDS for all the rows that the wavefront goes through; with the weights they become two
// factors an element, y = rs (x own + x' off), x' the pair's other element: a shuffle of 16 bytes.
//
// HBM bound: 22891 tokens of 28 + 2 x 4 heads x 128, bf16, 97 us, 4.4 TB/s of the 5.0 that a copy reaches (133 with
// every row's angles formed by its own lanes).  One token: 4.1 us, a few loads one after the other.
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
  int32_t num_tokens, num_append, num_qo_heads, num_kv_heads, head_dim, page_size, rotary_dim, pos_is_64;
  int32_t weight_f32, keep_k, parts, part_steps, items;  // items: of a token and a part of its steps
  float eps;
  // turns a position of pair i: g = 2^(i step); g / scale, or blended with g by smooth = slope g - bias
  double step, inv_scale, slope, bias;
  int32_t llama31;
};

enum : int { kNoCache = -1 };

template <int CTRL>
MI_DEVICE float dpp_add(float x) {
  return x + bitcast<float>((uint32_t)__builtin_amdgcn_update_dpp(0, (int)bitcast<uint32_t>(x), CTRL, 0xf, 0xf, false));
}
// Sum over the LPR adjacent lanes of a row, in all of them.
template <int LPR>
MI_DEVICE float row_sum(float x) {
  x = dpp_add<0xb1>(x);                        // quad_perm [1,0,3,2]
  x = dpp_add<0x4e>(x);                        // quad_perm [2,3,0,1]
  x = dpp_add<0x141>(x);                       // row_half_mirror
  if constexpr (LPR >= 16) x = dpp_add<0x140>(x);  // row_mirror
  if constexpr (LPR >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(x), bitcast<uint32_t>(x), false, false);
    x = bitcast<float>((uint32_t)a[0]) + bitcast<float>((uint32_t)a[1]);
  }
  if constexpr (LPR >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(x), bitcast<uint32_t>(x), false, false);
    x = bitcast<float>((uint32_t)a[0]) + bitcast<float>((uint32_t)a[1]);
  }
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

MI_DEVICE void read8(const float* src, float (&x)[8]) {
  const float4 a = ((const float4*)src)[0], b = ((const float4*)src)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// Of a step's rows: 0 q, 1 k, 2 v.
MI_DEVICE int kind_of(int st, int nq, int nk) { return st < nq ? 0 : st < nq + nk ? 1 : 2; }
// Element d0 of the row of head first + slot_row.
MI_DEVICE uint16_t* norm_row(const NormRopeParams& p, int kind, int64_t t, int first, int slot_row, int d0) {
  uint16_t* base = (uint16_t*)(kind == 0 ? p.q : kind == 1 ? p.k : const_cast<void*>(p.v));
  const int64_t tok = kind == 0 ? p.q_stride_tok : kind == 1 ? p.k_stride_tok : p.v_stride_tok;
  const int64_t head = kind == 0 ? p.q_stride_head : kind == 1 ? p.k_stride_head : p.v_stride_head;
  return base + (t * tok + first * head) + (slot_row * head + d0);
}

// A token's steps: its q heads, RPW at a time, then its k heads and, with a cache, its v heads.
template <typename MT, int DST, int LPR, bool INTERLEAVE>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRopeParams p) {
  constexpr int RPW = kWave / LPR, DIM = 8 * LPR, NP = (DIM / 2 + kWave - 1) / kWave, U = 4;
  __shared__ __attribute__((aligned(16))) float s_w[2][DIM];             // of q, of k
  __shared__ __attribute__((aligned(16))) float s_cos[4][DIM / 2], s_sin[4][DIM / 2];
  const int tid = (int)threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6), sub = lane % LPR, slot_row = lane / LPR;
  const int d0 = 8 * sub, hq = p.num_qo_heads, hkv = p.num_kv_heads, half = p.rotary_dim >> 1;
  const bool in_row = d0 < p.head_dim, rot = d0 < p.rotary_dim;
  // the lane that holds the other halves of this one's pairs
  const int other = INTERLEAVE || !rot ? 0 : d0 < half ? half / 8 : -(half / 8);
  const int nq = (hq + RPW - 1) / RPW, nk = (hkv + RPW - 1) / RPW, total = nq + (DST == kNoCache ? 1 : 2) * nk;
  for (int i = tid; i < 2 * DIM; i += 256) {
    const int d = i % DIM;
    const void* w = i < DIM ? p.q_weight : p.k_weight;
    s_w[0][i] = d >= p.head_dim ? 0.f : p.weight_f32 ? ((const float*)w)[d] : MT::to_f32(((const uint16_t*)w)[d]);
  }
  double turns[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const double g = exp2((double)(lane + kWave * j) * p.step);
    double f = g * p.inv_scale;
    if (p.llama31) {
      const double smooth = fmin(fmax(g * p.slope - p.bias, 0.0), 1.0);
      f = (1.0 - smooth) * f + smooth * g;
    }
    turns[j] = f * 0.15915494309189533577;
  }
  __syncthreads();
  const float inv_dim = 1.f / (float)p.head_dim;

  for (int item = (int)blockIdx.x * 4 + wave; item < p.items; item += (int)gridDim.x * 4) {
    const int token = p.parts == 1 ? item : (int)((unsigned)item / (unsigned)p.parts), s0 = (item - token * p.parts) * p.part_steps;
    const int s1 = min(s0 + p.part_steps, total);
    const int64_t t = token;
    auto load = [&](int st) {
      const int kind = kind_of(st, nq, nk), first = RPW * (st - (kind == 0 ? 0 : kind == 1 ? nq : nq + nk));
      const bool live = in_row && first + slot_row < (kind == 0 ? hq : hkv);
      return live ? *(const uint4*)norm_row(p, kind, t, first, slot_row, d0) : make_uint4(0, 0, 0, 0);
    };
    uint4 u[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (s0 + i < s1) u[i] = load(s0 + i);

    // the token's cache row (K half, head 0)
    int64_t page = -1, slot = 0;
    if (DST != kNoCache && s1 > nq && token < p.num_append) {
      const bool real = !p.num_tokens_device || token < *p.num_tokens_device;
      page = p.page_idx[t * p.idx_stride];
      slot = p.slot_idx[t * p.idx_stride];
      if (!real || page >= p.max_pages || slot < 0 || slot >= p.page_size) page = -1;
    }
    // every pair's cosine and sine once, to the wavefront's part of LDS
    if (s0 < nq + nk) {
      const double pos = p.pos_is_64 ? (double)((const int64_t*)p.pos)[t] : (double)((const int32_t*)p.pos)[t];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int pair = lane + kWave * j;
        if (pair < half) {
          const double a = pos * turns[j];
          float sn, cs;
          sincospif(2.f * (float)(a - rint(a)), &sn, &cs);
          s_cos[wave][pair] = cs;
          s_sin[wave][pair] = sn;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    float own[8], off[8];  // an element's factor in its own sum, and its partner's
    int kind = -1;
    auto factors = [&](int which) {
      read8(&s_w[which][d0], own);
      read8(&s_w[which][d0 + 8 * other], off);
      if (!rot) {
#pragma unroll
        for (int e = 0; e < 8; ++e) off[e] = 0.f;
        return;
      }
      if constexpr (INTERLEAVE) {
        const float4 c = *(const float4*)&s_cos[wave][d0 / 2], s = *(const float4*)&s_sin[wave][d0 / 2];
        const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          off[e] = -own[e + 1] * sn[e / 2];
          off[e + 1] = own[e] * sn[e / 2];
          own[e] *= cs[e / 2];
          own[e + 1] *= cs[e / 2];
        }
      } else {
        const int at = d0 < half ? d0 : d0 - half;
        float cs[8], sn[8];
        read8(&s_cos[wave][at], cs);
        read8(&s_sin[wave][at], sn);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          own[e] *= cs[e];
          off[e] *= d0 < half ? -sn[e] : sn[e];
        }
      }
    };
    auto process = [&](const uint4& in, int st) {
      const int now = kind_of(st, nq, nk), first = RPW * (st - (now == 0 ? 0 : now == 1 ? nq : nq + nk)), h = first + slot_row;
      const bool live = in_row && h < (now == 0 ? hq : hkv);
      if (now != kind && now < 2) factors(now);
      kind = now;
      const uint32_t w[4] = {in.x, in.y, in.z, in.w};
      float y[8];
      uint4 out = in;
      if (now < 2 || DST != MT::kDtype) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[2 * i] = MT::to_f32((uint16_t)(w[i] & 0xffffu));
          y[2 * i + 1] = MT::to_f32((uint16_t)(w[i] >> 16));
        }
      }
      if (now < 2) {
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sq = fmaf(y[e], y[e], sq);
        const float rs = rsqrtf(row_sum<LPR>(sq) * inv_dim + p.eps);
        if constexpr (INTERLEAVE) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float a = y[e], b = y[e + 1];
            y[e] = rs * (a * own[e] + b * off[e]);
            y[e + 1] = rs * (b * own[e + 1] + a * off[e + 1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t o = (uint32_t)__shfl((int)w[i], lane + other, kWave);
            y[2 * i] = rs * (y[2 * i] * own[2 * i] + MT::to_f32((uint16_t)(o & 0xffffu)) * off[2 * i]);
            y[2 * i + 1] = rs * (y[2 * i + 1] * own[2 * i + 1] + MT::to_f32((uint16_t)(o >> 16)) * off[2 * i + 1]);
          }
        }
        out = make_uint4(MT::pack2(y[0], y[1]), MT::pack2(y[2], y[3]), MT::pack2(y[4], y[5]), MT::pack2(y[6], y[7]));
        if (live && (now == 0 || p.keep_k)) *(uint4*)norm_row(p, now, t, first, slot_row, d0) = out;
      }
      if constexpr (DST != kNoCache) {
        if (now == 0 || page < 0 || !live) return;
        constexpr int ESZ = DST == MI_F32 ? 4 : DST == MI_BF16 || DST == MI_F16 ? 2 : 1;
        const bool is_v = now == 2;
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
    };
    for (int s = s0; s < s1; s += U) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (s + i >= s1) break;
        process(u[i], s + i);
        if (s + i + U < s1) u[i] = load(s + i + U);
      }
    }
  }
}

template <typename MT, int DST, int LPR>
static void launch_norm_lpr(const NormRopeParams& p, bool interleave, dim3 grid, hipStream_t s) {
  if (interleave) hipLaunchKernelGGL((qk_norm_rope_kernel<MT, DST, LPR, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<MT, DST, LPR, false>), grid, dim3(256), 0, s, p);
}

template <typename MT, int DST>
static int launch_norm(NormRopeParams& p, bool interleave, hipStream_t s) {
  const int lanes = p.head_dim / 8, lpr = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64, rpw = kWave / lpr;
  const int total = (p.num_qo_heads + rpw - 1) / rpw + (DST == kNoCache ? 1 : 2) * ((p.num_kv_heads + rpw - 1) / rpw);
  // wavefronts for every place of the chip first, then more steps to one, which its angles serve
  const int64_t places = 16LL * device_cu_count();
  const int64_t want = (places + p.num_tokens - 1) / p.num_tokens;
  p.part_steps = want >= total ? 1 : (int)((total + want - 1) / want);
  p.parts = (total + p.part_steps - 1) / p.part_steps;
  p.items = p.num_tokens * p.parts;  // parts > 1 only for fewer tokens than places
  const int64_t blocks = (p.items + 3LL) / 4, most = 8LL * device_cu_count();
  const dim3 grid((uint32_t)(blocks < most ? blocks : most));
  switch (lpr) {
    case 8: launch_norm_lpr<MT, DST, 8>(p, interleave, grid, s); break;
    case 16: launch_norm_lpr<MT, DST, 16>(p, interleave, grid, s); break;
    case 32: launch_norm_lpr<MT, DST, 32>(p, interleave, grid, s); break;
    default: launch_norm_lpr<MT, DST, 64>(p, interleave, grid, s); break;
  }
  return MI_OK;
}

template <typename MT>
static int launch_norm_dst(NormRopeParams& p, int dst, bool interleave, hipStream_t s) {
  switch (dst) {
    case kNoCache: return launch_norm<MT, kNoCache>(p, interleave, s);
    case MI_BF16: return launch_norm<MT, MI_BF16>(p, interleave, s);
    case MI_F16: return launch_norm<MT, MI_F16>(p, interleave, s);
    case MI_F32: return launch_norm<MT, MI_F32>(p, interleave, s);
    case MI_FP8_E4M3: return launch_norm<MT, MI_FP8_E4M3>(p, interleave, s);
    case MI_MXFP8: return launch_norm<MT, MI_MXFP8>(p, interleave, s);
    case MI_MXFP4: return launch_norm<MT, MI_MXFP4>(p, interleave, s);
    default: return MI_ERR_UNSUPPORTED;
  }
}

static bool rows_aligned_by8(const void* base, int64_t a, int64_t b) { return (uintptr_t)base % 16 == 0 && a % 8 == 0 && b % 8 == 0; }

}  // namespace mi

extern "C" int mi_qk_norm_rope_block(const mi_qk_norm_rope_args* args) {
  using namespace mi;
  if (!args) return MI_ERR_INVALID;
  const mi_qk_norm_rope_args& a = *args;
  if (a.num_tokens < 0 || a.num_qo_heads < 0 || a.num_kv_heads < 0 || a.num_append_tokens < 0) return MI_ERR_INVALID;
  if (a.num_tokens == 0 || a.num_qo_heads + a.num_kv_heads == 0) return MI_OK;
  if (!a.pos_ids || (a.num_qo_heads > 0 && (!a.q || !a.q_weight)) || (a.num_kv_heads > 0 && (!a.k || !a.k_weight))) return MI_ERR_INVALID;
  if (a.num_tokens > INT32_MAX - (1 << 20)) return MI_ERR_UNSUPPORTED;  // a grid's stride past the last one is still an int
  if (a.dtype != MI_BF16 && a.dtype != MI_F16) return MI_ERR_UNSUPPORTED;
  if (a.weight_dtype != a.dtype && a.weight_dtype != MI_F32) return MI_ERR_UNSUPPORTED;
  if (a.pos_dtype != MI_I32 && a.pos_dtype != MI_I64) return MI_ERR_UNSUPPORTED;
  if (a.head_dim <= 0 || a.head_dim % 8 || a.head_dim > kNormDimMax) return MI_ERR_UNSUPPORTED;
  // a half-split rotation pairs whole 16-byte pieces
  if (a.rotary_dim <= 0 || a.rotary_dim > a.head_dim || a.rotary_dim % (a.interleave ? 8 : 16)) return MI_ERR_UNSUPPORTED;
  if (!(a.rope_scale > 0.f) || !(a.rope_theta > 0.f) || !(a.eps >= 0.f)) return MI_ERR_INVALID;
  if (a.llama31 && (!(a.high_freq_factor > a.low_freq_factor) || !(a.low_freq_factor > 0.f))) return MI_ERR_INVALID;
  if (a.num_qo_heads > 0 && !rows_aligned_by8(a.q, a.q_stride_token, a.q_stride_head)) return MI_ERR_INVALID;
  if (a.num_kv_heads > 0 && !rows_aligned_by8(a.k, a.k_stride_token, a.k_stride_head)) return MI_ERR_INVALID;
  NormRopeParams p{};
  int dst = kNoCache;
  if (a.kv) {
    dst = a.kv->dtype;
    if (dst != MI_BF16 && dst != MI_F16 && dst != MI_F32 && !kv_is_scaled(dst)) return MI_ERR_UNSUPPORTED;
    if (!a.kv->data || !a.v || !a.page_idx || !a.slot_idx || a.idx_stride <= 0 || a.kv->page_size <= 0) return MI_ERR_INVALID;
    if (a.kv->num_kv_heads != a.num_kv_heads || a.kv->head_dim != a.head_dim || a.num_append_tokens > a.num_tokens) return MI_ERR_INVALID;
    if (kv_is_mx(dst) && a.head_dim % kMxBlock) return MI_ERR_UNSUPPORTED;
    if (!rows_aligned_by8(a.v, a.v_stride_token, a.v_stride_head) || !kv_scales_ok(a.kv)) return MI_ERR_INVALID;
    const int esz = kv_elem_bytes(dst);
    if ((a.kv->page_stride | a.kv->kv_stride | a.kv->token_stride | a.kv->head_stride) % 8 || (uintptr_t)a.kv->data % (8 * esz))
      return MI_ERR_INVALID;
    if (kv_is_mx(dst) && !kv_aligned16(a.kv)) return MI_ERR_INVALID;
    p.cache = (uint8_t*)a.kv->data;
    p.page_stride = a.kv->page_stride;
    p.kv_stride = a.kv->kv_stride;
    p.token_stride = a.kv->token_stride;
    p.head_stride = a.kv->head_stride;
    p.max_pages = a.kv->max_pages;
    p.k_scale = (void*)a.kv->k_scale;
    p.v_scale = (void*)a.kv->v_scale;
    p.page_idx = a.page_idx;
    p.slot_idx = a.slot_idx;
    p.idx_stride = a.idx_stride;
    p.num_tokens_device = a.num_tokens_device;
    p.num_append = a.num_append_tokens;
    p.page_size = a.kv->page_size;
  }
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.q_stride_tok = a.q_stride_token;
  p.q_stride_head = a.q_stride_head;
  p.k_stride_tok = a.k_stride_token;
  p.k_stride_head = a.k_stride_head;
  p.v_stride_tok = a.v_stride_token;
  p.v_stride_head = a.v_stride_head;
  // a side without heads reads the other's weight, and uses none of it
  p.q_weight = a.num_qo_heads ? a.q_weight : a.k_weight;
  p.k_weight = a.num_kv_heads ? a.k_weight : a.q_weight;
  p.pos = a.pos_ids;
  p.pos_is_64 = a.pos_dtype == MI_I64;
  p.num_tokens = a.num_tokens;
  p.num_qo_heads = a.num_qo_heads;
  p.num_kv_heads = a.num_kv_heads;
  p.head_dim = a.head_dim;
  p.rotary_dim = a.rotary_dim;
  p.weight_f32 = a.weight_dtype == MI_F32;
  p.keep_k = a.keep_k ? 1 : 0;
  p.eps = a.eps;
  const double two_pi = 6.283185307179586476925286766559, span = (double)a.high_freq_factor - (double)a.low_freq_factor;
  p.step = -2.0 / a.rotary_dim * std::log2((double)a.rope_theta);
  p.inv_scale = 1.0 / (double)a.rope_scale;
  p.llama31 = a.llama31 ? 1 : 0;
  p.slope = a.llama31 ? (double)a.old_context_len / two_pi / span : 0.0;
  p.bias = a.llama31 ? (double)a.low_freq_factor / span : 0.0;
  hipStream_t s = (hipStream_t)a.stream;
  const int st = a.dtype == MI_BF16 ? launch_norm_dst<BF16>(p, dst, a.interleave != 0, s) : launch_norm_dst<F16>(p, dst, a.interleave != 0, s);
  if (st != MI_OK) return st;
  MI_CHECK_LAUNCH();
  return MI_OK;
}

extern "C" int mi_qk_norm_rope(void* q, int64_t q_stride_token, int64_t q_stride_head, int32_t num_qo_heads, void* k,
                               int64_t k_stride_token, int64_t k_stride_head, int32_t num_kv_heads, const void* v,
                               int64_t v_stride_token, int64_t v_stride_head, int32_t dtype, int32_t head_dim,
                               const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps, int32_t keep_k,
                               const mi_paged_kv* kv, const int64_t* page_idx, const int64_t* slot_idx, int64_t idx_stride,
                               int32_t num_append_tokens, const int32_t* num_tokens_device, int32_t rotary_dim,
                               const void* pos_ids, int32_t pos_dtype, int32_t num_tokens, int32_t interleave,
                               float rope_scale, float rope_theta, int32_t llama31, float low_freq_factor,
                               float high_freq_factor, float old_context_len, void* stream) {
  const mi_qk_norm_rope_args args = {
      q, k, v, q_weight, k_weight, pos_ids, kv, page_idx, slot_idx, num_tokens_device, stream, q_stride_token, q_stride_head,
      k_stride_token, k_stride_head, v_stride_token, v_stride_head, idx_stride, num_qo_heads, num_kv_heads, dtype, head_dim,
      weight_dtype, keep_k, num_append_tokens, rotary_dim, pos_dtype, num_tokens, interleave, llama31, eps, rope_scale,
      rope_theta, low_freq_factor, high_freq_factor, old_context_len};
  return mi_qk_norm_rope_block(&args);
}
