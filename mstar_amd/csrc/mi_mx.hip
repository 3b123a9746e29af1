// The microscaled KV cache's own kernels: quantising rows as they are appended,
// and reading a batch's contexts back as values (which serves every cache format).
//
// Quantisation.  A block is 32 consecutive elements of one (token, kv-head) row of
// K or V.  Its exponent e is the least at which the largest magnitude a still
// rounds to a code: a <= T 2^e, T = 464 = 448 + half a step for e4m3, 7 = 6 + half
// a step for e2m1 (taking T = 448 or 6 would give up to twice the step to blocks
// just above it, taking the next power of two below would clip up to an eighth, a
// quarter, of a).  Codes are RNE(x 2^-e), formed by the hardware's scaled
// conversions.  e is held to at least -126 and at most 119 (e4m3) or 125 (e2m1), the
// highest at which every code is a finite float: a finite row reads as finite
// values, the largest magnitudes of its type as the largest code, and as fp16's
// largest value what is past it (f16_saturate).  Blocks of zeros have e = 0.  A block with a NaN or an infinity has scale byte 255 and reads as NaN
// throughout.
#include <type_traits>

#include "mi_internal.h"

namespace mi {

// ---------------------------------------------------------------- append
struct MxAppendParams {
  const void *k, *v;
  int64_t k_stride_tok, k_stride_head, v_stride_tok, v_stride_head;
  uint8_t* cache;
  int64_t page_stride, kv_stride, token_stride, head_stride, max_pages;
  uint8_t *k_scale, *v_scale;
  const int64_t* page_idx;
  const int64_t* slot_idx;
  int64_t idx_stride;
  const int32_t* num_tokens_device;
  int32_t num_tokens, num_kv_heads, head_dim, page_size;
};

template <int SRC>
MI_DEVICE void load8f(const void* base, int64_t off, float (&x)[8]) {
  if constexpr (SRC == MI_F32) {
    const float4 a = *(const float4*)((const float*)base + off), b = *(const float4*)((const float*)base + off + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 u = *(const uint4*)((const uint16_t*)base + off);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t lo = (uint16_t)(w[i] & 0xffffu), hi = (uint16_t)(w[i] >> 16);
      x[2 * i] = SRC == MI_BF16 ? bf16_to_f32(lo) : f16_to_f32(lo);
      x[2 * i + 1] = SRC == MI_BF16 ? bf16_to_f32(hi) : f16_to_f32(hi);
    }
  }
}

template <int KVT>
constexpr int kMxMaxExp = KVT == kKvMx8 ? 119 : 125;

// The scale byte of a block whose largest magnitude has these float bits.
template <int KVT>
MI_DEVICE uint32_t mx_scale_byte(uint32_t amax) {
  constexpr uint32_t kMantissa = KVT == kKvMx8 ? 0x680000u : 0x600000u;  // of T: 1.8125, 1.75
  constexpr int kExp = KVT == kKvMx8 ? 8 : 2;                            // T's exponent
  if (amax >= 0x7f800000u) return 255u;
  if (amax == 0) return 127u;
  // a subnormal a is below every 2^-126 T: it gets the least exponent
  const int e = (int)(amax >> 23) - kExp + ((amax & 0x7fffffu) > kMantissa ? 1 : 0);  // biased by 127
  return (uint32_t)min(max(e, 1), 127 + kMxMaxExp<KVT>);
}

// Eight elements of a block's four threads -> their codes and the block's scale byte.
template <int SRC, int KVT>
MI_DEVICE uint32_t mx_encode8(const void* src, int64_t off, uint32_t (&codes)[2]) {
  typedef __attribute__((ext_vector_type(2))) short s16x2;
  float x[8];
  load8f<SRC>(src, off, x);
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, bitcast<uint32_t>(x[i]) & 0x7fffffffu);  // floats order as ints, NaN on top
  a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0xb1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
  a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x4e, 0xf, 0xf, false));  // quad_perm [2,3,0,1]
  const uint32_t byte = mx_scale_byte<KVT>(a);
  const float scale = bitcast<float>(byte << 23);
  codes[0] = codes[1] = 0;
  if (byte == 255) return byte;
  if constexpr (KVT == kKvMx8) {
    if (byte == 127 + kMxMaxExp<KVT>) {  // the conversion gives NaN past 464 (e2m1's gives the largest code)
      const float top = 448.f * scale;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -top), top);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s16x2 w = {0, 0};
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i], x[4 * i + 1], scale, false);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i + 2], x[4 * i + 3], scale, true);
      codes[i] = bitcast<uint32_t>(w);
    }
  } else {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
    codes[0] = w;
  }
  return byte;
}

// One thread per 8 elements of a (token, kv-head), K then V; four adjacent
// threads share a block.
template <int SRC, int KVT>
__global__ __launch_bounds__(256) void mx_append_kernel(MxAppendParams p) {
  const int per_head = p.head_dim >> 3, per_token = p.num_kv_heads * per_head;
  const int64_t first = (int64_t)blockIdx.x * 256;
  const int t0 = (int)(first / per_token);  // uniform; the thread's own token by 32-bit arithmetic
  const int rest = (int)(first - (int64_t)t0 * per_token) + (int)threadIdx.x;
  const int i = t0 + rest / per_token;
  int n = p.num_tokens;
  if (p.num_tokens_device) n = min(n, *p.num_tokens_device);
  if (i >= n) return;
  const int rem = rest % per_token, hh = rem / per_head, d0 = (rem - hh * per_head) << 3;
  const int64_t page = p.page_idx[(int64_t)i * p.idx_stride];
  const int64_t slot = p.slot_idx[(int64_t)i * p.idx_stride];
  if (page < 0 || page >= p.max_pages || slot < 0 || slot >= p.page_size) return;
  uint8_t* row = p.cache + page * p.page_stride + slot * p.token_stride + hh * p.head_stride + (KVT == kKvMx8 ? d0 : d0 >> 1);
  const int nblk = p.head_dim / kMxBlock;
  const int64_t soff = page * (2LL * p.num_kv_heads * nblk * p.page_size) + (int64_t)(hh * nblk + d0 / kMxBlock) * p.page_size + slot;
  uint32_t kc[2], vc[2];
  const uint32_t ks = mx_encode8<SRC, KVT>(p.k, (int64_t)i * p.k_stride_tok + (int64_t)hh * p.k_stride_head + d0, kc);
  const uint32_t vs = mx_encode8<SRC, KVT>(p.v, (int64_t)i * p.v_stride_tok + (int64_t)hh * p.v_stride_head + d0, vc);
  if constexpr (KVT == kKvMx8) {
    *(uint2*)row = make_uint2(kc[0], kc[1]);
    *(uint2*)(row + p.kv_stride) = make_uint2(vc[0], vc[1]);
  } else {
    *(uint32_t*)row = kc[0];
    *(uint32_t*)(row + p.kv_stride) = vc[0];
  }
  if ((threadIdx.x & 3) == 0) {
    p.k_scale[soff] = (uint8_t)ks;
    p.v_scale[soff] = (uint8_t)vs;
  }
}

int mx_append_launch(const mi_paged_kv* kv, const void* k, const void* v, int32_t src_dtype, int64_t k_stride_token,
                     int64_t k_stride_head, int64_t v_stride_token, int64_t v_stride_head, const int64_t* page_idx,
                     const int64_t* slot_idx, int64_t idx_stride, int32_t num_tokens,
                     const int32_t* num_tokens_device, hipStream_t stream) {
  if (kv->head_dim % kMxBlock) return MI_ERR_UNSUPPORTED;
  if (!kv_scales_ok(kv) || !kv_aligned16(kv)) return MI_ERR_INVALID;
  const MxAppendParams p{k, v, k_stride_token, k_stride_head, v_stride_token, v_stride_head, (uint8_t*)kv->data,
                         kv->page_stride, kv->kv_stride, kv->token_stride, kv->head_stride, kv->max_pages,
                         (uint8_t*)kv->k_scale, (uint8_t*)kv->v_scale, page_idx, slot_idx, idx_stride, num_tokens_device,
                         num_tokens, kv->num_kv_heads, kv->head_dim, kv->page_size};
  const int64_t threads = (int64_t)num_tokens * kv->num_kv_heads * (kv->head_dim / 8), grid = (threads + 255) / 256;
  if (grid > INT32_MAX) return MI_ERR_UNSUPPORTED;
  const bool mx8 = kv->dtype == MI_MXFP8;
  const dim3 g((uint32_t)grid), b(256);
  switch (src_dtype) {
    case MI_BF16:
      if (mx8) hipLaunchKernelGGL((mx_append_kernel<MI_BF16, kKvMx8>), g, b, 0, stream, p);
      else hipLaunchKernelGGL((mx_append_kernel<MI_BF16, kKvMx4>), g, b, 0, stream, p);
      break;
    case MI_F16:
      if (mx8) hipLaunchKernelGGL((mx_append_kernel<MI_F16, kKvMx8>), g, b, 0, stream, p);
      else hipLaunchKernelGGL((mx_append_kernel<MI_F16, kKvMx4>), g, b, 0, stream, p);
      break;
    default:
      if (mx8) hipLaunchKernelGGL((mx_append_kernel<MI_F32, kKvMx8>), g, b, 0, stream, p);
      else hipLaunchKernelGGL((mx_append_kernel<MI_F32, kKvMx4>), g, b, 0, stream, p);
  }
  MI_CHECK_LAUNCH();
  return MI_OK;
}

// ------------------------------------------------------------------ read
struct ReadParams {
  const uint8_t* cache;
  int64_t page_stride, kv_stride, token_stride, head_stride, max_pages;
  const void *k_scale, *v_scale;
  const int32_t *kv_indptr, *kv_indices, *last_page_len;
  void *k_out, *v_out;
  int64_t out_tokens;
  int32_t batch, num_indices, num_kv_heads, head_dim, page_size, entries;
};

// Eight elements of a cached row as they lie in the pool, and its scale.
template <int CACHE>
struct Row8 {
  static constexpr int W = CACHE == MI_F32 ? 8 : CACHE == MI_BF16 || CACHE == MI_F16 ? 4 : CACHE == MI_MXFP4 ? 1 : 2;
  uint32_t w[W];
  float scale;  // fp8: the head's; microscaled: the block's
};

template <int CACHE>
MI_DEVICE void row8_load(Row8<CACHE>& r, const uint8_t* src, const void* scales, int64_t soff, int head) {
  if constexpr (Row8<CACHE>::W >= 4) {
#pragma unroll
    for (int i = 0; i < Row8<CACHE>::W; i += 4) {
      const uint4 u = ((const uint4*)src)[i / 4];
      r.w[i] = u.x, r.w[i + 1] = u.y, r.w[i + 2] = u.z, r.w[i + 3] = u.w;
    }
  } else if constexpr (Row8<CACHE>::W == 2) {
    const uint2 u = *(const uint2*)src;
    r.w[0] = u.x, r.w[1] = u.y;
  } else {
    r.w[0] = *(const uint32_t*)src;
  }
  if constexpr (CACHE == MI_MXFP8 || CACHE == MI_MXFP4) r.scale = bitcast<float>((uint32_t)((const uint8_t*)scales)[soff] << 23);
  if constexpr (CACHE == MI_FP8_E4M3) r.scale = ((const float*)scales)[head];
}

// Streamed out: the caller reads the values from memory later, and kept in the L2
// they push out what the other workgroups read (43 -> 29 us below).
MI_DEVICE void stream16(void* dst, const uint4& v) {
  __builtin_nontemporal_store(u32x4_t{v.x, v.y, v.z, v.w}, (u32x4_t*)dst);
}

template <int CACHE, int OUT>
MI_DEVICE void row8_store(const Row8<CACHE>& r, void* out, int64_t oo) {
  constexpr bool MX = CACHE == MI_MXFP8 || CACHE == MI_MXFP4;
  if constexpr (MX && OUT != MI_F32) {
    uint32_t o[4];
    constexpr int KVT = CACHE == MI_MXFP8 ? kKvMx8 : kKvMx4;
    mx_to_mt<std::conditional_t<OUT == MI_BF16, BF16, F16>, KVT>(r.w, r.scale, o);
    if constexpr (OUT == MI_F16)
      if (mx_past_f16<KVT>(bitcast<uint32_t>(r.scale) >> 23)) f16_saturate(o);
    stream16((uint16_t*)out + oo, make_uint4(o[0], o[1], o[2], o[3]));
  } else if constexpr (CACHE == OUT && OUT != MI_F32) {  // bit patterns kept
    stream16((uint16_t*)out + oo, make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]));
  } else {
    float x[8];
    if constexpr (CACHE == MI_MXFP8 || CACHE == MI_FP8_E4M3) {
      const float s = MX ? r.scale : 1.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(r.w[i], s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(r.w[i], s, true);
        x[4 * i] = a[0], x[4 * i + 1] = a[1], x[4 * i + 2] = b[0], x[4 * i + 3] = b[1];
      }
      if constexpr (!MX)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= r.scale;
    } else if constexpr (CACHE == MI_MXFP4) {
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.w[0], r.scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.w[0], r.scale, 1);
      const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.w[0], r.scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.w[0], r.scale, 3);
      x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1], x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
    } else if constexpr (CACHE == MI_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = bitcast<float>(r.w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t e = (uint16_t)(r.w[i / 2] >> (16 * (i & 1)));
        x[i] = CACHE == MI_BF16 ? bf16_to_f32(e) : f16_to_f32(e);
      }
    }
    if constexpr (OUT == MI_F32) {
      float* o = (float*)out + oo;
      stream16(o, bitcast<uint4>(make_float4(x[0], x[1], x[2], x[3])));
      stream16(o + 4, bitcast<uint4>(make_float4(x[4], x[5], x[6], x[7])));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = OUT == MI_BF16 ? f32_to_bf16_rne(x[2 * i]) : f32_to_f16_rne(x[2 * i]);
        const uint32_t hi = OUT == MI_BF16 ? f32_to_bf16_rne(x[2 * i + 1]) : f32_to_f16_rne(x[2 * i + 1]);
        w[i] = lo | hi << 16;
      }
      stream16((uint16_t*)out + oo, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
}

MI_DEVICE int request_len(const ReadParams& p, int b) {
  const int np = p.kv_indptr[b + 1] - p.kv_indptr[b];
  return np > 0 ? (np - 1) * p.page_size + p.last_page_len[b] : 0;
}

constexpr int kReadUnroll = 2;

// A workgroup reads a share (blockIdx.y of gridDim.y) of the elements of `entries`
// consecutive entries of the page list.  Where the first one's request begins in
// the output is a sum over the requests before it, which the workgroup's threads
// add up from the index arrays: no plan, no launch for a prefix sum.  A thread's U
// loads of K and V are in flight together.  HBM bound: 68k tokens at 4 kv heads x 128
// in 4 bits 29 us (175 MB, 6.0 TB/s); 2000 tokens at 8 x 128 in 8 bits 5.0 us (9.2
// with a page to a workgroup, 6.4 with four loads a thread).
template <int CACHE, int OUT>
__global__ __launch_bounds__(256) void read_kv_kernel(ReadParams p) {
  constexpr int ESZ = CACHE == MI_F32 ? 4 : CACHE == MI_BF16 || CACHE == MI_F16 ? 2 : 1, U = kReadUnroll;
  __shared__ int64_t s_sum[4];
  __shared__ int s_cnt[4];
  const int tid = (int)threadIdx.x, end = min(p.kv_indptr[p.batch], p.num_indices);
  const int e0 = (int)blockIdx.x * p.entries, e1 = min(e0 + p.entries, end);
  if (e0 >= e1) return;
  int64_t tokens = 0;
  int before = 0;  // requests whose pages end at or before e0
  for (int b = tid; b < p.batch; b += 256)
    if (p.kv_indptr[b + 1] <= e0) {
      tokens += request_len(p, b);
      ++before;
    }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    tokens += __shfl_xor(tokens, m, kWave);
    before += __shfl_xor(before, m, kWave);
  }
  if ((tid & 63) == 0) {
    s_sum[tid >> 6] = tokens;
    s_cnt[tid >> 6] = before;
  }
  __syncthreads();
  tokens = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  int r = uniform(s_cnt[0] + s_cnt[1] + s_cnt[2] + s_cnt[3]);
  const int per_head = p.head_dim >> 3, per_token = p.num_kv_heads * per_head, nblk = p.head_dim / kMxBlock;
  for (int e = e0; e < e1; ++e) {
    while (r < p.batch - 1 && p.kv_indptr[r + 1] <= e) tokens += request_len(p, r++);
    const int first = p.kv_indptr[r];
    const int64_t at = tokens + (int64_t)(e - first) * p.page_size;
    const int64_t left = p.out_tokens - at;
    if (left <= 0) return;
    if (at < 0) continue;  // entries before the first request's
    int slots = e == p.kv_indptr[r + 1] - 1 ? min(p.last_page_len[r], p.page_size) : p.page_size;
    if (slots > left) slots = (int)left;
    const int64_t page = p.kv_indices[e];
    if (page < 0 || page >= p.max_pages) continue;
    const int n = slots * per_token;
    for (int j0 = (int)blockIdx.y * 256 * U; j0 < n; j0 += (int)gridDim.y * 256 * U) {
      Row8<CACHE> k[U], v[U];
      int64_t oo[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + 256 * u + tid;
        if (j >= n) continue;
        const int slot = j / per_token, rem = j - slot * per_token, h = rem / per_head, d0 = (rem - h * per_head) << 3;
        const int64_t el = CACHE == MI_MXFP4 ? d0 >> 1 : d0;
        const uint8_t* src = p.cache + (page * p.page_stride + slot * p.token_stride + h * p.head_stride + el) * ESZ;
        const int64_t so = (page * 2 * p.num_kv_heads + h) * nblk * (int64_t)p.page_size + (int64_t)(d0 / kMxBlock) * p.page_size + slot;
        oo[u] = (at + slot) * ((int64_t)p.num_kv_heads * p.head_dim) + (int64_t)h * p.head_dim + d0;
        row8_load(k[u], src, p.k_scale, so, h);
        row8_load(v[u], src + p.kv_stride * ESZ, p.v_scale, so, h);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j0 + 256 * u + tid >= n) continue;
        row8_store<CACHE, OUT>(k[u], p.k_out, oo[u]);
        row8_store<CACHE, OUT>(v[u], p.v_out, oo[u]);
      }
    }
  }
}

template <int CACHE>
static int launch_read(const ReadParams& p, int out_dtype, dim3 grid, hipStream_t stream) {
  switch (out_dtype) {
    case MI_BF16: hipLaunchKernelGGL((read_kv_kernel<CACHE, MI_BF16>), grid, dim3(256), 0, stream, p); break;
    case MI_F16: hipLaunchKernelGGL((read_kv_kernel<CACHE, MI_F16>), grid, dim3(256), 0, stream, p); break;
    case MI_F32: hipLaunchKernelGGL((read_kv_kernel<CACHE, MI_F32>), grid, dim3(256), 0, stream, p); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

}  // namespace mi

extern "C" int mi_kv_read(const mi_paged_kv* kv, const int32_t* kv_indptr, const int32_t* kv_indices,
                          const int32_t* last_page_len, int32_t batch, int32_t num_indices, void* k_out, void* v_out,
                          int32_t out_dtype, int64_t out_tokens, void* stream) {
  using namespace mi;
  if (!kv || batch < 0 || num_indices < 0 || out_tokens < 0) return MI_ERR_INVALID;
  if (batch == 0 || num_indices == 0 || out_tokens == 0) return MI_OK;
  if (!kv->data || !kv_indptr || !kv_indices || !last_page_len || !k_out || !v_out) return MI_ERR_INVALID;
  if (kv->num_kv_heads <= 0 || kv->head_dim <= 0 || kv->page_size <= 0) return MI_ERR_INVALID;
  if (kv->head_dim % 8 || (kv_is_mx(kv->dtype) && kv->head_dim % kMxBlock)) return MI_ERR_UNSUPPORTED;
  if ((int64_t)kv->page_size * kv->num_kv_heads * kv->head_dim > INT32_MAX) return MI_ERR_UNSUPPORTED;
  if (!kv_scales_ok(kv) || !kv_aligned16(kv)) return MI_ERR_INVALID;
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return MI_ERR_INVALID;
  ReadParams p{(const uint8_t*)kv->data, kv->page_stride, kv->kv_stride, kv->token_stride, kv->head_stride, kv->max_pages,
               kv->k_scale, kv->v_scale, kv_indptr, kv_indices, last_page_len, k_out, v_out, out_tokens,
               batch, num_indices, kv->num_kv_heads, kv->head_dim, kv->page_size, 1};
  // about eight workgroups a CU: several pages each, or a share of a page's
  // elements (no less than what its threads load at once)
  const int64_t places = 8LL * device_cu_count(), once = 256 * kReadUnroll;
  const int64_t shares = ((int64_t)kv->page_size * kv->num_kv_heads * (kv->head_dim / 8) + once - 1) / once;
  p.entries = (int)((num_indices + places - 1) / places);
  const int64_t want = p.entries > 1 ? 1 : places / num_indices;
  const dim3 grid((num_indices + p.entries - 1) / p.entries, (uint32_t)(want < 1 ? 1 : want < shares ? want : shares));
  hipStream_t s = (hipStream_t)stream;
  int st;
  switch (kv->dtype) {
    case MI_BF16: st = launch_read<MI_BF16>(p, out_dtype, grid, s); break;
    case MI_F16: st = launch_read<MI_F16>(p, out_dtype, grid, s); break;
    case MI_F32: st = launch_read<MI_F32>(p, out_dtype, grid, s); break;
    case MI_FP8_E4M3: st = launch_read<MI_FP8_E4M3>(p, out_dtype, grid, s); break;
    case MI_MXFP8: st = launch_read<MI_MXFP8>(p, out_dtype, grid, s); break;
    case MI_MXFP4: st = launch_read<MI_MXFP4>(p, out_dtype, grid, s); break;
    default: return MI_ERR_UNSUPPORTED;
  }
  if (st != MI_OK) return st;
  MI_CHECK_LAUNCH();
  return MI_OK;
}
