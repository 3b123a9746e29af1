// Attention weights of cached tokens, accumulated (mi_attention_weights).
//
//   w[t, h] += sum over queries i and q heads g of kv head h of  exp(s_igt - lse_ig),
//   s_igt = sm_scale q_ig . k_th,   lse_ig = log sum_t exp(s_igt)  over the keys that query i sees,
//
// beginning at zero for the step's own tokens (the last qo_len of a request).  The
// sum needs every row's lse first, so the keys are gone through twice:
//
// * Requests of at most 16 rows (qo_len x group; decode): K is what costs, so it is read once. The first
//   launch writes the scores (group x 4 bytes a token and kv head, beside a row of K of 64 to 512 bytes) and
//   a log-sum-exp for each run of pages; the second joins those and sums the exponentials.  256 requests over
//   1.93M tokens, 4 heads x 128, bf16: 437 + 65 us.  K alone takes 320; any writing beside it brings reads and
//   writes together to a copy's 5 TB/s (a quarter of the scores: 399).  Small batches take one launch instead.
// * Longer ones: the products are what costs, and are done twice; a launch goes by rows with the
//   keys streaming past (lse), one by keys with the rows streaming past (sums).  4 chunks of 512 to 2048 tokens
//   over 22k, 28 / 4 heads x 128: 203 + 200 us (199 to 207, 196 to 200 by machine), 130 GFLOP each.
//
// Every sum has one order, from the index arrays and shapes alone: the same call gives the same bits.
// Work is found from the index arrays (unit_request): no plan is read, and any plan's workspace
// stays as it is.
#include "mi_weights_kernel.h"

namespace mi {

int weights_launch_16(const WeightsParams& p, int q_dtype, int head_dim, int which, dim3 grid, hipStream_t s) {
  return q_dtype == MI_BF16  ? launch_weights_kvt<BF16, kKv16>(p, head_dim, which, grid, s)
         : q_dtype == MI_F16 ? launch_weights_kvt<F16, kKv16>(p, head_dim, which, grid, s)
                             : launch_weights_kvt<F32, kKv16>(p, head_dim, which, grid, s);
}

// The second launch over short queries: four tokens to a thread.
__global__ __launch_bounds__(256) void weights_finish_kernel(WeightsParams p) {
  __shared__ float s_m[16][kWRows], s_l[16][kWRows], s_lse[kWRows];
  const int tid = (int)threadIdx.x, nkv = p.num_kv_heads;
  const int h = uniform((int)(blockIdx.x % nkv)), unit = uniform((int)(blockIdx.x / nkv));
  const int r = uniform(unit_request(p.kv_indptr, 1, p.finish_pages, p.batch, unit));
  if (r < 0) return;
  const WRequest q = w_request(p, r);
  if (q.rows <= 0 || q.rows > kWRows) return;
  const int tok0 = (unit - unit_begin(p.kv_indptr, 1, p.finish_pages, r)) * p.finish_pages * p.page_size;
  const int tok1 = min(tok0 + p.finish_pages * p.page_size, q.len), off = q.len - q.qo_len;
  if (tok0 >= tok1) return;
  constexpr int kAhead = 8;  // rows whose scores are loaded with the token's weight, the first time ahead of the join
  float4 s[kAhead], old;
  float* w;
  const float* src;
  auto load = [&](int t) {
    src = p.scores + (((((int64_t)q.first * p.page_size + t) >> 4) * nkv + h) * p.score_rows * 16 + (t & 15));
    const int e = (int)((unsigned)t / (unsigned)p.page_size);
    const int64_t page = p.kv_indices[q.first + e];
    w = page >= 0 && page < p.max_pages ? p.weights + (page * nkv + h) * p.page_size + t - e * p.page_size : nullptr;
#pragma unroll
    for (int row = 0; row < kAhead; ++row)
      if (row < q.rows) s[row] = *(const float4*)(src + 16 * row);
    old = w ? *(const float4*)w : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  int t = tok0 + 4 * tid;
  if (t < tok1) load(t);
  // the request's log-sum-exp: 16 threads a row go through its units of scores
  {
    const int row = tid & 15, part = tid >> 4, tokens = p.unit_pages * p.page_size, units = (q.len + tokens - 1) / tokens;
    const int begin = unit_begin(p.kv_indptr, 1, p.unit_pages, r);
    float m = -kWInf, l = 0.f;
    bool bad = false;
    for (int u0 = part; u0 < units; u0 += 16 * 8) {  // eight in flight
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        e[i] = u0 + 16 * i < units ? p.unit_lse[((int64_t)(begin + u0 + 16 * i) * nkv + h) * kWRows + row] : kWInf;
      float mn = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bad |= e[i] != e[i];
        if (e[i] == kWInf) e[i] = -kWInf;  // saw nothing there
        mn = fmaxf(mn, e[i]);
      }
      const float mu = mn == -kWInf ? 0.f : mn;
      l *= fast_exp2(m - mu);
#pragma unroll
      for (int i = 0; i < 8; ++i) l += fast_exp2(e[i] - mu);
      m = mn;
    }
    s_m[part][row] = m;
    s_l[part][row] = bad ? __builtin_nanf("") : l;
    __syncthreads();
    if (tid < kWRows) {
      float M = -kWInf, L = 0.f;
      for (int i = 0; i < 16; ++i) M = fmaxf(M, s_m[i][tid]);
      const float Mu = M == -kWInf ? 0.f : M;
      for (int i = 0; i < 16; ++i) L += s_l[i][tid] * fast_exp2(s_m[i][tid] - Mu);
      s_lse[tid] = w_lse(M, L);
    }
    __syncthreads();
  }
  while (t < tok1) {
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    // the first row that sees token t + i: those before it add nothing, also where their log-sum-exp is NaN
    auto first = [&](int i) { return p.causal ? max(0, t + i - off) * p.group : 0; };
    const int f0 = first(0), f1 = first(1), f2 = first(2), f3 = first(3);
    auto add = [&](const float4& x, int row) {
      const float e = s_lse[row];
      sum.x += row < f0 ? 0.f : fast_exp2(x.x - e);
      sum.y += row < f1 ? 0.f : fast_exp2(x.y - e);
      sum.z += row < f2 ? 0.f : fast_exp2(x.z - e);
      sum.w += row < f3 ? 0.f : fast_exp2(x.w - e);
    };
#pragma unroll
    for (int row = 0; row < kAhead; ++row)
      if (row < q.rows) add(s[row], row);
    for (int row = kAhead; row < q.rows; ++row) add(*(const float4*)(src + 16 * row), row);
    if (w) {
      if (t + 4 <= min(off, tok1)) {
        *(float4*)w = make_float4(old.x + sum.x, old.y + sum.y, old.z + sum.z, old.w + sum.w);
      } else {
        const float was[4] = {old.x, old.y, old.z, old.w}, more[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i < tok1) w[i] = t + i >= off ? more[i] : was[i] + more[i];
      }
    }
    t += 1024;
    if (t < tok1) load(t);
  }
}

constexpr int kMostRowSplits = 8;

// Joins the key shares' log-sum-exps of a row into the first.
__global__ __launch_bounds__(256) void weights_join_kernel(WeightsParams p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)p.num_kv_heads * p.total_rows;
  if (i >= n) return;
  float m = -kWInf, l = 0.f;
  bool bad = false;
  for (int s0 = 0; s0 < p.key_splits; s0 += 8) {  // eight in flight
    float e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = s0 + k < p.key_splits ? p.row_lse[(s0 + k) * n + i] : kWInf;
    float mn = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      bad |= e[k] != e[k];
      if (e[k] == kWInf) e[k] = -kWInf;  // saw nothing there
      mn = fmaxf(mn, e[k]);
    }
    const float mu = mn == -kWInf ? 0.f : mn;
    l *= fast_exp2(m - mu);
#pragma unroll
    for (int k = 0; k < 8; ++k) l += fast_exp2(e[k] - mu);
    m = mn;
  }
  p.row_lse[i] = w_lse(m, bad ? __builtin_nanf("") : l);
}

// Adds the row shares' sums of a token to its weight.
__global__ __launch_bounds__(256) void weights_sum_kernel(WeightsParams p) {
  const int nkv = p.num_kv_heads;
  const int h = uniform((int)(blockIdx.x % nkv)), unit = uniform((int)(blockIdx.x / nkv));
  const int r = uniform(unit_request(p.kv_indptr, 1, p.key_pages, p.batch, unit));
  if (r < 0) return;
  const WRequest q = w_request(p, r);
  if (q.rows <= kWRows) return;
  const int tok0 = (unit - unit_begin(p.kv_indptr, 1, p.key_pages, r)) * p.key_pages * p.page_size;
  const int tok1 = min(tok0 + p.key_pages * p.page_size, q.len), off = q.len - q.qo_len;
  for (int t = tok0 + (int)threadIdx.x; t < tok1; t += 256) {
    float x[kMostRowSplits], total = 0.f;
#pragma unroll
    for (int s = 0; s < kMostRowSplits; ++s)
      x[s] = s < p.row_splits ? p.sums[((int64_t)s * nkv + h) * p.places + (int64_t)q.first * p.page_size + t] : 0.f;
#pragma unroll
    for (int s = 0; s < kMostRowSplits; ++s) total += x[s];
    const int e = (int)((unsigned)t / (unsigned)p.page_size);
    const int64_t page = p.kv_indices[q.first + e];
    if (page < 0 || page >= p.max_pages) continue;
    float* w = p.weights + (page * nkv + h) * p.page_size + t - e * p.page_size;
    *w = t >= off ? total : *w + total;
  }
}

// One launch for short queries up to so many tokens in all, and a request on average: a workgroup
// streams a request alone, and a second launch costs 4 us (us a call, one / two launches: 4 requests of 100 to 400
// tokens 6.5 / 10.3, 16 of 20 to 90 6.5 / 10.2, one of 1000 11.6 / 10.2).
constexpr int64_t kOneTokens = 2048, kOneMean = 512;

// How a call is cut, from its shapes alone, and where its scratch lies.
struct WeightsCut {
  int32_t unit_pages, units, finish_pages, finish_units, score_rows;   // short
  bool one;                                                            // in one launch, without scratch
  int32_t row_units, key_splits, key_pages, key_units, row_splits;     // long
  int64_t scores, unit_lse, row_lse, sums, total;                      // bytes
};

// block: rows and keys of a workgroup of the long path's passes (the scratch does not depend on it).
static WeightsCut weights_cut(int32_t batch, int32_t max_qo_tokens, int32_t num_indices, int32_t page_size, int32_t nkv,
                              int32_t group, bool ragged, int parts, int block) {
  WeightsCut c{};
  const int64_t tokens = (int64_t)num_indices * page_size;
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  auto clamp = [](int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; };
  int64_t at = 0;
  // Runs of pages: about 4096 workgroups, of 64 tokens (one tile a wavefront) and more.
  c.unit_pages = (int32_t)up(clamp(up(tokens * nkv, 4096), 64, 1 << 24), page_size);
  c.units = (int32_t)(num_indices / c.unit_pages + batch);
  c.finish_pages = (int32_t)clamp(c.unit_pages, up(1024, page_size), INT32_MAX);  // as many tokens as its threads take at once
  c.finish_units = (int32_t)(num_indices / c.finish_pages + batch);
  c.score_rows = ragged ? kWRows : group;
  c.one = (parts & 1) && (int64_t)batch * nkv <= device_cu_count() && tokens <= kOneTokens && tokens <= kOneMean * batch &&
          (tokens + kOnePad) * c.score_rows <= kOneScores;
  if ((parts & 1) && !c.one) {
    c.scores = at;
    at = mi_align_up(at + 4 * tokens * nkv * c.score_rows, 256);
    c.unit_lse = at;
    at = mi_align_up(at + 4LL * c.units * nkv * kWRows, 256);
  }
  if (parts & 2) {
    const int64_t rows = (int64_t)max_qo_tokens * group, b = batch > 0 ? batch : 1;
    c.row_units = (int32_t)(rows / block + b);
    c.key_splits = (int32_t)clamp(2048 / ((rows / 256 + b) * nkv), 1, clamp(tokens / b / 256, 1, 16));
    c.key_pages = (int32_t)up(block, page_size);
    c.key_units = (int32_t)(num_indices / c.key_pages + b);
    c.row_splits = (int32_t)clamp(2048 / ((tokens / 256 + b) * nkv), 1, clamp(rows / b / 128, 1, kMostRowSplits));
    c.row_lse = at;
    at = mi_align_up(at + 4 * rows * nkv * c.key_splits, 256);
    c.sums = at;
    if (c.row_splits > 1) at = mi_align_up(at + 4 * tokens * nkv * c.row_splits, 256);
  }
  c.total = at;
  return c;
}

static bool weights_shapes_ok(int32_t batch, int32_t max_qo_tokens, int32_t num_indices, int32_t page_size, int32_t hq,
                              int32_t nkv, int32_t parts) {
  return batch >= 0 && max_qo_tokens >= 0 && num_indices >= 0 && page_size > 0 && nkv > 0 && hq > 0 && hq % nkv == 0 &&
         parts >= 1 && parts <= 3;
}

}  // namespace mi

extern "C" int64_t mi_attention_weights_bytes(int32_t batch, int32_t max_qo_tokens, int32_t num_indices, int32_t page_size,
                                              int32_t num_qo_heads, int32_t num_kv_heads, int32_t ragged, int32_t parts) {
  using namespace mi;
  if (!weights_shapes_ok(batch, max_qo_tokens, num_indices, page_size, num_qo_heads, num_kv_heads, parts)) return MI_ERR_INVALID;
  if (!ragged) parts = 1;
  return weights_cut(batch, max_qo_tokens, num_indices, page_size, num_kv_heads, num_qo_heads / num_kv_heads, ragged != 0, parts, kRowBlock).total;
}

extern "C" int mi_attention_weights_block(const mi_attention_weights_args* args) {
  using namespace mi;
  if (!args) return MI_ERR_INVALID;
  const mi_attention_weights_args& a = *args;
  if (!a.kv || !weights_shapes_ok(a.batch, a.max_qo_tokens, a.num_indices, a.kv->page_size, a.num_qo_heads, a.kv->num_kv_heads, a.parts))
    return MI_ERR_INVALID;
  if (a.batch == 0 || a.max_qo_tokens == 0 || a.num_indices == 0) return MI_OK;
  if (!a.q || !a.kv->data || !a.kv_indptr || !a.kv_indices || !a.last_page_len || !a.weights) return MI_ERR_INVALID;
  const int nkv = a.kv->num_kv_heads, D = a.kv->head_dim, group = a.num_qo_heads / nkv;
  if (group > kWRows || a.kv->page_size % 16 || (D != 64 && D != 128 && D != 256)) return MI_ERR_UNSUPPORTED;
  const bool scaled = kv_is_scaled(a.kv->dtype);
  if (a.q_dtype != MI_BF16 && a.q_dtype != MI_F16 && a.q_dtype != MI_F32) return MI_ERR_UNSUPPORTED;
  if (scaled ? a.q_dtype == MI_F32 : a.kv->dtype != a.q_dtype) return MI_ERR_UNSUPPORTED;
  if (!kv_scales_ok(a.kv)) return MI_ERR_INVALID;
  if (!rows_aligned16(a.q, a.q_stride_token, a.q_stride_head, a.q_dtype == MI_F32 ? 4 : 2) || !kv_aligned16(a.kv)) return MI_ERR_INVALID;
  if ((uintptr_t)a.weights % 16 || (uintptr_t)a.workspace % 16) return MI_ERR_INVALID;
  // places in the page list and rows are counted in 32 bits
  if ((int64_t)a.num_indices * a.kv->page_size > INT32_MAX - (1 << 25) || (int64_t)a.max_qo_tokens * group > INT32_MAX - 65536 ||
      a.kv->page_size > (1 << 24))
    return MI_ERR_UNSUPPORTED;
  // a wavefront's rows of a page are 32 bits apart
  if (a.kv->token_stride < 0 || a.kv->token_stride * kv_elem_bytes(a.kv->dtype) > (INT32_MAX >> 4)) return MI_ERR_UNSUPPORTED;
  const bool ragged = a.qo_indptr != nullptr;
  const int parts = ragged ? a.parts : 1;
  const WeightsCut c = weights_cut(a.batch, a.max_qo_tokens, a.num_indices, a.kv->page_size, nkv, group, ragged, parts,
                                   a.q_dtype == MI_F32 ? kRowBlock : mma_block(D));
  if (c.total > 0 && !a.workspace) return MI_ERR_INVALID;
  if (a.workspace_bytes < c.total) return MI_ERR_WORKSPACE;
  WeightsParams p{};
  p.q = a.q;
  p.q_stride_tok = a.q_stride_token;
  p.q_stride_head = a.q_stride_head;
  p.k = (const uint8_t*)a.kv->data;
  p.page_stride = a.kv->page_stride;
  p.token_stride = a.kv->token_stride;
  p.head_stride = a.kv->head_stride;
  p.max_pages = a.kv->max_pages;
  p.k_scale = a.kv->k_scale;
  p.qo_indptr = a.qo_indptr;
  p.kv_indptr = a.kv_indptr;
  p.kv_indices = a.kv_indices;
  p.last_page_len = a.last_page_len;
  p.weights = a.weights;
  uint8_t* ws = (uint8_t*)a.workspace;
  p.scores = (float*)(ws + c.scores);
  p.unit_lse = (float*)(ws + c.unit_lse);
  p.row_lse = (float*)(ws + c.row_lse);
  p.sums = (float*)(ws + c.sums);
  p.total_rows = (int64_t)a.max_qo_tokens * group;
  p.places = (int64_t)a.num_indices * a.kv->page_size;
  p.batch = a.batch;
  p.num_kv_heads = nkv;
  p.group = group;
  p.page_size = a.kv->page_size;
  p.causal = a.causal ? 1 : 0;
  p.max_tokens = a.max_qo_tokens;
  p.num_indices = a.num_indices;
  p.unit_pages = c.unit_pages;
  p.finish_pages = c.finish_pages;
  p.score_rows = c.score_rows;
  p.key_splits = c.key_splits;
  p.row_splits = c.row_splits;
  p.key_pages = c.key_pages;
  p.scale_log2 = a.sm_scale * 1.4426950408889634f;
  hipStream_t s = (hipStream_t)a.stream;
  const int kvt = kv_format(a.kv->dtype);
  auto launch = [&](int which, int64_t blocks) {
    if (blocks > INT32_MAX) return MI_ERR_UNSUPPORTED;
    const dim3 grid((uint32_t)blocks);
    return scaled ? weights_launch_scaled(p, a.q_dtype, kvt, D, which, grid, s) : weights_launch_16(p, a.q_dtype, D, which, grid, s);
  };
  if (c.one) {
    const int st = launch(kWOne, (int64_t)a.batch * nkv);
    if (st != MI_OK) return st;
  } else if (parts & 1) {
    const int st = launch(kWScores, (int64_t)c.units * nkv);
    if (st != MI_OK) return st;
    hipLaunchKernelGGL(weights_finish_kernel, dim3((uint32_t)(c.finish_units * nkv)), dim3(256), 0, s, p);
  }
  if (parts & 2) {
    int st = launch(kWRowsPass, (int64_t)c.row_units * nkv * c.key_splits);
    if (st != MI_OK) return st;
    if (c.key_splits > 1)
      hipLaunchKernelGGL(weights_join_kernel, dim3((uint32_t)((nkv * p.total_rows + 255) / 256)), dim3(256), 0, s, p);
    st = launch(kWColsPass, (int64_t)c.key_units * nkv * c.row_splits);
    if (st != MI_OK) return st;
    if (c.row_splits > 1)
      hipLaunchKernelGGL(weights_sum_kernel, dim3((uint32_t)(c.key_units * nkv)), dim3(256), 0, s, p);
  }
  MI_CHECK_LAUNCH();
  return MI_OK;
}

extern "C" int mi_attention_weights(const void* q, int32_t q_dtype, int64_t q_stride_token, int64_t q_stride_head,
                                    const mi_paged_kv* kv, const int32_t* qo_indptr, const int32_t* kv_indptr,
                                    const int32_t* kv_indices, const int32_t* last_page_len, int32_t batch,
                                    int32_t max_qo_tokens, int32_t num_indices, int32_t num_qo_heads, int32_t causal,
                                    float sm_scale, int32_t parts, float* weights, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  const mi_attention_weights_args args = {q, kv, qo_indptr, kv_indptr, kv_indices, last_page_len, weights, workspace, stream, q_stride_token, q_stride_head, workspace_bytes, q_dtype, batch, max_qo_tokens, num_indices, num_qo_heads, causal, parts, sm_scale};
  return mi_attention_weights_block(&args);
}
