// Log probabilities of given tokens, entropy and top alternatives of rows of logits, and the gradient.
//
//   m = max_j x_j,  S = sum_j exp(x_j - m),  T = sum_j (x_j - m) exp(x_j - m)
//   lse = m + log S        log p(token) = x_token - lse        H = -sum_j p_j log p_j = log S - T / S
//   d x_j = d_logp * ([j = token] - p_j) - d_H * p_j * (log p_j + H)
// T is summed over x - m, not over x: the terms stay small, and a ruled-out symbol (-1e9, or minus infinity) adds exactly 0.
#include "nst_common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// Order of the alternatives: value, then the lower index; a NaN ranks first, -0 equals +0.  The 64-bit keys of a row differ.
__device__ __forceinline__ uint64_t order_key(float x, int idx) {
  uint32_t u = __float_as_uint(x + 0.0f);
  u = (x != x) ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)(0xffffffffu - (uint32_t)idx);
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}

template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_kernel(const T* __restrict__ logits, const int64_t* __restrict__ tokens,
                                                             float* __restrict__ logp, float* __restrict__ entropy,
                                                             float* __restrict__ lse_out, float* __restrict__ top_logp,
                                                             int64_t* __restrict__ top_ids, int V, int64_t ldl, int top_n) {
  __shared__ float red[3][4];
  __shared__ uint64_t best[4];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ldl;
  const int tid = threadIdx.x;
  float m = -INFINITY;
  for (int j = tid; j < V; j += 256) m = fmaxf(m, to_f32<T>(x[j]));
  m = wave_max(m);
  if ((tid & 63) == 0) red[0][tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float s = 0.f, t = 0.f;
  for (int j = tid; j < V; j += 256) {
    const float d = to_f32<T>(x[j]) - m, e = exp2f(d * LOG2E);
    s += e;
    t += e == 0.f ? 0.f : d * e;
  }
  s = wave_sum(s);
  t = wave_sum(t);
  if ((tid & 63) == 0) {
    red[1][tid >> 6] = s;
    red[2][tid >> 6] = t;
  }
  __syncthreads();
  s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  t = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  const float lse = m + logf(s);
  if (tid == 0) {
    if (lse_out) lse_out[row] = lse;
    if (entropy) entropy[row] = logf(s) - t / s;
    if (logp) {
      const int64_t tok = tokens[row];
      logp[row] = tok >= 0 && tok < V ? to_f32<T>(x[tok]) - lse : 0.f;
    }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < top_n; ++k) {
    uint64_t b = 0;
    for (int j = tid; j < V; j += 256) {
      const uint64_t key = order_key(to_f32<T>(x[j]), j);
      if ((k == 0 || key < last) && key > b) b = key;
    }
    b = wave_max_u64(b);
    if ((tid & 63) == 0) best[tid >> 6] = b;
    __syncthreads();
    for (int w = 0; w < 4; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    __syncthreads();
    if (tid == 0) {
      const int id = (int)(0xffffffffu - (uint32_t)b);
      top_ids[row * top_n + k] = id;
      top_logp[row * top_n + k] = to_f32<T>(x[id]) - lse;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_bwd_kernel(const T* logits, const int64_t* __restrict__ tokens,
                                                                 const float* __restrict__ lse, const float* __restrict__ entropy,
                                                                 const float* __restrict__ dlogp, const float* __restrict__ dentropy,
                                                                 T* dlogits, int V, int64_t ldl, int64_t ldd) {
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ldl;
  T* g = dlogits + row * ldd;
  const int64_t tok = tokens ? tokens[row] : -1;
  const bool given = tok >= 0 && tok < V;
  const float L = lse[row], a = given && dlogp ? dlogp[row] : 0.f, b = dentropy ? dentropy[row] : 0.f, h = dentropy ? entropy[row] : 0.f;
  for (int j = threadIdx.x; j < V; j += 256) {
    const float lp = to_f32<T>(x[j]) - L, pr = exp2f(lp * LOG2E);
    float v = pr == 0.f ? 0.f : -pr * (a + b * (lp + h));
    if (given && j == tok) v += a;
    g[j] = from_f32<T>(v);
  }
}

}  // namespace

static int logprobs_check(const char* name, int64_t rows, int V, int64_t ldl, int top_n, int dtype) {
  NST_CHECK_ARG(dtype == NST_F32 || dtype == NST_BF16, "%s: dtype %d", name, dtype);
  NST_CHECK_ARG(rows >= 0 && rows <= 0x7fffffffLL && V > 0 && V <= (1 << 20), "%s: rows=%lld V=%d (1 .. 2^20)", name, (long long)rows, V);
  NST_CHECK_ARG(ldl >= 0 && top_n >= 0 && top_n <= 64 && top_n <= V, "%s: ldl=%lld top_n=%d (0 .. min(64, V))", name, (long long)ldl, top_n);
  return NST_OK;
}

extern "C" int64_t nst_token_logprobs_workspace_bytes(int64_t rows, int V, int top_n, int dtype) {
  const int rc = logprobs_check("nst_token_logprobs_workspace_bytes", rows, V, 0, top_n, dtype);
  return rc != NST_OK ? rc : 0;
}

extern "C" int nst_token_logprobs_fwd(const void* logits, const int64_t* tokens, float* logp, float* entropy, float* lse, float* top_logp,
                                      int64_t* top_ids, int64_t rows, int V, int64_t ldl, int top_n, int dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const int rc = logprobs_check("nst_token_logprobs_fwd", rows, V, ldl, top_n, dtype);
  if (rc != NST_OK) return rc;
  if (rows == 0) return NST_OK;
  NST_CHECK_ARG(logits && (!logp || tokens) && (top_n == 0 || (top_logp && top_ids)), "nst_token_logprobs_fwd: NULL pointer");
  (void)workspace; (void)workspace_bytes;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NST_BF16)
    token_logprobs_kernel<bf16_t><<<(unsigned)rows, 256, 0, st>>>((const bf16_t*)logits, tokens, logp, entropy, lse, top_logp, top_ids, V, ldl, top_n);
  else
    token_logprobs_kernel<float><<<(unsigned)rows, 256, 0, st>>>((const float*)logits, tokens, logp, entropy, lse, top_logp, top_ids, V, ldl, top_n);
  NST_CHECK_LAUNCH("nst_token_logprobs_fwd");
  return NST_OK;
}

extern "C" int nst_token_logprobs_bwd(const void* logits, const int64_t* tokens, const float* lse, const float* entropy, const float* dlogp,
                                      const float* dentropy, void* dlogits, int64_t rows, int V, int64_t ldl, int64_t ldd, int dtype,
                                      void* stream) {
  const int rc = logprobs_check("nst_token_logprobs_bwd", rows, V, ldl, 0, dtype);
  if (rc != NST_OK) return rc;
  if (rows == 0) return NST_OK;
  NST_CHECK_ARG(logits && lse && dlogits && (!dlogp || tokens) && (!dentropy || entropy), "nst_token_logprobs_bwd: NULL pointer");
  NST_CHECK_ARG(ldd >= V || rows == 1, "nst_token_logprobs_bwd: ldd=%lld < V=%d", (long long)ldd, V);
  NST_CHECK_ARG(dlogits != logits || ldd == ldl, "nst_token_logprobs_bwd: in place needs equal strides (%lld, %lld)", (long long)ldl,
                (long long)ldd);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NST_BF16)
    token_logprobs_bwd_kernel<bf16_t><<<(unsigned)rows, 256, 0, st>>>((const bf16_t*)logits, tokens, lse, entropy, dlogp, dentropy, (bf16_t*)dlogits, V, ldl, ldd);
  else
    token_logprobs_bwd_kernel<float><<<(unsigned)rows, 256, 0, st>>>((const float*)logits, tokens, lse, entropy, dlogp, dentropy, (float*)dlogits, V, ldl, ldd);
  NST_CHECK_LAUNCH("nst_token_logprobs_bwd");
  return NST_OK;
}
