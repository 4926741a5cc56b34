// Log probabilities of given tokens, entropy and top alternatives of rows of logits, and the gradient.
//
//   m = max_j x_j,  S = sum_j exp(x_j - m),  T = sum_j (x_j - m) exp(x_j - m)
//   lse = m + log S        log p(token) = (x_token - m) - log S        H = -sum_j p_j log p_j = log S - T / S
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

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}

template <typename T>
struct LV;
template <>
struct LV<bf16_t> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
};
template <>
struct LV<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&x)[4]) {
    x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};

constexpr int MAX_PARTS = 64, MAX_TOP = 64, CAND = 512;
constexpr float LOWEST = -3.402823466e38f;

struct LogprobParams {
  const void* logits;
  const int64_t* tokens;
  float *logp, *entropy, *lse, *top_logp;
  int64_t* top_ids;
  int64_t ldl;
  int V, top_n, nparts, part;     // part: elements of a part (a multiple of 16 bytes)
  float* stats;                   // nparts > 1: [rows][nparts][4]  m, S, T, -
  uint64_t* keys;                 //             [rows][nparts][top_n], descending, 0: none
};

// What a row's statistics give: one thread.  log p is (x - m) - log S, not x - lse: lse is rounded at its own size (3e-5 at 1000), while what the
// likely logits have in common with m drops out of x - m exactly.
template <typename T>
__device__ __forceinline__ void write_row(const LogprobParams& p, int64_t row, float m, float log_s, float ratio) {
  if (p.lse) p.lse[row] = m + log_s;
  if (p.entropy) p.entropy[row] = log_s - ratio;
  if (p.logp) {
    const int64_t tok = p.tokens[row];
    p.logp[row] = tok >= 0 && tok < p.V ? (to_f32<T>(((const T*)p.logits)[row * p.ldl + tok]) - m) - log_s : 0.f;
  }
}
__device__ __forceinline__ void write_top(const LogprobParams& p, int64_t row, int rank, uint64_t key, float m, float log_s) {
  p.top_ids[row * p.top_n + rank] = key_index(key);
  p.top_logp[row * p.top_n + rank] = (key_value(key) - m) - log_s;
}

// One workgroup holds a row, or a part of one (up to 256 * E * NV elements), in registers: every load is requested before the first is used and
// the logits are read once, for the statistics and for the alternatives.
// Bound by memory where there are rows enough (9600 x 8008 bf16: 27 us, 5.6 TB/s; an exponential and six more vector operations per element
// are 77 % of the time it takes to arrive, so not much closer), else by the latency of read -> maximum -> sum -> threshold -> ranking: 128 x
// 8008 bf16 with six alternatives 6.8 us, 4 x 128000 float32 with twenty 6.2 us and 5.5 us for the join.
// Alternatives: the top_n-th largest of the 256 threads' maxima (found by bisection over its bits) is a value that at least top_n
// elements reach, so only elements from it on are candidates -- a few more than top_n for ordinary rows; they are collected in LDS and ranked by
// counting.  Rows where too many elements tie at that value take the ties in index order; what overflows even then, and rows with NaN, fall
// back to one reduction per alternative.
template <typename T, int NV>
__global__ void __launch_bounds__(256) token_logprobs_kernel(LogprobParams p) {
  constexpr int E = LV<T>::E;
  __shared__ float red[3][4];
  __shared__ uint32_t s_max[256];
  __shared__ uint64_t cand[CAND];
  __shared__ uint64_t best[4];
  __shared__ int s_count, s_wave[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / p.nparts;
  const int part = (int)(blockIdx.x - row * p.nparts);
  const int j0 = part * p.part, n = min(p.part, p.V - j0);
  const T* x = (const T*)p.logits + row * p.ldl + j0;
  const int nfull = n / E, ntail = n - nfull * E;       // whole 16-byte pieces; the rest is one element for each of the first threads
  uint4 v[NV];
  if (nfull > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) __builtin_memcpy(&v[i], x + (int64_t)min(i * 256 + tid, nfull - 1) * E, 16);
  }
  const bool has_tail = tid < ntail;
  const float tail = has_tail ? to_f32<T>(x[nfull * E + tid]) : -INFINITY;
  float mt = tail;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * 256 + tid < nfull) {
      float e[E];
      LV<T>::unpack(v[i], e);
#pragma unroll
      for (int k = 0; k < E; ++k) mt = fmaxf(mt, e[k]);
    }
  const float mw = wave_max(mt);
  if (lane == 0) red[0][wave] = mw;
  if (tid == 0) s_count = 0;
  if (p.top_n > 0) s_max[tid] = tid < nfull || has_tail ? (uint32_t)(order_key(mt, 0) >> 32) : 0u;
  __syncthreads();
  const float m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float mu = m == -INFINITY ? 0.f : m;            // (a part of nothing but ruled-out symbols adds exactly nothing)
  float s = 0.f, t = 0.f;
  {
    const float d = tail - mu, e = __builtin_amdgcn_exp2f(d * LOG2E);
    s += e;
    t += fmaxf(d, LOWEST) * e;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * 256 + tid < nfull) {
      float e[E];
      LV<T>::unpack(v[i], e);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float d = e[k] - mu, w = __builtin_amdgcn_exp2f(d * LOG2E);
        s += w;
        t = fmaf(fmaxf(d, LOWEST), w, t);               // (a NaN is in w; minus infinity times 0 is kept out)
      }
    }
  s = wave_sum(s);
  t = wave_sum(t);
  if (lane == 0) {
    red[1][wave] = s;
    red[2][wave] = t;
  }
  __syncthreads();
  s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  t = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  const bool single = p.nparts == 1;
  const float log_s = m == -INFINITY ? NAN : logf(s);
  if (tid == 0) {
    if (single) {
      write_row<T>(p, row, m, log_s, t / s);
    } else {
      float* st = p.stats + (row * p.nparts + part) * 4;
      st[0] = m; st[1] = s; st[2] = t;
    }
  }
  if (p.top_n == 0) return;
  const int want = min(p.top_n, n);
  uint64_t* keys = single ? nullptr : p.keys + (row * p.nparts + part) * p.top_n;
  auto emit = [&](int rank, uint64_t key) __attribute__((always_inline)) {
    if (single) write_top(p, row, rank, key, m, log_s);
    else keys[rank] = key;
  };
  if (!single)
    for (int k = want + tid; k < p.top_n; k += 256) keys[k] = 0;
  // this thread's elements from `tau` on (`above`: only those above it) into the candidates.  Pieces are skipped by their largest element;
  // the comparison of values is that of the ordered words (a NaN does not come here, -0 equals +0).
  auto collect = [&](uint32_t tau, bool above) __attribute__((always_inline)) {
    const float tv = tau <= 0x007fffffu ? -INFINITY : key_value((uint64_t)tau << 32);
    auto take = [&](float e, int j) __attribute__((always_inline)) {
      if (above ? e > tv : e >= tv) {
        const int at = atomicAdd(&s_count, 1);
        if (at < CAND) cand[at] = order_key(e, j);
      }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * 256 + tid < nfull) {
        float e[E], most = -INFINITY;
        LV<T>::unpack(v[i], e);
#pragma unroll
        for (int k = 0; k < E; ++k) most = fmaxf(most, e[k]);
        if (most >= tv) {
#pragma unroll
          for (int k = 0; k < E; ++k) take(e[k], j0 + (i * 256 + tid) * E + k);
        }
      }
    if (has_tail) take(tail, j0 + nfull * E + tid);
  };
  // largest value (as an ordered word, cut to its upper `bits`) that at least `want` threads' maxima reach; 0 if there are fewer threads
  auto bisect = [&](int bits) __attribute__((always_inline)) {
    const uint32_t a = s_max[lane], b = s_max[64 + lane], c = s_max[128 + lane], d = s_max[192 + lane];
    uint32_t tau = 0;
    for (int bit = 31; bit >= 32 - bits; --bit) {
      const uint32_t probe = tau | (1u << bit);
      const int cnt = __popcll(__ballot(a >= probe)) + __popcll(__ballot(b >= probe)) + __popcll(__ballot(c >= probe)) +
                      __popcll(__ballot(d >= probe));
      if (cnt >= want) tau = probe;
    }
    return tau;
  };
  auto ranked = [&](int count) __attribute__((always_inline)) {      // the candidates, ranked by counting
    for (int i = tid; i < count; i += 256) {
      const uint64_t key = cand[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < count; ++j) rank += cand[j] > key;
      if (rank < want) emit(rank, key);
    }
  };
  const uint32_t my_max = s_max[tid];
  if (s == s) {
    uint32_t tau = bisect(16);
    if (my_max >= tau) collect(tau, false);
    __syncthreads();
    int count = s_count;
    if (count <= CAND) {
      ranked(count);
      return;
    }
    // too many: the value in full, what lies above it, and the ties in the order of their index
    tau = bisect(32);
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
    if (my_max > tau) collect(tau, true);
    __syncthreads();
    count = s_count;
    if (count <= CAND - MAX_TOP) {
      // (pieces of one index i lie in thread order; the elements behind them are the last round.  Read again: a register cannot be
      // chosen by a loop that ends early)
      int need = want - count, base = count;
      for (int i = 0; i <= NV && need > 0; ++i) {
        const bool tail_round = i == NV;
        const int first = tail_round ? nfull * E + tid : (i * 256 + tid) * E;
        const int here = tail_round ? (has_tail ? 1 : 0) : (i * 256 + tid < nfull ? E : 0);
        int ties = 0;
        for (int k = 0; k < here; ++k) ties += (uint32_t)(order_key(to_f32<T>(x[first + k]), 0) >> 32) == tau;
        int incl = ties;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int up = __shfl_up(incl, o, 64);
          if (lane >= o) incl += up;
        }
        if (lane == 63) s_wave[wave] = incl;
        __syncthreads();
        int before = incl - ties, total = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if (w < wave) before += s_wave[w];
          total += s_wave[w];
        }
        for (int k = 0; k < here && before < need; ++k) {
          const uint64_t key = order_key(to_f32<T>(x[first + k]), j0 + first + k);
          if ((uint32_t)(key >> 32) == tau) cand[base + before++] = key;
        }
        base += min(total, need);
        need -= total;
        __syncthreads();
      }
      ranked(base);
      return;
    }
    __syncthreads();
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < want; ++k) {
    uint64_t b = 0;
    for (int j = tid; j < n; j += 256) {
      const uint64_t key = order_key(to_f32<T>(x[j]), j0 + j);
      if ((k == 0 || key < last) && key > b) b = key;
    }
    b = wave_max_u64(b);
    if (lane == 0) best[wave] = b;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    if (tid == 0) emit(k, b);
    __syncthreads();
  }
}

// Joins the parts of a row: lane i of every wave has part i (four waves only so that the lists arrive at once).  Alternatives: with d entries
// of each list looked at (d * parts >= top_n), k = ceil(top_n / d) lists hold at least k * d >= top_n keys not below the k-th largest of the
// lists' d-th entries, so only keys from it on are candidates; they are ranked by counting.
template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_join_kernel(LogprobParams p) {
  extern __shared__ uint64_t lists[];                  // [nparts][top_n], then the lists' heads and, in their place, the candidates
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 63, np = p.nparts, n = p.top_n;
  const int64_t row = blockIdx.x;
  const float* st = p.stats + row * np * 4;
  float m = -INFINITY, s = 0.f, t = 0.f;
  if (lane < np) {
    const float4 q = reinterpret_cast<const float4*>(st)[lane];
    m = q.x; s = q.y; t = q.z;
  }
  uint64_t *heads = lists + np * n, *cand = heads;
  const int depth = n > 0 ? (n + np - 1) / np : 1, wanted = n > 0 ? (n + depth - 1) / depth : 0;      // d and k
  {
    const uint64_t* src = p.keys + row * np * n;
    const uint64_t head = n > 0 && lane < np ? src[lane * n + depth - 1] : 0;
    uint64_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i * 256 + tid < np * n ? src[i * 256 + tid] : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i * 256 + tid < np * n) lists[i * 256 + tid] = v[i];
    if (tid < MAX_PARTS) heads[tid] = head;
  }
  const float M = wave_max(m), mu = M == -INFINITY ? 0.f : M;
  const float d = m - mu, c = __builtin_amdgcn_exp2f(d * LOG2E);
  t = wave_sum(fmaf(c * fmaxf(d, LOWEST), s, c * t));      // (c first: d * s overflows where a part holds nothing but large finite masks, c is 0 there)
  s = wave_sum(c * s);
  const float log_s = M == -INFINITY ? NAN : logf(s);
  if (tid == 0) write_row<T>(p, row, M, log_s, t / s);
  if (n == 0) return;
  __syncthreads();
  const uint64_t head = heads[lane];
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < np; ++j) rank += heads[j] > head;
  // (keys differ, a key holds its index; lists that are shorter than d have 0 there: then there may be no k-th, and every key counts)
  const uint64_t nth = __ballot(lane < np && head != 0 && rank == wanted - 1);
  const uint64_t tau = nth ? heads[__ffsll((unsigned long long)nth) - 1] : 1;
  __syncthreads();                                      // the candidates take the heads' place
  if (tid < 64) {
    int cnt = 0;
    if (lane < np)
      while (cnt < n && lists[lane * n + cnt] >= tau) ++cnt;
    int incl = cnt;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(incl, o, 64);
      if (lane >= o) incl += up;
    }
    for (int k = 0; k < cnt; ++k) cand[incl - cnt + k] = lists[lane * n + k];
    if (lane == 63) s_count = incl;
  }
  __syncthreads();
  const int count = s_count;
  for (int i = tid; i < count; i += 256) {
    const uint64_t key = cand[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) r += cand[j] > key;
    if (r < n) write_top(p, row, r, key, M, log_s);
  }
}

// One read and one write of a row's length: 9600 x 8008 bf16 48 us, 6.4 TB/s (part of the logits still lie in the last-level cache when the
// gradient follows the forward pass).  Each thread owns four 16-byte pieces, all requested before the row's scalars are used.
constexpr int BWD_PIECES = 4;      // 16-byte pieces of a thread

template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_bwd_kernel(const T* logits, const int64_t* __restrict__ tokens,
                                                                 const float* __restrict__ lse, const float* __restrict__ entropy,
                                                                 const float* __restrict__ dlogp, const float* __restrict__ dentropy,
                                                                 T* dlogits, int V, int64_t ldl, int64_t ldd, int chunks) {
  constexpr int E = LV<T>::E;
  const int64_t row = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x - row * chunks), tid = threadIdx.x;
  const T* x = logits + row * ldl;
  T* gr = dlogits + row * ldd;
  const int nfull = V / E;
  uint4 v[BWD_PIECES];
  const int p0 = chunk * (256 * BWD_PIECES) + tid;
#pragma unroll
  for (int i = 0; i < BWD_PIECES; ++i)
    if (p0 + i * 256 < nfull) __builtin_memcpy(&v[i], x + (int64_t)(p0 + i * 256) * E, 16);
  const int64_t tok = tokens ? tokens[row] : -1;
  const bool given = tok >= 0 && tok < V;
  const float L = lse[row], a = given && dlogp ? dlogp[row] : 0.f, b = dentropy ? dentropy[row] : 0.f, h = dentropy ? entropy[row] : 0.f;
  auto grad = [&](float e) __attribute__((always_inline)) {
    const float lp = e - L;
    return -__builtin_amdgcn_exp2f(lp * LOG2E) * fmaf(b, fmaxf(lp, -1e4f) + h, a);     // (p is 0 long before log p = -1e4)
  };
#pragma unroll
  for (int i = 0; i < BWD_PIECES; ++i) {
    const int piece = p0 + i * 256;
    if (piece >= nfull) break;
    float e[E];
    LV<T>::unpack(v[i], e);
#pragma unroll
    for (int k = 0; k < E; ++k) e[k] = grad(e[k]);
    if (given && tok / E == piece) {
#pragma unroll
      for (int k = 0; k < E; ++k) e[k] += k == (int)(tok % E) ? a : 0.f;
    }
    const uint4 r = LV<T>::pack(e);
    __builtin_memcpy(gr + (int64_t)piece * E, &r, 16);
  }
  const int j = nfull * E + tid;
  if (chunk == chunks - 1 && j < V) gr[j] = from_f32<T>(grad(to_f32<T>(x[j])) + (given && j == tok ? a : 0.f));
}

struct LogprobSplit {
  int nparts, part, pieces;     // pieces: of a thread
};
// Rows of up to 32768 elements stay whole.  Against parts of 1024 .. 16384 elements and a second launch (device time without / with six
// alternatives): 16 rows of 8008 bf16 3.6 / 6.2 against 5.6 / 9.5 us, 127 rows of 32000 5.7 / 9.9 against 7.3 / 12.3 us, 1000 rows of
// 32000 14.5 / 19.1 against 16.8 / 23.5 us, and a launch less for the host.  Longer ones are cut into at most 64 parts of at most 16384
// elements (1000 rows of 50000 float32 34 us, in parts of up to 32768 35 us) -- of at least 1024 where there are so few rows that they
// would not reach every CU otherwise.
static LogprobSplit logprob_split(int64_t rows, int V, int dtype) {
  const int E = dtype == NST_BF16 ? 8 : 4, most = 16384;
  int64_t want = V <= 2 * most || rows >= 128 ? 1 : rows > 0 ? (256 + rows - 1) / rows : 1;
  if (want > (V + 1023) / 1024) want = (V + 1023) / 1024;
  if (V > 2 * most && want < (V + most - 1) / most) want = (V + most - 1) / most;
  if (want > MAX_PARTS) want = MAX_PARTS;
  LogprobSplit s;
  s.part = (int)(((V + want - 1) / want + E - 1) / E * E);
  s.nparts = (V + s.part - 1) / s.part;
  s.pieces = (s.part + 256 * E - 1) / (256 * E);
  return s;
}

template <typename T>
void logprobs_launch(const LogprobParams& p, int pieces, unsigned grid, hipStream_t st) {
  constexpr int MOST = 32768 / (256 * LV<T>::E);           // pieces of a thread in the longest whole row: 16 of bf16, 32 of f32
  if (pieces <= 1) token_logprobs_kernel<T, 1><<<grid, 256, 0, st>>>(p);
  else if (pieces <= 2) token_logprobs_kernel<T, 2><<<grid, 256, 0, st>>>(p);
  else if (pieces <= 4) token_logprobs_kernel<T, 4><<<grid, 256, 0, st>>>(p);
  else if (pieces <= 8) token_logprobs_kernel<T, 8><<<grid, 256, 0, st>>>(p);
  else if (pieces <= 16) token_logprobs_kernel<T, 16><<<grid, 256, 0, st>>>(p);
  else token_logprobs_kernel<T, MOST><<<grid, 256, 0, st>>>(p);
}

}  // namespace

static int logprobs_check(const char* name, int64_t rows, int V, int64_t ldl, int top_n, int dtype) {
  NST_CHECK_ARG(dtype == NST_F32 || dtype == NST_BF16, "%s: dtype %d", name, dtype);
  NST_CHECK_ARG(rows >= 0 && rows <= 0x7fffffffLL && V > 0 && V <= (1 << 20), "%s: rows=%lld V=%d (1 .. 2^20)", name, (long long)rows, V);
  NST_CHECK_ARG(ldl >= 0 && top_n >= 0 && top_n <= 64 && top_n <= V, "%s: ldl=%lld top_n=%d (0 .. min(64, V))", name, (long long)ldl, top_n);
  return NST_OK;
}

static int64_t logprobs_workspace(int64_t rows, int V, int top_n, int dtype) {
  const int n = logprob_split(rows, V, dtype).nparts;
  return n > 1 ? rows * n * (16 + 8LL * top_n) : 0;
}

extern "C" int64_t nst_token_logprobs_workspace_bytes(int64_t rows, int V, int top_n, int dtype) {
  const int rc = logprobs_check("nst_token_logprobs_workspace_bytes", rows, V, 0, top_n, dtype);
  return rc != NST_OK ? rc : logprobs_workspace(rows, V, top_n, dtype);
}

extern "C" int nst_token_logprobs_fwd(const void* logits, const int64_t* tokens, float* logp, float* entropy, float* lse, float* top_logp,
                                      int64_t* top_ids, int64_t rows, int V, int64_t ldl, int top_n, int dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const int rc = logprobs_check("nst_token_logprobs_fwd", rows, V, ldl, top_n, dtype);
  if (rc != NST_OK) return rc;
  if (rows == 0) return NST_OK;
  NST_CHECK_ARG(logits && (!logp || tokens) && (top_n == 0 || (top_logp && top_ids)), "nst_token_logprobs_fwd: NULL pointer");
  const LogprobSplit sp = logprob_split(rows, V, dtype);
  LogprobParams p = {logits, tokens, logp, entropy, lse, top_logp, top_ids, ldl, V, top_n, sp.nparts, sp.part, nullptr, nullptr};
  if (sp.nparts > 1) {
    const int64_t need = logprobs_workspace(rows, V, top_n, dtype);
    if (!workspace || workspace_bytes < need || !nst_aligned16(workspace)) {
      nst_set_error("nst_token_logprobs_fwd: workspace of %lld bytes, needs %lld (16-byte aligned)", (long long)workspace_bytes, (long long)need);
      return NST_ERR_WORKSPACE;
    }
    p.stats = (float*)workspace;
    p.keys = (uint64_t*)(p.stats + rows * sp.nparts * 4);
  }
  NST_CHECK_ARG(rows * sp.nparts <= 0x7fffffffLL, "nst_token_logprobs_fwd: %lld rows of %d parts", (long long)rows, sp.nparts);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NST_BF16) logprobs_launch<bf16_t>(p, sp.pieces, (unsigned)(rows * sp.nparts), st);
  else logprobs_launch<float>(p, sp.pieces, (unsigned)(rows * sp.nparts), st);
  if (sp.nparts > 1) {
    NST_CHECK_LAUNCH("nst_token_logprobs_fwd");
    // (64 parts of 64 alternatives: 64 KiB, and the kernel's own word of LDS, of the 160 KiB of a CU)
    const size_t held = (size_t)sp.nparts * top_n, lds = sizeof(uint64_t) * (held + (held > MAX_PARTS ? held : MAX_PARTS));
    if (dtype == NST_BF16) token_logprobs_join_kernel<bf16_t><<<(unsigned)rows, 256, lds, st>>>(p);
    else token_logprobs_join_kernel<float><<<(unsigned)rows, 256, lds, st>>>(p);
  }
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
  const int per = (dtype == NST_BF16 ? 8 : 4) * 256 * BWD_PIECES, chunks = (V + per - 1) / per;
  NST_CHECK_ARG(rows * chunks <= 0x7fffffffLL, "nst_token_logprobs_bwd: %lld rows of %d", (long long)rows, V);
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)(rows * chunks);
  if (dtype == NST_BF16)
    token_logprobs_bwd_kernel<bf16_t><<<grid, 256, 0, st>>>((const bf16_t*)logits, tokens, lse, entropy, dlogp, dentropy,
                                                            (bf16_t*)dlogits, V, ldl, ldd, chunks);
  else
    token_logprobs_bwd_kernel<float><<<grid, 256, 0, st>>>((const float*)logits, tokens, lse, entropy, dlogp, dentropy, (float*)dlogits, V,
                                                           ldl, ldd, chunks);
  NST_CHECK_LAUNCH("nst_token_logprobs_bwd");
  return NST_OK;
}
