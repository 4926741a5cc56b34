// Paged key / value caches: page assignment from request lengths, rows to slots, attention of one new token over the pages,
// re-ordering behind a beam-search step.
//
// A cache holds `num_pages` pages of `page_size` token rows; page p of request b's sequence is block_table[b][p].  The slot of a
// token is page * page_size + position % page_size.  Every entry read from a table, a slot map, a free list or a list of parents
// is checked against its range on the device before it becomes an address: an entry outside contributes nothing.
#include <type_traits>

#include "nst_common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float LOWEST = -3.402823466e38f;
constexpr int64_t MAX_POSITIONS = 1 << 30;     // of one request: position arithmetic, a tile or two past the end included, stays in 32 bits

// t / d for 0 <= t < 2^31 by one multiplication: with s = ceil(log2 d) and magic = floor(2^(31 + s) / d) + 1 the error of t * magic / 2^(31 + s)
// stays below 1 / d, so the quotient is exact.  magic == 0: d == 1.
struct FastDiv {
  uint32_t d, magic;
  int shift;
  __device__ __forceinline__ uint32_t div(uint32_t t) const { return magic ? __umulhi(t, magic) >> shift : t; }
  __device__ __forceinline__ uint32_t up(uint32_t t) const { return div(t + d - 1); }      // (t + d - 1 < 2^31 too)
};
FastDiv fast_div(int d) {
  FastDiv f = {(uint32_t)d, 0, 0};
  int s = 0;
  while ((1LL << s) < d) ++s;
  if (s > 0) {
    f.magic = (uint32_t)((1ULL << (31 + s)) / (uint64_t)d + 1);
    f.shift = s - 1;
  }
  return f;
}

// ---------------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------------
struct PlanParams {
  const int32_t *cached, *fresh;
  int B, max_pages;
  FastDiv page;
  int32_t* table;
  int64_t table_stride;
  const int32_t* free_pages;
  int n_free;
  const int32_t* cursor_in;
  int64_t* slots;
  int max_tokens;
  int32_t *seq_lens, *cu_new, *cursor_out;
  int per_group;   // requests of one workgroup (<= 64)
};

struct PlanRequest {
  int cached, fresh, held, need;   // tokens there / to come, pages held / wanted (as far as the table row reaches)
};
__device__ __forceinline__ PlanRequest plan_request(const PlanParams& p, int b) {
  PlanRequest r;
  const int cap = p.max_pages * (int)p.page.d;             // <= 2^30
  r.cached = min(max(p.cached[b], 0), cap);
  r.fresh = max(p.fresh[b], 0);
  r.held = (int)p.page.up(r.cached);
  r.need = (int)p.page.up(r.cached + min(r.fresh, cap - r.cached)) - r.held;
  return r;
}
__device__ __forceinline__ int64_t wave_sum_i64(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Every workgroup sums the wishes of the requests in front of its own (8 bytes each, from the cache: cheaper than a launch that scans
// them first) while its first wave scans its own; then its threads walk the group's pages and tokens as one flat range, so that one long
// prompt among many short requests keeps all of them busy.  blockIdx.y splits the tokens of a group further.
// Bound by latency: two reads from the cache and two barriers before the first slot is known.
// 128 requests of one token: 4.5 us; 2047 prompts with 1.05 M tokens (8.9 MB): 12 us, 24 us when a thread looked up one token at a time.
__global__ void __launch_bounds__(256) paged_plan_kernel(PlanParams p) {
  __shared__ int64_t red[2][4];
  __shared__ int tok_off[65], page_off[65];                // saturated at 2^31 - 1: nothing behind that is used
  __shared__ int s_cached[64], s_held[64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int b0 = blockIdx.x * p.per_group, nb = min(p.per_group, p.B - b0);
  const int cursor = max(*p.cursor_in, 0);
  int64_t tok = 0, pages = 0;
  int b = tid;
  for (; b + 768 < b0; b += 1024) {                        // (four at a time: the reads are independent)
    PlanRequest r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = plan_request(p, b + k * 256);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      tok += r[k].fresh;
      pages += r[k].need;
    }
  }
  for (; b < b0; b += 256) {
    const PlanRequest r = plan_request(p, b);
    tok += r.fresh;
    pages += r.need;
  }
  tok = wave_sum_i64(tok);
  pages = wave_sum_i64(pages);
  if (lane == 0) {
    red[0][tid >> 6] = tok;
    red[1][tid >> 6] = pages;
  }
  PlanRequest mine = {0, 0, 0, 0};
  if (tid < 64) {
    if (tid < nb) mine = plan_request(p, b0 + tid);
    int64_t a = mine.fresh, c = mine.need;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {                     // inclusive scan
      const int64_t ua = __shfl_up(a, o, 64), uc = __shfl_up(c, o, 64);
      if (lane >= o) {
        a += ua;
        c += uc;
      }
    }
    s_cached[tid] = mine.cached;
    s_held[tid] = mine.held;
    tok_off[tid + 1] = (int)min(a, (int64_t)0x7fffffff);
    page_off[tid + 1] = (int)min(c, (int64_t)0x7fffffff);
    if (tid == 0) tok_off[0] = page_off[0] = 0;
  }
  __syncthreads();
  const int64_t tok_base = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
  const int64_t page_base = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]) + cursor;
  const int n_tok = tok_off[nb], n_page = page_off[nb];
  auto find = [&](const int* off, int i) __attribute__((always_inline)) {   // last request whose range starts at or before i
    int lo = 0, hi = nb - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (off[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  if (blockIdx.y == 0) {
    if (tid < nb) {
      int64_t got = (int64_t)p.n_free - (page_base + page_off[tid]);
      got = got < 0 ? 0 : (got < mine.need ? got : mine.need);
      const int64_t room = max((int64_t)p.max_tokens - (tok_base + tok_off[tid]), (int64_t)0);       // slots left for its tokens
      const int64_t cap = (mine.held + got) * p.page.d, want = mine.cached + (mine.fresh < room ? mine.fresh : room);
      p.seq_lens[b0 + tid] = (int)(want < cap ? want : cap);
      p.cu_new[b0 + tid] = (int)(tok_base + tok_off[tid]);
    }
    const int64_t left = p.n_free - page_base;             // pages behind these do not exist: a senseless length costs no walk
    for (int64_t i = tid; i < n_page && i < left; i += 256) {
      // (an entry that names no page takes the place of whatever the row held here before: that page may be another request's by now)
      const int r = find(page_off, (int)i);
      p.table[(int64_t)(b0 + r) * p.table_stride + s_held[r] + (i - page_off[r])] = max(p.free_pages[page_base + i], -1);
    }
  }
  // (64 bits: the last step of a walk over nearly 2^31 tokens passes them; four tokens at a time, so that their pages are looked up together)
  const int64_t room = p.max_tokens - tok_base, stop = n_tok < room ? n_tok : room;
  auto entry_of = [&](int i, int& off) __attribute__((always_inline)) {
    const int r = find(tok_off, i);
    const int64_t pos = (int64_t)s_cached[r] + (i - tok_off[r]);
    off = 0;
    if (pos >= (int64_t)p.max_pages * p.page.d) return (const int32_t*)nullptr;
    const int j = (int)p.page.div((uint32_t)pos);
    off = (int)pos - j * (int)p.page.d;
    if (j < s_held[r]) return (const int32_t*)p.table + (int64_t)(b0 + r) * p.table_stride + j;
    const int64_t at = page_base + page_off[r] + (j - s_held[r]);
    return at < p.n_free ? p.free_pages + at : (const int32_t*)nullptr;
  };
  auto slot_of = [&](int page, int off) __attribute__((always_inline)) { return page < 0 ? (int64_t)-1 : (int64_t)page * p.page.d + off; };
  int64_t k = (int64_t)blockIdx.y * 1024 + tid;
  for (; k + 768 < stop; k += (int64_t)gridDim.y * 1024) {
    int page[4], off[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int32_t* e = entry_of((int)k + u * 256, off[u]);
      page[u] = e ? *e : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) p.slots[tok_base + k + u * 256] = slot_of(page[u], off[u]);
  }
  for (int u = 0; u < 4 && k < stop; ++u, k += 256) {
    int off;
    const int32_t* e = entry_of((int)k, off);
    const int page = e ? *e : -1;
    p.slots[tok_base + k] = slot_of(page, off);
  }
  if (b0 + nb == p.B) {
    const int64_t total = tok_base + n_tok;
    if (blockIdx.y == 0 && tid == 0) {
      p.cu_new[p.B] = (int)total;
      const int64_t at = page_base + n_page, most = cursor > p.n_free ? cursor : p.n_free;
      *p.cursor_out = (int)(at < most ? at : most);
    }
    for (int64_t i = total + (int64_t)blockIdx.y * 256 + tid; i < p.max_tokens; i += (int64_t)gridDim.y * 256) p.slots[i] = -1;
  }
}

// ---------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------
// A thread moves the same 16 bytes (or, where rows do not allow that, the same element) of a token's k and v row.  Bound by memory:
// 40961 tokens of 8 x 128 bf16 (335 MB read and written) 59 us, 5.7 TB/s; 128 tokens of 4 x 64 2.8 us, a launch.
struct AppendParams {
  const char *k, *v;
  char *kp, *vp;
  const int64_t* slots;
  int64_t T, n_slots;
  int H, row, page_size;                                    // heads, vectors of one head
  int64_t k_tok, k_head, v_tok, v_head;                     // bytes
  int64_t kp_page, kp_tok, kp_head, vp_page, vp_tok, vp_head;
};
template <typename V>
__global__ void __launch_bounds__(256) paged_append_kernel(AppendParams p) {
  const int per = p.H * p.row;
  const int64_t n = p.T * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per;
    const int c = (int)(i - t * per), h = c / p.row, e = c - h * p.row;
    const int64_t slot = p.slots[t];
    if (slot < 0 || slot >= p.n_slots) continue;
    const int64_t page = slot / p.page_size, at = slot - page * p.page_size;
    const V kv = *reinterpret_cast<const V*>(p.k + t * p.k_tok + h * p.k_head + (int64_t)e * sizeof(V));
    const V vv = *reinterpret_cast<const V*>(p.v + t * p.v_tok + h * p.v_head + (int64_t)e * sizeof(V));
    *reinterpret_cast<V*>(p.kp + page * p.kp_page + at * p.kp_tok + h * p.kp_head + (int64_t)e * sizeof(V)) = kv;
    *reinterpret_cast<V*>(p.vp + page * p.vp_page + at * p.vp_tok + h * p.vp_head + (int64_t)e * sizeof(V)) = vv;
  }
}

// ---------------------------------------------------------------------------------------------
// attention of one new token
// ---------------------------------------------------------------------------------------------
// A workgroup owns one part of one request's tokens for one key / value head and up to 16 of the query heads that share it; its four
// waves take tiles of 16 * NF tokens in turn, each with a running maximum and sum of its own, and are joined in LDS at the end.
// Parts of a request are joined by a second small kernel.
//   scores   S^T[token][head] = K . Q^T   the 16 x 16 accumulator block of a wave keeps, in lane l, head l & 15 and tokens 4 (l >> 4) + 0..3:
//   output   O^T[dim][head] += V^T . P^T  ... which is the operand layout of the second product, so the weights stay in registers.
// K goes from memory straight into operand registers (lane: token l & 15, 16 bytes of its row).  bf16: V rows go through LDS, because
// their operand needs 8 tokens of one dim per lane (ds_read_b64_tr_b16); f32: the 16x16x4 product takes ONE token per lane, so 16-byte
// pieces of V rows are operands as they come and nothing passes through LDS.  The waves never wait for each other inside the loop.
// A tile's rows are requested while the one before is multiplied, the page entries a tile earlier still.  All loads are unconditional: under
// masks the compiler loses count of what is in flight and drains everything at every wait (64 requests of 1 .. 8192 tokens: 1250 us).
// With one query head per key / value head 15 of 16 columns of the products are idle: the products take a twentieth of the time a tile
// needs to arrive, and vector code would have to unpack and multiply every element instead.
// Bound by memory: 64 requests of 1 .. 8192 tokens, 32 heads of 128 over 8, bf16 (1.07 GB): 220 us and 5 us for the join, 4.9 TB/s (equally
// long requests 5.4 .. 5.7); 24 requests of up to 2047 tokens, 8 heads of 64, f32 (105 MB): 27 + 4 us; 128 requests of up to 75
// tokens, 4 heads of 64: 5.4 us, the latency of length -> entry -> rows -> join.  More than 16 query heads for a key / value head read it
// once per 16.
constexpr int MIN_PART = 128;      // tokens: a tile for each wave; parts are multiples of it

__host__ __device__ __forceinline__ int part_tokens(int len, int nsplit) {
  const int even = (int)(((int64_t)len + nsplit - 1) / nsplit), p = (even + MIN_PART - 1) / MIN_PART * MIN_PART;
  return p < MIN_PART ? MIN_PART : p;
}

struct PagedAttnParams {
  const char *q, *k, *v;
  char* out;
  float* lse;
  const int32_t *table, *lens;
  int B, H, Hkv, dh, page_size, num_pages, max_pages;
  int64_t q_row, q_head, o_row, o_head, table_stride;               // elements
  uint32_t k_page, k_tok, v_page, v_tok;                            // elements, below 2^31
  int64_t k_head, v_head;
  float scale_log2;
  int nsplit, qchunks, by_xcd;
  FastDiv page;
  float* part_ml;          // [B * H][nsplit][2]: maximum and sum of a part
  float* part_o;           // [B * H][nsplit][dh rounded up to 4]: its output
};

template <typename T>
struct PA;
template <>
struct PA<bf16_t> { static constexpr int E = 8; };
template <>
struct PA<float> { static constexpr int E = 4; };

// 16 bytes of a row from element d on.  A piece behind the row's end (d >= dh) repeats its first one: the loads have no masks, so that
// the compiler can keep count of what is in flight; what they may not contribute is zeroed where it is used.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 row_chunk(const T* row, int d, int dh) {
  if (VEC) return *reinterpret_cast<const uint4*>(row + (d < dh ? d : 0));
  T e[PA<T>::E];
#pragma unroll
  for (int i = 0; i < PA<T>::E; ++i) {
    const T v = row[d + i < dh ? d + i : 0];
    e[i] = d + i < dh ? v : T(0);
  }
  uint4 r;
  memcpy(&r, e, 16);
  return r;
}
__device__ __forceinline__ uint4 keep_if(uint4 v, bool ok) { return make_uint4(ok ? v.x : 0u, ok ? v.y : 0u, ok ? v.z : 0u, ok ? v.w : 0u); }

// DP: head size padded to the tile (32, 64, 128, 256); NF: 16-token blocks of a tile
// VEC: rows are whole 16-byte pieces; EXACT: dh == DP
template <typename T, int DP, int NF, bool VEC, bool EXACT>
__global__ void __launch_bounds__(256) paged_attn_kernel(PagedAttnParams p) {
  const int dh = EXACT ? DP : p.dh;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int TK = 16 * NF;                          // tokens of a tile
  constexpr int RSV = DP * 2 + 32;                     // LDS row of V (bf16): rows spread over the banks for the transpose read
  constexpr int KC = DP * (int)sizeof(T) / 64;         // 16-byte pieces of a K row per lane
  constexpr int VC = BF ? TK * DP / 8 / 64 : 0;        // 16-byte pieces of the V tile per lane
  constexpr int NA = DP / 16;                          // accumulator blocks
  constexpr int WAVE_BYTES = BF ? TK * RSV : 0, JOIN_BYTES = 4 * 16 * (DP + 4) * 4;
  constexpr int LDS_BYTES = 4 * WAVE_BYTES > JOIN_BYTES ? 4 * WAVE_BYTES : JOIN_BYTES;
  __shared__ __attribute__((aligned(16))) char lds[LDS_BYTES];
  __shared__ float s_ml[2][4][16];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, lc = lane & 15;
  const int heads = p.Hkv * p.qchunks;
  int hq = blockIdx.x % heads, rest = blockIdx.x / heads;
  if (p.by_xcd) {          // (see paged_attention_by_xcd)
    const int turn = blockIdx.x >> 3;
    hq = turn % heads;
    rest = turn / heads * 8 + (blockIdx.x & 7);
    if (rest >= p.B * p.nsplit) return;
  }
  const int split = rest % p.nsplit, b = rest / p.nsplit;
  const int hk = hq / p.qchunks, qc = hq % p.qchunks, group = p.H / p.Hkv;
  const int h0 = hk * group + qc * 16, nh = min(16, group - qc * 16);
  const int cap = p.max_pages * p.page_size;
  const int len = min(max(p.lens[b], 0), cap);
  const int part = part_tokens(len, p.nsplit), t_begin = split * part, t_end = min(len, t_begin + part);
  if (t_begin >= len && (p.nsplit > 1 || len > 0)) return;      // (an empty request with one part writes its zeros below)
  const int32_t* table = p.table + (int64_t)b * p.table_stride;
  const T* kbase = (const T*)p.k + hk * p.k_head;
  const T* vbase = (const T*)p.v + hk * p.v_head;

  uint4 qf[KC];
  {
    const T* q = (const T*)p.q + (int64_t)b * p.q_row + (int64_t)(h0 + min(lc, nh - 1)) * p.q_head;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int d = c * (64 / (int)sizeof(T)) + g * PA<T>::E;
      qf[c] = keep_if(row_chunk<T, VEC>(q, d, dh), lc < nh && d < dh);
    }
  }
  floatx4_t acc[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) acc[i] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  float m = LOWEST, l = 0.f;
  uint4 kr[NF][KC], vr[BF ? VC : NF * 4 * (DP / 64 > 0 ? DP / 64 : 1)];

  // Lane i looks up the page of token t0 + i % TK.  The entry is checked where it is used, a tile later: a check here would wait for it,
  // and with it for all rows requested before.
  const int tl = lane % TK;
  auto look = [&](int t0, int& entry, int& off) __attribute__((always_inline)) {
    const int t = min(t0 + tl, t_end - 1);
    const int j = (int)p.page.div((uint32_t)t);
    off = t - j * p.page_size;
    entry = table[j];
  };
  // page of this lane's token, 0 (whose rows exist) with the token out of `valid` when it has none
  auto resolve = [&](int t0, int entry, uint64_t& valid) __attribute__((always_inline)) {
    const bool ok = t0 + tl < t_end && entry >= 0 && entry < p.num_pages;
    valid = __ballot(ok);
    return ok ? entry : 0;
  };
  auto load_k = [&](int page, int off) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const uint32_t pg = __shfl(page, f * 16 + lc, 64), of = __shfl(off, f * 16 + lc, 64);
      const T* row = kbase + ((uint64_t)pg * p.k_page + (uint64_t)of * p.k_tok);
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[f][c] = row_chunk<T, VEC>(row, c * (64 / (int)sizeof(T)) + g * PA<T>::E, dh);
    }
  };
  auto load_v = [&](int page, int off) __attribute__((always_inline)) {
    if constexpr (BF) {
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        const int r = (i * 64 + lane) / (DP / 8), col = (i * 64 + lane) % (DP / 8);
        const uint32_t pg = __shfl(page, r, 64), of = __shfl(off, r, 64);
        vr[i] = row_chunk<T, VEC>(vbase + ((uint64_t)pg * p.v_page + (uint64_t)of * p.v_tok), col * 8, dh);
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = f * 16 + g * 4 + r;
          const uint32_t pg = __shfl(page, key, 64), of = __shfl(off, key, 64);
          const T* row = vbase + ((uint64_t)pg * p.v_page + (uint64_t)of * p.v_tok);
#pragma unroll
          for (int c = 0; c < DP / 64; ++c) vr[(f * 4 + r) * (DP / 64) + c] = row_chunk<T, VEC>(row, c * 64 + lc * 4, dh);
        }
    }
  };
  constexpr uint64_t ALL = ~0ull;      // (lanes i and i + TK hold the same token)

  char* vt = lds + wave * WAVE_BYTES;
  int t0 = t_begin + wave * TK;
  uint64_t next_valid = 0;
  int entry, off;
  if (t0 < t_end) {
    look(t0, entry, off);
    const int page = resolve(t0, entry, next_valid);
    const int o = off;
    look(t0 + 4 * TK, entry, off);
    load_k(page, o);
    load_v(page, o);
  }
  for (; t0 < t_end; t0 += 4 * TK) {
    const uint64_t valid = next_valid;
    // ---- S^T = K . Q^T
    floatx4_t s[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      s[f] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        uint4 kc = kr[f][c];
        if (VEC && !EXACT) kc = keep_if(kc, c * (64 / (int)sizeof(T)) + g * PA<T>::E < dh);
        if constexpr (BF) {
          s[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kc), __builtin_bit_cast(bf16x8_t, qf[c]), s[f], 0, 0, 0);
        } else {
          const floatx4_t a = __builtin_bit_cast(floatx4_t, kc), q4 = __builtin_bit_cast(floatx4_t, qf[c]);
#pragma unroll
          for (int j = 0; j < 4; ++j) s[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], q4[j], s[f], 0, 0, 0);
        }
      }
    }
    // ---- this tile's V out of the load registers (rows that are no tokens as zeros: their weight is 0, but what lies there may be NaN)
    if (valid != ALL) {
      if constexpr (BF) {
#pragma unroll
        for (int i = 0; i < VC; ++i) vr[i] = keep_if(vr[i], (valid >> ((i * 64 + lane) / (DP / 8))) & 1);
      } else {
#pragma unroll
        for (int i = 0; i < NF * 4 * (DP / 64); ++i) {
          const int r = i / (DP / 64);
          vr[i] = keep_if(vr[i], (valid >> ((r >> 2) * 16 + g * 4 + (r & 3))) & 1);
        }
      }
    }
    if constexpr (BF) {
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        const int r = (i * 64 + lane) / (DP / 8), col = (i * 64 + lane) % (DP / 8);
        *reinterpret_cast<uint4*>(vt + r * RSV + col * 16) = vr[i];
      }
    }
    // ---- the next tile's rows on their way, and the pages of the one behind it (past the end: rows and entries that exist, unused).
    // f32 keeps V in its load registers until the second product: a copy would cost half of the waves a SIMD can hold
    const int next_page = resolve(t0 + 4 * TK, entry, next_valid), next_off = off;
    look(t0 + 8 * TK, entry, off);
    load_k(next_page, next_off);
    if constexpr (BF) load_v(next_page, next_off);
    // ---- weights
    float mx = -INFINITY;
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[f][r] = s[f][r] * p.scale_log2;
        if (valid != ALL) s[f][r] = (valid >> (f * 16 + g * 4 + r)) & 1 ? s[f][r] : -INFINITY;
        mx = fmaxf(mx, s[f][r]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx), back = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[f][r] = __builtin_amdgcn_exp2f(s[f][r] - mn);
        sum += s[f][r];
      }
    l = l * back + sum;
#pragma unroll
    for (int i = 0; i < NA; ++i) acc[i] *= back;
    // ---- O^T += V^T . P^T
    if constexpr (BF) {
      static_assert(NF == 2 || !BF, "a bf16 product takes 32 tokens");
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      typedef short4_t __attribute__((address_space(3))) * lds_ptr_t;
      // a weight is the sum of two bf16 numbers: rounded to one it would add as much error to the output as the output's own rounding
      // (6.3e-4 against 5.0e-4 of the largest value over 64 requests), and the second product is free, the kernel waits for memory
      union { uint32_t u[4]; bf16x8_t f; } w, rest;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = s[i < 2 ? 0 : NF - 1][(i & 1) * 2], y = s[i < 2 ? 0 : NF - 1][(i & 1) * 2 + 1];
        w.u[i] = pack_bf16x2(x, y);
        rest.u[i] = pack_bf16x2(x - __uint_as_float(w.u[i] << 16), y - __uint_as_float(w.u[i] & 0xffff0000u));
      }
      const char* base = vt + (g * 4 + (lc >> 2)) * RSV + (lc & 3) * 8;
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        union { short4_t h[2]; bf16x8_t f; } a;
        a.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr_t)(base + i * 32));
        a.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr_t)(base + i * 32 + 16 * RSV));
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.f, w.f, acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.f, rest.f, acc[i], 0, 0, 0);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[c * 4 + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(floatx4_t, vr[(f * 4 + r) * (DP / 64) + c])[j], s[f][r],
                                                                    acc[c * 4 + j], 0, 0, 0);
      load_v(next_page, next_off);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  // ---- join the waves: O[wave][head][dim] in LDS
  __syncthreads();
  float* jo = reinterpret_cast<float*>(lds);
  if (lane < 16) {
    s_ml[0][wave][lc] = m;
    s_ml[1][wave][lc] = l;
  }
  if (lc < nh) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // f32: block c * 4 + j holds dims c * 64 + 4 * row + j
        const int d = BF ? i * 16 + g * 4 + r : (i >> 2) * 64 + 4 * (g * 4 + r) + (i & 3);
        jo[(wave * 16 + lc) * (DP + 4) + d] = acc[i][r];
      }
  }
  __syncthreads();
  for (int e = tid; e < nh * DP; e += 256) {
    const int h = e / DP, d = e % DP;
    if (d >= dh) continue;
    const float mj = fmaxf(fmaxf(s_ml[0][0][h], s_ml[0][1][h]), fmaxf(s_ml[0][2][h], s_ml[0][3][h]));
    float lj = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float c = __builtin_amdgcn_exp2f(s_ml[0][w][h] - mj);
      lj += c * s_ml[1][w][h];
      o += c * jo[(w * 16 + h) * (DP + 4) + d];
    }
    const int64_t row = (int64_t)b * p.H + h0 + h;
    if (p.nsplit > 1) {
      const int64_t at = row * p.nsplit + split;
      p.part_o[at * ((dh + 3) & ~3) + d] = o;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mj, lj);
    } else {
      ((T*)p.out)[b * p.o_row + (h0 + h) * p.o_head + d] = from_f32<T>(lj == 0.f ? 0.f : o / lj);
      if (d == 0 && p.lse) p.lse[row] = lj == 0.f ? -INFINITY : (mj + log2f(lj)) * LN2;
    }
  }
}

// Joins the parts of a request: one workgroup per (request, head).  The weights of all parts first (they need every maximum), then threads
// of four dims each share the parts, eight reads of each in flight: with 256 parts this is all the time there is.
constexpr int MAX_SPLITS = 2048;
template <typename T>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(PagedAttnParams p) {
  __shared__ float s_w[MAX_SPLITS], s_red[2][4];
  __shared__ float4 s_o[256];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const int b = (int)(row / p.H), h = (int)(row - (int64_t)b * p.H);
  const int len = min(max(p.lens[b], 0), p.max_pages * (int)p.page.d);
  const int part = part_tokens(len, p.nsplit), n = (int)(((int64_t)len + part - 1) / part);
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row * p.nsplit;
  float m = LOWEST;
  for (int i = tid; i < n; i += 256) m = fmaxf(m, ml[i].x);
  m = wave_max(m);
  if (lane == 0) s_red[0][wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  float l = 0.f;
  for (int i = tid; i < n; i += 256) {
    const float2 v = ml[i];
    const float w = __builtin_amdgcn_exp2f(v.x - m);
    s_w[i] = w;
    l += w * v.y;
  }
  l = wave_sum(l);
  if (lane == 0) s_red[1][wave] = l;
  __syncthreads();
  l = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  const int dv = (p.dh + 3) / 4;                           // threads of one part (<= 64); `groups` parts at a time
  const int groups = 256 / dv, grp = tid / dv, c = tid - grp * dv;
  const float4* src = reinterpret_cast<const float4*>(p.part_o) + row * p.nsplit * dv + c;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < groups) {
    for (int i = grp; i < n; i += groups * 8) {
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = src[(int64_t)min(i + k * groups, n - 1) * dv];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = i + k * groups < n ? s_w[i + k * groups] : 0.f;
        o.x += w * v[k].x; o.y += w * v[k].y; o.z += w * v[k].z; o.w += w * v[k].w;
      }
    }
  }
  s_o[tid] = o;
  __syncthreads();
  if (tid < dv) {
    for (int k = 1; k < groups; ++k) {
      const float4 v = s_o[k * dv + tid];
      o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
    }
    const float r[4] = {o.x, o.y, o.z, o.w};
    T* dst = (T*)p.out + b * p.o_row + h * p.o_head + tid * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (tid * 4 + k < p.dh) dst[k] = from_f32<T>(l == 0.f ? 0.f : r[k] / l);
  }
  if (tid == 0 && p.lse) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// The same for at most FEW_SPLITS parts: a wave for each (request, head), no barriers; lane i weighs part i.
constexpr int FEW_SPLITS = 16;
template <typename T>
__global__ void __launch_bounds__(256) paged_attn_join_few_kernel(PagedAttnParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)p.B * p.H) return;
  const int b = (int)(row / p.H), h = (int)(row - (int64_t)b * p.H);
  const int len = min(max(p.lens[b], 0), p.max_pages * (int)p.page.d);
  const int part = part_tokens(len, p.nsplit), n = (int)(((int64_t)len + part - 1) / part);
  const float2 ml = lane < n ? reinterpret_cast<const float2*>(p.part_ml)[row * p.nsplit + lane] : make_float2(LOWEST, 0.f);
  const int dv = (p.dh + 3) / 4, groups = 64 / dv, grp = lane / dv, c = lane - grp * dv;
  const float4* src = reinterpret_cast<const float4*>(p.part_o) + row * p.nsplit * dv + c;
  float4 v[4], o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto fetch = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = src[(int64_t)min(k + u * groups + min(grp, groups - 1), max(n - 1, 0)) * dv];
  };
  fetch(0);                                                // (on its way while the weights are found)
  const float m = wave_max(ml.x), w = __builtin_amdgcn_exp2f(ml.x - m), l = wave_sum_fast(w * ml.y);
  for (int k = 0; k < n; k += groups * 4) {
    if (k > 0) fetch(k);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = k + u * groups + grp;
      const float wi = __shfl(w, min(i, 63), 64);
      if (i < n && grp < groups) {
        o.x += wi * v[u].x; o.y += wi * v[u].y; o.z += wi * v[u].z; o.w += wi * v[u].w;
      }
    }
  }
  float4 sum = o;
  for (int k = 1; k < groups; ++k) {
    const int from = min(c + k * dv, 63);
    sum.x += __shfl(o.x, from, 64); sum.y += __shfl(o.y, from, 64); sum.z += __shfl(o.z, from, 64); sum.w += __shfl(o.w, from, 64);
  }
  if (lane < dv) {
    const float r[4] = {sum.x, sum.y, sum.z, sum.w};
    T* dst = (T*)p.out + b * p.o_row + h * p.o_head + lane * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane * 4 + k < p.dh) dst[k] = from_f32<T>(l == 0.f ? 0.f : r[k] / l);
  }
  if (lane == 0 && p.lse) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

template <typename T>
void paged_attn_join(const PagedAttnParams& p, hipStream_t st) {
  const int rows = p.B * p.H;
  if (p.nsplit <= FEW_SPLITS) paged_attn_join_few_kernel<T><<<(rows + 3) / 4, 256, 0, st>>>(p);
  else paged_attn_join_kernel<T><<<rows, 256, 0, st>>>(p);
}

template <typename T, int DP, int NF>
void paged_attn_launch(const PagedAttnParams& p, bool vec, unsigned grid, hipStream_t st) {
  if (vec && p.dh == DP) paged_attn_kernel<T, DP, NF, true, true><<<grid, 256, 0, st>>>(p);
  else if (vec) paged_attn_kernel<T, DP, NF, true, false><<<grid, 256, 0, st>>>(p);
  else paged_attn_kernel<T, DP, NF, false, false><<<grid, 256, 0, st>>>(p);
}

// ---------------------------------------------------------------------------------------------
// reorder
// ---------------------------------------------------------------------------------------------
// One workgroup per row and plane; the first plane's also write the row's table.  Rows that continue themselves leave at once.  Bound by memory:
// 256 rows of 512 bf16 in pages of 32, 12 planes (92 MB): 16 us, 5.7 TB/s; 128 rows of 256 in pages of 16: 4.6 us.
struct ReorderParams {
  char* pool;
  int planes, page_size, num_pages, max_pages, R;
  int64_t plane_stride, page_stride;     // bytes
  int64_t tok_bytes;                     // bytes of one token row (pages are dense)
  const int32_t* table_in;
  int32_t* table_out;
  int64_t in_stride, out_stride;
  const int32_t* lens;
  const int64_t* parents;
  const int32_t* spare_in;
  int32_t* spare_out;
};
struct ReorderRow {
  int64_t parent;
  int len, src, dst;     // src >= 0: copy the filled part of page src into page dst
};
// A row whose parent does not exist or has another length keeps its own sequence.
__device__ __forceinline__ ReorderRow reorder_row(const ReorderParams& p, int r) {
  ReorderRow o;
  const int cap = p.max_pages * p.page_size;
  o.len = min(max(p.lens[r], 0), cap);
  o.parent = p.parents[r];
  if (o.parent < 0 || o.parent >= p.R || min(max(p.lens[o.parent], 0), cap) != o.len) o.parent = r;
  o.src = o.dst = -1;
  if (o.parent != r && o.len % p.page_size) {
    const int src = p.table_in[o.parent * p.in_stride + o.len / p.page_size], dst = p.spare_in[r];
    if (src >= 0 && src < p.num_pages && dst >= 0 && dst < p.num_pages) {
      o.src = src;
      o.dst = dst;
    } else {
      o.parent = r;
    }
  }
  return o;
}
template <typename V>
__global__ void __launch_bounds__(256) paged_reorder_kernel(ReorderParams p) {
  const int r = blockIdx.x, tid = threadIdx.x;
  const ReorderRow row = reorder_row(p, r);
  if (blockIdx.y == 0) {
    const int used = (row.len + p.page_size - 1) / p.page_size, last = row.len / p.page_size;
    for (int j = tid; j < p.max_pages; j += 256) {
      int page = j < used ? p.table_in[row.parent * p.in_stride + j] : -1;
      if (row.src >= 0 && j == last) page = row.dst;
      p.table_out[r * p.out_stride + j] = page;
    }
    if (tid == 0) p.spare_out[r] = row.src >= 0 ? p.table_in[r * p.in_stride + last] : p.spare_in[r];
  }
  if (row.src < 0) return;
  const int64_t n = (int64_t)(row.len % p.page_size) * p.tok_bytes / sizeof(V);
  const int64_t base = blockIdx.y * p.plane_stride;
  const V* src = reinterpret_cast<const V*>(p.pool + base + row.src * p.page_stride);
  V* dst = reinterpret_cast<V*>(p.pool + base + row.dst * p.page_stride);
  for (int64_t i = tid; i < n; i += 256) dst[i] = src[i];
}

}  // namespace

// ---------------------------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------------------------
extern "C" int nst_paged_plan(const int32_t* cached_lens, const int32_t* new_lens, int B, int32_t* block_table, int64_t table_stride,
                              int max_pages, const int32_t* free_pages, int n_free, const int32_t* cursor_in, int page_size,
                              int64_t* slots, int64_t max_tokens, int32_t* seq_lens, int32_t* cu_new, int32_t* cursor_out,
                              void* stream) {
  NST_CHECK_ARG(B >= 0 && max_pages > 0 && page_size > 0 && n_free >= 0 && max_tokens >= 0,
                "nst_paged_plan: B=%d max_pages=%d page_size=%d n_free=%d max_tokens=%lld", B, max_pages, page_size, n_free,
                (long long)max_tokens);
  NST_CHECK_ARG((int64_t)max_pages * page_size <= MAX_POSITIONS, "nst_paged_plan: %d pages of %d tokens pass 2^30 positions", max_pages,
                page_size);
  NST_CHECK_ARG(max_tokens <= 0x7fffffffLL, "nst_paged_plan: max_tokens=%lld (at most 2^31 - 1)", (long long)max_tokens);
  NST_CHECK_ARG(cursor_in && cu_new && cursor_out && (slots || max_tokens == 0) && (free_pages || n_free == 0),
                "nst_paged_plan: NULL pointer");
  NST_CHECK_ARG(B == 0 || (cached_lens && new_lens && block_table && seq_lens && table_stride >= max_pages),
                "nst_paged_plan: NULL pointer or table stride %lld < %d", (long long)table_stride, max_pages);
  NST_CHECK_ARG(cursor_in != cursor_out && (B == 0 || (seq_lens != cached_lens && seq_lens != new_lens)),
                "nst_paged_plan: the outputs may not overlap the inputs (other workgroups still read them)");
  PlanParams p = {cached_lens, new_lens, B, max_pages, fast_div(page_size), block_table, table_stride, free_pages, n_free, cursor_in,
                  slots, (int)max_tokens, seq_lens, cu_new, cursor_out, 1};
  int64_t per = max_tokens > 0 ? (1024LL * B + max_tokens - 1) / max_tokens : 64;      // about 1024 tokens for a workgroup
  p.per_group = (int)(per < 1 ? 1 : per > 64 ? 64 : per);
  const int gx = B > 0 ? (B + p.per_group - 1) / p.per_group : 1;
  int64_t gy = max_tokens / ((int64_t)gx * 1024);
  gy = gy < 1 ? 1 : gy > 64 ? 64 : gy;
  paged_plan_kernel<<<dim3(gx, (unsigned)gy), 256, 0, (hipStream_t)stream>>>(p);
  NST_CHECK_LAUNCH("nst_paged_plan");
  return NST_OK;
}

extern "C" int nst_paged_append(const void* k, const void* v, int64_t tokens, int kv_heads, int dh, int64_t k_token_stride,
                                int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, void* k_pool, void* v_pool,
                                const NstPagedPool* pool, const int64_t* slots, void* stream) {
  NST_CHECK_ARG(pool && tokens >= 0 && kv_heads > 0 && dh > 0, "nst_paged_append: tokens=%lld kv_heads=%d dh=%d", (long long)tokens,
                kv_heads, dh);
  NST_CHECK_ARG(pool->dtype == NST_F32 || pool->dtype == NST_BF16, "nst_paged_append: dtype %d", pool->dtype);
  NST_CHECK_ARG(pool->page_size > 0 && pool->num_pages >= 0, "nst_paged_append: %d pages of %d tokens", pool->num_pages, pool->page_size);
  if (tokens == 0 || pool->num_pages == 0) return NST_OK;
  NST_CHECK_ARG(k && v && k_pool && v_pool && slots, "nst_paged_append: NULL pointer");
  const int64_t es = nst_dtype_size(pool->dtype);
  AppendParams p;
  p.k = (const char*)k; p.v = (const char*)v; p.kp = (char*)k_pool; p.vp = (char*)v_pool;
  p.slots = slots; p.T = tokens; p.n_slots = (int64_t)pool->num_pages * pool->page_size;
  p.H = kv_heads; p.page_size = pool->page_size;
  const int64_t st[10] = {k_token_stride, k_head_stride, v_token_stride, v_head_stride, pool->k_page_stride, pool->k_token_stride,
                          pool->k_head_stride, pool->v_page_stride, pool->v_token_stride, pool->v_head_stride};
  int64_t* to[10] = {&p.k_tok, &p.k_head, &p.v_tok, &p.v_head, &p.kp_page, &p.kp_tok, &p.kp_head, &p.vp_page, &p.vp_tok, &p.vp_head};
  bool wide = nst_aligned16(k) && nst_aligned16(v) && nst_aligned16(k_pool) && nst_aligned16(v_pool) && (dh * es) % 16 == 0;
  for (int i = 0; i < 10; ++i) {
    *to[i] = st[i] * es;
    wide = wide && (st[i] * es) % 16 == 0;
  }
  p.row = wide ? (int)(dh * es / 16) : dh;
  const int64_t n = tokens * kv_heads * p.row, blocks = (n + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
  hipStream_t st_ = (hipStream_t)stream;
  if (wide) paged_append_kernel<uint4><<<grid, 256, 0, st_>>>(p);
  else if (es == 4) paged_append_kernel<uint32_t><<<grid, 256, 0, st_>>>(p);
  else paged_append_kernel<uint16_t><<<grid, 256, 0, st_>>>(p);
  NST_CHECK_LAUNCH("nst_paged_append");
  return NST_OK;
}

static int paged_attention_check(const NstPagedAttnDesc* d) {
  NST_CHECK_ARG(d, "nst_paged_attention: NULL descriptor");
  const NstPagedPool& pl = d->pool;
  NST_CHECK_ARG(pl.dtype == NST_F32 || pl.dtype == NST_BF16, "nst_paged_attention: dtype %d", pl.dtype);
  NST_CHECK_ARG(d->B >= 0 && d->H > 0 && d->Hkv > 0 && d->H % d->Hkv == 0, "nst_paged_attention: B=%d, %d heads over %d key / value heads",
                d->B, d->H, d->Hkv);
  NST_CHECK_ARG(d->dh > 0 && d->dh <= 256, "nst_paged_attention: head size %d (1 .. 256)", d->dh);
  NST_CHECK_ARG(pl.page_size > 0 && pl.num_pages >= 0 && d->max_pages > 0 && d->table_stride >= d->max_pages && d->max_len >= 0,
                "nst_paged_attention: page_size=%d num_pages=%d max_pages=%d table stride %lld max_len=%d", pl.page_size, pl.num_pages,
                d->max_pages, (long long)d->table_stride, d->max_len);
  NST_CHECK_ARG((int64_t)d->max_pages * pl.page_size <= MAX_POSITIONS, "nst_paged_attention: %d pages of %d tokens pass 2^30 positions",
                d->max_pages, pl.page_size);
  const int64_t rows[4] = {pl.k_page_stride, pl.k_token_stride, pl.v_page_stride, pl.v_token_stride};
  for (int i = 0; i < 4; ++i)
    NST_CHECK_ARG(rows[i] >= 0 && rows[i] <= 0x7fffffffLL, "nst_paged_attention: page or token stride %lld (0 .. 2^31 - 1 elements)",
                  (long long)rows[i]);
  NST_CHECK_ARG((int64_t)d->B * d->H <= 0x7fffffffLL, "nst_paged_attention: %d x %d rows", d->B, d->H);
  return NST_OK;
}

// How many parts a request is cut into at most.
//   768 workgroups: what the chip holds at once (three for a CU at 128 .. 168 registers).  24 x 8 float32 heads of up to 2047 tokens: 512 / 768
//     / 1024 / 2048 workgroups 36.7 / 32.4 / 34.0 / 35.3 us.
//   Parts of at most 2048 tokens, or the last long requests of a ragged batch run alone (64 requests of 1 .. 8192 tokens, 8 heads: 240 us
//     without this bound, 223 us with it, 230 us with half of it), and of at least 256 in a request as long as the bound (a shorter one of
//     the batch may come into as many parts, of at least MIN_PART tokens: part_tokens).
//   Up to 512 tokens a request stays whole (16 x 8 heads: 10.3 us, in parts with the second launch 12.1 us, and a launch less for the host;
//     up to 256 of float32 with tiles of 16 tokens: 29 x 2 heads of 80, 512 tokens 24.9 us whole, 18.8 in parts),
//     up to 1024 where there are 128 rows of heads or more (64 x 4: 14.0 against 18.7 us; 8 x 4: 18.3 against 11.6 us, so not for fewer).
static int paged_attention_splits(const NstPagedAttnDesc* d) {
  const int64_t cap = (int64_t)d->max_pages * d->pool.page_size, bound = d->max_len > 0 && d->max_len < cap ? d->max_len : cap;
  const int64_t units = (int64_t)d->B * d->Hkv * ((d->H / d->Hkv + 15) / 16);
  const int64_t whole = d->pool.dtype == NST_F32 && d->dh > 64 ? 256 : 512;
  if (bound <= whole || (bound <= 1024 && units >= 128)) return 1;
  const int64_t most = (bound + 255) / 256, few = (768 + units - 1) / units, ragged = (bound + 2047) / 2048;
  const int64_t want = few > ragged ? few : ragged, n = want < most ? want : most;
  return (int)(n > MAX_SPLITS ? MAX_SPLITS : n);
}

// Workgroups go to the eight XCDs in turn.  All heads of a part of a request on ONE of them find in its cache what their rows share: cache lines,
// where a head's row is not a multiple of 128 bytes (16 requests, 8 heads of 40 bf16: 90 -> 57 us; 32 requests, 8 heads of 32: 88 -> 54 us),
// and whole rows, where more than 16 query heads read them (128 over one, 256 wide: 314 -> 221 us); others do not care (64 x 8 heads of 128:
// 396, 392 us).  From 64 parts on: below, eight XCDs would have unequally many.
static bool paged_attention_by_xcd(int64_t parts) { return parts >= 64; }

static int64_t paged_attention_ml_bytes(const NstPagedAttnDesc* d, int nsplit) {      // (the outputs behind it start 16-byte aligned)
  return ((int64_t)d->B * d->H * nsplit * 8 + 15) / 16 * 16;
}
static int64_t paged_attention_workspace(const NstPagedAttnDesc* d, int nsplit) {
  return nsplit > 1 ? paged_attention_ml_bytes(d, nsplit) + (int64_t)d->B * d->H * nsplit * ((d->dh + 3) / 4 * 16) : 0;
}

extern "C" int64_t nst_paged_attention_workspace_bytes(const NstPagedAttnDesc* d) {
  const int rc = paged_attention_check(d);
  if (rc != NST_OK) return rc;
  return d->B > 0 ? paged_attention_workspace(d, paged_attention_splits(d)) : 0;
}

extern "C" int nst_paged_attention(const NstPagedAttnDesc* d, const void* q, const void* k_pool, const void* v_pool,
                                   const int32_t* block_table, const int32_t* seq_lens, void* out, float* lse, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  const int rc = paged_attention_check(d);
  if (rc != NST_OK) return rc;
  if (d->B == 0) return NST_OK;
  NST_CHECK_ARG(q && block_table && seq_lens && out && ((k_pool && v_pool) || d->pool.num_pages == 0), "nst_paged_attention: NULL pointer");
  const NstPagedPool& pl = d->pool;
  PagedAttnParams p;
  memset(&p, 0, sizeof(p));
  p.q = (const char*)q; p.k = (const char*)k_pool; p.v = (const char*)v_pool; p.out = (char*)out; p.lse = lse;
  p.table = block_table; p.lens = seq_lens;
  p.B = d->B; p.H = d->H; p.Hkv = d->Hkv; p.dh = d->dh;
  p.page_size = pl.page_size; p.num_pages = pl.num_pages; p.max_pages = d->max_pages;
  p.q_row = d->q_row_stride; p.q_head = d->q_head_stride; p.o_row = d->o_row_stride; p.o_head = d->o_head_stride;
  p.table_stride = d->table_stride;
  if (pl.num_pages > 0) {
    p.k_page = (uint32_t)pl.k_page_stride; p.k_tok = (uint32_t)pl.k_token_stride; p.k_head = pl.k_head_stride;
    p.v_page = (uint32_t)pl.v_page_stride; p.v_tok = (uint32_t)pl.v_token_stride; p.v_head = pl.v_head_stride;
  } else {
    p.k = p.v = p.q;       // no page exists: every row the kernel touches (and ignores) is the first row of q
  }
  p.scale_log2 = d->scale * LOG2E;
  p.qchunks = (d->H / d->Hkv + 15) / 16;
  p.nsplit = paged_attention_splits(d);
  p.page = fast_div(pl.page_size);
  if (p.nsplit > 1) {
    const int64_t need = paged_attention_workspace(d, p.nsplit);
    if (!workspace || workspace_bytes < need || !nst_aligned16(workspace)) {
      nst_set_error("nst_paged_attention: workspace of %lld bytes, needs %lld (16-byte aligned)", (long long)workspace_bytes, (long long)need);
      return NST_ERR_WORKSPACE;
    }
    p.part_ml = (float*)workspace;
    p.part_o = (float*)((char*)workspace + paged_attention_ml_bytes(d, p.nsplit));
  }
  const int64_t parts = (int64_t)d->B * p.nsplit;
  p.by_xcd = paged_attention_by_xcd(parts);
  const int64_t blocks = (p.by_xcd ? (parts + 7) / 8 * 8 : parts) * d->Hkv * p.qchunks;
  NST_CHECK_ARG(blocks <= 0x7fffffffLL, "nst_paged_attention: %lld workgroups", (long long)blocks);
  const int es = nst_dtype_size(pl.dtype);
  bool vec = nst_aligned16(q) && nst_aligned16(p.k) && nst_aligned16(p.v) && (d->dh * es) % 16 == 0;
  const int64_t strides[8] = {p.q_row, p.q_head, p.k_page, p.k_tok, p.k_head, p.v_page, p.v_tok, p.v_head};
  for (int i = 0; i < 8; ++i) vec = vec && (strides[i] * es) % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)blocks;
  if (pl.dtype == NST_BF16) {
    if (d->dh <= 32) paged_attn_launch<bf16_t, 32, 2>(p, vec, grid, st);
    else if (d->dh <= 64) paged_attn_launch<bf16_t, 64, 2>(p, vec, grid, st);
    else if (d->dh <= 128) paged_attn_launch<bf16_t, 128, 2>(p, vec, grid, st);
    else paged_attn_launch<bf16_t, 256, 2>(p, vec, grid, st);
  } else {
    // (tiles of 16 tokens from 65 on: with 32 a wave needs more than 256 registers and a SIMD holds one; 13 x 8 heads of 80: 78, 61 us)
    if (d->dh <= 64) paged_attn_launch<float, 64, 2>(p, vec, grid, st);
    else if (d->dh <= 128) paged_attn_launch<float, 128, 1>(p, vec, grid, st);
    else paged_attn_launch<float, 256, 1>(p, vec, grid, st);
  }
  if (p.nsplit > 1) {
    NST_CHECK_LAUNCH("nst_paged_attention");
    if (pl.dtype == NST_BF16) paged_attn_join<bf16_t>(p, st);
    else paged_attn_join<float>(p, st);
  }
  NST_CHECK_LAUNCH("nst_paged_attention");
  return NST_OK;
}

extern "C" int nst_paged_reorder(void* pool, int planes, int64_t plane_stride, int num_pages, int64_t page_stride, int page_size,
                                 int64_t token_bytes, const int32_t* table_in, int64_t in_stride, int32_t* table_out,
                                 int64_t out_stride, int max_pages, int rows, const int32_t* seq_lens, const int64_t* parents,
                                 const int32_t* spare_in, int32_t* spare_out, void* stream) {
  NST_CHECK_ARG(planes > 0 && planes <= 65535 && num_pages >= 0 && page_size > 0 && token_bytes > 0 && max_pages > 0 && rows >= 0,
                "nst_paged_reorder: planes=%d num_pages=%d page_size=%d token_bytes=%lld max_pages=%d rows=%d", planes, num_pages,
                page_size, (long long)token_bytes, max_pages, rows);
  NST_CHECK_ARG((int64_t)max_pages * page_size <= MAX_POSITIONS, "nst_paged_reorder: %d pages of %d tokens pass 2^30 positions", max_pages,
                page_size);
  NST_CHECK_ARG(page_stride >= token_bytes * page_size || num_pages <= 1, "nst_paged_reorder: pages of %lld bytes %lld bytes apart",
                (long long)(token_bytes * page_size), (long long)page_stride);
  if (rows == 0) return NST_OK;
  NST_CHECK_ARG((pool || num_pages == 0) && table_in && table_out && seq_lens && parents && spare_in && spare_out,
                "nst_paged_reorder: NULL pointer");
  NST_CHECK_ARG(in_stride >= max_pages && out_stride >= max_pages, "nst_paged_reorder: table strides %lld / %lld < %d", (long long)in_stride,
                (long long)out_stride, max_pages);
  NST_CHECK_ARG(table_in != table_out && spare_in != spare_out, "nst_paged_reorder: the outputs may not overlap the inputs");
  ReorderParams p = {(char*)pool, planes, page_size, num_pages, max_pages, rows, plane_stride, page_stride, token_bytes,
                     table_in, table_out, in_stride, out_stride, seq_lens, parents, spare_in, spare_out};
  const dim3 grid(rows, planes);
  hipStream_t st = (hipStream_t)stream;
  const int64_t all = (int64_t)(uintptr_t)pool | plane_stride | page_stride | token_bytes;
  if (all % 16 == 0) paged_reorder_kernel<uint4><<<grid, 256, 0, st>>>(p);
  else if (all % 4 == 0) paged_reorder_kernel<uint32_t><<<grid, 256, 0, st>>>(p);
  else if (all % 2 == 0) paged_reorder_kernel<uint16_t><<<grid, 256, 0, st>>>(p);
  else paged_reorder_kernel<uint8_t><<<grid, 256, 0, st>>>(p);
  NST_CHECK_LAUNCH("nst_paged_reorder");
  return NST_OK;
}
