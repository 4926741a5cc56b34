// Paged key / value caches: page assignment from request lengths, rows to slots, attention of one new token over the pages,
// re-ordering behind a beam-search step.
//
// A cache holds `num_pages` pages of `page_size` token rows; page p of request b's sequence is block_table[b][p].  The slot of a
// token is page * page_size + position % page_size.  Every entry read from a table, a slot map, a free list or a list of parents
// is checked against its range on the device before it becomes an address: an entry outside contributes nothing.
#include "nst_common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// ---------------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------------
struct PlanParams {
  const int32_t *cached, *fresh;
  int B, page_size, max_pages;
  int32_t* table;
  int64_t table_stride;
  const int32_t* free_pages;
  int n_free;
  const int32_t* cursor_in;
  int64_t* slots;
  int64_t max_tokens;
  int32_t *seq_lens, *cu_new, *cursor_out;
  int per_group;   // requests of one workgroup (<= 256)
};

struct PlanRequest {
  int cached, fresh, held, need;   // tokens there / to come, pages held / wanted (as far as the table row reaches)
};
__device__ __forceinline__ PlanRequest plan_request(const PlanParams& p, int b) {
  PlanRequest r;
  const int64_t cap = (int64_t)p.max_pages * p.page_size;
  const int64_t c = max(p.cached[b], 0), n = max(p.fresh[b], 0);
  r.cached = (int)(c < cap ? c : cap);
  r.fresh = (int)n;
  const int64_t end = r.cached + n < cap ? r.cached + n : cap;
  r.held = (int)((r.cached + p.page_size - 1) / p.page_size);
  r.need = (int)((end + p.page_size - 1) / p.page_size) - r.held;
  return r;
}

// Every workgroup sums the wishes of the requests in front of its own (B * 8 bytes from the cache: cheaper than a launch that
// scans them first) and scans its own; then its threads walk the group's pages and tokens as one flat range, so that one long
// prompt among many short requests keeps all of them busy.  blockIdx.y splits the tokens of a group further.
__global__ void __launch_bounds__(256) paged_plan_kernel(PlanParams p) {
  __shared__ int64_t red[2][256];
  __shared__ int64_t tok_off[257], page_off[257];
  __shared__ int s_cached[256], s_held[256];
  const int tid = threadIdx.x;
  const int b0 = blockIdx.x * p.per_group, nb = min(p.per_group, p.B - b0);
  int64_t tok = 0, pages = 0;
  for (int b = tid; b < b0; b += 256) {
    const PlanRequest r = plan_request(p, b);
    tok += r.fresh;
    pages += r.need;
  }
  red[0][tid] = tok;
  red[1][tid] = pages;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (tid < o) {
      red[0][tid] += red[0][tid + o];
      red[1][tid] += red[1][tid + o];
    }
    __syncthreads();
  }
  const int64_t tok_base = red[0][0], page_base = red[1][0] + max(*p.cursor_in, 0);
  __syncthreads();
  PlanRequest mine = {0, 0, 0, 0};
  if (tid < nb) mine = plan_request(p, b0 + tid);
  s_cached[tid] = mine.cached;
  s_held[tid] = mine.held;
  red[0][tid] = mine.fresh;
  red[1][tid] = mine.need;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {     // inclusive scan
    const int64_t a = tid >= o ? red[0][tid - o] : 0, b = tid >= o ? red[1][tid - o] : 0;
    __syncthreads();
    red[0][tid] += a;
    red[1][tid] += b;
    __syncthreads();
  }
  tok_off[tid + 1] = red[0][tid];
  page_off[tid + 1] = red[1][tid];
  if (tid == 0) tok_off[0] = page_off[0] = 0;
  __syncthreads();
  const int64_t n_tok = tok_off[nb], n_page = page_off[nb];
  auto find = [&](const int64_t* off, int64_t i) {   // last request whose range starts at or before i
    int lo = 0, hi = nb - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (off[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  auto free_page = [&](int64_t at) { return at < p.n_free ? p.free_pages[at] : -1; };
  if (blockIdx.y == 0) {
    if (tid < nb) {
      const int64_t at = page_base + page_off[tid];
      int64_t got = (int64_t)p.n_free - at;
      got = got < 0 ? 0 : (got < mine.need ? got : mine.need);
      const int64_t cap = (mine.held + got) * p.page_size, want = (int64_t)mine.cached + mine.fresh;
      p.seq_lens[b0 + tid] = (int)(want < cap ? want : cap);
      p.cu_new[b0 + tid] = (int)(tok_base + tok_off[tid]);
    }
    for (int64_t i = tid; i < n_page; i += 256) {
      const int r = find(page_off, i);
      const int page = free_page(page_base + i);
      if (page >= 0) p.table[(int64_t)(b0 + r) * p.table_stride + s_held[r] + (i - page_off[r])] = page;
    }
  }
  for (int64_t i = (int64_t)blockIdx.y * 256 + tid; i < n_tok; i += (int64_t)gridDim.y * 256) {
    if (tok_base + i >= p.max_tokens) break;
    const int r = find(tok_off, i);
    const int64_t pos = s_cached[r] + (i - tok_off[r]), j = pos / p.page_size;
    int page = -1;
    if (j < s_held[r]) page = p.table[(int64_t)(b0 + r) * p.table_stride + j];
    else if (j < p.max_pages) page = free_page(page_base + page_off[r] + (j - s_held[r]));
    p.slots[tok_base + i] = page < 0 ? -1 : (int64_t)page * p.page_size + pos % p.page_size;
  }
  if (b0 + nb == p.B) {
    const int64_t total = tok_base + n_tok;
    if (blockIdx.y == 0 && tid == 0) {
      p.cu_new[p.B] = (int)total;
      const int64_t at = page_base + n_page, start = *p.cursor_in;
      *p.cursor_out = (int)(at < p.n_free ? at : (start > p.n_free ? start : p.n_free));
    }
    for (int64_t i = total + (int64_t)blockIdx.y * 256 + tid; i < p.max_tokens; i += (int64_t)gridDim.y * 256) p.slots[i] = -1;
  }
}

// ---------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------
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
struct PagedAttnParams {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int32_t *table, *lens;
  int B, H, Hkv, dh, page_size, num_pages, max_pages;
  int64_t q_row, q_head, o_row, o_head, table_stride;
  int64_t k_page, k_tok, k_head, v_page, v_tok, v_head;
  float scale;
};

// One wave per (request, head): a lane scores one key of a 64-key step, the lanes then share the head's columns.
template <typename T>
__global__ void __launch_bounds__(64) paged_attn_kernel(PagedAttnParams p) {
  __shared__ float s_p[64];
  __shared__ int64_t s_v[64];
  const int lane = threadIdx.x, h = blockIdx.x % p.H, b = blockIdx.x / p.H, hk = h / (p.H / p.Hkv);
  const T* q = (const T*)p.q + b * p.q_row + h * p.q_head;
  const int len = min(max(p.lens[b], 0), p.max_pages * p.page_size);
  float m = -3.402823466e38f, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < len; t0 += 64) {
    const int t = t0 + lane;
    int page = -1;
    if (t < len) page = p.table[b * p.table_stride + t / p.page_size];
    const bool ok = page >= 0 && page < p.num_pages;
    float s = -INFINITY;
    if (ok) {
      const T* k = (const T*)p.k + page * p.k_page + (t % p.page_size) * p.k_tok + hk * p.k_head;
      s = 0.f;
      for (int d = 0; d < p.dh; ++d) s += to_f32<T>(q[d]) * to_f32<T>(k[d]);
      s *= p.scale * LOG2E;
    }
    const float mn = fmaxf(m, wave_max(s)), pr = ok ? exp2f(s - mn) : 0.f, back = exp2f(m - mn);
    l = l * back + pr;
    m = mn;
    s_p[lane] = pr;
    s_v[lane] = ok ? page * p.v_page + (t % p.page_size) * p.v_tok + hk * p.v_head : -1;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d = c * 64 + lane;
      if (d < p.dh) {
        float a = acc[c] * back;
        for (int i = 0; i < min(64, len - t0); ++i)
          if (s_v[i] >= 0) a += s_p[i] * to_f32<T>(((const T*)p.v)[s_v[i] + d]);
        acc[c] = a;
      }
    }
    __syncthreads();
  }
  l = wave_sum(l);
  T* o = (T*)p.out + b * p.o_row + h * p.o_head;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c * 64 + lane < p.dh) o[c * 64 + lane] = from_f32<T>(l == 0.f ? 0.f : acc[c] / l);
  if (p.lse && lane == 0) p.lse[(int64_t)b * p.H + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// ---------------------------------------------------------------------------------------------
// reorder
// ---------------------------------------------------------------------------------------------
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
  NST_CHECK_ARG((int64_t)max_pages * page_size <= 0x7fffffffLL, "nst_paged_plan: %d pages of %d tokens pass 2^31 - 1 positions", max_pages,
                page_size);
  NST_CHECK_ARG(cursor_in && cu_new && cursor_out && (slots || max_tokens == 0) && (free_pages || n_free == 0),
                "nst_paged_plan: NULL pointer");
  NST_CHECK_ARG(B == 0 || (cached_lens && new_lens && block_table && seq_lens && table_stride >= max_pages),
                "nst_paged_plan: NULL pointer or table stride %lld < %d", (long long)table_stride, max_pages);
  NST_CHECK_ARG(cursor_in != cursor_out && (B == 0 || (seq_lens != cached_lens && seq_lens != new_lens)),
                "nst_paged_plan: the outputs may not overlap the inputs (other workgroups still read them)");
  PlanParams p = {cached_lens, new_lens, B, page_size, max_pages, block_table, table_stride, free_pages, n_free, cursor_in,
                  slots, max_tokens, seq_lens, cu_new, cursor_out, 1};
  int64_t per = max_tokens > 0 ? (4096LL * B + max_tokens - 1) / max_tokens : 256;     // about 4096 tokens for a workgroup
  p.per_group = (int)(per < 1 ? 1 : per > 256 ? 256 : per);
  const int gx = B > 0 ? (B + p.per_group - 1) / p.per_group : 1;
  int64_t gy = max_tokens / ((int64_t)gx * 4096);
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
  NST_CHECK_ARG((int64_t)d->max_pages * pl.page_size <= 0x7fffffffLL, "nst_paged_attention: %d pages of %d tokens pass 2^31 - 1 positions",
                d->max_pages, pl.page_size);
  NST_CHECK_ARG((int64_t)d->B * d->H <= 0x7fffffffLL, "nst_paged_attention: %d x %d rows", d->B, d->H);
  return NST_OK;
}

extern "C" int64_t nst_paged_attention_workspace_bytes(const NstPagedAttnDesc* d) {
  const int rc = paged_attention_check(d);
  return rc != NST_OK ? rc : 0;
}

extern "C" int nst_paged_attention(const NstPagedAttnDesc* d, const void* q, const void* k_pool, const void* v_pool,
                                   const int32_t* block_table, const int32_t* seq_lens, void* out, float* lse, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  const int rc = paged_attention_check(d);
  if (rc != NST_OK) return rc;
  if (d->B == 0) return NST_OK;
  NST_CHECK_ARG(q && block_table && seq_lens && out && ((k_pool && v_pool) || d->pool.num_pages == 0), "nst_paged_attention: NULL pointer");
  (void)workspace; (void)workspace_bytes;
  const NstPagedPool& pl = d->pool;
  PagedAttnParams p = {q, k_pool, v_pool, out, lse, block_table, seq_lens, d->B, d->H, d->Hkv, d->dh, pl.page_size, pl.num_pages,
                       d->max_pages, d->q_row_stride, d->q_head_stride, d->o_row_stride, d->o_head_stride, d->table_stride,
                       pl.k_page_stride, pl.k_token_stride, pl.k_head_stride, pl.v_page_stride, pl.v_token_stride, pl.v_head_stride,
                       d->scale};
  if (pl.dtype == NST_BF16) paged_attn_kernel<bf16_t><<<d->B * d->H, 64, 0, (hipStream_t)stream>>>(p);
  else paged_attn_kernel<float><<<d->B * d->H, 64, 0, (hipStream_t)stream>>>(p);
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
  NST_CHECK_ARG((int64_t)max_pages * page_size <= 0x7fffffffLL, "nst_paged_reorder: %d pages of %d tokens pass 2^31 - 1 positions", max_pages,
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
