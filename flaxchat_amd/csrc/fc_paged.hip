// A paged KV cache whose rows may share a prefix: the page bookkeeping on the
// GPU, the write of new K and V into the pages, and the attention over them.
// No counterpart in the reference, which keeps one contiguous cache per row
// (flaxchat/engine.py:26-48); the attention's mathematics is the one of
// flaxchat/engine.py:128-156, as in fc_attn.hip.
//
// A page holds `page` positions (a multiple of 32) of every KV head of one
// layer, in the caches' own 32-position blocks (include/flaxchat_amd.h), so
// that a layer of a contiguous cache is a pool whose rows are its pages.
// Position p of a row: below prefix_len the shared prefix, entry
// p / page of prefix_pages; from there on entry (p - prefix_len) / page of the
// row's table. An entry outside [0, n_pages) holds no keys.
#include "fc_common.h"
#include "fc_internal.h"

// Smallest b in [0, n) with off[b + 1] > t; n if there is none. Ends for any
// contents of off.
__device__ __forceinline__ int row_of(const int* off, int n, int t) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (off[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// Page tables
// ---------------------------------------------------------------------------
// What a batch's step does to its pages is a handful of prefix sums over the
// rows (pages given back, pages needed, tokens), so one workgroup does it all,
// in place: every row is read before the first is written. Sums saturate at
// 2^30 (they are only compared with capacities below that), which keeps them
// associative and in 32 bits whatever the arrays hold. Bound by latency: two
// scans over 16 waves, four dependent passes over global memory.
#define PT_ROWS 4096     // rows a call may have: 4 per thread
#define PT_SAT (1u << 30)
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, PT_SAT); }

// Exclusive scan over the workgroup's 1024 threads of two values at once.
__device__ __forceinline__ void scan2(uint32_t& a, uint32_t& b, uint2* red, uint2& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t x = a, y = b;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t xo = __shfl_up(x, o, WAVE), yo = __shfl_up(y, o, WAVE);
    if (lane >= o) {
      x = sat_add(x, xo);
      y = sat_add(y, yo);
    }
  }
  if (lane == 63) red[w] = make_uint2(x, y);
  uint32_t xe = __shfl_up(x, 1, WAVE), ye = __shfl_up(y, 1, WAVE);
  if (lane == 0) xe = ye = 0;
  __syncthreads();
  uint32_t px = 0, py = 0, tx = 0, ty = 0;
  for (int i = 0; i < 16; ++i) {
    const uint2 r = red[i];
    if (i < w) px = sat_add(px, r.x), py = sat_add(py, r.y);
    tx = sat_add(tx, r.x);
    ty = sat_add(ty, r.y);
  }
  __syncthreads();  // red is free again
  a = sat_add(px, xe);
  b = sat_add(py, ye);
  total = make_uint2(tx, ty);
}

// Row, position and slot of token t of the packed chunk; off: the rows'
// offsets (batch + 1).
__device__ __forceinline__ void slot_of(int t, const int* off, int batch, int W, int page, int prefix,
                                        const int* tables, const int* __restrict__ length,
                                        int* __restrict__ tok_row, int* __restrict__ tok_pos,
                                        int* __restrict__ slots) {
  int row = -1, pos = -1, slot = -1;
  if (t < off[batch]) {
    row = row_of(off, batch, t);
    const int at = length[row] + t - off[row];
    const int64_t id = tables[(int64_t)row * W + at / page];
    pos = prefix + at;
    if (id >= 0 && (id + 1) * page <= 0x7fffffff) slot = (int)id * page + at % page;
  }
  tok_row[t] = row;
  tok_pos[t] = pos;
  slots[t] = slot;
}

__global__ __launch_bounds__(1024) void k_page_tables(int batch, int W, int page, int prefix, int F, int max_tokens,
                                                      int fill, int* tables, int* held, int* stack, int* n_free,
                                                      const int* __restrict__ length, const int* __restrict__ n_new,
                                                      int* __restrict__ row_off, int* __restrict__ start,
                                                      int* __restrict__ tok_row, int* __restrict__ tok_pos,
                                                      int* __restrict__ slots) {
  __shared__ int s_off[PT_ROWS + 1], s_take[PT_ROWS + 1], s_give[PT_ROWS + 1];
  __shared__ uint2 red[16];
  const int tid = threadIdx.x, b0 = 4 * tid;
  const int64_t width = (int64_t)W * page;
  int hb[4], nb[4], lb[4];
  uint32_t need[4], give[4];
  bool asks[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = b0 + i < batch;
    hb[i] = in ? held[b0 + i] : 0;
    nb[i] = in ? n_new[b0 + i] : 0;
    lb[i] = in ? length[b0 + i] : 0;
  }
  const int nf = min(max(n_free[0], 0), F);
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t end = (int64_t)lb[i] + nb[i];
    asks[i] = nb[i] > 0 && lb[i] >= 0 && end <= width && hb[i] <= W && ((int64_t)lb[i] + page - 1) / page <= hb[i];
    need[i] = asks[i] ? (uint32_t)max((int64_t)0, min((end + page - 1) / page - hb[i], (int64_t)PT_SAT)) : 0;
    give[i] = nb[i] < 0 ? (uint32_t)min(max(hb[i], 0), W) : 0;
    a = sat_add(a, need[i]);
    b = sat_add(b, give[i]);
  }
  uint2 tot;
  scan2(a, b, red, tot);
  const int given = (int)min(tot.y, (uint32_t)(F - nf));  // no more than the stack has room for
  const int avail = nf + given;
  // rows whose pages fit the stack, then rows whose tokens fit the chunk
  uint32_t c = 0, d = 0;
  bool fits[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s_give[b0 + i] = (int)b;
    b = sat_add(b, give[i]);
    a = sat_add(a, need[i]);
    fits[i] = asks[i] && (need[i] == 0 || a <= (uint32_t)avail);
    c = sat_add(c, fits[i] ? (uint32_t)nb[i] : 0);
    d = sat_add(d, fits[i] ? need[i] : 0);
  }
  scan2(c, d, red, tot);
  // Past the first row whose tokens do not fit, none fit (the sum only grows), so the sums up to it are
  // those over the rows that are in.
  bool in[4];
  uint32_t in_n = 0, in_p = 0;  // the sums after this thread's last row that is in
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c0 = c, d0 = d;
    c = sat_add(c, fits[i] ? (uint32_t)nb[i] : 0);
    d = sat_add(d, fits[i] ? need[i] : 0);
    in[i] = fits[i] && c <= (uint32_t)max_tokens;
    if (in[i]) in_n = c, in_p = d;
    s_off[b0 + i] = (int)min(c0, (uint32_t)max_tokens + 1);
    s_take[b0 + i] = (int)d0;
  }
  // totals over the rows that are in
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    in_n = max(in_n, __shfl_xor(in_n, o, WAVE));
    in_p = max(in_p, __shfl_xor(in_p, o, WAVE));
  }
  if ((tid & 63) == 0) red[tid >> 6] = make_uint2(in_n, in_p);
  __syncthreads();
  for (int i = 0; i < 16; ++i) {
    in_n = max(in_n, red[i].x);
    in_p = max(in_p, red[i].y);
  }
  // rows past the last one that is in start at its end
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s_off[b0 + i] = min(s_off[b0 + i], (int)in_n);
    s_take[b0 + i] = min(s_take[b0 + i], (int)in_p);
  }
  if (tid == 0) {
    s_off[PT_ROWS] = (int)in_n;
    s_take[PT_ROWS] = (int)in_p;
    s_give[PT_ROWS] = (int)tot.y;
  }
  __syncthreads();
  // rows past the batch give, take and feed nothing, so entry `batch` of each array is its total
  for (int i = tid; i < given; i += 1024) {
    const int r = row_of(s_give, batch - 1, i);  // (the last row needs no bound of its own)
    stack[nf + i] = tables[(int64_t)r * W + i - s_give[r]];
  }
  __syncthreads();
  for (int i = tid; i < (int)in_p; i += 1024) {
    const int r = row_of(s_take, batch - 1, i);
    tables[(int64_t)r * W + held[r] + i - s_take[r]] = stack[avail - 1 - i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (b0 + i < batch) {
      held[b0 + i] = nb[i] < 0 ? 0 : in[i] ? hb[i] + (int)need[i] : hb[i];
      start[b0 + i] = prefix + (nb[i] < 0 ? 0 : lb[i]);
      row_off[b0 + i] = s_off[b0 + i];
    }
  if (tid == 0) {
    row_off[batch] = (int)in_n;
    n_free[0] = avail - (int)in_p;
  }
  if (!fill) return;
  for (int t = tid; t < max_tokens; t += 1024)
    slot_of(t, s_off, batch, W, page, prefix, tables, length, tok_row, tok_pos, slots);
}

// The tokens of a large chunk, once the rows are settled: one workgroup per
// 1024 tokens.
__global__ __launch_bounds__(256) void k_page_slots(int batch, int W, int page, int prefix, int max_tokens,
                                                    const int* __restrict__ tables, const int* __restrict__ length,
                                                    const int* __restrict__ row_off, int* __restrict__ tok_row,
                                                    int* __restrict__ tok_pos, int* __restrict__ slots) {
  __shared__ int s_off[PT_ROWS + 1];
  for (int i = threadIdx.x; i <= batch; i += 256) s_off[i] = row_off[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = blockIdx.x * 1024 + 256 * i + threadIdx.x;
    if (t < max_tokens) slot_of(t, s_off, batch, W, page, prefix, tables, length, tok_row, tok_pos, slots);
  }
}

// tokens up to which the settling workgroup writes them itself
#define PT_INLINE 2048

extern "C" int32_t fc_page_tables(int32_t* tables, int32_t* held, int32_t* free_pages, int32_t* n_free,
                                  const int32_t* length, const int32_t* n_new, int32_t* row_off, int32_t* start,
                                  int32_t* tok_row, int32_t* tok_pos, int32_t* slots, int32_t batch, int32_t width,
                                  int32_t free_cap, int32_t max_tokens, int32_t page, int32_t prefix_len,
                                  void* stream) {
  FC_CHECK_ARG(tables && held && free_pages && n_free && length && n_new && row_off && start && tok_row && tok_pos &&
                   slots, "null pointer");
  FC_CHECK_ARG(batch > 0 && batch <= PT_ROWS, "batch must be in [1, 4096]");
  FC_CHECK_ARG(page > 0 && page % 32 == 0, "page must be a multiple of 32");
  FC_CHECK_ARG(width > 0 && prefix_len >= 0 && (int64_t)width * page + prefix_len <= 0x7fffffff,
               "positions must fit 31 bits");
  FC_CHECK_ARG(free_cap > 0 && free_cap < (int32_t)PT_SAT && max_tokens > 0 && max_tokens < (int32_t)PT_SAT,
               "free_cap and max_tokens must be in [1, 2^30)");
  const hipStream_t s = (hipStream_t)stream;
  const int fill = max_tokens <= PT_INLINE;
  hipLaunchKernelGGL(k_page_tables, dim3(1), dim3(1024), 0, s, batch, width, page, prefix_len, free_cap, max_tokens,
                     fill, tables, held, free_pages, n_free, length, n_new, row_off, start, tok_row, tok_pos, slots);
  FC_LAUNCH_CHECK();
  if (!fill) {
    hipLaunchKernelGGL(k_page_slots, dim3((max_tokens + 1023) / 1024), dim3(256), 0, s, batch, width, page, prefix_len,
                       max_tokens, tables, length, row_off, tok_row, tok_pos, slots);
    FC_LAUNCH_CHECK();
  }
  return FC_OK;
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// What the kernels need of an fc_pages.
struct PageView {
  int64_t ks, vs;  // elements between pages
  int N, G, page, hd;
  int kblk;        // K blocks in the matrix-core order
};
static PageView page_view(const fc_pages* p) {
  return PageView{p->k_stride, p->v_stride, p->n_pages, p->n_kv_head, p->page, p->head_dim,
                  p->dtype == FC_BF16 && p->head_dim == 128};
}
static int check_pages(const fc_pages* p) {
  FC_CHECK_ARG(p && p->k && p->v, "null pointer");
  FC_CHECK_ARG(p->dtype == FC_F32 || p->dtype == FC_BF16, "dtype");
  FC_CHECK_ARG(p->n_pages > 0 && p->n_kv_head > 0 && p->head_dim > 0 && p->head_dim <= 256,
               "n_pages, n_kv_head and head_dim (at most 256) must be positive");
  FC_CHECK_ARG(p->page > 0 && p->page % 32 == 0, "page must be a multiple of 32");
  const int64_t elems = (int64_t)p->n_kv_head * p->page * p->head_dim;
  FC_CHECK_ARG(p->k_stride >= elems && p->v_stride >= elems, "page strides below a page's elements");
  return FC_OK;
}
__device__ __forceinline__ int64_t k_elem(const PageView& pv, int id, int g, int at, int d) {
  const int64_t base = (int64_t)id * pv.ks + (int64_t)g * pv.page * pv.hd;
  return base + (pv.kblk ? kblk_idx(at, d) : (int64_t)at * pv.hd + d);
}
__device__ __forceinline__ int64_t v_elem(const PageView& pv, int id, int g, int at, int d) {
  return (int64_t)id * pv.vs + (int64_t)g * pv.page * pv.hd + (int64_t)(at >> 5) * 32 * pv.hd + d * 32 + (at & 31);
}

template <typename T, typename S>
__global__ __launch_bounds__(256) void k_page_append(PageView pv, T* __restrict__ kp, T* __restrict__ vp,
                                                     const S* __restrict__ k, const S* __restrict__ v, int64_t kst,
                                                     int64_t ksh, int64_t vst, int64_t vsh,
                                                     const int* __restrict__ slots, int M) {
  const int64_t per = (int64_t)pv.G * pv.hd;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < M * per; i += (int64_t)gridDim.x * 256) {
    const int m = (int)(i / per), r = (int)(i - m * per), g = r / pv.hd, d = r - g * pv.hd;
    const int slot = slots[m];
    if (slot < 0 || slot / pv.page >= pv.N) continue;
    const int id = slot / pv.page, at = slot - id * pv.page;
    st<T>(kp, k_elem(pv, id, g, at, d), ld<S>(k, m * kst + g * ksh + d));
    st<T>(vp, v_elem(pv, id, g, at, d), ld<S>(v, m * vst + g * vsh + d));
  }
}

extern "C" int32_t fc_page_append(const fc_pages* pages, const void* k, const void* v, int64_t k_token_stride,
                                  int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                  int32_t src_dtype, const int32_t* slots, int32_t M, void* stream) {
  const int rc = check_pages(pages);
  if (rc != FC_OK) return rc;
  FC_CHECK_ARG(M >= 0, "M");
  FC_CHECK_ARG(src_dtype == FC_F32 || src_dtype == FC_BF16, "src_dtype");
  FC_CHECK_ARG(src_dtype == pages->dtype || src_dtype == FC_F32, "bf16 values into fp32 pages");
  if (M == 0) return FC_OK;
  FC_CHECK_ARG(k && v && slots, "null pointer");
  const PageView pv = page_view(pages);
  const hipStream_t s = (hipStream_t)stream;
  const int64_t n = (int64_t)M * pv.G * pv.hd;
  const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 65536));
#define APPEND(T, S)                                                                                                 \
  hipLaunchKernelGGL((k_page_append<T, S>), grid, dim3(256), 0, s, pv, (T*)pages->k, (T*)pages->v, (const S*)k,      \
                     (const S*)v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots, M)
  if (pages->dtype == FC_F32) APPEND(float, float);
  else if (src_dtype == FC_F32) APPEND(bf16_t, float);
  else APPEND(bf16_t, bf16_t);
#undef APPEND
  FC_LAUNCH_CHECK();
  return FC_OK;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// One chunk's attention as the kernels see it.
struct PagedChunk {
  PageView pv;
  const int *tables, *row_off, *start, *pre;
  int B, H, W, P, window, max_per_row, Mcap, flags;
  int64_t qst, qsh;  // query strides (elements): token, head
  float scale;
};

// Any head size, type and alignment: one workgroup per (token, head), keys in
// blocks of 256 (a thread scores one key, then sums one dimension), with the
// running maximum and sum of the softmax.
template <typename T>
__global__ __launch_bounds__(256) void k_paged_any(PagedChunk c, const T* __restrict__ q, const T* __restrict__ kp,
                                                   const T* __restrict__ vp, T* __restrict__ y) {
  __shared__ float qs[256], ps[256], red[16];
  const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, hd = c.pv.hd;
  T* yo = y + ((int64_t)t * c.H + h) * hd;
  const int b = row_of(c.row_off, c.B, t);
  RowSpan sp{0, 0};
  if (b < c.B) sp = row_span(c.row_off, b, c.max_per_row, c.Mcap);
  if (t < sp.base || t >= sp.base + sp.n) {
    if ((c.flags & FC_PAGED_ZERO_TAIL) && t >= c.row_off[c.B])
      for (int d = tid; d < hd; d += 256) st<T>(yo, d, 0.f);
    return;
  }
  const int g = h / (c.H / c.pv.G);
  // keys [lo, hi]: the prefix's positions, then the table's
  const int64_t pos = (int64_t)c.start[b] + (t - sp.base);
  const int64_t lo = c.window > 0 ? max((int64_t)0, pos - c.window) : 0;
  const int64_t hi = min(pos, (int64_t)c.P + (int64_t)c.W * c.pv.page - 1);
  for (int d = tid; d < hd; d += 256) qs[d] = ld<T>(q, t * c.qst + h * c.qsh + d);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int64_t k0 = lo; k0 <= hi; k0 += 256) {
    const int64_t key = k0 + tid;
    int id = -1, at = 0;
    if (key <= hi) {
      const int w = (int)(key < c.P ? key : key - c.P);
      id = key < c.P ? c.pre[w / c.pv.page] : c.tables[(int64_t)b * c.W + w / c.pv.page];
      at = w % c.pv.page;
    }
    const bool ok = (unsigned)id < (unsigned)c.pv.N;
    float s = -INFINITY;
    if (ok) {
      float acc = 0.f;
      for (int d = 0; d < hd; ++d) acc += qs[d] * ld<T>(kp, k_elem(c.pv, id, g, at, d));
      s = acc * c.scale;
    }
    const float mn = fmaxf(m, block_max(s, red)), mu = mn == -INFINITY ? 0.f : mn;
    const float p = ok ? expf(s - mu) : 0.f;
    const float alpha = expf(m - mu);
    l = l * alpha + block_sum(p, red);
    m = mn;
    ps[tid] = ok ? p : -1.f;  // -1: not a key, whose V is left alone
    __syncthreads();
    o *= alpha;
    if (tid < hd)
      for (int i = 0; i < 256; ++i) {
        if (ps[i] < 0.f) continue;
        const int64_t key2 = k0 + i;
        const int w = (int)(key2 < c.P ? key2 : key2 - c.P);
        const int id2 = key2 < c.P ? c.pre[w / c.pv.page] : c.tables[(int64_t)b * c.W + w / c.pv.page];
        o += ps[i] * ld<T>(vp, v_elem(c.pv, id2, g, w % c.pv.page, tid));
      }
    __syncthreads();
  }
  if (tid < hd) st<T>(yo, tid, l == 0.f ? 0.f : o / l);  // 0: no key
}

extern "C" int64_t fc_paged_attention_workspace_bytes(const fc_pages* pages, int32_t batch, int32_t max_tokens,
                                                      int32_t max_per_row, int32_t n_head, int32_t width,
                                                      int32_t prefix_len, int32_t window) {
  return 0;
}

extern "C" int32_t fc_paged_attention(const fc_pages* pages, const void* q, int64_t q_token_stride,
                                      int64_t q_head_stride, void* y, int32_t batch, int32_t max_tokens,
                                      int32_t max_per_row, int32_t n_head, const int32_t* tables, int32_t width,
                                      const int32_t* row_off, const int32_t* start, const int32_t* prefix_pages,
                                      int32_t prefix_len, int32_t window, int32_t flags, void* work,
                                      int64_t work_bytes, void* stream) {
  const int rc = check_pages(pages);
  if (rc != FC_OK) return rc;
  FC_CHECK_ARG(q && y && tables && row_off && start, "null pointer");
  FC_CHECK_ARG(batch > 0 && batch <= PT_ROWS, "batch must be in [1, 4096]");
  FC_CHECK_ARG(max_tokens > 0 && max_per_row > 0 && n_head > 0 && n_head % pages->n_kv_head == 0,
               "max_tokens, max_per_row, n_head (a multiple of n_kv_head)");
  FC_CHECK_ARG(n_head <= 65535, "n_head must be <= 65535");
  FC_CHECK_ARG(window >= 0 && prefix_len >= 0 && (prefix_len == 0 || prefix_pages), "window, prefix");
  FC_CHECK_ARG(width > 0 && (int64_t)width * pages->page + prefix_len <= 0x7fffffff, "positions must fit 31 bits");
  PagedChunk c{page_view(pages), tables, row_off, start, prefix_pages, batch, n_head, width, prefix_len, window,
               max_per_row, max_tokens, flags, q_token_stride, q_head_stride,
               1.f / sqrtf((float)pages->head_dim)};
  const hipStream_t s = (hipStream_t)stream;
  if (pages->dtype == FC_BF16)
    hipLaunchKernelGGL(k_paged_any<bf16_t>, dim3(max_tokens, n_head), dim3(256), 0, s, c, (const bf16_t*)q,
                       (const bf16_t*)pages->k, (const bf16_t*)pages->v, (bf16_t*)y);
  else
    hipLaunchKernelGGL(k_paged_any<float>, dim3(max_tokens, n_head), dim3(256), 0, s, c, (const float*)q,
                       (const float*)pages->k, (const float*)pages->v, (float*)y);
  FC_LAUNCH_CHECK();
  return FC_OK;
}
