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
#include "fc_paged.h"
#include <cmath>
#include <type_traits>

// K and V of a row's own pages are read once a call: non-temporal loads keep
// them from displacing lines that are read again.
typedef uint32_t kv_u32x4 __attribute__((ext_vector_type(4)));
#define KV_LD(p) __builtin_bit_cast(uint4, __builtin_nontemporal_load((const kv_u32x4*)(p)))

// ---------------------------------------------------------------------------
// Page tables
// ---------------------------------------------------------------------------
// The rows' offsets into LDS, by 256 threads, four loads under way at once.
__device__ __forceinline__ void stage_offsets(int* off, const int* __restrict__ row_off, int batch) {
  for (int i0 = threadIdx.x; i0 <= batch; i0 += 1024) {
    int x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = row_off[min(i0 + 256 * k, batch)];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i0 + 256 * k <= batch) off[i0 + 256 * k] = x[k];
  }
}

// What a batch's step does to its pages is a handful of prefix sums over the
// rows (pages given back, pages needed, tokens), so one workgroup does it all,
// in place: every row is read before the first is written. Sums saturate at
// 2^30 (they are only compared with capacities below that), which keeps them
// associative and in 32 bits whatever the arrays hold. Bound by latency: four
// dependent passes over global memory and two scans, hence no more waves than
// there are rows or tokens for (64 rows with 16 waves: 7.8 us, with one: 6.5).
#define PT_SAT (1u << 30)
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, PT_SAT); }

// Exclusive scan over the workgroup's threads of two values at once.
__device__ __forceinline__ void scan2(uint32_t& a, uint32_t& b, uint2* red, uint2& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
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
  for (int i = 0; i < nw; ++i) {
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

// Rows, positions and slots of four tokens of the packed chunk, t0 + i * step;
// off: the rows' offsets (batch + 1). Their searches and loads go side by side.
__device__ __forceinline__ void slots_of(int t0, int step, int max_tokens, const int* off, int batch, int W, int page,
                                         int prefix, const int* tables, const int* __restrict__ length,
                                         int* __restrict__ tok_row, int* __restrict__ tok_pos,
                                         int* __restrict__ slots) {
  const int total = off[batch];
  int row[4] = {0, 0, 0, 0}, at[4], id[4];
  for (int s = 1 << (31 - __builtin_clz(batch)); s > 0; s >>= 1)  // the last row that begins at the token or before
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (row[i] + s < batch && off[row[i] + s] <= t0 + i * step) row[i] += s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + i * step;
    at[i] = t < total ? length[row[i]] + t - off[row[i]] : 0;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) id[i] = t0 + i * step < total ? tables[(int64_t)row[i] * W + at[i] / page] : -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + i * step;
    if (t >= max_tokens) continue;
    const bool in = t < total;
    tok_row[t] = in ? row[i] : -1;
    tok_pos[t] = in ? prefix + at[i] : -1;
    slots[t] = id[i] >= 0 && ((int64_t)id[i] + 1) * page <= 0x7fffffff ? id[i] * page + at[i] % page : -1;
  }
}

struct TableArgs {
  int batch, W, page, prefix, F, max_tokens, fill;
  int *tables, *held, *stack, *n_free;
  const int *length, *n_new;
  int *row_off, *start, *tok_row, *tok_pos, *slots;
};
__global__ __launch_bounds__(1024) void k_page_tables(TableArgs t) {
  const int batch = t.batch, W = t.W, page = t.page, F = t.F, max_tokens = t.max_tokens;
  int *tables = t.tables, *held = t.held, *stack = t.stack;
  __shared__ int s_off[PT_ROWS + 1], s_take[PT_ROWS + 1], s_give[PT_ROWS];
  __shared__ uint2 red[16];
  const int tid = threadIdx.x, b0 = 4 * tid;
  const int64_t width = (int64_t)W * page;
  int hb[4], nb[4], lb[4];
  uint32_t ask[4], need[4], give[4];  // tokens asked for, pages they need, pages given back
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = b0 + i < batch;
    hb[i] = in ? held[b0 + i] : 0;
    nb[i] = in ? t.n_new[b0 + i] : 0;
    lb[i] = in ? t.length[b0 + i] : 0;
  }
  const int nf = min(max(t.n_free[0], 0), F);
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t end = (int64_t)lb[i] + nb[i];
    const bool asks =
        nb[i] > 0 && lb[i] >= 0 && end <= width && hb[i] <= W && ((int64_t)lb[i] + page - 1) / page <= hb[i];
    ask[i] = asks ? (uint32_t)nb[i] : 0;
    need[i] = asks ? (uint32_t)max((int64_t)0, min((end + page - 1) / page - hb[i], (int64_t)PT_SAT)) : 0;
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
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s_give[b0 + i] = (int)b;
    b = sat_add(b, give[i]);
    a = sat_add(a, need[i]);
    if (need[i] > 0 && a > (uint32_t)avail) ask[i] = need[i] = 0;
    c = sat_add(c, ask[i]);
    d = sat_add(d, need[i]);
  }
  scan2(c, d, red, tot);
  // Past the first row whose tokens do not fit, none fit (the sum only grows), so the sums up to it are
  // those over the rows that are in.
  uint32_t in_n = 0, in_p = 0;  // the sums after this thread's last row that is in
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s_off[b0 + i] = (int)min(c, (uint32_t)max_tokens + 1);
    s_take[b0 + i] = (int)d;
    c = sat_add(c, ask[i]);
    d = sat_add(d, need[i]);
    if (c > (uint32_t)max_tokens) need[i] = 0;
    else if (ask[i] > 0) in_n = c, in_p = d;
  }
  // totals over the rows that are in
  const int nw = blockDim.x >> 6, step = blockDim.x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    in_n = max(in_n, __shfl_xor(in_n, o, WAVE));
    in_p = max(in_p, __shfl_xor(in_p, o, WAVE));
  }
  if ((tid & 63) == 0) red[tid >> 6] = make_uint2(in_n, in_p);
  __syncthreads();
  for (int i = 0; i < nw; ++i) {
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
    s_off[4 * step] = (int)in_n;
    s_take[4 * step] = (int)in_p;
  }
  __syncthreads();
  // (the last row needs no bound of its own, hence batch - 1; rows past the batch give, take and feed nothing)
  for (int i = tid; i < given; i += step) {
    const int r = row_of(s_give, batch - 1, i);
    stack[nf + i] = tables[(int64_t)r * W + i - s_give[r]];
  }
  __syncthreads();
  for (int i = tid; i < (int)in_p; i += step) {
    const int r = row_of(s_take, batch - 1, i);
    tables[(int64_t)r * W + held[r] + i - s_take[r]] = stack[avail - 1 - i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (b0 + i < batch) {
      held[b0 + i] = nb[i] < 0 ? 0 : hb[i] + (int)need[i];
      t.start[b0 + i] = t.prefix + (nb[i] < 0 ? 0 : lb[i]);
      t.row_off[b0 + i] = s_off[b0 + i];
    }
  if (tid == 0) {
    t.row_off[batch] = (int)in_n;
    t.n_free[0] = avail - (int)in_p;
  }
  if (!t.fill) return;
  for (int k = tid; k < max_tokens; k += 4 * step)
    slots_of(k, step, max_tokens, s_off, batch, W, page, t.prefix, tables, t.length, t.tok_row, t.tok_pos, t.slots);
}

// The tokens of a large chunk, once the rows are settled: 1024 per workgroup.
__global__ __launch_bounds__(256) void k_page_slots(int batch, int W, int page, int prefix, int max_tokens,
                                                    const int* __restrict__ tables, const int* __restrict__ length,
                                                    const int* __restrict__ row_off, int* __restrict__ tok_row,
                                                    int* __restrict__ tok_pos, int* __restrict__ slots) {
  __shared__ int s_off[PT_ROWS + 1];
  stage_offsets(s_off, row_off, batch);
  __syncthreads();
  slots_of(blockIdx.x * 1024 + threadIdx.x, 256, max_tokens, s_off, batch, W, page, prefix, tables, length, tok_row,
           tok_pos, slots);
}

// Tokens up to which the settling workgroup writes them itself: 64 rows and their 64 tokens are 6.5 us that way and
// 4.3 + 4 in two launches, 1000 rows with 7000 tokens 16.4 us or 6.1 + 7.2.
#define PT_INLINE 512

extern "C" int32_t fc_page_tables(int32_t* tables, int32_t* held, int32_t* free_pages, int32_t* n_free,
                                  const int32_t* length, const int32_t* n_new, int32_t* row_off, int32_t* start,
                                  int32_t* tok_row, int32_t* tok_pos, int32_t* slots, int32_t batch, int32_t width,
                                  int32_t free_cap, int32_t max_tokens, int32_t page, int32_t prefix_len,
                                  void* stream) {
  FC_CHECK_ARG(tables && held && (free_pages || free_cap == 0) && n_free && length && n_new && row_off && start &&
                   tok_row && tok_pos && slots, "null pointer");
  FC_CHECK_ARG(batch > 0 && batch <= PT_ROWS, "batch must be in [1, 4096]");
  FC_CHECK_ARG(page > 0 && page % 32 == 0, "page must be a multiple of 32");
  FC_CHECK_ARG(width > 0 && prefix_len >= 0 && (int64_t)width * page + prefix_len <= 0x7fffffff,
               "positions must fit 31 bits");
  FC_CHECK_ARG(free_cap >= 0 && free_cap < (int32_t)PT_SAT && max_tokens > 0 && max_tokens < (int32_t)PT_SAT,
               "free_cap must be in [0, 2^30), max_tokens in [1, 2^30)");
  const hipStream_t s = (hipStream_t)stream;
  const int fill = max_tokens <= PT_INLINE;
  const TableArgs t{batch, width, page, prefix_len, free_cap, max_tokens, fill, tables, held, free_pages, n_free,
                    length, n_new, row_off, start, tok_row, tok_pos, slots};
  const int threads = std::max((batch + 3) / 4, fill ? (max_tokens + 3) / 4 : 0);
  hipLaunchKernelGGL(k_page_tables, dim3(1), dim3(std::min(1024, (threads + 63) / 64 * 64)), 0, s, t);
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
// Any head size and alignment: an element per thread.
template <typename T, typename S>
__global__ __launch_bounds__(256) void k_page_append_any(PageView pv, T* __restrict__ kp, T* __restrict__ vp,
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

// About 32 tokens of one KV head per workgroup, 16 bytes per load and store.
// K: 8 dims of a position are 16 bytes of its block; lanes are dealt so that the
// positions next to each other in it are next to each other in the wave. V is
// stored dim by dim: through LDS, and where 8 tokens fill an aligned run of 8
// positions (a prompt's, save its ends) they are one store, element by element
// elsewhere (2-byte stores to rows 64 bytes apart take a cycle per lane). Hence a
// workgroup's tokens begin where a run of 8 does, if one is near. Bound by the
// copy of K and V in a prompt: 16000 tokens of 4 heads 21 us (3.1 TB/s moved, a plain
// copy 4.9); 448 tokens in runs of up to 7, 12 heads, 11 us, of which most is the
// waits for slots, values and LDS one after the other.
#define PA_TILE 32
#define PA_MOST (PA_TILE + 7)
// First token of tile i: the first one from 32 i on that begins a run of 8
// positions, or does not follow the one before it.
__device__ __forceinline__ int append_from(const int* __restrict__ slots, int M, int i) {
  const int64_t t = (int64_t)PA_TILE * i;
  if (i == 0 || t >= M) return (int)min(t, (int64_t)M);
  const int k = threadIdx.x & 7;
  const int a = t + k < M ? slots[t + k] : -1, b = t + k - 1 < M ? slots[t + k - 1] : -1;
  const uint64_t cut = __ballot(a < 0 || (a & 7) == 0 || a != b + 1);
  return (int)t + __builtin_ctzll(cut);  // of 8 that follow each other one begins a run
}

template <typename T, typename S, bool KBLK>
__global__ __launch_bounds__(256) void k_page_append(PageView pv, T* __restrict__ kp, T* __restrict__ vp,
                                                     const S* __restrict__ k, const S* __restrict__ v, int64_t kst,
                                                     int64_t ksh, int64_t vst, int64_t vsh,
                                                     const int* __restrict__ slots, int M) {
  extern __shared__ char lds[];  // the tile's V, [token][hd + pad]
  __shared__ int s_slot[64], s_run[8], s_one[64], s_n[2];
  const int g = blockIdx.y, tid = threadIdx.x, n8 = pv.hd >> 3, ldv = pv.hd + 2;
  T* tv = (T*)lds;
  const int t0 = append_from(slots, M, blockIdx.x), n = append_from(slots, M, blockIdx.x + 1) - t0;
  if (n <= 0) return;
  if (tid < 64) {
    int slot = tid < n ? slots[t0 + tid] : -1;
    if (slot < 0 || slot / pv.page >= pv.N) slot = -1;
    s_slot[tid] = slot;
    // runs of 8 positions whose tokens are all here, and the tokens outside them
    uint64_t run = __ballot(slot >= 0 && (slot & 7) == 0), ok = __ballot(slot >= 0);
    const uint64_t next = __ballot(slot >= 0 && slot == __shfl_up(slot, 1, WAVE) + 1);  // follows the lane before
#pragma unroll
    for (int i = 1; i < 8; ++i) run &= next >> i;
    uint64_t in = run;
#pragma unroll
    for (int i = 1; i < 8; ++i) in |= run << i;
    const uint64_t below = (1ull << tid) - 1, one = ok & ~in;
    if ((run >> tid) & 1) s_run[__popcll(run & below)] = tid;
    if ((one >> tid) & 1) s_one[__popcll(one & below)] = tid;
    if (tid == 0) {
      s_n[0] = __popcll(run);
      s_n[1] = __popcll(one);
    }
  }
  for (int i = tid; i < n * n8; i += 256) {
    const int t = i / n8, d = 8 * (i - t * n8);
    float x[8];
    load8(v + (t0 + t) * vst + g * vsh + d, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) st<T>(tv, t * ldv + d + e, x[e]);
  }
  __syncthreads();
  // K: chunk i is 8 dims of a token; in the matrix-core order 16 lanes take every token of a half block
  const int chunks = KBLK ? ((n + 31) >> 5) * 512 : n * n8;
  for (int i = tid; i < chunks; i += 256) {
    int t, d;
    if constexpr (KBLK) {
      const int r = i & 15;
      t = 32 * (i >> 9) + 8 * (r >> 2) + (r & 3) + 4 * ((i >> 6) & 1);
      d = 32 * ((i >> 7) & 3) + 8 * ((i >> 4) & 3);
    } else {
      t = i / n8;
      d = 8 * (i - t * n8);
    }
    const int slot = t < n ? s_slot[t] : -1;
    if (slot < 0) continue;
    float x[8];
    load8(k + (t0 + t) * kst + g * ksh + d, x);
    const int id = slot / pv.page;
    store8(kp + k_elem(pv, id, g, slot - id * pv.page, d), x, 1.f);
  }
  // V: four runs of a block side by side are a row of 64 bytes
  const int nr = s_n[0], no = s_n[1];
  for (int i = tid; i < ((nr + 3) & ~3) * pv.hd; i += 256) {
    const int q = (i & 3) + 4 * (i / (4 * pv.hd)), d = (i >> 2) % pv.hd;
    if (q >= nr) continue;
    const int t = s_run[q], slot = s_slot[t], id = slot / pv.page;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = ld<T>(tv, (t + e) * ldv + d);
    store8(vp + v_elem(pv, id, g, slot - id * pv.page, d), x, 1.f);
  }
  for (int i = tid; i < no * pv.hd; i += 256) {
    const int q = i / pv.hd, d = i - q * pv.hd, t = s_one[q], slot = s_slot[t], id = slot / pv.page;
    st<T>(vp, v_elem(pv, id, g, slot - id * pv.page, d), ld<T>(tv, t * ldv + d));
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
  const int per = src_dtype == FC_BF16 ? 8 : 4, per_page = pages->dtype == FC_BF16 ? 8 : 4;
  const uintptr_t at = (uintptr_t)pages->k | (uintptr_t)pages->v | (uintptr_t)k | (uintptr_t)v;
  const int64_t strides = k_token_stride | k_head_stride | v_token_stride | v_head_stride;
  const int64_t tiles = ((int64_t)M + PA_TILE - 1) / PA_TILE;
  const bool vec = (at & 15) == 0 && strides % per == 0 && (pages->k_stride | pages->v_stride) % per_page == 0 &&
                   pv.hd % 8 == 0 && pv.G <= 65535 && tiles < 1 << 24;  // (a launch's threads are counted in 32 bits)
  const int64_t n = (int64_t)M * pv.G * pv.hd;
#define APPEND(T, S, KBLK)                                                                                           \
  if (vec)                                                                                                           \
    hipLaunchKernelGGL((k_page_append<T, S, KBLK>), dim3((int)tiles, pv.G), dim3(256),                               \
                       PA_MOST * (pv.hd + 2) * sizeof(T), s, pv, (T*)pages->k, (T*)pages->v, (const S*)k, (const S*)v,\
                       k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots, M);                      \
  else                                                                                                               \
    hipLaunchKernelGGL((k_page_append_any<T, S>), dim3((unsigned)std::min<int64_t>((n + 255) / 256, 65536)),         \
                       dim3(256), 0, s, pv, (T*)pages->k, (T*)pages->v, (const S*)k, (const S*)v, k_token_stride,    \
                       k_head_stride, v_token_stride, v_head_stride, slots, M)
  if (pages->dtype == FC_F32) {
    APPEND(float, float, false);
  } else if (src_dtype == FC_F32) {
    if (pv.kblk) {
      APPEND(bf16_t, float, true);
    } else {
      APPEND(bf16_t, float, false);
    }
  } else {
    if (pv.kblk) {
      APPEND(bf16_t, bf16_t, true);
    } else {
      APPEND(bf16_t, bf16_t, false);
    }
  }
#undef APPEND
  FC_LAUNCH_CHECK();
  return FC_OK;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// tree: a chunk's tokens are the nodes of trees, each with its position and a row
// of bits that says which of the row's nodes it sees. Every node's walk reaches the
// last node's key, the range of keys that all of its columns see ends before the
// first node's, and only tiles and steps behind that ask for bits: a lane's 8 keys of
// a tile are 8 bits next to each other, a load of one word or two. The bound is the
// one of plain chunks (128 trees of up to 25 nodes, 12 heads on 4, behind 6144 keys,
// 50-2000 of their own: 144 us with the merge; a library product does the 69 GFLOP
// in 56).
//
// One chunk's attention as the kernels see it.
struct PagedChunk {
  PageView pv;
  const int *tables, *row_off, *start, *pre;
  int B, H, W, P, window, max_per_row, Mcap, flags;
  int64_t qst, qsh;  // query strides (elements): token, head
  float scale;
  // key splits: most of a row's own keys, of the prefix, keys of each of these; workgroups that the own keys are to
  // be spread over
  int S_own, S_pre, pre_chunk, target;
  int joint;  // the rows' walks begin with the prefix, P rounded up to 32; 0: it is walked for itself, or there is none
  // partials of split s (the own ones first): po[(s Mcap + token) H + head][hd] unnormalised, pml (max, sum)
  float* po;
  float2* pml;
  int* items;  // of more than ROWS_SCAN rows: the chunk's length, and every 64 rows' first item
  const void *q, *kp, *vp;
  void* y;
  // a tree's chunk: each token's row of bits (`words` of them) and its position
  const uint64_t* mask;
  const int* tok_pos;
  int words, pre_blk;
};

// The chunk, read from the kernel's arguments (its first) at this point and not
// kept from earlier. What is kept of it through a whole walk, with the constants
// that the compiler makes of it for its divisions, is more than the scalar
// registers hold, and a spill of theirs is not to be had here: a part of one came
// back wrong (the lower half of a pointer), so the kernels here are to have none: the
// build fails if one has.
template <typename P>
__device__ __forceinline__ P* in_global(P* p) {
  return (P*)(__attribute__((address_space(1))) P*)p;
}
template <typename P>
__device__ __forceinline__ P* scalar(P* p) {  // the same in every lane, and known to be
  const uint64_t u = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return in_global((P*)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ PagedChunk chunk_args() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  PagedChunk c;
  __builtin_memcpy(&c, (const void*)p, sizeof(c));
  c.tables = in_global(c.tables);
  c.row_off = in_global(c.row_off);
  c.start = in_global(c.start);
  c.pre = in_global(c.pre);
  c.po = in_global(c.po);
  c.pml = in_global(c.pml);
  c.items = in_global(c.items);
  c.q = in_global(c.q);
  c.kp = in_global(c.kp);
  c.vp = in_global(c.vp);
  c.y = in_global(c.y);
  c.mask = in_global(c.mask);
  c.tok_pos = in_global(c.tok_pos);
  return c;
}

// Any head size, type and alignment: one workgroup per (token, head), keys in
// blocks of 256 (a thread scores one key, then sums one dimension), with the
// running maximum and sum of the softmax. Without matrix instructions and with keys
// read once per query head, it is for shapes that no model here has: 64 rows of 300
// keys, 12 heads of 96, 175 us (12 of 128: 25).
//
// tree: a key before the row's start is seen by the window that ends at the token's
// position, one of the chunk's own if the token's row of bits says so.
template <typename T, bool tree>
__global__ __launch_bounds__(256) void k_paged_any(PagedChunk c) {
  const T *q = (const T*)c.q, *kp = (const T*)c.kp, *vp = (const T*)c.vp;
  T* y = (T*)c.y;
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
  const int64_t first = c.start[b], last = (int64_t)c.P + (int64_t)c.W * c.pv.page - 1;
  const int64_t pos = tree ? max(first, (int64_t)c.tok_pos[t]) : first + (t - sp.base);
  const int64_t from = tree ? min(pos - c.window, first) : pos - c.window;
  const int64_t lo = c.window > 0 ? max((int64_t)0, from) : 0;
  const int64_t hi = min(tree ? first + sp.n - 1 : pos, last);
  const uint64_t* bits = c.mask + (int64_t)t * c.words;
  for (int d = tid; d < hd; d += 256) qs[d] = ld<T>(q, t * c.qst + h * c.qsh + d);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int64_t k0 = lo; k0 <= hi; k0 += 256) {
    const int64_t key = k0 + tid;
    int id = -1, at = 0;
    if (key <= hi && (!tree || key < first ||
                      (key >= c.P && (bits[(key - first) >> 6] >> ((key - first) & 63) & 1)))) {
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

// Table entries are read through the constant address space: scalar loads,
// whose result can be a scalar base of the direct LDS loads below.
typedef const __attribute__((address_space(4))) int* const_ints;
#define CONST_INTS(p) ((const_ints)(uint64_t)(p))

__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                  0, 0);
}
__device__ __forceinline__ float exp2a(float x) { return __builtin_amdgcn_exp2f(x); }
// Two keys' worth of a V operand word: all ones where the key is in [lo, hi].
// (Keys are compared as constants with bounds relative to the lane's first
// key: the other way round the sums, one per key, are kept in registers
// through the whole walk.)
__device__ __forceinline__ uint32_t key_mask(int key, int lo, int hi) {
  return (key >= lo && key <= hi ? 0xffffu : 0u) | (key + 1 >= lo && key + 1 <= hi ? 0xffff0000u : 0u);
}
// The larger magnitudes of two pairs of bf16, as 15-bit numbers: an infinity
// or NaN is one of 0x7f80 and more.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 max_magnitude(u16x2 a, uint32_t w) {
  return __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, w & 0x7fff7fffu));
}
__device__ __forceinline__ bool any_odd(u16x2 m) { return __any(m.x >= 0x7f80 || m.y >= 0x7f80); }
// Reductions over the lanes of a wave in registers (rotations within 16 lanes,
// swaps of rows and halves): the shuffles through LDS take ~5 times as long, and
// a workgroup's first loads wait for these.
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}
template <int N, typename F>
__device__ __forceinline__ int lanes_reduce(int v, F f) {  // over groups of N = 16, 32 or 64 lanes, in every lane
  v = f(v, dpp<0x128>(v));
  v = f(v, dpp<0x124>(v));
  v = f(v, dpp<0x122>(v));
  v = f(v, dpp<0x121>(v));
  if constexpr (N > 16) {
    const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = f((int)h[0], (int)h[1]);
  }
  if constexpr (N > 32) {
    const auto h = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    v = f((int)h[0], (int)h[1]);
  }
  return v;
}
template <int N>
__device__ __forceinline__ int lanes_min(int v) {
  return __builtin_amdgcn_readfirstlane(lanes_reduce<N>(v, [](int a, int b) { return min(a, b); }));
}
template <int N>
__device__ __forceinline__ int lanes_max(int v) {
  return __builtin_amdgcn_readfirstlane(lanes_reduce<N>(v, [](int a, int b) { return max(a, b); }));
}
__device__ __forceinline__ float lanes_sum(float v) {
  return __uint_as_float(lanes_reduce<64>(__float_as_uint(v), [](int a, int b) {
    return (int)__float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
// maximum over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float rows_max(float v) {
  const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
  const auto g = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(g[0]), __uint_as_float(g[1]));
}
// inclusive sum over the lanes up to this one (up to 2^31)
__device__ __forceinline__ int lanes_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // a row's last lane onto the next row
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // the lower half's onto the upper
  return v;
}

// Keys of a job are counted from 0: the prefix's positions, or a row's own
// ones (position - P, which is their place in the row's table).
// A query: its position, and, of a tree, its row's start and nodes.
struct Query {
  int64_t pos, first;
  int n;
};
// Query j of a row of n that starts at `first`; t: its token.
template <bool tree>
__device__ __forceinline__ Query query_at(const PagedChunk& c, int64_t first, int n, int j, int t) {
  return Query{tree ? max(first, (int64_t)c.tok_pos[t]) : first + j, first, n};
}
// The keys [lo, hi] that a query sees; hi < lo: none. Of a tree: what the row
// holds before its start, as far as the window reaches, and all of its nodes'
// keys, of which the query's bits say more.
template <bool tree>
__device__ __forceinline__ void key_range(const PagedChunk& c, const Query& q, bool pre, int& lo, int& hi) {
  const int64_t off = pre ? 0 : c.P, last = pre ? (int64_t)c.P - 1 : (int64_t)c.W * c.pv.page - 1;
  const int64_t end = !tree ? q.pos : pre ? q.first - 1 : q.first + q.n - 1;
  const int64_t from = tree ? min(q.pos - c.window, q.first) : q.pos - c.window;
  hi = (int)max((int64_t)-1, min(end - off, last));
  lo = c.window > 0 ? (int)max((int64_t)0, min(from - off, (int64_t)0x7fffffff)) : 0;
}
// Where the nodes' keys begin in a walk whose keys are counted from `off`. (Below -FC_TREE_MOST no node has one.)
__device__ __forceinline__ int nodes_from(int64_t first, int64_t off) {
  return (int)max(first - off, (int64_t)-2 * FC_TREE_MOST);
}
// Bits j0 .. j0 + 7 of a token's row of `words` words; those before 0, for what the row holds before its nodes, are
// set, those behind the words are not.
__device__ __forceinline__ uint32_t bits8(const uint64_t* row, int words, int j0) {
  const int w = j0 >> 6, sh = j0 & 63;
  const uint64_t a = w < 0 ? ~0ull : w < words ? row[w] : 0ull;
  uint64_t x = a >> sh;
  if (sh > 56) x |= (w + 1 < 0 ? ~0ull : w + 1 < words ? row[w + 1] : 0ull) << (64 - sh);
  return (uint32_t)x & 0xffu;
}

// How a workgroup walks: over a row's own keys, over the prefix for all rows, or
// over a row's keys and, if c.joint, the prefix ahead of them. In the last, keys are
// counted from the prefix's first, and own ones from c.joint: no key lies between.
enum Walk { OWN_KEYS, PREFIX_KEYS, ROW_KEYS };
template <int walk, bool tree>
__device__ __forceinline__ void walk_range(const PagedChunk& c, const Query& q, int& lo, int& hi) {
  key_range<tree>(c, q, walk == PREFIX_KEYS, lo, hi);
  if constexpr (walk == ROW_KEYS) {
    int plo, phi;
    key_range<tree>(c, q, true, plo, phi);
    if (c.joint > 0) {
      lo = plo < c.P ? plo : (int)min((int64_t)lo + c.joint, (int64_t)0x7fffffff);
      hi = hi >= 0 ? hi + c.joint : phi;
    }
  }
}

// A piece of work: a column block of row b (or, for the prefix, of all tokens)
// and KV group g against `len` keys from `skip` keys on behind the 32-key block
// of the row's first key; the `split`th of the block's nsplit pieces.
struct Item {
  int b, blk, g, split, nsplit, len;
  int64_t skip;
};
// keys of row r's walk, from the 32-key block of its first query's first key, and its column blocks; -1: no query
struct RowKeys {
  int len, blocks;
};
template <int CB, int walk, bool tree>
__device__ __forceinline__ RowKeys row_keys(const PagedChunk& c, int r) {
  const int64_t at = c.start[min(r, c.B - 1)];  // (its load goes beside those of the offsets)
  const RowSpan sp = row_span(c.row_off, min(r, c.B - 1), c.max_per_row, c.Mcap);
  int lo, hi, lo1, hi1;  // (no node of a tree is before its row's start, and all reach its last node's key)
  walk_range<walk, tree>(c, Query{at, at, sp.n}, lo, hi);
  walk_range<walk, tree>(c, Query{at + sp.n - 1, at, sp.n}, lo1, hi1);
  if (r >= c.B || sp.n == 0) return {-1, 0};
  return {hi1 < lo ? 0 : hi1 + 1 - (lo & ~31), (sp.n * (c.H / c.pv.G) + CB - 1) / CB};
}

// Rows are of unequal length: with a number of key splits for all, the longest
// row's would be left for last and the short rows' have nothing to do. So the
// rows' own keys are a list of items (row, column block, key split, KV group), cut
// by one chunk length for all rows, and every workgroup looks its own one up, by
// its number, from all rows' lengths (each wave reads them all; the result is the
// same everywhere). The chunk is what spreads the keys over about c.target items,
// at least 128 (a tile for each of four waves), in the streaming kernel no more
// than CHUNK_MAX (several rounds of items: their times differ then; a cut column
// block of the wide kernel costs more than that, 16 rows of 512 at 8000 keys 633 us
// with the limit and 560 without) and at least what makes c.S_own splits of the
// longest row; a row's pieces are then of one length (64 rows of 4800 keys, 12 heads:
// 302 us, and 356 with 4096 and 704). (One share of all keys for each workgroup that fits
// the card, whatever rows it crosses, took 10-15% longer: a workgroup then waits
// at every border, where two on a CU hide each other's.)
// Up to ROWS_SCAN rows every wave looks through all of them. With more the reading
// of so many lengths would be most of a workgroup's time (4096 rows of up to 200
// keys: 1448 us, 215 with the list): a kernel ahead of the walk finds the chunk and
// where every 64 rows' items begin.
#define CHUNK_MAX 4096
#define CHUNK_WIDE 1000000000
#define ROWS_SCAN 256
// A tree's rows without a prefix, in the streaming kernel: none is cut if the longest is no longer than a share of 256
// items, a workgroup for every CU, as a cut costs a start (32 rows at 1280 keys, 12 heads, not cut and in two: trees of 16
// 49 and 52 us, of 32 54 and 64; 22 rows at 8000 keys, cut to c.target all the same, 190, and 199 with CHUNK_MAX). Where
// rows are cut it is to c.target and not to 256 (32 rows of 100 to 4000 keys 81 and 86 us, 8 rows at 8000 73 and 88).
template <int CB, bool tree>
__device__ __forceinline__ int chunk_length(const PagedChunk& c, float total, int longest) {
  const float all = total * (float)c.pv.G;
  float share = ceilf(all / (float)c.target);
  if (tree && CB < 64 && c.P == 0 && longest <= CHUNK_MAX && (float)longest * 256.f <= all) share = (float)longest;
  // (unsigned: a row may have up to 2^31 - 32 keys)
  const uint32_t least = max(128u, ((uint32_t)longest + c.S_own - 1) / c.S_own);
  const uint32_t len = (max((uint32_t)fminf(share, (float)(CB >= 64 ? CHUNK_WIDE : CHUNK_MAX)), least) + 63) & ~63u;
  return __builtin_amdgcn_readfirstlane((int)min(len, 0x7fffffe0u));
}
// pieces of a row: its keys / chunk, at least one (past 2^24 keys it may be one too few, never too many)
__device__ __forceinline__ int row_pieces(const RowKeys& r, int chunk) {
  const uint32_t len = max(r.len, 0), by = chunk;
  uint32_t ns = (uint32_t)((float)len * (1.f / (float)chunk));
  ns += ns * by < len;
  return max(1, (int)(ns - (ns > 1 && (ns - 1) * by >= len)));
}
// The item numbered `at` from the 64 rows' first on, lane l holding row r0 + l; false: it is behind them, and at less
// by theirs.
__device__ __forceinline__ bool item_of(const PagedChunk& c, int& at, int r0, const RowKeys& r, int chunk, Item& it) {
  const int ns = row_pieces(r, chunk), mine = ns * r.blocks * c.pv.G, upto = lanes_scan(mine);
  const uint64_t past = __ballot(upto > at);
  if (past == 0) {
    at -= __builtin_amdgcn_readlane(upto, 63);
    return false;
  }
  const int l = __builtin_ctzll(past);
  at -= __builtin_amdgcn_readlane(upto - mine, l);
  // (the walk's addresses are scalar: said so here, since the compiler loses track of it where the ways here meet)
  it.b = __builtin_amdgcn_readfirstlane(r0 + l);
  it.nsplit = __builtin_amdgcn_readlane(ns, l);
  // pieces of one length, that of the row's keys and not of the chunk (about no longer than it, so none is empty); a
  // row's only piece takes all
  it.len = it.nsplit > 1 ? ((__builtin_amdgcn_readlane(r.len, l) - 1) / it.nsplit + 64) & ~63 : 0x7fffffe0;
  const int unit = __builtin_amdgcn_readfirstlane(at) / c.pv.G;
  it.g = __builtin_amdgcn_readfirstlane(at) - unit * c.pv.G;
  it.blk = __builtin_amdgcn_readlane(r.blocks, l) - 1 - unit / it.nsplit;  // (later queries see more keys: first)
  it.split = unit % it.nsplit;
  it.skip = (int64_t)it.split * it.len;
  return true;
}
template <int CB, int walk, bool tree, int N>
__device__ __forceinline__ bool find_among(const PagedChunk& c, int at, Item& it) {
  const int lane = threadIdx.x & 63;
  RowKeys r[N];
  float total = 0.f;
  int longest = 1;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r[i] = row_keys<CB, walk, tree>(c, 64 * i + lane);
    total += (float)max(r[i].len, 0) * (float)r[i].blocks;
    longest = max(longest, r[i].len);
  }
  const int chunk = chunk_length<CB, tree>(c, lanes_sum(total), lanes_max<64>(longest));
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (item_of(c, at, 64 * i, r[i], chunk, it)) return true;
  return false;
}
template <int CB, int walk, bool tree>
__device__ __forceinline__ bool find_item(const PagedChunk& c, int at, Item& it) {
  if (c.B <= 64) return find_among<CB, walk, tree, 1>(c, at, it);
  if (c.B <= ROWS_SCAN) return find_among<CB, walk, tree, ROWS_SCAN / 64>(c, at, it);
  const int lane = threadIdx.x & 63, n = (c.B + 63) >> 6;
  const int chunk = __builtin_amdgcn_readfirstlane(c.items[0]), first = c.items[1 + min(lane, n)];
  const int k = __builtin_popcountll(__ballot(lane < n && first <= at)) - 1;
  at -= __builtin_amdgcn_readlane(first, k);
  return item_of(c, at, 64 * k, row_keys<CB, walk, tree>(c, 64 * k + lane), chunk, it);
}
template <int CB, int walk, bool tree>
__global__ __launch_bounds__(1024) void k_paged_items(PagedChunk c) {
  constexpr int N = PT_ROWS / 1024;
  __shared__ float s_total[16];
  __shared__ int s_longest[16], s_items[64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  RowKeys r[N];
  float total = 0.f;
  int longest = 1;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r[i] = row_keys<CB, walk, tree>(c, 64 * (wave + 16 * i) + lane);
    total += (float)max(r[i].len, 0) * (float)r[i].blocks;
    longest = max(longest, r[i].len);
  }
  total = lanes_sum(total);
  longest = lanes_max<64>(longest);
  if (lane == 0) s_total[wave] = total, s_longest[wave] = longest;
  __syncthreads();
  total = 0.f;
  for (int i = 0; i < 16; ++i) total += s_total[i], longest = max(longest, s_longest[i]);
  const int chunk = chunk_length<CB, tree>(c, total, longest);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int upto = lanes_scan(row_pieces(r[i], chunk) * r[i].blocks * c.pv.G);
    if (lane == 63) s_items[wave + 16 * i] = upto;
  }
  __syncthreads();
  if (wave > 0) return;
  const int mine = s_items[lane], n = (c.B + 63) >> 6;
  if (lane < n) c.items[1 + lane] = lanes_scan(mine) - mine;
  if (lane == 0) c.items[0] = chunk;
}
// The partials of a row's column that no split writes: the item of its last split marks them.
__device__ __forceinline__ void mark_unused(const PagedChunk& c, const Item& it, int64_t pair) {
  if (it.split == it.nsplit - 1)
    for (int s = it.nsplit; s < c.S_own; ++s) c.pml[(int64_t)s * c.Mcap * c.H + pair] = make_float2(-INFINITY, 0.f);
}

// An item that holds all of its columns' keys writes their outputs itself. Where other rows are split it says so in
// place of the first partial's sum, which is never negative.
__device__ __forceinline__ bool whole(const PagedChunk& c, const Item& it) {
  return c.S_pre == 0 && it.nsplit == 1;
}
__device__ __forceinline__ void mark_whole(const PagedChunk& c, int64_t pair) {
  if (c.S_own > 1) c.pml[pair] = make_float2(0.f, -1.f);
}

// Tokens past the last row: set to 0 by the launch's workgroups in turn.
template <typename T>
__device__ __forceinline__ void zero_tail(int wg, int nwg) {
  const PagedChunk c = chunk_args();
  if (c.S_own + c.S_pre > 1 || !(c.flags & FC_PAGED_ZERO_TAIL)) return;
  const int n8 = c.H * c.pv.hd * (int)sizeof(T) / 16;
  for (int64_t t = max(0, c.row_off[c.B]) + (int64_t)wg; t < c.Mcap; t += nwg)
    for (int i = threadIdx.x; i < n8; i += blockDim.x) ((uint4*)c.y)[t * n8 + i] = uint4{0u, 0u, 0u, 0u};
}

// The matrix product multiplies a key's V by the weight 0 of a column that
// does not see the key: NaN if V is not finite. Both kernels clear the keys
// that no column of theirs sees, look for such values among the rest where the
// columns differ (`odd`) and, if there are any, hand the workgroup's columns
// [c_lo, c_hi) over to this plain form, one wave per column, over the keys
// [kbeg, kend). (Anything done about them in the walk itself costs every call
// registers, and spills.)
template <typename T, int HD, bool tree>
__device__ __forceinline__ void redo_columns(int walk, const Item& it, int base, int c_lo, int c_hi, int kbeg, int kend,
                                             int wave) {
  const PagedChunk c = chunk_args();
  const T *q = (const T*)c.q, *kp = (const T*)c.kp, *vp = (const T*)c.vp;
  T* y = (T*)c.y;
  const bool pre = walk == PREFIX_KEYS;
  const int sg = pre ? c.S_own + it.split : it.split;
  const int lane = threadIdx.x & 63, rep = c.H / c.pv.G, b = it.b, g = it.g;
  for (int col = c_lo + wave; col < c_hi; col += 4) {
    const int j = col / rep, head = g * rep + col - j * rep;
    int r = b;
    if (pre) {
      r = row_of(c.row_off, c.B, j);
      if (r >= c.B) continue;
    }
    const RowSpan sp = row_span(c.row_off, r, c.max_per_row, c.Mcap);
    if (pre && (j < sp.base || j >= sp.base + sp.n)) continue;
    const Query qy = query_at<tree>(c, c.start[r], sp.n, pre ? j - sp.base : j, base + j);
    const uint64_t* bits = c.mask + (int64_t)(base + j) * c.words;
    int v_lo, v_hi;
    if (walk == ROW_KEYS) walk_range<ROW_KEYS, tree>(c, qy, v_lo, v_hi);
    else key_range<tree>(c, qy, pre, v_lo, v_hi);
    v_lo = max(v_lo, kbeg);
    v_hi = min(v_hi, kend - 1);
    const T* qr = q + (base + j) * c.qst + head * c.qsh;
    float m = -INFINITY, l = 0.f, o[HD / 64] = {};
#pragma unroll 1
    for (int part = walk == ROW_KEYS && c.joint > 0 ? 0 : 1; part < 2; ++part) {  // the prefix, the row's own keys
      const int from = part == 1 && walk == ROW_KEYS ? c.joint : 0;
      const int lo = max(v_lo - from, 0), hi = part == 0 ? min(v_hi, c.P - 1) : v_hi - from;
      const int* list = pre || part == 0 ? c.pre : c.tables + (int64_t)b * c.W;
      // (counted by what is left: a key behind hi may not fit 31 bits)
      for (int left = hi - lo + 1; left > 0; left -= 64) {
        const int key = hi + 1 - left + min(lane, left - 1), pg = key / c.pv.page, at = key - pg * c.pv.page;
        const int id = list[pg];
        bool ok = lane < left && (unsigned)id < (unsigned)c.pv.N;
        if constexpr (tree) {
          const bool own = !pre && part == 1;  // (of the prefix, what is before the start)
          const int node = key - nodes_from(qy.first, own ? c.P : 0);
          ok = ok && (node < 0 || (own && node < qy.n && (bits[node >> 6] >> (node & 63) & 1)));
        }
        if (!__any(ok)) continue;
        float s = -INFINITY;
        if (ok) {
          float a = 0.f;
#pragma unroll 1
          for (int d = 0; d < HD; ++d) a += ld<T>(qr, d) * ld<T>(kp, k_elem(c.pv, id, g, at, d));
          s = a * c.scale * 1.4426950408889634f;
        }
        const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
        const float p = ok ? exp2a(s - mu) : 0.f, alpha = exp2a(m - mu);
        l = l * alpha + wave_sum(p);
        m = mn;
#pragma unroll
        for (int t = 0; t < HD / 64; ++t) o[t] *= alpha;
#pragma unroll 1
        for (int i = 0; i < 64; ++i) {
          const int idi = __shfl(ok ? id : -1, i, WAVE), ati = __shfl(at, i, WAVE);
          const float w = __shfl(p, i, WAVE);
          if (idi < 0) continue;
#pragma unroll
          for (int t = 0; t < HD / 64; ++t) o[t] += w * ld<T>(vp, v_elem(c.pv, idi, g, ati, lane + 64 * t));
        }
      }
    }
    const int64_t pair = (int64_t)(base + j) * c.H + head;
    if (whole(c, it)) {
      if (lane == 0) mark_whole(c, pair);
      for (int t = 0; t < HD / 64; ++t) st<T>(y, pair * HD + lane + 64 * t, l == 0.f ? 0.f : o[t] / l);
    } else {
      const int64_t at = (int64_t)sg * c.Mcap * c.H + pair;
      for (int t = 0; t < HD / 64; ++t) c.po[at * HD + lane + 64 * t] = o[t];
      if (lane == 0) {
        c.pml[at] = make_float2(m, l);
        if (!pre) mark_unused(c, it, pair);
      }
    }
  }
}

// The matrix operands of one 32-key tile and 16 query columns, in registers:
// lane l = cl + 16 g4 holds operand row cl. K row cl of half cc is key
// 8 (cl / 4) + cl % 4 + 4 cc, so that the scores leave a lane with keys 8 g4 ..
// +7 of its column: the P operand as they stand.
__device__ __forceinline__ f32x4 mfma16f(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
template <typename T, int HD>
struct Tile;
// bf16: 16x16x32 products, 8 values of k a lane
template <int HD>
struct Tile<bf16_t, HD> {
  uint4 k[2][HD / 32], v[HD / 16];
  struct Q {
    uint4 q[HD / 32];
    __device__ __forceinline__ void load(const bf16_t* row, int g4, bool ok) {
      const uint32_t keep = ok ? 0xffffffffu : 0u;  // (a select of the address would make these flat loads)
#pragma unroll
      for (int s = 0; s < HD / 32; ++s) {
        const uint4 x = *(const uint4*)(row + 32 * s + 8 * g4);
        q[s] = uint4{x.x & keep, x.y & keep, x.z & keep, x.w & keep};
      }
    }
  };
  __device__ __forceinline__ void load(const bf16_t* kt, const bf16_t* vt, int lane) {
    const int cl = lane & 15, g4 = lane >> 4;
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int s = 0; s < HD / 32; ++s)
        k[cc][s] = KV_LD((const uint4*)(HD == 128 ? kt + lane * 8 + (s * 2 + cc) * 512
                                                  : kt + (8 * (cl >> 2) + (cl & 3) + 4 * cc) * HD + 32 * s + 8 * g4));
#pragma unroll
    for (int db = 0; db < HD / 16; ++db) v[db] = KV_LD((const uint4*)(vt + cl * 32 + 8 * g4 + db * 512));
  }
  // V = 0 for keys outside [zl, zh] (counted from the lane's first); whether any other value is not finite
  __device__ __forceinline__ bool clear(int zl, int zh) {
    const uint32_t m0 = key_mask(0, zl, zh), m1 = key_mask(2, zl, zh), m2 = key_mask(4, zl, zh),
                   m3 = key_mask(6, zl, zh);
    u16x2 mag = {0, 0};
#pragma unroll
    for (int db = 0; db < HD / 16; ++db) {
      v[db] = uint4{v[db].x & m0, v[db].y & m1, v[db].z & m2, v[db].w & m3};
      mag = max_magnitude(max_magnitude(mag, v[db].x), v[db].y);
      mag = max_magnitude(max_magnitude(mag, v[db].z), v[db].w);
    }
    return any_odd(mag);
  }
  __device__ __forceinline__ void scores(const Q& q, f32x4 (&sc)[2]) const {
#pragma unroll
    for (int s = 0; s < HD / 32; ++s)
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) sc[cc] = mfma16(k[cc][s], q.q[s], sc[cc]);
  }
  // the weights go into the product rounded to bf16 (half a step, 2^-8, of each), as the matrix cores take both operands
  // in V's type; their sum keeps fp32. (Outputs are 0.0018-0.0021 of their root mean square off the 64-bit ones; their own
  // rounding is 0.0017.)
  __device__ __forceinline__ void add(const float (&p)[8], f32x4 (&O)[HD / 16]) const {
    const uint4 pf = {pack2bf(p[0], p[1]), pack2bf(p[2], p[3]), pack2bf(p[4], p[5]), pack2bf(p[6], p[7])};
#pragma unroll
    for (int db = 0; db < HD / 16; ++db) O[db] = mfma16(v[db], pf, O[db]);
  }
};
// fp32: 16x16x4 products, one value of k a lane; 16-byte loads give it four products' worth
template <int HD>
struct Tile<float, HD> {
  f32x4 k[2][HD / 16], v[HD / 16][2];
  struct Q {
    f32x4 q[HD / 16];
    __device__ __forceinline__ void load(const float* row, int g4, bool ok) {
#pragma unroll
      for (int s = 0; s < HD / 16; ++s) {
        const f32x4 x = *(const f32x4*)(row + 16 * s + 4 * g4);
#pragma unroll
        for (int i = 0; i < 4; ++i) q[s][i] = ok ? x[i] : 0.f;
      }
    }
  };
  __device__ __forceinline__ void load(const float* kt, const float* vt, int lane) {
    const int cl = lane & 15, g4 = lane >> 4;
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int s = 0; s < HD / 16; ++s)
        k[cc][s] = *(const f32x4*)(kt + (8 * (cl >> 2) + (cl & 3) + 4 * cc) * HD + 16 * s + 4 * g4);
#pragma unroll
    for (int db = 0; db < HD / 16; ++db)
#pragma unroll
      for (int h = 0; h < 2; ++h) v[db][h] = *(const f32x4*)(vt + db * 512 + cl * 32 + 8 * g4 + 4 * h);
  }
  __device__ __forceinline__ bool clear(int zl, int zh) {
    uint32_t mag = 0;
#pragma unroll
    for (int db = 0; db < HD / 16; ++db)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = i >= zl && i <= zh ? v[db][i >> 2][i & 3] : 0.f;
        mag = max(mag, __float_as_uint(x) & 0x7fffffffu);
        v[db][i >> 2][i & 3] = x;
      }
    return __any(mag >= 0x7f800000u);
  }
  __device__ __forceinline__ void scores(const Q& q, f32x4 (&sc)[2]) const {
#pragma unroll
    for (int s = 0; s < HD / 16; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) sc[cc] = mfma16f(k[cc][s][i], q.q[s][i], sc[cc]);
  }
  __device__ __forceinline__ void add(const float (&p)[8], f32x4 (&O)[HD / 16]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int db = 0; db < HD / 16; ++db) O[db] = mfma16f(v[db][i >> 2][i & 3], p[i], O[db]);
  }
};

// One tile of one wave for 16 query columns: S^T = K Q^T, the running softmax,
// O^T += V^T P^T. lo, hi: the keys that this lane's column sees, and, of a tree,
// the bits of the lane's 8; the tile's V is 0 for those that none sees.
template <bool tree, typename T, int HD>
__device__ __forceinline__ void tile16(const Tile<T, HD>& t, const typename Tile<T, HD>::Q& q, int kb, int g4, int lo,
                                       int hi, uint32_t bits, float scale_log2, float& m_run, float& l_run,
                                       f32x4 (&O)[HD / 16]) {
  f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  t.scores(q, sc);
  float p[8], mt = -INFINITY;
#pragma unroll
  for (int jj = 0; jj < 8; ++jj) {
    const bool seen = jj >= lo - kb - 8 * g4 && jj <= hi - kb - 8 * g4 && (!tree || (bits >> jj & 1));
    p[jj] = seen ? sc[jj >> 2][jj & 3] * scale_log2 : -INFINITY;
    mt = fmaxf(mt, p[jj]);
  }
  const float m_new = fmaxf(m_run, rows_max(mt));
  if (__any(m_new > m_run)) {
    const float alpha = exp2a(m_run - (m_new == -INFINITY ? 0.f : m_new));
    l_run *= alpha;
#pragma unroll
    for (int db = 0; db < HD / 16; ++db) O[db] *= alpha;
    m_run = m_new;
  }
  const float mu = m_run == -INFINITY ? 0.f : m_run;  // no key yet: every term exp2(-inf) = 0
#pragma unroll
  for (int jj = 0; jj < 8; ++jj) {
    p[jj] = exp2a(p[jj] - mu);
    l_run += p[jj];
  }
  t.add(p, O);
}

// Few query columns (token, head in group), or fp32: a workgroup takes 16 QB of
// a row and KV group, or, for the prefix (`pre`), of all rows together, and one
// key split; its four waves every fourth 32-key tile, straight from memory into
// registers, each tile applied to all QB blocks of 16 columns, and are merged in
// LDS.
//
// Bound by the reading of K and V: 17 rows of about 114000 keys (8 KV heads of 128)
// take 1.26 ms, 6.4 TB/s of the 7.1 that a plain read reaches, 64 rows of 2400 keys
// (12 heads) 152 us, 6.2 TB/s. Short rows are bound by what a workgroup waits for
// one after the other (the rows' offsets, the table, the keys): 64 rows of 300 keys
// 25 us, 4.8 TB/s. fp32 takes four times the matrix instructions of bf16 for as
// many keys: 8 rows of 5 tokens, 6 heads, behind 1000 keys 17 us.
template <int HD>
struct StreamLds {
  float o[4][16][HD + 4];
  float m[4][16], l[4][16];
};
template <typename T, int HD, int QB, bool pre, bool tree>
__device__ __forceinline__ void stream_item(const PagedChunk& w, StreamLds<HD>& lds, const Item& it, int base,
                                            int ncol) {
  constexpr int NW = 4, NT = 2 * HD;  // threads that own 8 dims of a column after the merge
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cl = lane & 15, g4 = lane >> 4;
  const int b = it.b, g = it.g, col0 = it.blk * 16 * QB;
  typename Tile<T, HD>::Q qf[QB];
  int lo[QB], hi[QB], tok[QB];
  int w_lo = 0x7fffffff, w_hi = -1, f_lo = 0, f_hi = 0x7fffffff, nodes = 0x7fffffff;
  int64_t kbeg, kend;
  {
    const PagedChunk& c = w;
    const int rep = c.H / c.pv.G;
    // this lane's columns
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      const int col = col0 + 16 * u + cl;
      bool ok = col < ncol;
      const int j = ok ? col / rep : 0, head = g * rep + (ok ? col - j * rep : 0);
      Query qy{0, 0, 0};
      if (pre) {
        const int* off = (const int*)&lds;
        const int r = row_of(off, c.B, j);
        RowSpan sp{0, 0};
        if (r < c.B) sp = row_span(off, r, c.max_per_row, c.Mcap);
        ok = ok && j >= sp.base && j < sp.base + sp.n;
        if (ok) qy = query_at<tree>(c, c.start[r], sp.n, j - sp.base, j);
      } else {
        qy = query_at<tree>(c, c.start[b], ncol / rep, j, base + j);
      }
      tok[u] = base + j;
      key_range<tree>(c, qy, pre, lo[u], hi[u]);
      if (!ok) lo[u] = 0x7fffffff, hi[u] = -1;
      const bool some = lo[u] <= hi[u];  // columns that see nothing do not widen the range
      w_lo = min(w_lo, some ? lo[u] : 0x7fffffff);
      w_hi = max(w_hi, some ? hi[u] : -1);
      f_lo = max(f_lo, ok ? lo[u] : 0);
      f_hi = min(f_hi, ok ? hi[u] : 0x7fffffff);
      qf[u].load((const T*)c.q + (base + j) * c.qst + head * c.qsh, g4, ok);
    }
    w_lo = lanes_min<16>(w_lo);
    w_hi = lanes_max<16>(w_hi);
    f_lo = lanes_max<16>(f_lo);
    f_hi = lanes_min<16>(f_hi);
    if constexpr (tree && !pre) {
      nodes = nodes_from(c.start[b], c.P);
      f_hi = min(f_hi, nodes - 1);
    }
    // (a row's splits are counted from its first column's first key in every one of its blocks)
    int from = w_lo, unused;
    if (!pre && c.window > 0) key_range<tree>(c, Query{c.start[b], c.start[b], 1}, false, from, unused);
    const int64_t s_beg = (int64_t)(from & ~31) + it.skip;
    kbeg = max(s_beg, (int64_t)(w_lo & ~31));
    kend = min((int64_t)w_hi + 1, s_beg + it.len);
  }
  if (kbeg >= kend && w.S_own + w.S_pre > 1) {
    const int col = col0 + threadIdx.x, rep = w.H / w.pv.G;
    if (threadIdx.x < 16 * QB && col < ncol) {
      const int j = col / rep;
      const int64_t pair = (int64_t)(base + j) * w.H + g * rep + col - j * rep;
      w.pml[(int64_t)(pre ? w.S_own + it.split : it.split) * w.Mcap * w.H + pair] = make_float2(-INFINITY, 0.f);
      if (!pre) mark_unused(w, it, pair);
    }
    return;
  }
  const float scale_log2 = w.scale * 1.4426950408889634f;
  const int tpp = w.pv.page >> 5, tend = kbeg >= kend ? 0 : (int)((kend + 31) >> 5);
  const const_ints list = CONST_INTS(pre ? w.pre : w.tables + (int64_t)b * w.W);
  const int64_t gofs = (int64_t)g * w.pv.page * HD;
  int tile = (int)(min(kbeg, (int64_t)w_hi + 1) >> 5) + wave;
  int pg = tile / tpp, r = tile - pg * tpp;
  float m_run[QB], l_run[QB];
  f32x4 O[QB][HD / 16];
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    m_run[u] = -INFINITY;
    l_run[u] = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) O[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int id = tile < tend ? list[pg] : -1;
  bool odd = false;
  while (tile < tend) {
    const int kb = 32 * tile, id0 = id, r0 = r;
    // the next tile's page, ahead of this one's work
    tile += NW;
    r += NW;
    while (r >= tpp) r -= tpp, ++pg;
    id = tile < tend ? list[pg] : -1;
    if ((unsigned)id0 >= (unsigned)w.pv.N) continue;
    Tile<T, HD> t;
    const int64_t in = gofs + r0 * (32 * HD);
    t.load((const T*)w.kp + (int64_t)id0 * w.pv.ks + in, (const T*)w.vp + (int64_t)id0 * w.pv.vs + in, lane);
    uint32_t bits[QB];
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      bits[u] = 0xff;
      if (tree && !pre && kb + 31 >= nodes)
        bits[u] = bits8(w.mask + (int64_t)tok[u] * w.words, w.words, kb + 8 * g4 - nodes);
    }
    if (!(kb >= f_lo && kb + 31 <= f_hi)) odd |= t.clear(w_lo - kb - 8 * g4, w_hi - kb - 8 * g4);
#pragma unroll
    for (int u = 0; u < QB; ++u)
      tile16<tree && !pre, T, HD>(t, qf[u], kb, g4, lo[u], hi[u], bits[u], scale_log2, m_run[u], l_run[u], O[u]);
  }
  if (__syncthreads_or(odd)) {  // (also: the readers of the LDS are done with it)
    redo_columns<T, HD, tree>(pre ? PREFIX_KEYS : OWN_KEYS, it, base, col0, min(col0 + 16 * QB, ncol), (int)min(kbeg, kend),
                        (int)kend, wave);
    return;
  }
  const PagedChunk c = chunk_args();
  const int rep = c.H / c.pv.G, sg = pre ? c.S_own + it.split : it.split;
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    if (col0 + 16 * u < ncol) {  // uniform; a guard, not a break, so that u stays a constant
      l_run[u] += __shfl_xor(l_run[u], 16, WAVE);
      l_run[u] += __shfl_xor(l_run[u], 32, WAVE);
      if (u > 0) __syncthreads();  // the readers of the LDS are done with it
      if (g4 == 0) {
        lds.m[wave][cl] = m_run[u];
        lds.l[wave][cl] = l_run[u];
      }
#pragma unroll
      for (int db = 0; db < HD / 16; ++db) *(f32x4*)&lds.o[wave][cl][16 * db + 4 * g4] = O[u][db];
      __syncthreads();
      const int qc = threadIdx.x / (HD / 8), d0 = (threadIdx.x % (HD / 8)) * 8, col = col0 + 16 * u + qc;
      if (threadIdx.x < NT && col < ncol) {
        float M = -INFINITY, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, lds.m[w][qc]);
        const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float a = exp2a(lds.m[w][qc] - mu);
          L += a * lds.l[w][qc];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] += a * lds.o[w][qc][d0 + i];
        }
        const int j = col / rep, head = g * rep + col - j * rep;
        if (!pre && whole(c, it)) {
          if (d0 == 0) mark_whole(c, (int64_t)(base + j) * c.H + head);
          store8((T*)c.y + ((int64_t)(base + j) * c.H + head) * HD + d0, o, L == 0.f ? 0.f : 1.f / L);
        } else {
          const int64_t slot = ((int64_t)sg * c.Mcap + base + j) * c.H + head;
          float4* po = (float4*)(c.po + slot * HD + d0);
          po[0] = make_float4(o[0], o[1], o[2], o[3]);
          po[1] = make_float4(o[4], o[5], o[6], o[7]);
          if (d0 == 0) {
            c.pml[slot] = make_float2(M, L);
            if (!pre) mark_unused(c, it, (int64_t)(base + j) * c.H + head);
          }
        }
      }
    }
  }
}

// The workgroup numbered `at`: an item of the list, or a split of the prefix.
template <typename T, int HD, int QB, bool pre, bool tree>
__device__ __forceinline__ void stream_keys(const PagedChunk& c, StreamLds<HD>& lds, int at) {
  Item it;
  int base = 0, ncol;
  if constexpr (pre) {
    static_assert(sizeof(lds) >= (PT_ROWS + 1) * 4, "the rows' offsets");
    it = Item{0, 0, at % c.pv.G, 0, 1, c.pre_chunk, 0};
    at /= c.pv.G;
    it.split = at % c.S_pre;
    it.blk = at / c.S_pre;
    it.skip = (int64_t)it.split * it.len;
    if (it.split == c.S_pre - 1) it.len = c.P;
    ncol = min(max(c.row_off[c.B], 0), c.Mcap) * (c.H / c.pv.G);
    if (it.blk * 16 * QB >= ncol) return;
    int* off = (int*)&lds;
    stage_offsets(off, c.row_off, c.B);
    __syncthreads();
  } else {
    if (!find_item<16 * QB, OWN_KEYS, tree>(c, at, it)) return;
    const RowSpan sp = row_span(c.row_off, it.b, c.max_per_row, c.Mcap);
    base = sp.base;
    ncol = sp.n * (c.H / c.pv.G);
  }
  stream_item<T, HD, QB, pre, tree>(c, lds, it, base, ncol);
}

// Merge of the key splits of one (token, head), HD / 8 threads with 8
// dimensions each: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s. The
// splits' (max, sum) are read side by side, ahead of the token's row; then the
// outputs of those that hold keys, CB at a time. Bound by the reading of the
// partials: 4482 tokens of 12 heads with three of them 17 us, 5.7 TB/s; with few
// tokens by the launch and three waits, 5 us.
template <typename T, int HD, int CB>
__global__ __launch_bounds__(256) void k_paged_merge(PagedChunk c) {
  __shared__ int off[PT_ROWS + 1];
  constexpr int TP = HD / 8;
  const int64_t pair = (int64_t)blockIdx.x * (256 / TP) + threadIdx.x / TP, pairs = (int64_t)c.Mcap * c.H;
  const int tp = threadIdx.x % TP, d0 = tp * 8, S = c.S_own + c.S_pre, own = c.S_own;
  const int64_t at = min(pair, pairs - 1);
  const int off0 = c.row_off[min((int)threadIdx.x, c.B)];  // its wait goes beside the next loads'
  float M = -INFINITY;
  int used = 0;  // own splits with keys: the first ones
  const bool done = c.pml[at].y < 0.f;  // by a whole item
  for (int s = tp; s < S; s += TP) {
    const float2 e = c.pml[(int64_t)s * pairs + at];
    M = fmaxf(M, e.x);
    if (s < own && (e.x != -INFINITY || e.y != 0.f)) used = s + 1;
  }
  if ((int)threadIdx.x <= c.B) off[threadIdx.x] = off0;
  for (int i = threadIdx.x + 256; i <= c.B; i += 256) off[i] = c.row_off[i];
#pragma unroll
  for (int o = TP / 2; o > 0; o >>= 1) {
    M = fmaxf(M, __shfl_xor(M, o, WAVE));
    used = max(used, __shfl_xor(used, o, WAVE));
  }
  // CB splits' partials, under way while the token's row is looked up
  const int n = used + c.S_pre;
  float2 e[CB];
  float4 u[CB][2];
  auto load = [&](int s0) {
#pragma unroll
    for (int k = 0; k < CB; ++k) {
      const int s = min(s0 + k, n - 1);
      const int64_t i = (int64_t)(s < used ? s : s - used + own) * pairs + at;
      e[k] = c.pml[i];
      u[k][0] = *(const float4*)(c.po + i * HD + d0);
      u[k][1] = *(const float4*)(c.po + i * HD + d0 + 4);
    }
  };
  if (!done && n > 0) load(0);  // (n = 0: no split holds a key, or a token of no row)
  __syncthreads();
  if (pair >= pairs) return;
  const int t = (int)(pair / c.H), b = row_of(off, c.B, t);
  RowSpan sp{0, 0};
  if (b < c.B) sp = row_span(off, b, c.max_per_row, c.Mcap);
  T* yo = (T*)c.y + pair * HD + d0;
  if (t < sp.base || t >= sp.base + sp.n) {
    if ((c.flags & FC_PAGED_ZERO_TAIL) && t >= off[c.B])
      store8(yo, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, 1.f);
    return;
  }
  if (done) return;
  const float mu = M == -INFINITY ? 0.f : M;
  float L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < n; s0 += CB) {
    if (s0 > 0) load(s0);
#pragma unroll
    for (int k = 0; k < CB; ++k) {
      // a split without keys holds (-inf, 0) and no output
      if (s0 + k >= n || (e[k].x == -INFINITY && e[k].y == 0.f)) continue;
      const float a = exp2a(e[k].x - mu);
      L += a * e[k].y;
      o[0] += a * u[k][0].x; o[1] += a * u[k][0].y; o[2] += a * u[k][0].z; o[3] += a * u[k][0].w;
      o[4] += a * u[k][1].x; o[5] += a * u[k][1].y; o[6] += a * u[k][1].z; o[7] += a * u[k][1].w;
    }
  }
  store8(yo, o, L == 0.f ? 0.f : 1.f / L);
}

// Many query columns: 128 per workgroup, 32 per wave, on the 32x32x16 MFMA, of
// one row and KV group, or, for the prefix (`pre`), of all rows' tokens side by
// side, so that its keys are read once per 128 columns whatever rows they
// belong to. The walk, the operand order in LDS and the softmax are those of
// fc_attn.hip's prefill kernel: 64 keys a step through two LDS stages filled
// by direct loads, scores and outputs in registers.
//
// Workgroups: the items of the list, or, for the prefix, group x key split x
// column block, all blocks of a split on one XCD, whose L2 then holds its keys.
//
// Bound by the matrix cores and the softmax's arithmetic together: a step of a wave
// is 1024 cycles of the first and about 1300 of the second, of which two waves a
// SIMD hide a part (16 rows of 512 tokens behind 8000 shared keys 510 us, 0.81
// PFLOP/s; a library matrix product reaches 1.23). With few steps a workgroup the
// start and the end weigh in: behind 4001 keys, 4482 tokens of unequal rows, 205 us,
// 0.61 PFLOP/s. Tried: the maximum left behind by up to 2^8, to scale the sums less
// often, gave 4% and cost precision, as the largest weight is then no longer 1.
template <int HD>
struct WideStage {
  uint4 k[2][HD / 16][64];  // [32-key tile][16-dim slice][lane]
  uint4 v[2][HD / 16][64];  // [32-key tile][2 (dim / 32) + key half][lane]
};
template <int HD>
struct WideLds {
  WideStage<HD> stg[2];
  int rng[4][2];
};
// CB = 64: blocks of 64 columns, two waves on each of a step's two tiles, joined at
// the end: a step is then half as long, and the next one's loads go out the sooner.
// (32 trees of 64 nodes at 1024-1536 keys, 12 heads, 60 us and 4.6 TB/s without the merge,
// 67 in blocks of 128; at 300 keys 25 and 29.)
template <int HD, int walk, bool tree, int CB = 128>
__device__ __forceinline__ void wide_keys(const PagedChunk& w, WideLds<HD>& lds, int at) {
  constexpr int DS = HD / 16, DD = HD / 32;  // 16-dim slices, 32-dim output blocks
  constexpr bool halves = CB == 64;
  constexpr int NU = halves ? 1 : 2;  // tiles of a step that a wave takes
  static_assert(!halves || walk == OWN_KEYS, "a row's own keys");
  constexpr bool pre = walk == PREFIX_KEYS;
  WideStage<HD>(&stg)[2] = lds.stg;
  static_assert(sizeof(lds.stg) >= (PT_ROWS + 1) * 4, "the rows' offsets");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, kk = lane & 31;
  const int cw = halves ? wave & 1 : wave, u0 = halves ? wave >> 1 : 0;  // its 32 columns, its first tile
  Item it;
  int base = 0, ncol, lo_c, hi_c, w_lo, w_hi, tok = 0;
  int64_t kbeg64, kend64;
  bool ok;
  v4u qf[DS];  // dims 16 h + 8 hl .. +7 of this lane's query
  {
    const PagedChunk& c = w;
    const int rep = c.H / c.pv.G;
    it = Item{0, 0, 0, 0, 1, c.pre_chunk, 0};
    if constexpr (pre) {
      const int nunit = c.pv.G * c.S_pre;
      int unit;
      // a tree's chunk: the blocks unit by unit, an eighth of them on each XCD. (By whole units one XCD may get two and
      // the next one: 37 blocks of 4 groups against 6144 keys in 3 splits 140 us so, 99 in equal numbers. Each order with
      // its model of the splits, trees as plain rows are: up to 25 nodes in 128 rows, 12 heads on 4, behind 6144 keys
      // alone 118 us and 95, with 50-2000 of their own 140 and 147; 200 rows of 3, 12 heads, behind 3000 76 and 70; 500
      // rows of one behind 2000 80 and 85.)
      // Plain chunks keep the order by units and its model, also where equal numbers would be the better: other splits
      // would round their sums in another way. (The same shapes: 118 us and 98, 163 and 158, 73 and 70, 78 and 83.)
      if constexpr (tree) {
        const int nb = c.pre_blk, per = (nunit * nb + 7) >> 3, idx = (at & 7) * per + (at >> 3);
        unit = idx / nb;
        if ((at >> 3) >= per || unit >= nunit) return;
        it.blk = idx - unit * nb;
      } else {
        const int nul = (nunit + 7) >> 3, jj = at >> 3;
        unit = (jj % nul) * 8 + (at & 7);
        if (unit >= nunit) return;
        it.blk = jj / nul;
      }
      it.g = unit / c.S_pre;
      it.split = unit - it.g * c.S_pre;
      it.skip = (int64_t)it.split * it.len;
      if (it.split == c.S_pre - 1) it.len = c.P;
      ncol = min(max(c.row_off[c.B], 0), c.Mcap) * rep;
      if (it.blk * 128 >= ncol) return;
      int* off = (int*)stg;
      stage_offsets(off, c.row_off, c.B);
      __syncthreads();
    } else {
      if (!find_item<CB, walk, tree>(c, at, it)) return;
      const RowSpan sp = row_span(c.row_off, it.b, c.max_per_row, c.Mcap);
      base = sp.base;
      ncol = sp.n * rep;
    }
    const int c0 = it.blk * CB;
    // this lane's column
    const int col = c0 + 32 * cw + kk;
    ok = col < ncol;
    const int j = ok ? col / rep : 0, head = it.g * rep + (ok ? col - j * rep : 0);
    Query qy{0, 0, 0};
    if (pre) {
      const int* off = (const int*)stg;
      const int r = row_of(off, c.B, j);
      RowSpan sp{0, 0};
      if (r < c.B) sp = row_span(off, r, c.max_per_row, c.Mcap);
      ok = ok && j >= sp.base && j < sp.base + sp.n;
      if (ok) qy = query_at<tree>(c, c.start[r], sp.n, j - sp.base, j);
    } else {
      tok = base + j;
      qy = query_at<tree>(c, c.start[it.b], ncol / rep, j, tok);
    }
    {
      const bf16_t* qr = (const bf16_t*)c.q + (base + j) * c.qst + head * c.qsh + 8 * hl;
      const uint32_t keep = ok ? 0xffffffffu : 0u;
#pragma unroll
      for (int h = 0; h < DS; ++h) qf[h] = *(const v4u*)(qr + 16 * h) & keep;
    }
    walk_range<walk, tree>(c, qy, lo_c, hi_c);
    if (!ok) lo_c = 0x7fffffff, hi_c = -1;
    // the keys that some column of the workgroup sees
    w_lo = lanes_min<32>(lo_c <= hi_c ? lo_c : 0x7fffffff);
    w_hi = lanes_max<32>(lo_c <= hi_c ? hi_c : -1);
    if (lane == 0) {
      lds.rng[wave][0] = w_lo;
      lds.rng[wave][1] = w_hi;
    }
    __syncthreads();
    int g_lo = 0x7fffffff, g_hi = -1;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      g_lo = min(g_lo, lds.rng[w][0]);
      g_hi = max(g_hi, lds.rng[w][1]);
    }
    g_lo = __builtin_amdgcn_readfirstlane(g_lo);
    g_hi = __builtin_amdgcn_readfirstlane(g_hi);
    // (a row's splits are counted from its first column's first key in every one of its blocks)
    int row_lo = g_lo, unused;
    if (!pre && c.window > 0) walk_range<walk, tree>(c, Query{c.start[it.b], c.start[it.b], 1}, row_lo, unused);
    const int64_t s_beg = (int64_t)(row_lo & ~31) + it.skip;
    kend64 = min((int64_t)g_hi + 1, s_beg + it.len);
    kbeg64 = max(s_beg, (int64_t)(g_lo & ~31));
  }
  const int b = it.b, g = it.g, c0 = it.blk * CB;
  const bool none = kbeg64 >= kend64;
  if (none && w.S_own + w.S_pre > 1) {
    const int cx = c0 + threadIdx.x, rep = w.H / w.pv.G;
    if (threadIdx.x < CB && cx < ncol) {
      const int jx = cx / rep;
      const int64_t pair = (int64_t)(base + jx) * w.H + g * rep + cx - jx * rep;
      w.pml[(int64_t)(pre ? w.S_own + it.split : it.split) * w.Mcap * w.H + pair] = make_float2(-INFINITY, 0.f);
      if (!pre) mark_unused(w, it, pair);
    }
    return;
  }
  const int kbeg = none ? 0 : (int)kbeg64, kend = none ? 0 : (int)kend64;
  // byte offsets of this lane's 16 bytes of the operands: K row kk is key
  // 16 (kk / 16) + 8 ((kk / 4) % 2) + 4 ((kk / 8) % 2) + kk % 4 of the tile, V row kk is dim kk of 32
  const int key = ((kk >> 4) << 4) | (((kk >> 2) & 1) << 3) | (((kk >> 3) & 1) << 2) | (kk & 3);
  const uint32_t koff = HD == 128 ? 16u * (uint32_t)((((key >> 2) & 1) << 6) + ((key >> 3) << 2) + (key & 3) + 16 * hl)
                                  : (uint32_t)(key * (2 * HD) + 16 * hl);
  const uint32_t voff = 16u * (uint32_t)(4 * kk + hl);
  const int64_t gofs = (int64_t)g * w.pv.page * HD;
  const float scale_log2 = w.scale * 1.4426950408889634f;
  const char *kp = (const char*)scalar(w.kp), *vp = (const char*)scalar(w.vp);
  const int tpp = w.pv.page >> 5;
  f32x16 O[DD];
#pragma unroll
  for (int dd = 0; dd < DD; ++dd)
#pragma unroll
    for (int x = 0; x < 16; ++x) O[dd][x] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  bool odd = false;
  __syncthreads();  // the rows' offsets in the stages have been read
  // each wave's loads of a tile: a quarter of K's slices and of V's dims
#define WIDE_ISSUE(S_)                                                                                       \
  next = 0;                                                                                                  \
  _Pragma("unroll") for (int u = 0; u < 2; ++u) {                                                            \
    const bool is = (unsigned)id < (unsigned)w.pv.N;                                                         \
    next |= (int)is << u;                                                                                    \
    const int64_t pid = is ? id : 0; /* no page: page 0's place is read and masked */                        \
    const bf16_t* kt = (const bf16_t*)kp + pid * w.pv.ks + gofs + tr * (32 * HD);                            \
    const bf16_t* vt = (const bf16_t*)vp + pid * w.pv.vs + gofs + tr * (32 * HD);                            \
    if constexpr (HD == 128) {                                                                               \
      const uint32_t lk = LDS_ADDR(S_.k[u][0]) + 2048 * wave, lv = LDS_ADDR(S_.v[u][0]) + 2048 * wave;       \
      lds_load_1k(kt + 1024 * wave, koff, lk);                                                               \
      lds_load_1k(kt + 1024 * wave + 256, koff, lk + 1024);                                                  \
      lds_load_1k(vt + 1024 * wave, voff, lv);                                                               \
      lds_load_1k(vt + 1024 * wave + 16, voff, lv + 1024);                                                   \
    } else {                                                                                                 \
      lds_load_1k(kt + 16 * wave, koff, LDS_ADDR(S_.k[u][0]) + 1024 * wave);                                 \
      lds_load_1k(vt + 1024 * (wave >> 1) + 16 * (wave & 1), voff, LDS_ADDR(S_.v[u][0]) + 1024 * wave);      \
    }                                                                                                        \
    if (tile < tlast) {                                                                                      \
      ++tile;                                                                                                \
      if (++tr == tpp) {                                                                                     \
        tr = 0;                                                                                              \
        id = id_next;                                                                                        \
        ++pg;                                                                                                \
        id_next = list[min(pg + 1, pg_last)];                                                                \
      }                                                                                                      \
    }                                                                                                        \
  }
#define WIDE_SYNC()                                                                                          \
  {                                                                                                          \
    __builtin_amdgcn_sched_barrier(0);                                                                       \
    __builtin_amdgcn_s_waitcnt(0); /* this step's loads, issued a step ago, and this wave's LDS reads */     \
    __atomic_signal_fence(__ATOMIC_SEQ_CST);                                                                 \
    __builtin_amdgcn_sched_barrier(0);                                                                       \
    __builtin_amdgcn_s_barrier();                                                                            \
    __builtin_amdgcn_sched_barrier(0);                                                                       \
    __atomic_signal_fence(__ATOMIC_SEQ_CST);                                                                 \
  }
  // the prefix and then the row's own keys, or the one of them that this walk is over
#pragma unroll 1
  for (int part = walk == ROW_KEYS && w.joint > 0 ? 0 : 1; part < 2; ++part) {
    const int from = part == 1 && walk == ROW_KEYS ? w.joint : 0;
    const int t0 = max(kbeg - from, 0), t1 = part == 0 ? min(kend, w.P) : kend - from;
    if (t0 >= t1) continue;
    const int ntiles = (t1 - t0 + 31) >> 5, nstep = (ntiles + 1) >> 1;
    const int tlast = (t0 >> 5) + ntiles - 1, pg0 = (t0 >> 5) / tpp, pg_last = tlast / tpp;
    const const_ints list = CONST_INTS(pre || part == 0 ? w.pre : w.tables + (int64_t)b * w.W);
    // keys that the column sees, that one of the wave does, that all of them do; behind t1 a step repeats its last tile
    const int lo = lo_c - from, hi = min(hi_c - from, t1 - 1), a_lo = w_lo - from, a_hi = min(w_hi - from, t1 - 1);
    const int f_lo = lanes_max<32>(ok ? lo : 0), h_hi = lanes_min<32>(ok ? hi : 0x7fffffff);
    // a tree's nodes: their keys' first, and the words of bits that say who sees which (in the prefix, none)
    const int nodes = tree && !pre ? nodes_from(w.start[b], part == 0 ? 0 : w.P) : 0x7fffffff;
    const int f_hi = tree && !pre ? min(h_hi, nodes - 1) : h_hi;
    // the walk over the pages, one tile at a time; the next page's entry is under way a page ahead
    int tile = t0 >> 5, pg = pg0, tr = tile - pg * tpp;
    int id = list[pg], id_next = list[min(pg + 1, pg_last)];
    int now = 0, next = 0;  // bit u: the page of tile u of the step is one of the pool's
    auto step = [&](const WideStage<HD>& S_, int in, int i) {
      const int kb = t0 + 64 * i;
      if (!(kb <= a_hi && kb + 63 >= a_lo)) return;
      uint32_t bits = 0xffffffffu;  // which of the lane's keys a tree's node may see, 16 of either tile
      if (tree && !pre && kb + 63 >= nodes) {
        const uint64_t* row = w.mask + (int64_t)tok * w.words;
        const int words = part == 0 ? 0 : w.words, k0 = kb + 32 * u0 + 8 * hl - nodes;
        bits = bits8(row, words, k0) | bits8(row, words, k0 + 16) << 8;
        if (!halves) bits |= bits8(row, words, k0 + 32) << 16 | bits8(row, words, k0 + 48) << 24;
      }
      f32x16 sc[NU];
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int x = 0; x < 16; ++x) sc[u][x] = 0.f;
      v4u kf[DS][NU], vf[NU][DS];
#pragma unroll
      for (int h = 0; h < DS; ++h)
#pragma unroll
        for (int u = 0; u < NU; ++u) kf[h][u] = __builtin_bit_cast(v4u, S_.k[u0 + u][h][lane]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < DS; ++h)
#pragma unroll
        for (int u = 0; u < NU; ++u) sc[u] = mfma32(kf[h][u], qf[h], sc[u]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int f = 0; f < DS; ++f) vf[u][f] = __builtin_bit_cast(v4u, S_.v[u0 + u][f][lane]);
      __builtin_amdgcn_sched_barrier(0);
      if (!(kb >= f_lo && kb + 63 <= f_hi && in == 3)) {
        u16x2 mag = {0, 0};
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const bool there = (in >> (u0 + u)) & 1;
          const int k0 = kb + 32 * (u0 + u) + 8 * hl;
          const int lr = there ? lo - k0 : 64, hr = hi - k0;
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int kx = 16 * (x >> 3) + (x & 7);
            if (!(kx >= lr && kx <= hr && (!tree || pre || (bits >> (16 * u + x) & 1)))) sc[u][x] = -INFINITY;
          }
          // keys that no column of the wave sees: their weights are 0, and so have their V to be, which may be
          // anything; then whether any is left that is not finite
          const int zl = there ? a_lo - k0 : 64, zh = a_hi - k0;
#pragma unroll
          for (int f = 0; f < DS; ++f) {
            const int kx = 16 * (f & 1);
            v4u v = vf[u][f];
            v.x &= key_mask(kx, zl, zh);
            v.y &= key_mask(kx + 2, zl, zh);
            v.z &= key_mask(kx + 4, zl, zh);
            v.w &= key_mask(kx + 6, zl, zh);
            mag = max_magnitude(max_magnitude(mag, v.x), v.y);
            mag = max_magnitude(max_magnitude(mag, v.z), v.w);
            vf[u][f] = v;
          }
        }
        odd |= any_odd(mag);
      }
      float m4[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) m4[x] = fmaxf(sc[0][x], sc[NU - 1][x]);
#pragma unroll
      for (int x = 4; x < 16; ++x) m4[x & 3] = fmaxf(m4[x & 3], fmaxf(sc[0][x], sc[NU - 1][x]));
      float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      {
        const auto h2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
        mt = fmaxf(__uint_as_float(h2[0]), __uint_as_float(h2[1]));  // lanes l and l ^ 32: the column's two key halves
      }
      const float m_new = fmaxf(m_run, mt * scale_log2);
      if (__any(m_new > m_run)) {
        const float alpha = exp2a(m_run - (m_new == -INFINITY ? 0.f : m_new));
        l_run *= alpha;
#pragma unroll
        for (int dd = 0; dd < DD; ++dd) O[dd] *= alpha;
        m_run = m_new;
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run;  // no key yet: every term exp2(-inf) = 0
      float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          float pv[8];  // rounded to bf16 for the product, not in the sum (see Tile<bf16_t>::add)
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            pv[x] = exp2a(fmaf(sc[u][8 * kh + x], scale_log2, -m_use));
            ps[x & 3] += pv[x];
          }
          const v4u pb =
              v4u{pack2bf(pv[0], pv[1]), pack2bf(pv[2], pv[3]), pack2bf(pv[4], pv[5]), pack2bf(pv[6], pv[7])};
#pragma unroll
          for (int dd = 0; dd < DD; ++dd) O[dd] = mfma32(vf[u][2 * dd + kh], pb, O[dd]);
        }
      l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
    };
    WIDE_ISSUE(stg[0]);
    for (int i = 0; i < nstep; ++i) {
      now = next;
      WIDE_SYNC();
      WIDE_ISSUE(stg[(i + 1) & 1]);
      step(stg[i & 1], now, i);
    }
    WIDE_SYNC();  // no direct load outlives its stage, no reader is left in the stages
  }
#undef WIDE_SYNC
#undef WIDE_ISSUE
  if (__syncthreads_or(odd)) {
    redo_columns<bf16_t, HD, tree>(walk, it, base, c0, min(c0 + CB, ncol), kbeg, kend, wave);
    return;
  }
  if constexpr (halves) {
    // the second tiles' waves hand over: the sums through the second stage, maximum and sum through what the taking wave
    // writes its outputs through later
    float* sums = (float*)&stg[1] + cw * (DD * 16 * 64) + lane;
    float2* ml = (float2*)((bf16_t*)&stg[0] + cw * 32 * (HD + 8)) + lane;
    static_assert(sizeof(WideStage<HD>) >= 2 * DD * 16 * 64 * 4, "two waves' sums");
    if (u0 == 1) {
#pragma unroll
      for (int dd = 0; dd < DD; ++dd)
#pragma unroll
        for (int x = 0; x < 16; ++x) sums[(16 * dd + x) * 64] = O[dd][x];
      *ml = make_float2(m_run, l_run);
    }
    __syncthreads();
    if (u0 == 1) return;
    const float2 e = *ml;
    const float m_new = fmaxf(m_run, e.x), mu = m_new == -INFINITY ? 0.f : m_new;
    const float a0 = exp2a(m_run - mu), a1 = exp2a(e.x - mu);
    l_run = l_run * a0 + e.y * a1;
    m_run = m_new;
#pragma unroll
    for (int dd = 0; dd < DD; ++dd)
#pragma unroll
      for (int x = 0; x < 16; ++x) O[dd][x] = O[dd][x] * a0 + sums[(16 * dd + x) * 64] * a1;
  }
  const PagedChunk c = chunk_args();
  const int rep = c.H / c.pv.G, sg = pre ? c.S_own + it.split : it.split;
  const int col = c0 + 32 * cw + kk, j = ok ? col / rep : 0, head = g * rep + (ok ? col - j * rep : 0);
  const float l_tot = l_run + __shfl_xor(l_run, 32, WAVE);
  // lane: column kk; register 4 i4 + x of O[dd] is dim 32 dd + 8 i4 + 4 hl + x
  if (pre || !whole(c, it)) {
    if (ok) {
      const int64_t slot = ((int64_t)sg * c.Mcap + base + j) * c.H + head;
      float* po = c.po + slot * HD + 4 * hl;
#pragma unroll
      for (int dd = 0; dd < DD; ++dd)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          *(float4*)(po + 32 * dd + 8 * i4) =
              make_float4(O[dd][4 * i4], O[dd][4 * i4 + 1], O[dd][4 * i4 + 2], O[dd][4 * i4 + 3]);
      if (hl == 0) {
        c.pml[slot] = make_float2(m_run, l_tot);
        if (!pre) mark_unused(c, it, (int64_t)(base + j) * c.H + head);
      }
    }
  } else {
    if (ok && hl == 0) mark_whole(c, (int64_t)(base + j) * c.H + head);
    // through LDS, so that a lane writes 8 dims of a column
    const float inv = l_tot == 0.f ? 0.f : 1.f / l_tot;
    constexpr int LD = HD + 8;
    bf16_t* T = (bf16_t*)&stg[wave >> 1] + (wave & 1) * 32 * LD;
    static_assert(sizeof(WideStage<HD>) >= 2 * 32 * LD * 2, "two waves' scratch");
#pragma unroll
    for (int dd = 0; dd < DD; ++dd)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        uint2 pk;
        pk.x = pack2bf(O[dd][4 * i4] * inv, O[dd][4 * i4 + 1] * inv);
        pk.y = pack2bf(O[dd][4 * i4 + 2] * inv, O[dd][4 * i4 + 3] * inv);
        *(uint2*)(T + kk * LD + 32 * dd + 8 * i4 + 4 * hl) = pk;
      }
    __builtin_amdgcn_wave_barrier();
    constexpr int TP = HD / 8, CP = 64 / TP;  // lanes per column, columns per pass
#pragma unroll
    for (int it = 0; it < 32 / CP; ++it) {
      const int cc = CP * it + lane / TP, d0 = 8 * (lane % TP), co = c0 + 32 * cw + cc, jo = co / rep;
      const uint4 val = *(const uint4*)(T + cc * LD + d0);
      if (co < ncol) *(uint4*)((bf16_t*)c.y + ((int64_t)(base + jo) * c.H + g * rep + co - jo * rep) * HD + d0) = val;
    }
  }
}

// The prefix (PRE: 16-column blocks of the streaming kernel, 0: the wide one,
// -1: no prefix) and the rows' own keys (OWN likewise, 64: the wide one with blocks of
// 64 columns) in one launch: the first is bound by the matrix cores where many rows
// share it, the second by memory, and each hides the other's start and end. 256 workgroups of either in turn, so that a CU
// holds one of each. (64 samples behind 5000 keys: 41 us with the merge, the rows' own
// keys alone 29, the prefix alone 15.) Without a prefix the streaming kernel runs
// three to a CU, which hides more of the waits at an item's start (64 rows of 300 keys
// 25 us, two to a CU 30; rows of 100000 keys 1262 us, and 1243).
template <typename T, int HD, int PRE, int OWN, bool tree>
__global__ __launch_bounds__(256, PRE < 0 && OWN == 1 && sizeof(T) == 2 ? 3 : 2) void k_paged_attn(PagedChunk c,
                                                                                                int npre, int nown) {
  union Lds {
    StreamLds<HD> s;
    std::conditional_t<PRE == 0 || OWN == 0 || OWN == 64, WideLds<HD>, char> w;
  };
  __shared__ Lds lds;
  int at = blockIdx.x;
  if constexpr (PRE < 0) zero_tail<T>(blockIdx.x, gridDim.x);
  if constexpr (PRE >= 0) {
    const int both = min((npre + 255) >> 8, (nown + 255) >> 8);
    bool pre;
    if ((at >> 8) < 2 * both) {
      pre = !((at >> 8) & 1);
      at = ((at >> 9) << 8) | (at & 255);
    } else {
      at -= both << 8;
      pre = npre > nown;
    }
    if (pre) {
      if (at >= npre) return;
      if constexpr (PRE == 0) wide_keys<HD, PREFIX_KEYS, tree>(c, lds.w, at);
      else stream_keys<T, HD, PRE, true, tree>(c, lds.s, at);
      return;
    }
    if (at >= nown) return;
  }
  const PagedChunk o = PRE >= 0 ? chunk_args() : c;
  if constexpr (OWN == 64) wide_keys<HD, OWN_KEYS, tree, 64>(o, lds.w, at);
  else if constexpr (OWN == 0) wide_keys<HD, PRE < 0 ? ROW_KEYS : OWN_KEYS, tree>(o, lds.w, at);
  else stream_keys<T, HD, OWN, false, tree>(o, lds.s, at);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {
// Bytes of partials that the own keys' splits are cut down to, and those of the prefix for themselves: together up to
// twice that. One split of each there is whatever its size. (16000 tokens of 12 heads of 128 behind 4000 keys ask for up
// to 381 MiB, two splits of either, 95 MiB each; 100000 such tokens in 4000 rows for 1.2 GiB, one of either.)
constexpr int64_t kPartMax = 256ll << 20;
// How a call is cut: the kernels of the rows' own keys and of the prefix (query
// blocks of 16 columns in a workgroup of the streaming kernel, 0: the wide one),
// their column blocks, and the key splits.
struct PagedPlan {
  bool mfma, even;  // even: the prefix's workgroups go to the XCDs in equal numbers, not by units
  int own_qb, own_cb, own_blk, pre_qb, pre_blk;
  int S_own, S_pre, pre_chunk, target, joint;
  int64_t items;  // of the rows' own keys, at most: every row's last chunk may be short, none has more than S_own
  int64_t part_bytes, ml_bytes, item_bytes;
};
// Key splits of the prefix. With S of them, in us: the time that their workgroups
// take on the XCD with the most of them (a unit's column blocks share one; 64 run
// at once there, two a CU), 2 us for a step of 64 keys, twice that in fp32, and six
// steps for a workgroup's start and end; half of one workgroup's time alone (1.2 us a
// step: the rows' own keys hide some of it); 5 TB/s for the partials, and 0.2 of
// the merge. Against the best of S = 1 .. 40 its choice costs 5% or less in 10 of 13
// measured shapes and 16% at most (prefixes of 1000 to 16000 keys under 1 to 4482
// tokens: 18 to 212 us).
int pre_splits(int64_t P, int G, int blk, int64_t part_bytes, int most, bool fp32) {
  int best = 1;
  double least = 1e30;
  for (int S = 1; S <= std::min<int64_t>(most, (P + 127) / 128); ++S) {
    const int64_t on = (int64_t)((G * S + 7) / 8) * blk;
    const double steps = (double)(((P + S - 1) / S + 63) / 64 * (fp32 ? 2 : 1) + 6);
    const double t = on * steps * 2.0 / 64 + steps * 0.6 + S * (0.2 + (double)part_bytes * 2 / 5e6);
    if (t < least) least = t, best = S;
  }
  return best;
}
// The same where the workgroups go to the XCDs in equal numbers (`even`), beside `items` of the rows' own keys. A step of
// a workgroup alone on its CU is 1.5 us, of one of two 2.4, and with more than two for every CU the last ones are a
// round of their own, or fill the gaps of others, half and half; a start and an end are four steps. As far as the own
// keys' items fill the card, the prefix's time counts half, and the sum of its steps for the rest. Its choice costs 4% or
// less against the best of S = 1 .. 10 in 9 of 10 measured shapes, 17% in the other (prefixes of 500 to 16000 keys under
// 40 to 1600 nodes, 17 to 148 us).
int pre_splits_even(int64_t P, int G, int blk, int64_t part_bytes, int most, int64_t items) {
  const double fill = std::min(1.0, (double)items / 512);
  int best = 1;
  double least = 1e30;
  for (int S = 1; S <= std::min<int64_t>(most, (P + 127) / 128); ++S) {
    const int64_t on = ((int64_t)G * S * blk + 7) / 8;
    const double steps = (double)(((P + S - 1) / S + 63) / 64), rounds = (double)on / 64;
    const double step = on <= 24 ? 1.5 : on <= 40 ? 1.5 + 0.9 * (double)(on - 24) / 16
                        : on <= 64 ? 2.4 : 2.4 * (rounds + std::ceil(rounds)) / 2;
    const double t = (steps + 4) * step * (1 - fill / 2) + (double)on * (steps + 6) * 2.0 / 64 * fill +
                     S * (0.2 + (double)part_bytes * 2 / 5e6);
    if (t < least) least = t, best = S;
  }
  return best;
}
PagedPlan paged_plan(const fc_pages* p, int B, int T, int max_per_row, int H, int W, int P, int window, bool tree) {
  PagedPlan a{};
  a.mfma = p->head_dim == 64 || p->head_dim == 128;
  if (!a.mfma) return a;
  const int G = p->n_kv_head, rep = H / G;
  auto kernel = [&](int64_t ncol, int& qb, int& blk) {
    qb = ncol <= 16 || p->dtype == FC_F32 ? 1 : ncol <= 32 ? 2 : 0;
    blk = (int)(qb ? (ncol + 16 * qb - 1) / (16 * qb) : (ncol + 127) / 128);
  };
  const int64_t cols = (int64_t)std::min(max_per_row, T) * rep;
  kernel(cols, a.own_qb, a.own_blk);
  a.own_cb = a.own_qb ? 16 * a.own_qb : tree && cols <= 64 ? 64 : 128;
  kernel((int64_t)T * rep, a.pre_qb, a.pre_blk);
  a.mfma = (!a.own_qb || a.own_blk <= 65535) && (!a.pre_qb || a.pre_blk <= 65535);
  if (!a.mfma) return a;
  const int64_t width = (int64_t)W * p->page, pad = ((int64_t)P + 31) / 32 * 32;
  // (a row's last block may be short, so the tokens make up to one more block a row than they would side by side)
  const int64_t units = G * std::min((int64_t)B * a.own_blk, (int64_t)T * rep / a.own_cb + B);
  // Rows that fill column blocks of the wide kernel may walk the prefix themselves, which saves its partials and the
  // merge, but cuts the work coarser and leaves the rows' last blocks part empty: done where they see little of it, or
  // the blocks are several rounds of the card's 512 workgroups and not many more than the tokens fill. (92 rows of 490
  // tokens, 8 heads on one, behind 7 keys: 167 us so, and 726 with the prefix walked for itself; 64 rows of up to 512,
  // 12 heads, behind 2000: 441 and 542; but 16 such rows behind 4001, 516 blocks, 264 and 205, and 100 rows of up to
  // 130 behind 8000 627 and 422.)
  const int64_t full = G * ((int64_t)T * rep / 128);
  const bool rounds = units >= 3 * 512 && units <= full + full * 3 / 5;
  const int seen = window > 0 ? std::min(P, window) : P;  // by tokens behind the prefix
  if (P > 0 && !a.own_qb && cols >= 128 && (seen <= 1024 || rounds) && pad + width <= 0x7fffffff) a.joint = (int)pad;
  // the rows' walks
  const int64_t all = width + a.joint;
  const int64_t longest = window > 0 ? std::min(all, (int64_t)window + max_per_row + 64) : all;
  const int64_t one = (int64_t)T * H * (p->head_dim + 2) * 4;
  const int64_t room = std::max<int64_t>(1, kPartMax / one);
  a.S_own = (int)std::min({(longest + 127) / 128, room, (int64_t)64});
  // Where the rows alone make several items for every workgroup, no more than it takes to cut the longest into pieces
  // of 512 keys (1024 in the wide kernel): every (token, head) has a sum for each. (16 rows of up to 512 tokens at up
  // to 2000 keys: 97 us without this rule and with partials of rows that are not split, 84 so.)
  const int fill = a.own_qb ? 4 * 768 : 512, piece = a.own_qb ? 512 : 1024;
  a.S_own = (int)std::min<int64_t>(a.S_own, std::max((longest + piece - 1) / piece, (fill - 1 + units) / units));
  // short rows without a prefix: one split, and no merge (one row of 640 keys, 6 heads: one launch of 10.6 us, or 6.8
  // and 3.4 with the gap between them; 17 us or 21 from one call to the next)
  if (P == 0 && longest <= 1024) a.S_own = 1;
  a.target = a.own_qb ? 768 : 256;
  if (tree) {
    // Without a prefix chunk_length decides, by the rows' lengths, whether any is cut. A rule here could only go by the
    // slots for rows and the tables' width: it would save rows of one length the merge (32 rows of 64 nodes at 1280 keys,
    // 12 heads, 60 us, 63 with it) and leave one live row of 64 at 3900 keys, or one among 31 of 100-300, to a workgroup
    // a head (70 and 28 us; 73 and 32).
    // Behind a prefix in the wide kernel long rows are cut to the mean's length (128 rows of 50 to 2000 keys, up to 25
    // nodes of 12 heads on 4, behind 6144 keys: 148 us, 158 uncut).
    if (P > 0 && !a.own_qb) a.target = 512;
  }
  const int64_t cut = units * longest / (a.own_qb ? CHUNK_MAX : CHUNK_WIDE) + 1;
  a.items = std::min(units * a.S_own, units + std::max<int64_t>(a.target, cut));
  a.even = tree && !a.pre_qb;
  if (P > 0 && a.joint == 0) {
    // The splits are counted from the first key that a column block sees: all of the prefix, or, by tokens behind it,
    // the window's end. The last one takes what is left, for rows that begin within the prefix. (7 rows of 9 tokens, 8
    // heads on one, fp32, a window of 1024 over 12268 keys: 85 us with splits of the whole prefix, 25 so.)
    // (in 64 bits: a prefix may have up to 2^31 - 33 positions)
    const int64_t over = window > 0 ? std::min<int64_t>(P, (int64_t)window + 32) : P;
    const int most = (int)std::min<int64_t>(room, 128);
    const int S = a.even ? pre_splits_even(over, G, a.pre_blk, one, most, a.items)
                         : pre_splits(over, G, a.pre_blk, one, most, p->dtype == FC_F32);
    const int64_t chunk = ((over + S - 1) / S + 63) / 64 * 64;
    a.S_pre = (int)((over + chunk - 1) / chunk);
    a.pre_chunk = (int)std::min<int64_t>(chunk, 0x7fffffc0);  // (below the chunk with one split alone, which takes all)
  }
  if (a.S_own + a.S_pre > 1) {
    const int64_t pairs = (int64_t)T * H * (a.S_own + a.S_pre);
    a.part_bytes = fc_align(pairs * p->head_dim * 4);
    a.ml_bytes = fc_align(pairs * 8);
  }
  if (B > ROWS_SCAN) a.item_bytes = fc_align((1 + PT_ROWS / 64) * 4);
  return a;
}

// workgroups of the prefix: in the wide kernel's order its units go to the XCDs in turn
int64_t prefix_groups(const PagedPlan& a, int G) {
  const int units = G * a.S_pre;
  if (a.even) return ((int64_t)units * a.pre_blk + 7) / 8 * 8;
  return (int64_t)(a.pre_qb ? units : (units + 7) / 8 * 8) * a.pre_blk;
}

template <typename T, int HD, bool tree>
int launch_mfma(const PagedChunk& c, const PagedPlan& a, hipStream_t s) {
  const int nown = (int)a.items, npre = (int)prefix_groups(a, c.pv.G);
  if (c.B > ROWS_SCAN) {
    if (tree && a.own_cb == 64) hipLaunchKernelGGL((k_paged_items<64, OWN_KEYS, tree>), dim3(1), dim3(1024), 0, s, c);
    else if (a.own_qb == 0) hipLaunchKernelGGL((k_paged_items<128, ROW_KEYS, tree>), dim3(1), dim3(1024), 0, s, c);
    else if (a.own_qb == 2) hipLaunchKernelGGL((k_paged_items<32, OWN_KEYS, tree>), dim3(1), dim3(1024), 0, s, c);
    else hipLaunchKernelGGL((k_paged_items<16, OWN_KEYS, tree>), dim3(1), dim3(1024), 0, s, c);
    FC_LAUNCH_CHECK();
  }
  const dim3 grid(npre == 0 ? nown : 256 * ((npre + 255) / 256 + (nown + 255) / 256));
#define PAGED(PRE, OWN)                                                                                             \
  hipLaunchKernelGGL((k_paged_attn<T, HD, PRE, OWN, tree>), grid, dim3(256), 0, s, c, npre, nown)
  if constexpr (sizeof(T) == 4) {
    if (npre == 0) PAGED(-1, 1);
    else PAGED(1, 1);
  } else if (npre == 0) {
    if (a.own_qb == 1) PAGED(-1, 1);
    else if (a.own_qb == 2) PAGED(-1, 2);
    else if (tree && a.own_cb == 64) PAGED(-1, tree ? 64 : 0);
    else PAGED(-1, 0);
  } else if (a.own_qb == 0) {
    if (tree && a.own_cb == 64) PAGED(0, tree ? 64 : 0);
    else PAGED(0, 0);
  } else if (a.own_qb == 2) {
    if (a.pre_qb == 2) PAGED(2, 2);
    else PAGED(0, 2);
  } else {
    if (a.pre_qb == 1) PAGED(1, 1);
    else if (a.pre_qb == 2) PAGED(2, 1);
    else PAGED(0, 1);
  }
#undef PAGED
  FC_LAUNCH_CHECK();
  const int S = a.S_own + a.S_pre;
  if (S > 1) {
    const int64_t threads = (int64_t)c.Mcap * c.H * (HD / 8);
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (S <= 2) hipLaunchKernelGGL((k_paged_merge<T, HD, 2>), grid, dim3(256), 0, s, c);
    else if (S <= 4) hipLaunchKernelGGL((k_paged_merge<T, HD, 4>), grid, dim3(256), 0, s, c);
    else hipLaunchKernelGGL((k_paged_merge<T, HD, 8>), grid, dim3(256), 0, s, c);
    FC_LAUNCH_CHECK();
  }
  return FC_OK;
}
}  // namespace

namespace {
// A tree's nodes as bits; none: a chunk's tokens follow one another.
struct TreeBits {
  const uint64_t* mask;
  const int32_t* tok_pos;
};
}  // namespace

// What the plan's arithmetic and the launches are made for. (A launch's threads are counted in 32 bits along x, its
// workgroups in 16 along y.)
static constexpr int64_t kMostGroups = (1 << 24) - 1024;
static int check_sizes(const fc_pages* p, int32_t batch, int32_t max_tokens, int32_t max_per_row, int32_t n_head,
                       int32_t width, int32_t prefix_len, int32_t window) {
  FC_CHECK_ARG(batch > 0 && batch <= PT_ROWS, "batch must be in [1, 4096]");
  FC_CHECK_ARG(max_tokens > 0 && max_per_row > 0 && n_head > 0 && n_head % p->n_kv_head == 0,
               "max_tokens, max_per_row, n_head (a multiple of n_kv_head)");
  FC_CHECK_ARG(n_head <= 65535, "n_head must be <= 65535");
  FC_CHECK_ARG(window >= 0 && prefix_len >= 0, "window, prefix");
  FC_CHECK_ARG(width > 0 && (int64_t)width * p->page + prefix_len <= 0x7fffffff, "positions must fit 31 bits");
  const int64_t merge = (int64_t)max_tokens * n_head * (p->head_dim / 8) / 256;
  FC_CHECK_ARG(std::max<int64_t>(merge, max_tokens) < kMostGroups, "too many tokens or heads");
  return FC_OK;
}

static int64_t workspace_bytes(const fc_pages* pages, int32_t batch, int32_t max_tokens, int32_t max_per_row,
                               int32_t n_head, int32_t width, int32_t prefix_len, int32_t window, bool tree) {
  if (check_pages(pages) != FC_OK ||
      check_sizes(pages, batch, max_tokens, max_per_row, n_head, width, prefix_len, window) != FC_OK)
    return FC_ERR_ARG;
  const PagedPlan a = paged_plan(pages, batch, max_tokens, max_per_row, n_head, width, prefix_len, window, tree);
  return a.part_bytes + a.ml_bytes + a.item_bytes;
}

extern "C" int64_t fc_paged_attention_workspace_bytes(const fc_pages* pages, int32_t batch, int32_t max_tokens,
                                                      int32_t max_per_row, int32_t n_head, int32_t width,
                                                      int32_t prefix_len, int32_t window) {
  return workspace_bytes(pages, batch, max_tokens, max_per_row, n_head, width, prefix_len, window, false);
}

static int attention(const fc_pages* pages, const void* q, int64_t q_token_stride, int64_t q_head_stride, void* y,
                     int32_t batch, int32_t max_tokens, int32_t max_per_row, int32_t n_head, const int32_t* tables,
                     int32_t width, const int32_t* row_off, const int32_t* start, const int32_t* prefix_pages,
                     int32_t prefix_len, int32_t window, int32_t flags, void* work, int64_t work_bytes, void* stream,
                     const TreeBits* tree) {
  int rc = check_pages(pages);
  if (rc != FC_OK) return rc;
  FC_CHECK_ARG(q && y && tables && row_off && start, "null pointer");
  rc = check_sizes(pages, batch, max_tokens, max_per_row, n_head, width, prefix_len, window);
  if (rc != FC_OK) return rc;
  FC_CHECK_ARG(prefix_len == 0 || prefix_pages, "window, prefix");
  const PagedPlan a =
      paged_plan(pages, batch, max_tokens, max_per_row, n_head, width, prefix_len, window, tree != nullptr);
  FC_CHECK_ARG(a.items + prefix_groups(a, pages->n_kv_head) < kMostGroups, "too many tokens, rows or heads");
  const int64_t need = a.part_bytes + a.ml_bytes + a.item_bytes;
  FC_CHECK_ARG(need == 0 || (work && work_bytes >= need), "workspace too small");
  PagedChunk c{page_view(pages), tables, row_off, start, prefix_pages, batch, n_head, width, prefix_len, window,
               max_per_row, max_tokens, flags, q_token_stride, q_head_stride,
               1.f / sqrtf((float)pages->head_dim), a.S_own, a.S_pre, a.pre_chunk, a.target, a.joint, (float*)work,
               (float2*)((char*)work + a.part_bytes), (int*)((char*)work + a.part_bytes + a.ml_bytes),
               q, pages->k, pages->v, y, tree ? tree->mask : nullptr, tree ? tree->tok_pos : nullptr,
               tree ? (max_per_row + 63) / 64 : 0, a.pre_blk};  // (of plain chunks max_per_row may be 2^31 - 1)
  const hipStream_t s = (hipStream_t)stream;
  // the matrix-core kernels load 16 bytes at a time
  const int64_t strides = q_token_stride | q_head_stride | pages->k_stride | pages->v_stride;
  const bool vec = (((uintptr_t)q | (uintptr_t)pages->k | (uintptr_t)pages->v | (uintptr_t)y | (uintptr_t)work) & 15) ==
                       0 && (strides & (pages->dtype == FC_BF16 ? 7 : 3)) == 0;
  if (a.mfma && vec) {
    const bool bf = pages->dtype == FC_BF16, wide = pages->head_dim == 128;
    if (tree)
      return bf ? wide ? launch_mfma<bf16_t, 128, true>(c, a, s) : launch_mfma<bf16_t, 64, true>(c, a, s)
                : wide ? launch_mfma<float, 128, true>(c, a, s) : launch_mfma<float, 64, true>(c, a, s);
    return bf ? wide ? launch_mfma<bf16_t, 128, false>(c, a, s) : launch_mfma<bf16_t, 64, false>(c, a, s)
              : wide ? launch_mfma<float, 128, false>(c, a, s) : launch_mfma<float, 64, false>(c, a, s);
  }
  const dim3 grid(max_tokens, n_head);
  if (tree) {
    if (pages->dtype == FC_BF16) hipLaunchKernelGGL((k_paged_any<bf16_t, true>), grid, dim3(256), 0, s, c);
    else hipLaunchKernelGGL((k_paged_any<float, true>), grid, dim3(256), 0, s, c);
  } else {
    if (pages->dtype == FC_BF16) hipLaunchKernelGGL((k_paged_any<bf16_t, false>), grid, dim3(256), 0, s, c);
    else hipLaunchKernelGGL((k_paged_any<float, false>), grid, dim3(256), 0, s, c);
  }
  FC_LAUNCH_CHECK();
  return FC_OK;
}

extern "C" int32_t fc_paged_attention(const fc_pages* pages, const void* q, int64_t q_token_stride,
                                      int64_t q_head_stride, void* y, int32_t batch, int32_t max_tokens,
                                      int32_t max_per_row, int32_t n_head, const int32_t* tables, int32_t width,
                                      const int32_t* row_off, const int32_t* start, const int32_t* prefix_pages,
                                      int32_t prefix_len, int32_t window, int32_t flags, void* work,
                                      int64_t work_bytes, void* stream) {
  return attention(pages, q, q_token_stride, q_head_stride, y, batch, max_tokens, max_per_row, n_head, tables, width,
                   row_off, start, prefix_pages, prefix_len, window, flags, work, work_bytes, stream, nullptr);
}

static int check_tree_sizes(int32_t max_per_row) {
  FC_CHECK_ARG(max_per_row <= FC_TREE_MOST, "max_per_row must be in [1, 512]");
  return FC_OK;
}

extern "C" int64_t fc_tree_attention_workspace_bytes(const fc_pages* pages, int32_t batch, int32_t max_tokens,
                                                     int32_t max_per_row, int32_t n_head, int32_t width,
                                                     int32_t prefix_len, int32_t window) {
  if (check_tree_sizes(max_per_row) != FC_OK) return FC_ERR_ARG;
  return workspace_bytes(pages, batch, max_tokens, max_per_row, n_head, width, prefix_len, window, true);
}

extern "C" int32_t fc_tree_attention(const fc_pages* pages, const void* q, int64_t q_token_stride,
                                     int64_t q_head_stride, void* y, int32_t batch, int32_t max_tokens,
                                     int32_t max_per_row, int32_t n_head, const int32_t* tables, int32_t width,
                                     const int32_t* row_off, const int32_t* start, const uint64_t* mask,
                                     const int32_t* tok_pos, const int32_t* prefix_pages, int32_t prefix_len,
                                     int32_t window, int32_t flags, void* work, int64_t work_bytes, void* stream) {
  FC_CHECK_ARG(mask && tok_pos, "null pointer");
  const int rc = check_tree_sizes(max_per_row);
  if (rc != FC_OK) return rc;
  const TreeBits t{mask, tok_pos};
  return attention(pages, q, q_token_stride, q_head_stride, y, batch, max_tokens, max_per_row, n_head, tables, width,
                   row_off, start, prefix_pages, prefix_len, window, flags, work, work_bytes, stream, &t);
}
