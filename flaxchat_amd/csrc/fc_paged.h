// What the kernels over the paged KV cache share: the rows of a packed chunk
// and the places of K and V in a pool (include/flaxchat_amd.h).
#pragma once
#include "fc_internal.h"

#define PT_ROWS 4096  // rows a call may have

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

// What the kernels need of an fc_pages.
struct PageView {
  int64_t ks, vs;  // elements between pages
  int N, G, page, hd;
  int kblk;        // K blocks in the matrix-core order
};
static inline PageView page_view(const fc_pages* p) {
  return PageView{p->k_stride, p->v_stride, p->n_pages, p->n_kv_head, p->page, p->head_dim,
                  p->dtype == FC_BF16 && p->head_dim == 128};
}
static inline int check_pages(const fc_pages* p) {
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

// 8 consecutive values as fp32, and back (rounded to nearest even)
__device__ __forceinline__ void load8(const bf16_t* p, float (&x)[8]) {
  const uint4 u = *(const uint4*)p;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
// 8 results of a row, times f
__device__ __forceinline__ void store8(bf16_t* y, const float (&o)[8], float f) {
  *(uint4*)y = uint4{pack2bf(o[0] * f, o[1] * f), pack2bf(o[2] * f, o[3] * f), pack2bf(o[4] * f, o[5] * f),
                     pack2bf(o[6] * f, o[7] * f)};
}
__device__ __forceinline__ void store8(float* y, const float (&o)[8], float f) {
  ((float4*)y)[0] = make_float4(o[0] * f, o[1] * f, o[2] * f, o[3] * f);
  ((float4*)y)[1] = make_float4(o[4] * f, o[5] * f, o[6] * f, o[7] * f);
}
