// Decoding with trees of drafted tokens over the paged KV cache: the trees'
// bookkeeping, the append with rotation, the accepted path and its way back
// to consecutive positions. (The attention is fc_paged.hip's.) No counterpart
// in the reference, which verifies one drafted chain, token by token
// (flaxchat/engine.py:484-606); rotation and norm are those of
// flaxchat/gpt.py:52-71 and flaxchat/engine.py:108-126.
//
// Row b's chunk is tokens row_off[b] .. row_off[b+1]-1, its nodes; node i's
// parent is an earlier node of the row, anything else makes it a root. Node i
// sits in the cache at position start[b] + i, whatever its depth.
#include "fc_paged.h"
#include <type_traits>

// ---------------------------------------------------------------------------
// Ancestors
// ---------------------------------------------------------------------------
// Node i and the nodes above it, as bits: word w holds nodes 64 w .. 64 w + 63.
// Within a block of 64 nodes, a lane each, by doubling: with the ancestors up
// to 2^r steps above in m and the 2^r-th in p, m |= m[p] and p = p[p] give
// 2^(r+1) steps. Six rounds at most, whatever the tree's shape.
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int from) {
  const uint32_t lo = __shfl((uint32_t)v, from, WAVE), hi = __shfl((uint32_t)(v >> 32), from, WAVE);
  return (uint64_t)hi << 32 | lo;
}
// p: the lane's parent within the block, -1: none there
__device__ __forceinline__ uint64_t block_ancestors(int p) {
  uint64_t m = 1ull << (threadIdx.x & 63);
  for (int r = 0; r < 6 && __any(p >= 0); ++r) {
    const uint64_t mo = shfl64(m, max(p, 0));
    const int po = __shfl(p, max(p, 0), WAVE);
    if (p >= 0) {
      m |= mo;
      p = po;
    }
  }
  return m;
}
__device__ __forceinline__ int parent_of(const int* __restrict__ parent, int base, int i, int n) {
  const int p = i < n ? parent[base + i] : -1;
  return p >= 0 && p < i ? p : -1;
}

// All of a row's nodes, by a workgroup, into LDS: mask[node][W]. First every
// block of 64 for itself, with the node by which each lane's chain leaves it;
// then, block by block, the words of that node. Bits of nodes past n: only
// their own.
struct RowTree {
  uint64_t* mask;  // [64 W][W]
  int* up;         // [64 W] the first ancestor in an earlier block, -1: none
};
__device__ __forceinline__ RowTree row_tree(char* lds, int W) {
  return RowTree{(uint64_t*)lds, (int*)(lds + (size_t)64 * W * W * 8)};
}
static size_t row_tree_bytes(int W) { return (size_t)64 * W * (W * 8 + 4); }
__device__ __forceinline__ void row_ancestors(const RowTree& t, const int* __restrict__ parent, int base, int n,
                                              int W) {
  const int lane = threadIdx.x & 63, nb = (n + 63) >> 6;
  for (int k = threadIdx.x >> 6; k < nb; k += blockDim.x >> 6) {
    const int i = 64 * k + lane, p = parent_of(parent, base, i, n);
    const uint64_t m = block_ancestors(p >= 64 * k ? p - 64 * k : -1);
    t.mask[i * W + k] = m;
    const int above = __shfl(p, __builtin_ctzll(m), WAVE);  // the chain's topmost node here has the lowest index
    t.up[i] = above;
    for (int w = k + 1; w < W; ++w) t.mask[i * W + w] = 0;
  }
  __syncthreads();
  for (int k = 1; k < nb; ++k) {
    for (int x = threadIdx.x; x < 64 * k; x += blockDim.x) {
      const int i = 64 * k + x / k, w = x % k, u = t.up[i];
      t.mask[i * W + w] = u >= 0 ? t.mask[u * W + w] : 0;
    }
    __syncthreads();
  }
}

// Tokens of no row: behind the last one, before the first, or of a row that is treated as empty.
template <typename F>
__device__ __forceinline__ void each_unowned(const int* __restrict__ row_off, int b, int B, int max_tokens, int n,
                                             F f) {
  const int lo = max(row_off[b], 0), hi = min(row_off[b + 1], max_tokens);
  if (n == 0)
    for (int t = lo + threadIdx.x; t < hi; t += blockDim.x) f(t);
  if (b == 0)
    for (int t = threadIdx.x; t < min(lo, max_tokens); t += blockDim.x) f(t);
  for (int64_t t = max(row_off[B], 0) + (int64_t)b * blockDim.x + threadIdx.x; t < max_tokens;
       t += (int64_t)B * blockDim.x)
    f((int)t);
}

// m without its lowest k bits that are set: above the position below which there are k of them, found in six halvings.
__device__ __forceinline__ uint64_t without_lowest(uint64_t m, int k) {
  if (k >= __popcll(m)) return 0;
  int at = 0;
#pragma unroll
  for (int step = 32; step > 0; step >>= 1)
    if (__popcll(m & ((1ull << (at + step)) - 1)) <= k) at += step;
  return m >> at << at;
}

// window > 0: of a node's ancestors those at most `window` positions above it. Parents
// come before their children, so a node's bits lie in the order of its ancestors'
// depths, and the ones that are too far are its lowest.
//
// A row per workgroup; rows of up to 64 nodes in one wave's registers (ONE). Bound
// by latency: offsets, parents, at most six rounds of shuffles, the stores; 64 rows
// of 64 nodes 3.0 us. Longer rows, four waves a row: a round of LDS and a barrier
// for each block of 64 nodes; 500 rows of up to 300 nodes 6.2 us, 3.7 MB at 0.6 TB/s.
// A window that most nodes reach past adds 0.1 us to the first, 0.9 to the second.
template <bool ONE>
__global__ __launch_bounds__(256) void k_tree_tables(const int* __restrict__ parent, const int* __restrict__ row_off,
                                                     const int* __restrict__ start, uint64_t* __restrict__ mask,
                                                     int* __restrict__ tok_pos, int B, int max_tokens,
                                                     int max_per_row, int W, int window) {
  extern __shared__ char lds[];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int at = start[b];
  const RowSpan sp = row_span(row_off, b, max_per_row, max_tokens);
  each_unowned(row_off, b, B, max_tokens, sp.n, [&](int t) {
    for (int w = 0; w < W; ++w) mask[(int64_t)t * W + w] = 0;
    tok_pos[t] = -1;
  });
  if (sp.n == 0) return;
  if constexpr (ONE) {
    const uint64_t m = block_ancestors(parent_of(parent, sp.base, tid, sp.n));
    if (tid < sp.n) {
      const int deep = __popcll(m) - 1;
      mask[sp.base + tid] = window > 0 && deep > window ? without_lowest(m, deep - window) : m;
      tok_pos[sp.base + tid] = at + deep;
    }
  } else {
    const RowTree t = row_tree(lds, W);
    row_ancestors(t, parent, sp.base, sp.n, W);
    for (int i = tid; i < sp.n; i += blockDim.x) {
      int deep = -1;
      for (int w = 0; w <= i >> 6; ++w) deep += __popcll(t.mask[i * W + w]);
      tok_pos[sp.base + i] = at + deep;
      if (window > 0)
        for (int w = 0, far = deep - window; far > 0; ++w) {  // (far <= deep: it ends before the node's own word does)
          const uint64_t m = t.mask[i * W + w];
          t.mask[i * W + w] = without_lowest(m, far);
          far -= __popcll(m);
        }
    }
    if (window > 0) __syncthreads();
    for (int x = tid; x < sp.n * W; x += blockDim.x) mask[(int64_t)sp.base * W + x] = t.mask[x];
  }
}

static int check_tree(int32_t batch, int32_t max_tokens, int32_t max_per_row) {
  FC_CHECK_ARG(batch > 0 && batch <= PT_ROWS, "batch must be in [1, 4096]");
  FC_CHECK_ARG(max_tokens > 0 && max_tokens < 1 << 30, "max_tokens must be in [1, 2^30)");
  FC_CHECK_ARG(max_per_row > 0 && max_per_row <= FC_TREE_MOST, "max_per_row must be in [1, 512]");
  return FC_OK;
}

extern "C" int32_t fc_tree_tables_window(const int32_t* parent, const int32_t* row_off, const int32_t* start,
                                         uint64_t* mask, int32_t* tok_pos, int32_t batch, int32_t max_tokens,
                                         int32_t max_per_row, int32_t window, void* stream) {
  FC_CHECK_ARG(parent && row_off && start && mask && tok_pos, "null pointer");
  const int rc = check_tree(batch, max_tokens, max_per_row);
  if (rc != FC_OK) return rc;
  FC_CHECK_ARG(window >= 0, "window");
  const int W = (max_per_row + 63) / 64;
  const hipStream_t s = (hipStream_t)stream;
  if (W == 1)
    hipLaunchKernelGGL(k_tree_tables<true>, dim3(batch), dim3(64), 0, s, parent, row_off, start, mask, tok_pos, batch,
                       max_tokens, max_per_row, W, window);
  else
    hipLaunchKernelGGL(k_tree_tables<false>, dim3(batch), dim3(256), row_tree_bytes(W), s, parent, row_off, start,
                       mask, tok_pos, batch, max_tokens, max_per_row, W, window);
  FC_LAUNCH_CHECK();
  return FC_OK;
}
extern "C" int32_t fc_tree_tables(const int32_t* parent, const int32_t* row_off, const int32_t* start, uint64_t* mask,
                                  int32_t* tok_pos, int32_t batch, int32_t max_tokens, int32_t max_per_row,
                                  void* stream) {
  return fc_tree_tables_window(parent, row_off, start, mask, tok_pos, batch, max_tokens, max_per_row, 0, stream);
}

// ---------------------------------------------------------------------------
// Accept
// ---------------------------------------------------------------------------
// A node agrees if it is a root or its token is the target's choice at its
// parent; it is accepted if it and all nodes above it agree, that is, if none of
// its mask's bits is outside the agreeing nodes' set. The accepted node with the
// most nodes above it, the lowest index among equals, ends the path. The masks are
// made again (six shuffles) and not read: they would be the call's longest array, and
// a caller that only wants the path need not have them. Latency, as above: 64 rows of
// 64 nodes 3.2 us, 500 of up to 300 6.9.
template <bool ONE>
__global__ __launch_bounds__(256) void k_tree_accept(const int* __restrict__ parent, const int* __restrict__ tokens,
                                                     const int* __restrict__ target, const int* __restrict__ row_off,
                                                     int* __restrict__ n_accepted, int* __restrict__ next_token,
                                                     int* __restrict__ path, int B, int max_tokens, int max_per_row,
                                                     int W) {
  extern __shared__ char lds[];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const RowSpan sp = row_span(row_off, b, max_per_row, max_tokens);
  each_unowned(row_off, b, B, max_tokens, sp.n, [&](int t) { path[t] = -1; });
  if (sp.n == 0) {
    if (tid == 0) {
      n_accepted[b] = 0;
      next_token[b] = -1;
    }
    return;
  }
  const int *tok = tokens + sp.base, *tgt = target + sp.base;
  int* out = path + sp.base;
  // (count of the path, 511 - index): the larger is better, and one bit at least is set
  if constexpr (ONE) {
    const int p = parent_of(parent, sp.base, lane, sp.n);
    const int mine = lane < sp.n ? tok[lane] : 0, chosen = lane < sp.n ? tgt[lane] : 0;
    const int above = __shfl(chosen, max(p, 0), WAVE);
    const uint64_t agree = __ballot(lane < sp.n && (p < 0 || mine == above)), m = block_ancestors(p);
    const int count = (m & ~agree) == 0 ? __popcll(m) : 0;
    int key = count > 0 ? count << 9 | (511 - lane) : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) key = max(key, __shfl_xor(key, o, WAVE));
    const int best = 511 - (key & 511), most = key >> 9;  // (node 0 is a root: most > 0)
    const uint64_t line = shfl64(m, best);
    if ((line >> lane) & 1) out[__popcll(line & ((1ull << lane) - 1))] = lane;
    if (lane >= most && lane < sp.n) out[lane] = -1;
    if (lane == best) {
      n_accepted[b] = most;
      next_token[b] = chosen;
    }
  } else {
    __shared__ uint64_t agree[FC_TREE_MOST / 64];
    __shared__ int keys[4];
    const RowTree t = row_tree(lds, W);
    row_ancestors(t, parent, sp.base, sp.n, W);
    const int nb = (sp.n + 63) >> 6;
    for (int k = tid >> 6; k < nb; k += blockDim.x >> 6) {
      const int i = 64 * k + lane, p = parent_of(parent, sp.base, i, sp.n);
      const uint64_t a = __ballot(i < sp.n && (p < 0 || tok[i] == tgt[p]));
      if (lane == 0) agree[k] = a;
    }
    __syncthreads();
    int key = 0;
    for (int i = tid; i < sp.n; i += blockDim.x) {
      int count = 0;
      bool ok = true;
      for (int w = 0; w <= i >> 6; ++w) {
        const uint64_t m = t.mask[i * W + w];
        ok = ok && (m & ~agree[w]) == 0;
        count += __popcll(m);
      }
      if (ok) key = max(key, count << 9 | (511 - i));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) key = max(key, __shfl_xor(key, o, WAVE));
    if (lane == 0) keys[tid >> 6] = key;
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) key = max(key, keys[w]);
    const int best = 511 - (key & 511), most = key >> 9;
    const uint64_t* line = t.mask + best * W;
    for (int i = tid; i < sp.n; i += blockDim.x) {
      if ((line[i >> 6] >> (i & 63)) & 1) {
        int place = __popcll(line[i >> 6] & ((1ull << (i & 63)) - 1));
        for (int w = 0; w < i >> 6; ++w) place += __popcll(line[w]);
        out[place] = i;
      }
      if (i >= most) out[i] = -1;
    }
    if (tid == 0) {
      n_accepted[b] = most;
      next_token[b] = tgt[best];
    }
  }
}

extern "C" int32_t fc_tree_accept(const int32_t* parent, const int32_t* tokens, const int32_t* target,
                                  const int32_t* row_off, int32_t* n_accepted, int32_t* next_token, int32_t* path,
                                  int32_t batch, int32_t max_tokens, int32_t max_per_row, void* stream) {
  FC_CHECK_ARG(parent && tokens && target && row_off && n_accepted && next_token && path, "null pointer");
  const int rc = check_tree(batch, max_tokens, max_per_row);
  if (rc != FC_OK) return rc;
  const int W = (max_per_row + 63) / 64;
  const hipStream_t s = (hipStream_t)stream;
  if (W == 1)
    hipLaunchKernelGGL(k_tree_accept<true>, dim3(batch), dim3(64), 0, s, parent, tokens, target, row_off, n_accepted,
                       next_token, path, batch, max_tokens, max_per_row, W);
  else
    hipLaunchKernelGGL(k_tree_accept<false>, dim3(batch), dim3(256), row_tree_bytes(W), s, parent, tokens, target,
                       row_off, n_accepted, next_token, path, batch, max_tokens, max_per_row, W);
  FC_LAUNCH_CHECK();
  return FC_OK;
}

// ---------------------------------------------------------------------------
// Commit
// ---------------------------------------------------------------------------
// Place j of a row's chunk takes K and V of node path[j] > j; an entry that is not
// behind its place moves nothing. In ascending order no move reads what an earlier one
// wrote (its source lies behind every place before it), so the places are done in
// batches, each read before it is written: the result is that of reading all first.
//
// A workgroup lists a row's moves once and makes them for some of the layers' KV
// heads, U at a time. The moves lie along the lanes: V is stored dim by dim, and those
// of one 32-position block then share the 64-byte rows of a load or store; of K,
// 8 dims of a position are 16 bytes of its block (VEC). With the dims along the lanes
// each value of V was a request of its own: 24 layers, 64 rows, 4 heads of 128 in bf16
// 126 us, and 50 so. What is left there are the lines: a place and its source are 2 bytes
// in each of V's hd rows of 64, and 16 in each of K's. Counted from the slots of eight such
// inputs, on average 41 MB of keys and values lie in 182 MB of such rows: of V 80 read and
// 56 written, of K 32 and 14.
// One layer (32 rows, 12 heads): 10.3 us, path and slots, values, stores in turn.
#define MOVES 16  // a batch
template <typename T, bool VEC, int E>  // E: V's elements of a batch per thread, head_dim <= 16 E
__global__ __launch_bounds__(256) void k_tree_commit(PageView pv, T* kp, T* vp, int64_t kls, int64_t vls,
                                                     const int* __restrict__ path, const int* __restrict__ slots,
                                                     const int* __restrict__ row_off, int max_tokens,
                                                     int max_per_row, int units) {
  constexpr int U = E <= 8 ? 2 : 1, KE = VEC ? (sizeof(T) == 2 ? (E + 7) / 8 : (E + 3) / 4) : E;
  constexpr int KD = VEC ? 16 / (int)sizeof(T) : 1;  // dims of a piece of K
  using Piece = std::conditional_t<VEC, uint4, T>;
  __shared__ int s_path[FC_TREE_MOST], s_slot[FC_TREE_MOST], s_src[FC_TREE_MOST], s_dst[FC_TREE_MOST], s_n;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, hd = pv.hd;
  const RowSpan sp = row_span(row_off, b, max_per_row, max_tokens);
  if (sp.n == 0) return;
  for (int j = tid; j < sp.n; j += 256) {  // (so that the sources' slots are not a trip to memory behind the path's)
    s_path[j] = path[sp.base + j];
    s_slot[j] = slots[sp.base + j];
  }
  __syncthreads();
  if (tid < 64) {  // the moves, in order of their places
    const int pool = (int)min((int64_t)pv.N * pv.page, (int64_t)0x7fffffff);
    int total = 0;
    for (int j0 = 0; j0 < sp.n; j0 += 64) {
      const int j = j0 + lane, p = j < sp.n ? s_path[j] : -1, dst = j < sp.n ? s_slot[j] : -1;
      bool is = p > j && p < sp.n;
      const int src = is ? s_slot[p] : -1;
      is = src >= 0 && src < pool && dst >= 0 && dst < pool;
      const uint64_t who = __ballot(is);
      if (is) {
        const int at = total + __popcll(who & ((1ull << lane) - 1));
        s_src[at] = src;
        s_dst[at] = dst;
      }
      total += __popcll(who);
    }
    if (lane == 0) s_n = total;
  }
  __syncthreads();
  const int total = s_n, jm = tid % MOVES, d0 = tid / MOVES;
  for (int m0 = 0; m0 < total; m0 += MOVES) {
    const bool is = m0 + jm < total;
    const int src = is ? s_src[m0 + jm] : 0, dst = is ? s_dst[m0 + jm] : 0;
    const int si = src / pv.page, sa = src - si * pv.page, di = dst / pv.page, da = dst - di * pv.page;
    const int64_t vs = v_elem(pv, si, 0, sa, d0), vd = v_elem(pv, di, 0, da, d0);
    for (int u0 = blockIdx.y; u0 < units; u0 += U * gridDim.y) {
      Piece k[U][KE];
      T v[U][E];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int unit = u0 + u * gridDim.y, layer = unit / pv.G, g = unit - layer * pv.G;
        if (!is || unit >= units) continue;
        const int64_t head = (int64_t)g * pv.page * hd;
        const T *kl = kp + layer * kls + head, *vl = vp + layer * vls + head;
#pragma unroll
        for (int e = 0; e < KE; ++e)
          if ((d0 + 16 * e) * KD < hd) k[u][e] = *(const Piece*)(kl + k_elem(pv, si, 0, sa, (d0 + 16 * e) * KD));
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (d0 + 16 * e < hd) v[u][e] = vl[vs + 16 * e * 32];
      }
      __builtin_amdgcn_s_waitcnt(0);  // all is read ...
      __syncthreads();                // ... before any is written
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int unit = u0 + u * gridDim.y, layer = unit / pv.G, g = unit - layer * pv.G;
        if (!is || unit >= units) continue;
        const int64_t head = (int64_t)g * pv.page * hd;
        T *kl = kp + layer * kls + head, *vl = vp + layer * vls + head;
#pragma unroll
        for (int e = 0; e < KE; ++e)
          if ((d0 + 16 * e) * KD < hd) *(Piece*)(kl + k_elem(pv, di, 0, da, (d0 + 16 * e) * KD)) = k[u][e];
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (d0 + 16 * e < hd) vl[vd + 16 * e * 32] = v[u][e];
      }
    }
  }
}

extern "C" int32_t fc_tree_commit(const fc_pages* pages, int32_t n_layer, int64_t k_layer_stride,
                                  int64_t v_layer_stride, const int32_t* path, const int32_t* slots,
                                  const int32_t* row_off, int32_t batch, int32_t max_tokens, int32_t max_per_row,
                                  void* stream) {
  int rc = check_pages(pages);
  if (rc != FC_OK) return rc;
  FC_CHECK_ARG(path && slots && row_off, "null pointer");
  rc = check_tree(batch, max_tokens, max_per_row);
  if (rc != FC_OK) return rc;
  FC_CHECK_ARG(n_layer > 0 && n_layer <= 65535 && pages->n_kv_head <= 65535, "n_layer and n_kv_head in [1, 65535]");
  const PageView pv = page_view(pages);
  const hipStream_t s = (hipStream_t)stream;
  // each takes every grid.y-th KV head of all layers; two or more if few workgroups are enough, as listing the moves
  // weighs more then (32 rows of 12 heads in one layer 10.5 us, 11.1 with one each; one row in 24 layers of 12 heads 8.1, 9.9)
  const int64_t units = (int64_t)n_layer * pv.G, each = units * batch > 4096 ? 1 : 2;
  FC_CHECK_ARG(units < 1 << 30, "too many layers and heads");
  const dim3 grid(batch, (unsigned)std::max<int64_t>(1, std::min<int64_t>({(units + each - 1) / each, 8192 / batch, 65535})));
  const int per = pages->dtype == FC_BF16 ? 8 : 4;
  const bool vec = ((uintptr_t)pages->k & 15) == 0 && (k_layer_stride | pages->k_stride) % per == 0 && pv.hd % per == 0;
#define COMMIT_E(T, VEC, E)                                                                                           \
  hipLaunchKernelGGL((k_tree_commit<T, VEC, E>), grid, dim3(256), 0, s, pv, (T*)pages->k, (T*)pages->v, k_layer_stride,\
                     v_layer_stride, path, slots, row_off, max_tokens, max_per_row, (int)units)
#define COMMIT(T)                            \
  if (!vec) COMMIT_E(T, false, 16);          \
  else if (pv.hd <= 64) COMMIT_E(T, true, 4);  \
  else if (pv.hd <= 128) COMMIT_E(T, true, 8); \
  else COMMIT_E(T, true, 16)
  if (pages->dtype == FC_BF16) {
    COMMIT(bf16_t);
  } else {
    COMMIT(float);
  }
#undef COMMIT
#undef COMMIT_E
  FC_LAUNCH_CHECK();
  return FC_OK;
}

// ---------------------------------------------------------------------------
// Append with rotation
// ---------------------------------------------------------------------------
struct RopeArgs {
  PageView pv;
  void *kp, *vp, *out;
  const void *q, *k, *v;
  int64_t qst, qsh, kst, ksh, vst, vsh;
  const int *tok_pos, *slots;
  const float *cos, *sin;
  int M, H, len, rot, interleaved;
  float norm;
};

// Any head size and alignment: a wave per token and head of q, k or v, up to two pairs of dims per lane, and the dims
// that are not rotated beside them. V's values are stored one by one, a line each, also where it is the rotation or the
// tables' alignment that k_rope_append does not take. No model here has such shapes (16000 tokens of 12 + 4 + 4 heads of
// 128 in bf16, 40 dims rotated 175 us, 64 rotated 39 in k_rope_append; of 10 + 2 + 2 heads of 96, all rotated, 82).
template <typename T, typename S>
__global__ __launch_bounds__(256) void k_rope_append_any(RopeArgs a) {
  const PageView& pv = a.pv;
  const int lane = threadIdx.x & 63, hd = pv.hd, half = a.rot >> 1, jobs = a.H + 2 * pv.G;
  const int64_t all = (int64_t)a.M * jobs, nw = (int64_t)gridDim.x * 4;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < all; i += nw) {
    const int m = (int)(i / jobs), job = (int)(i - (int64_t)m * jobs);
    const int pos = a.tok_pos[m], slot = a.slots[m];
    const bool there = pos >= 0 && pos < a.len;
    const int id = slot >= 0 && slot / pv.page < pv.N ? slot / pv.page : -1, at = slot - id * pv.page;
    if (job >= a.H && (id < 0 || !there)) continue;
    if (job >= a.H + pv.G) {
      const int g = job - a.H - pv.G;
      for (int d = lane; d < hd; d += 64)
        st<T>((T*)a.vp, v_elem(pv, id, g, at, d), ld<S>((const S*)a.v, m * a.vst + g * a.vsh + d));
      continue;
    }
    const int g = job < a.H ? job : job - a.H;
    const S* x = job < a.H ? (const S*)a.q + m * a.qst + g * a.qsh : (const S*)a.k + m * a.kst + g * a.ksh;
    // pairs lane and lane + 64, then the dims that stay
    float y1[2], y2[2], y0[4], ss = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int p = lane + 64 * t;
      y1[t] = y2[t] = 0.f;
      if (p < half && there) {
        const float c = a.cos[(int64_t)pos * half + p], s = a.sin[(int64_t)pos * half + p];
        const float x1 = ld<S>(x, a.interleaved ? 2 * p : p), x2 = ld<S>(x, a.interleaved ? 2 * p + 1 : p + half);
        y1[t] = x1 * c + x2 * s;
        y2[t] = x2 * c - x1 * s;
        ss += y1[t] * y1[t] + y2[t] * y2[t];
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int d = a.rot + lane + 64 * t;
      y0[t] = d < hd && there ? ld<S>(x, d) : 0.f;
      ss += y0[t] * y0[t];
    }
    const float f = a.norm > 0.f ? a.norm / sqrtf(wave_sum(ss) / (float)hd + 1e-6f) : 1.f;
    auto put = [&](int d, float v) {
      if (job < a.H) st<T>((T*)a.out, ((int64_t)m * a.H + g) * hd + d, v * f);
      else st<T>((T*)a.kp, k_elem(pv, id, g, at, d), v * f);
    };
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int p = lane + 64 * t;
      if (p < half) {
        put(a.interleaved ? 2 * p : p, y1[t]);
        put(a.interleaved ? 2 * p + 1 : p + half, y2[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (a.rot + lane + 64 * t < hd) put(a.rot + lane + 64 * t, y0[t]);
  }
}

// Heads of 64 and 128, rotated in multiples of 16 dims, arrays aligned to 16
// bytes. A workgroup takes 4096 / HD tokens and either `per` heads of q and k
// or one head of v.
//
// q and k: HD / 16 lanes a token, 16 dims each: with the halves of `rot` paired,
// 8 of either half; cos and sin stay in registers for all of the workgroup's
// heads. K goes out as it comes, 16 bytes a lane: in the matrix-core order four
// positions' pieces are 64 bytes next to each other. V is stored dim by dim: it is
// turned through LDS and written with the positions along the lanes, so that a
// wave's 2-byte stores fill the 64-byte rows that they lie in, whatever the slots'
// alignment (with the dims along the lanes each store is a line of its own).
//
// Bound by memory, and a workgroup's loads and stores do not overlap, several on a CU
// do: 16000 tokens of 12 + 4 + 4 heads in bf16 39 us, 168 MB at 4.3 TB/s (a copy: 4.9).
// Tokens in runs of 8 fill 16 bytes of V's rows of 64 at a time: 4000 tokens of
// 12 + 12 + 12 heads, fp32 to bf16, 83 us for 110 MB.
template <int L>
__device__ __forceinline__ float group_sum(float v) {  // over groups of L = 4 or 8 lanes, in every lane
#define ROPE_STEP(CTRL) \
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, false))
  ROPE_STEP(0xb1);                            // lanes l ^ 1
  ROPE_STEP(0x4e);                            // l ^ 2
  if constexpr (L == 8) ROPE_STEP(0x141);     // 7 - l: the other four
#undef ROPE_STEP
  return v;
}
__device__ __forceinline__ void load4(const float* p, float (&x)[8], int at) {
  const float4 a = *(const float4*)p;
  x[at] = a.x; x[at + 1] = a.y; x[at + 2] = a.z; x[at + 3] = a.w;
}
template <typename T, typename S, int HD>
__device__ __forceinline__ void rope_rows(const RopeArgs& a, int t0, int h0, int h1) {
  constexpr int L = HD / 16, U = sizeof(S) == 2 ? 4 : 2;  // heads whose loads are under way at once
  const int tid = threadIdx.x, l = tid % L, m = t0 + tid / L, half = a.rot >> 1;
  if (m >= a.M) return;
  const int pos = a.tok_pos[m], slot = a.slots[m];
  const bool there = pos >= 0 && pos < a.len, turns = 16 * l < a.rot;
  const int da = turns && !a.interleaved ? 8 * l : 16 * l, db = turns && !a.interleaved ? half + 8 * l : 16 * l + 8;
  float c[8], s[8];
  if (there && turns) {
    const int64_t at = (int64_t)pos * half + 8 * l;
    load4(a.cos + at, c, 0);
    load4(a.cos + at + 4, c, 4);
    load4(a.sin + at, s, 0);
    load4(a.sin + at + 4, s, 4);
  }
  const int id = slot >= 0 && slot / a.pv.page < a.pv.N ? slot / a.pv.page : -1, in = slot - id * a.pv.page;
  const bool keeps = there && id >= 0;
  const int64_t ka = keeps ? k_elem(a.pv, id, 0, in, da) : 0, kb = keeps ? k_elem(a.pv, id, 0, in, db) : 0;
  for (int h = h0; h < h1; h += U) {
    float x[U][8], y[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hu = min(h + u, h1 - 1);
      const S* p = hu < a.H ? (const S*)a.q + m * a.qst + hu * a.qsh : (const S*)a.k + m * a.kst + (hu - a.H) * a.ksh;
      load8(p + da, x[u]);
      load8(p + db, y[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u >= h1) break;
      if (turns) {
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x1 = x[u][2 * i], x2 = x[u][2 * i + 1], y1 = y[u][2 * i], y2 = y[u][2 * i + 1];
            x[u][2 * i] = x1 * c[i] + x2 * s[i];
            x[u][2 * i + 1] = x2 * c[i] - x1 * s[i];
            y[u][2 * i] = y1 * c[4 + i] + y2 * s[4 + i];
            y[u][2 * i + 1] = y2 * c[4 + i] - y1 * s[4 + i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x1 = x[u][i], x2 = y[u][i];
            x[u][i] = x1 * c[i] + x2 * s[i];
            y[u][i] = x2 * c[i] - x1 * s[i];
          }
        }
      }
      float f = 1.f;
      if (a.norm > 0.f) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[u][i] * x[u][i] + y[u][i] * y[u][i];
        f = a.norm / sqrtf(group_sum<L>(ss) * (1.f / HD) + 1e-6f);
      }
      if (h + u < a.H) {
        T* o = (T*)a.out + ((int64_t)m * a.H + h + u) * HD;
        if (!there) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[u][i] = y[u][i] = 0.f;
          f = 1.f;
        }
        store8(o + da, x[u], f);
        store8(o + db, y[u], f);
      } else if (keeps) {
        T* o = (T*)a.kp + (int64_t)(h + u - a.H) * a.pv.page * HD;
        store8(o + ka, x[u], f);
        store8(o + kb, y[u], f);
      }
    }
  }
}
template <typename T, typename S, int HD>
__device__ __forceinline__ void append_v(const RopeArgs& a, T* lds, int t0, int g) {
  constexpr int TT = 4096 / HD, LD = HD + (sizeof(T) == 2 ? 2 : 1), C = HD / 8;
  const int tid = threadIdx.x, t = tid % TT, m = t0 + t;
  int slot = m < a.M ? a.slots[m] : -1;
  const int pos = m < a.M ? a.tok_pos[m] : -1;
  float x[2][8];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = tid + 256 * e, tok = min(t0 + i / C, a.M - 1);
    load8((const S*)a.v + tok * a.vst + g * a.vsh + 8 * (i % C), x[e]);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = tid + 256 * e;
    T* w = lds + i / C * LD + 8 * (i % C);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int k = 0; k < 4; ++k) *(uint32_t*)(w + 2 * k) = pack2bf(x[e][2 * k], x[e][2 * k + 1]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = x[e][k];
    }
  }
  __syncthreads();
  const int id = slot >= 0 ? slot / a.pv.page : a.pv.N;
  if (id >= a.pv.N || pos < 0 || pos >= a.len) return;
  T* o = (T*)a.vp + v_elem(a.pv, id, g, slot - id * a.pv.page, tid / TT);
  const T* r = lds + t * LD + tid / TT;
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e * (256 / TT) * 32] = r[e * (256 / TT)];
}
template <typename T, typename S, int HD>
__global__ __launch_bounds__(256) void k_rope_append(RopeArgs a, int per, int groups) {
  __shared__ T lds[(4096 / HD) * (HD + (sizeof(T) == 2 ? 2 : 1))];
  // v's jobs, then q's and k's, an eighth of either kind on each XCD, next to each other: of V, a head's tiles one behind
  // the other, since the 64-byte rows in which two tiles meet are put together in the XCD's L2; of q and k, a tile's
  // heads, which read the same rows of cos and sin. (16000 tokens of 12 + 4 + 4 heads, half rotated, dealt out in turn:
  // 42 us; V's so 41, both 39. All of each head rotated: 43, 42, 38.)
  const int G = a.pv.G, tiles = (a.M + 4096 / HD - 1) / (4096 / HD), each = (G * tiles + 7) >> 3;
  const int r = (int)blockIdx.x - 8 * each;
  if (r >= 0) {
    const int each_qk = (tiles * groups + 7) >> 3, job = (r & 7) * each_qk + (r >> 3), at = job % groups * per;
    if (job < tiles * groups) rope_rows<T, S, HD>(a, job / groups * (4096 / HD), at, min(at + per, a.H + G));
  } else {
    const int job = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if (job < G * tiles) append_v<T, S, HD>(a, lds, job % tiles * (4096 / HD), job / tiles);
  }
}

extern "C" int32_t fc_rope_append(const fc_pages* pages, const void* q, const void* k, const void* v,
                                  int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                                  int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                  int32_t src_dtype, const int32_t* tok_pos, const int32_t* slots, const float* cos,
                                  const float* sin, int32_t rope_len, int32_t rot, int32_t interleaved, float norm,
                                  void* q_out, int32_t n_head, int32_t M, void* stream) {
  const int rc = check_pages(pages);
  if (rc != FC_OK) return rc;
  FC_CHECK_ARG(M >= 0 && n_head > 0 && n_head <= 65535 && pages->n_kv_head <= 65535,
               "M, n_head and n_kv_head in [1, 65535]");
  FC_CHECK_ARG(src_dtype == FC_F32 || src_dtype == FC_BF16, "src_dtype");
  FC_CHECK_ARG(src_dtype == pages->dtype || src_dtype == FC_F32, "bf16 values into fp32 pages");
  FC_CHECK_ARG(rot > 0 && rot % 2 == 0 && rot <= pages->head_dim, "rot must be even, in [2, head_dim]");
  FC_CHECK_ARG(rope_len > 0, "rope_len");
  // (norm / sqrt(0 + 1e-6) is finite, so that a head of zeros stays one)
  FC_CHECK_ARG(norm >= 0.f && norm <= 3.0e35f, "norm must be in [0, 3e35]");
  if (M == 0) return FC_OK;
  FC_CHECK_ARG(q && k && v && tok_pos && slots && cos && sin && q_out, "null pointer");
  const RopeArgs a{page_view(pages), pages->k, pages->v, q_out, q, k, v, q_token_stride, q_head_stride,
                   k_token_stride, k_head_stride, v_token_stride, v_head_stride, tok_pos, slots, cos, sin,
                   M, n_head, rope_len, rot, interleaved != 0, norm};
  const hipStream_t s = (hipStream_t)stream;
  const int G = pages->n_kv_head, hd = pages->head_dim;
  // 16 bytes at a time: everything aligned to them
  const int src = src_dtype == FC_BF16 ? 8 : 4, dst = pages->dtype == FC_BF16 ? 8 : 4;
  const uintptr_t at = (uintptr_t)pages->k | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out |
                       (uintptr_t)cos | (uintptr_t)sin;
  const int64_t strides = q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride |
                          v_head_stride;
  if ((hd == 64 || hd == 128) && rot % 16 == 0 && (at & 15) == 0 && strides % src == 0 && pages->k_stride % dst == 0) {
    // as many heads of q and k a workgroup as leave six for every CU, up to 4 (16000 tokens of 12 + 4 heads: one each 49
    // us, two 41, four 39, eight 41, all 57)
    const int64_t tiles = ((int64_t)M * hd + 4095) / 4096, heads = n_head + G;
    const int per = (int)std::max<int64_t>(1, std::min<int64_t>(4, tiles * heads / 1536));
    const int64_t groups = (heads + per - 1) / per, all = (tiles * groups + 7) / 8 * 8 + (tiles * G + 7) / 8 * 8;
    if (all < 1 << 24) {  // (a launch's threads are counted in 32 bits)
#define ROPE(T, S, HD) \
  hipLaunchKernelGGL((k_rope_append<T, S, HD>), dim3((int)all), dim3(256), 0, s, a, per, (int)groups)
#define ROPE_HD(T, S)          \
  if (hd == 64) ROPE(T, S, 64); \
  else ROPE(T, S, 128)
      if (pages->dtype == FC_F32) {
        ROPE_HD(float, float);
      } else if (src_dtype == FC_F32) {
        ROPE_HD(bf16_t, float);
      } else {
        ROPE_HD(bf16_t, bf16_t);
      }
#undef ROPE_HD
#undef ROPE
      FC_LAUNCH_CHECK();
      return FC_OK;
    }
  }
  const int64_t waves = (int64_t)M * (n_head + 2 * G);
  const dim3 grid((unsigned)std::min<int64_t>((waves + 3) / 4, 65536));
  if (pages->dtype == FC_F32) hipLaunchKernelGGL((k_rope_append_any<float, float>), grid, dim3(256), 0, s, a);
  else if (src_dtype == FC_F32) hipLaunchKernelGGL((k_rope_append_any<bf16_t, float>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_rope_append_any<bf16_t, bf16_t>), grid, dim3(256), 0, s, a);
  FC_LAUNCH_CHECK();
  return FC_OK;
}
