// What the 16-bit attention kernels (few_rows.cuh) share: the problem they are
// given, which keys a query row sees, and the plain evaluation of one row.
//
// Both operators are one formula.  Batch element b holds len(b) keys; query token t stands at
// index off(b) + t.  A token is valid when 0 <= index < len(b); an invalid token's output is zero.
//   chain:  token t sees key j        iff  j <= index(t)  and  (index(t) - j < window  or  j < sinks)
//   tree:   the keys from off(b) on are the drafted tokens themselves, each with a parent among the
//           tokens before it (or none); position(t) = off(b) + number of tokens above t.  Token t sees
//           the context (j < off(b)) and itself and the tokens above it, both subject to
//           position(t) - position(key) < window or position(key) < sinks.
// Output: softmax over the visible keys of scale * q.k, times V; a row that sees no key is zero.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "pk_internal.h"
#include "pk_ptx.cuh"

namespace pk {

constexpr int kAttendTile = 64;      // keys per step of the few-row kernel
constexpr int kMaxTreeTokens = 64;   // a token's visible drafted tokens are one 64-bit mask
constexpr int kNoWindow = 1 << 30;   // larger than any index

// K/V of the problem for the plain row evaluation and the copy maps.  Paged: [layers, pages,
// kv_heads, page, D] contiguous; dense: element strides of batch, head and key.
struct AttendParams {
  const void* q;
  int64_t q_stride[3];  // batch, head, token (elements)
  int q_vec;            // rows start on 16-byte boundaries
  void* out;            // [batch, heads, tokens, D]
  int batch, heads, kv_heads, group, tokens, rows, row_blocks;
  const int32_t* lengths;  // may be null (dense): every batch element holds kv_len keys
  const int32_t* starts;   // null (dense): off(b) = offset
  int kv_len, offset;
  const int32_t* table;  // [batch, width] pages; null: dense
  int width, page, page_shift, pages, page_base;  // page_base: first page of the layer in the pool
  const void* k;
  const void* v;
  int64_t k_stride[3], v_stride[3];  // dense
  const float* k_scale;  // 8-bit cache: one scale per row, from the layer's first page
  const float* v_scale;
  const int32_t* tree;  // [batch, tokens] parents, or null
  int64_t tree_stride;
  int window, sinks;
  float scale_log2;  // softmax scale * log2(e)
  float* partial;    // pieces of rows whose keys are shared by several CTAs
  int workers;
  int32_t* host_status;  // pinned word that takes the site of an abandoned wait
};

__device__ __forceinline__ int attend_len(const AttendParams& p, int b) {
  const int most = p.table ? p.width * p.page : p.kv_len;
  if (!p.lengths) return most;
  return max(0, min(p.lengths[b], most));
}
__device__ __forceinline__ int attend_off(const AttendParams& p, int b, int len) {
  return p.starts ? max(0, min(p.starts[b], len)) : p.offset;
}
// Page of key j of batch element b, or -1 where the table leads nowhere.
__device__ __forceinline__ int attend_page(const AttendParams& p, int b, int j) {
  const int page = p.table[static_cast<int64_t>(b) * p.width + (j >> p.page_shift)];
  return (page >= 0 && page < p.pages) ? page : -1;
}

// The drafted tokens that each token of one batch element sees, as bit masks, and each token's
// depth; shared memory, filled by one warp.  Ancestors by pointer doubling: six rounds reach 64
// levels.  A parent outside [-1, t) counts as -1 (no parent), so that no walk can go in circles.
struct TreeMasks {
  uint64_t sees[kMaxTreeTokens];
  int depth[kMaxTreeTokens];
};
__device__ __forceinline__ void build_tree(const AttendParams& p, int b, int off, int lane, TreeMasks* tm) {
  const int32_t* parents = p.tree + b * p.tree_stride;
  uint64_t mask[2];
  int up[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = lane + 32 * i;
    mask[i] = 1ull << t;
    up[i] = t < p.tokens ? parents[t] : -1;
    if (up[i] < 0 || up[i] >= t) up[i] = -1;
  }
#pragma unroll
  for (int round = 0; round < 6; ++round) {
    uint64_t next[2];
    int nup[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int src = up[i] < 0 ? 0 : up[i];
      const uint64_t m0 = __shfl_sync(0xffffffffu, mask[0], src & 31), m1 = __shfl_sync(0xffffffffu, mask[1], src & 31);
      const int u0 = __shfl_sync(0xffffffffu, up[0], src & 31), u1 = __shfl_sync(0xffffffffu, up[1], src & 31);
      next[i] = up[i] < 0 ? mask[i] : mask[i] | (src < 32 ? m0 : m1);
      nup[i] = up[i] < 0 ? -1 : (src < 32 ? u0 : u1);
    }
    mask[0] = next[0], mask[1] = next[1];
    up[0] = nup[0], up[1] = nup[1];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) tm->depth[lane + 32 * i] = __popcll(mask[i]) - 1;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = lane + 32 * i, mine = __popcll(mask[i]) - 1;
    uint64_t m = mask[i], keep = 0;
    while (m) {  // at most one turn per level
      const int a = __ffsll(static_cast<long long>(m)) - 1;
      m &= m - 1;
      const int d = tm->depth[a];
      if (mine - d < p.window || off + d < p.sinks) keep |= 1ull << a;
    }
    tm->sees[t] = keep;
  }
  __syncwarp();
}

// What one query row sees: keys below `lim`, those above `low` or below the sinks; in a tree also
// the drafted tokens of `mask`.
struct RowView {
  int lim, low;
  uint64_t mask;
};
__device__ __forceinline__ RowView row_view(const AttendParams& p, int off, int len, int t, const TreeMasks* tm) {
  RowView v{0, 0, 0};
  const int index = off + t;
  if (t >= p.tokens || index < 0 || index >= len) return v;
  if (tm) {
    v.lim = off;
    v.low = off + tm->depth[t] - p.window;
    v.mask = tm->sees[t];
  } else {
    v.lim = index + 1;
    v.low = index - p.window;
  }
  return v;
}
// Key j is known to be below len.
template <bool TREE>
__device__ __forceinline__ bool sees(const RowView& v, int j, int off, int sinks) {
  if (TREE && j >= off) {
    const int a = j - off;
    return a < kMaxTreeTokens && ((v.mask >> a) & 1);
  }
  return j < v.lim && (j > v.low || j < sinks);
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);  // one rounding to 16 bits each, nearest even
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ T from_f32(float a);
template <>
__device__ __forceinline__ __half from_f32(float a) { return __float2half_rn(a); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float a) { return __float2bfloat16_rn(a); }

// One output row from its visible keys alone, one key after the other, by one warp; lane i holds
// features [i * D/32, (i+1) * D/32).  The tiled kernels multiply whole tiles, so that an infinity
// or NaN in a V row that this query row must not see would still reach it (0 * NaN); a row that
// comes out of them with a value that is not finite is evaluated again here.  Rare, and slow.
template <typename T, bool I8, int D>
__device__ __noinline__ void plain_row(const AttendParams& p, int b, int kvh, int row, int off, int len, RowView view, bool tree) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, t = row / p.group, head = kvh * p.group + row % p.group;
  const T* q = static_cast<const T*>(p.q) + b * p.q_stride[0] + head * p.q_stride[1] + t * p.q_stride[2] + lane * E;
  float qf[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) qf[e] = to_f32(q[e]) * p.scale_log2, acc[e] = 0.f;
  const int end = tree ? min(len, off + kMaxTreeTokens) : min(len, view.lim);
  for (int j = 0; j < end; ++j) {
    const bool visible = tree ? sees<true>(view, j, off, p.sinks) : sees<false>(view, j, off, p.sinks);
    if (!visible) continue;  // the same for all lanes
    int64_t at_k, at_v, at_s = 0;
    if (p.table) {
      const int page = attend_page(p, b, j);
      if (page < 0) continue;
      at_s = (static_cast<int64_t>(page) * p.kv_heads + kvh) * p.page + (j & (p.page - 1));
      at_k = at_v = (at_s + static_cast<int64_t>(p.page_base) * p.kv_heads * p.page) * D;
    } else {
      at_k = b * p.k_stride[0] + kvh * p.k_stride[1] + j * p.k_stride[2];
      at_v = b * p.v_stride[0] + kvh * p.v_stride[1] + j * p.v_stride[2];
    }
    float s = 0.f, vf[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (I8) {
        s = fmaf(qf[e], static_cast<float>(static_cast<const int8_t*>(p.k)[at_k + lane * E + e]), s);
        vf[e] = static_cast<float>(static_cast<const int8_t*>(p.v)[at_v + lane * E + e]);
      } else {
        s = fmaf(qf[e], to_f32(static_cast<const T*>(p.k)[at_k + lane * E + e]), s);
        vf[e] = to_f32(static_cast<const T*>(p.v)[at_v + lane * E + e]);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (I8) {
      s *= p.k_scale[at_s];
      const float vs = p.v_scale[at_s];
#pragma unroll
      for (int e = 0; e < E; ++e) vf[e] *= vs;
    }
    // fmaxf drops a NaN: a score that is one stays visible through the sum
    const float mn = fmaxf(m, s);
    const float keep = m == mn ? 1.f : exp2f(m - mn), w = s == -INFINITY && mn == -INFINITY ? 0.f : exp2f(s - mn);
    l = l * keep + w;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * keep + w * vf[e];
    m = mn;
  }
  T* out = static_cast<T*>(p.out) + ((static_cast<int64_t>(b) * p.heads + head) * p.tokens + t) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = from_f32<T>(l == 0.f ? 0.f : acc[e] / l);
}

// Copy map of K or V: [line, key, lines of a row, head, batch element or page], boxes of `box` keys.
// `stride`: dense element strides (batch, head, key); paged caches are contiguous.
int attend_map(CUtensorMap* m, const AttendParams& p, const void* base, const int64_t* stride, int line, int lines, int esz, int box);

// few_rows.cuh
int launch_few_rows_f16(const AttendParams& p, int head_dim, bool i8, int device, cudaStream_t st);
int launch_few_rows_bf16(const AttendParams& p, int head_dim, bool i8, int device, cudaStream_t st);
uint64_t few_rows_workspace(int rows, int head_dim);

}  // namespace pk
