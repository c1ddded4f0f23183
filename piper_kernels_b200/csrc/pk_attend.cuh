// What the 16-bit attention kernels (few_rows.cuh, wide_rows.cuh) share: the problem they are
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
  uint64_t group_inv;  // ceil(2^64 / group): row / group is the high half of row * group_inv (group > 1)
  const int32_t* lengths;  // may be null (dense): every batch element holds kv_len keys
  const int32_t* starts;   // null (dense): off(b) = offset
  int kv_len, offset;
  const int32_t* table;  // [batch, width] pages; null: dense
  int width, page, page_shift, pages, page_base, pool_pages;  // page_base: first page of the layer in the pool of pool_pages
  const void* k;
  const void* v;
  int64_t k_stride[3], v_stride[3];  // dense
  const float* k_scale;  // 8-bit cache: one scale per row, from the layer's first page
  const float* v_scale;
  const int32_t* tree;  // [batch, tokens] parents, or null
  int64_t tree_stride;
  int window, sinks;
  int key_align;     // tiles begin on multiples of this: 8, or what keeps a tile's copies within pages
  float scale_log2;  // softmax scale * log2(e)
  // Units (group, key head) from first_unit on are shared out by tiles over `workers` CTAs (0: none is);
  // pieces of their rows: [2 * workers][rows of a unit][D + 4] (numerators, maximum, sum, -, -).
  float* partial;
  struct Pieces* pieces;  // per unit
  int workers, first_unit;
  int cluster;  // few rows: CTAs that share one unit and join its pieces themselves, or 0
  int32_t* host_status;  // pinned word that takes the site of an abandoned wait
  long long wait_cycles;  // a wait inside a kernel is given up after this many cycles
  int skip_copy;          // drill: every CTA leaves out its copy of this number, so that a wait runs out (-1: none)
  const CUtensorMap* maps;  // host: K and V maps for 64- and 128-key tiles of few rows and for many rows, or null
};

// Token of a row (its query head within the group is the remainder).
__device__ __forceinline__ int token_of(const AttendParams& p, int row) {
  return p.group == 1 ? row : static_cast<int>(__umul64hi(static_cast<uint64_t>(row), p.group_inv));
}
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
    uint64_t m = p.window < kNoWindow ? mask[i] : 0, keep = p.window < kNoWindow ? 0 : mask[i];
    while (m) {  // a window: at most one turn per level
      const int a = __ffsll(static_cast<long long>(m)) - 1;
      m &= m - 1;
      const int d = tm->depth[a];
      if (mine - d < p.window || off + d < p.sinks) keep |= 1ull << a;
    }
    tm->sees[t] = keep;
  }
  __syncwarp();
}

// A bounded wait with little code (it is in every role's loop): gives up after p.wait_cycles, or when another wait has
// been given up.  While a warp is away evaluating rows one by one (plain_row), which may take longer, it keeps the time
// at `busy`, and the wait counts from there.
__device__ __forceinline__ bool attend_wait(const AttendParams& p, uint32_t bar, uint32_t parity, volatile int* abort_flag, volatile long long* busy, int where) {
  long long since = 0;
  for (int n = 0; !mbar_try_wait(bar, parity); ++n) {
    if ((n & 63) != 63) continue;
    if (*abort_flag != 0) return false;
    const long long now = clock64();
    if (since == 0) since = now;
    if (now - since <= p.wait_cycles) continue;
    since = *busy;
    if (now - since <= p.wait_cycles) continue;
    *abort_flag = where;
    return false;
  }
  return true;
}

// Barrier of all threads of a cluster; what they wrote before it, they all read after it.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Barrier `id` of `threads` threads; true when `good` holds in all of them.
__device__ __forceinline__ bool vote_barrier(int id, int threads, bool good) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(good))
      : "memory");
  return all != 0;
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

// Whether a result is a number that T holds.  The sums take the probabilities as they are and the products take
// them rounded to T, relative to a reference that may lie far below the maximum: so the quotient may pass the
// largest |v| by half a step of T, and where that is T's largest number (65504; from 65520 on float16 rounds to
// infinity) the rounded result would be infinite.  Such a row is evaluated again.
template <typename T>
__device__ __forceinline__ bool holds(float x);
template <>
__device__ __forceinline__ bool holds<__half>(float x) { return fabsf(x) < 65520.f; }
template <>
__device__ __forceinline__ bool holds<__nv_bfloat16>(float x) { return fabsf(x) <= 3.0e38f; }

// One output row from its visible keys alone, one key after the other, by one warp; lane i holds
// features [i * D/32, (i+1) * D/32).  The tiled kernels multiply whole tiles, so that an infinity
// or NaN in a V row that this query row must not see would still reach it (0 * NaN); a row that
// comes out of them with a value that its type does not hold is evaluated again here (its features
// [first, last) are written).  Rare, and slow: 1000 to 2000 cycles a key.  `busy` (if any) takes the time
// meanwhile, for the waits of other warps.  EARLY: ends when the row is NaN throughout, so that inputs full of NaN are done
// with soon.  Not in the joins: the loop's second exit costs them the code around the call (two sequences of 16 tokens,
// 64 rows of 64 features, over 2000 8-bit rows: 22.7 against 18.1 us).
template <typename T, bool I8, int D, bool EARLY>
__device__ __noinline__ void plain_row(const AttendParams& p, int b, int kvh, int row, int off, int len, RowView view, bool tree, volatile long long* busy = nullptr,
                                       int first = 0, int last = D) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, t = token_of(p, row), head = kvh * p.group + row - t * p.group;
  const T* q = static_cast<const T*>(p.q) + b * p.q_stride[0] + head * p.q_stride[1] + t * p.q_stride[2] + lane * E;
  float qf[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) qf[e] = to_f32(q[e]) * p.scale_log2, acc[e] = 0.f;
  const int end = tree ? min(len, off + kMaxTreeTokens) : min(len, view.lim);
  for (int j = 0; j < end; ++j) {
    if (busy && lane == 0 && (j & 63) == 0) *busy = clock64();
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
    bool nan = EARLY;
#pragma unroll
    for (int e = 0; e < E; ++e) nan = nan && acc[e] != acc[e];
    if (EARLY && __all_sync(0xffffffffu, nan)) break;
  }
  T* out = static_cast<T*>(p.out) + ((static_cast<int64_t>(b) * p.heads + head) * p.tokens + t) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane * E + e >= first && lane * E + e < last) out[e] = from_f32<T>(l == 0.f ? 0.f : acc[e] / l);
}

// ---------------------------------------------------------------------------------------
// Sharing the work: the keys of all groups of query rows and key heads form one list of TILE-key
// tiles, of which every CTA takes an equal, contiguous part.
// ---------------------------------------------------------------------------------------
// One group of query rows (batch element, row block; the same for every key head) and the key tiles
// that any of its rows sees: `ns` tiles of sinks, then those from key `begin` on.
struct Span {
  int b, rb, off, len, ns, begin, n;
  int full_lo, full_hi;  // keys that every row sees
};

template <bool TREE, int TILE, int ROWS>
__device__ __forceinline__ Span span_of(const AttendParams& p, int g) {
  Span s;
  s.b = g / p.row_blocks;
  s.rb = g % p.row_blocks;
  s.len = attend_len(p, s.b);
  s.off = attend_off(p, s.b, s.len);
  const int r0 = s.rb * ROWS, r1 = min(r0 + ROWS, p.rows) - 1;
  const int t0 = token_of(p, r0), t1 = token_of(p, r1);
  int hi, lo;
  if (TREE) {
    hi = min(s.len, s.off + p.tokens);
    lo = s.off - p.window + 1;
    s.full_hi = min(s.len, s.off);
    s.full_lo = s.off + p.tokens - p.window;
  } else {
    hi = min(s.len, s.off + t1 + 1);
    lo = s.off + t0 - p.window + 1;
    s.full_hi = min(s.len, s.off + t0 + 1);
    s.full_lo = s.off + t1 - p.window + 1;
  }
  if (s.off + t0 >= s.len) hi = 0;  // no valid row
  hi = max(hi, 0);
  lo = min(max(lo, 0), hi);
  s.ns = (min(p.sinks, lo) + TILE - 1) / TILE;
  s.begin = max(lo & -p.key_align, s.ns * TILE);
  s.n = s.ns + max(0, (hi - s.begin + TILE - 1) / TILE);
  if (s.n == 0) s.n = 1, s.ns = 0, s.begin = 0;  // rows that see nothing still have to be written
  return s;
}

// First key of tile i.
template <int TILE>
__device__ __forceinline__ int key_of_tile(const Span& s, int i) {
  return i < s.ns ? i * TILE : s.begin + (i - s.ns) * TILE;
}

// First tile of worker w, when `total` tiles are shared out (fewer than 2^31: checked on the host).
__device__ __forceinline__ uint32_t share_begin(uint32_t total, uint32_t workers, uint32_t w) {
  return total / workers * w + min(w, total % workers);
}
__device__ __forceinline__ uint32_t owner_of(uint32_t total, uint32_t workers, uint32_t tile) {
  const uint32_t base = total / workers, extra = total % workers, big = extra * (base + 1);
  return tile < big ? tile / (base + 1) : extra + (tile - big) / base;
}

constexpr int kCounters = 128;  // threads that count tiles

struct Found {  // a group and the tiles in front of it
  uint32_t before;
  int group;
};

// Tiles of the groups [from, upto), all key heads; by the whole CTA, threads [0, 128) count.
template <bool TREE, int TILE, int ROWS>
__device__ __forceinline__ uint32_t sum_tiles(const AttendParams& p, int from, int upto, uint32_t* red) {
  uint32_t mine = 0;
  if (threadIdx.x < kCounters)
    for (int g = from + threadIdx.x; g < upto; g += kCounters) mine += span_of<TREE, TILE, ROWS>(p, g).n;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0 && threadIdx.x < kCounters) red[threadIdx.x >> 5] = mine;
  __syncthreads();
  const uint32_t sum = red[0] + red[1] + red[2] + red[3];
  __syncthreads();
  return sum * p.kv_heads;
}

// Finds the group that holds tile `at` of those from group `from` on, 128 groups at a time.
template <bool TREE, int TILE, int ROWS>
__device__ __forceinline__ Found find_group(const AttendParams& p, int from, uint32_t at, uint32_t* red, Found* out) {
  const int groups = p.batch * p.row_blocks, lane = threadIdx.x & 31;
  uint32_t before = 0;
  if (threadIdx.x == 0) out->group = -1;
  __syncthreads();
  for (int g0 = from; g0 < groups; g0 += kCounters) {
    const int g = g0 + threadIdx.x;
    uint32_t n = 0;
    if (threadIdx.x < kCounters && g < groups) n = span_of<TREE, TILE, ROWS>(p, g).n * p.kv_heads;
    uint32_t incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31 && threadIdx.x < kCounters) red[threadIdx.x >> 5] = incl;
    __syncthreads();
    if (threadIdx.x < kCounters) {
      uint32_t base = before;
      for (int w = 0; w < (threadIdx.x >> 5); ++w) base += red[w];
      const uint32_t b0 = base + incl - n;
      if (n > 0 && at >= b0 && at < b0 + n) out->group = g, out->before = b0;
    }
    before += red[0] + red[1] + red[2] + red[3];
    __syncthreads();
    if (out->group >= 0) break;  // the same for every thread: written before the barrier
  }
  return *out;
}

// Where the pieces of a unit (group, key head) are, written by the CTA that has its first tile: CTAs
// c0 .. c1, each in slot 0 of its two, but for c0 when `late` (it began with another unit).  c0 == c1:
// one CTA finished the unit.
struct Pieces {
  int c0, c1, late, pad;
};

// What a CTA that gave up a wait has not finished, for other code to see: rows of NaN, and pieces whose sum is
// negative, from which the join makes rows of NaN.
constexpr float kUndone = -1.f;
// Features [first, first + N) of a query row.
template <typename T, int D, int N>
__device__ __forceinline__ void nan_row(const AttendParams& p, int b, int kvh, int row, int first) {
  const int t = token_of(p, row), head = kvh * p.group + row - t * p.group;
  T* out = static_cast<T*>(p.out) + ((static_cast<int64_t>(b) * p.heads + head) * p.tokens + t) * D + first;
  const uint32_t w = pack2<T>(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
#pragma unroll 1
  for (int i = 0; i < N; i += 8) *reinterpret_cast<uint4*>(out + i) = make_uint4(w, w, w, w);
}

template <bool TREE, int TILE, int ROWS>
struct Walk {  // position in the list of tiles
  Span s;
  int g, h, tile;
  __device__ __forceinline__ void start(const AttendParams& p, const Found& f, uint32_t at) {
    g = f.group;
    s = span_of<TREE, TILE, ROWS>(p, g);
    const uint32_t rel = at - f.before;
    h = static_cast<int>(rel / s.n);
    tile = static_cast<int>(rel % s.n);
  }
  __device__ __forceinline__ void next(const AttendParams& p) {
    if (++tile < s.n) return;
    tile = 0;
    if (++h < p.kv_heads) return;
    h = 0;
    if (++g < p.batch * p.row_blocks) s = span_of<TREE, TILE, ROWS>(p, g);
  }
  __device__ __forceinline__ int key() const { return key_of_tile<TILE>(s, tile); }
};

// Joins the pieces of row r of a unit (group g, key head h): a warp per row, its pieces' weights first (a
// lane per piece), then their numerators, several loads in flight.
template <typename T, bool I8, int D, bool TREE, int ROWS>
__device__ __forceinline__ void join_row(const AttendParams& p, const Pieces at, int g, int h, int r, TreeMasks* tm) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, row = g % p.row_blocks * ROWS + r;
  if (row >= p.rows) return;  // the same for the warp
  // (a piece's slot) * ROWS + r, in rows of D + 4 words
  auto slot = [&](int c) { return (static_cast<int64_t>(2 * c + (c == at.c0 ? at.late : 0)) * ROWS + r) * (D + 4); };
  float mx = -INFINITY, sum = 0.f, acc[E];
  float2 first = make_float2(-INFINITY, 0.f);  // maximum and sum of this lane's first piece
  if (at.c0 + lane <= at.c1) first = *reinterpret_cast<const float2*>(p.partial + slot(at.c0 + lane) + D);
  mx = first.x;
  bool undone = first.y < 0.f;
  for (int c = at.c0 + 32 + lane; c <= at.c1; c += 32) {
    const float2 st = *reinterpret_cast<const float2*>(p.partial + slot(c) + D);
    mx = fmaxf(mx, st.x);
    undone |= st.y < 0.f;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int c0 = at.c0; c0 <= at.c1; c0 += 32) {
    float w = 0.f;
    if (c0 + lane <= at.c1) {
      const float2 st = c0 == at.c0 ? first : *reinterpret_cast<const float2*>(p.partial + slot(c0 + lane) + D);
      w = st.x == mx ? 1.f : ex2_approx(st.x - mx);
      sum = fmaf(st.y, w, sum);
    }
    const int n = min(32, at.c1 - c0 + 1);
#pragma unroll 8
    for (int c = 0; c < n; ++c) {
      const float wgt = __shfl_sync(0xffffffffu, w, c);
      const float* src = p.partial + slot(c0 + c) + lane * E;
      if (E == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        acc[0] = fmaf(v.x, wgt, acc[0]), acc[1] = fmaf(v.y, wgt, acc[1]), acc[E - 2] = fmaf(v.z, wgt, acc[E - 2]), acc[E - 1] = fmaf(v.w, wgt, acc[E - 1]);
      } else {
        const float2 v = *reinterpret_cast<const float2*>(src);
        acc[0] = fmaf(v.x, wgt, acc[0]), acc[1] = fmaf(v.y, wgt, acc[1]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  undone = __any_sync(0xffffffffu, undone);
  if (undone) sum = __int_as_float(0x7fc00000);
  const int b = g / p.row_blocks, len = attend_len(p, b), off = attend_off(p, b, len);
  const int t = token_of(p, row), idx = off + t;
  const bool valid = idx >= 0 && idx < len;
  const float inv = valid && sum != 0.f ? 1.f / sum : 0.f;
  T* dst = static_cast<T*>(p.out) + ((static_cast<int64_t>(b) * p.heads + h * p.group + row - t * p.group) * p.tokens + t) * D + lane * E;
  bool bad = valid && !(sum <= 3.0e38f);  // 1 / infinity would make zeros of a row of NaN
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const float x = inv == 0.f ? 0.f : acc[e] * inv, y = inv == 0.f ? 0.f : acc[e + 1] * inv;
    bad |= !holds<T>(x) || !holds<T>(y);
    *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(x, y);
  }
  __syncwarp();
  if (undone || !__any_sync(0xffffffffu, bad)) return;
  if (TREE) build_tree(p, b, off, lane, tm);  // warps of one CTA write the same values
  plain_row<T, I8, D, false>(p, b, h, row, off, len, row_view(p, off, len, t, TREE ? tm : nullptr), TREE);
}

// Joins the pieces of every unit that more than one CTA worked on.
constexpr int kJoinRows = 4;

template <typename T, bool I8, int D, bool TREE, int TILE, int ROWS>
__global__ void __launch_bounds__(32 * kJoinRows) join_kernel(const __grid_constant__ AttendParams p) {
  __shared__ TreeMasks tm;
  constexpr int BLOCKS = ROWS / kJoinRows;
  const int unit = p.first_unit + blockIdx.x / BLOCKS, g = unit / p.kv_heads;
  cudaGridDependencySynchronize();
  const Pieces at = p.pieces[unit];
  if (at.c0 == at.c1 || at.c0 < 0 || at.c1 < at.c0 || at.c1 >= p.workers) return;  // one CTA's; never written (a wait was abandoned)
  join_row<T, I8, D, TREE, ROWS>(p, at, g, unit - g * p.kv_heads, blockIdx.x % BLOCKS * kJoinRows + (threadIdx.x >> 5), &tm);
}

// Copy map of K or V: [line, key, lines of a row, head, batch element or page], boxes of `box` keys and
// `box_lines` lines.
// `stride`: dense element strides (batch, head, key); paged caches are contiguous.
int attend_map(CUtensorMap* m, const AttendParams& p, const void* base, const int64_t* stride, int line, int lines, int esz, int box, int box_lines);
// Maps of K and V for tiles of `tile` keys: the prepared ones (number `which`), or new ones.
int attend_maps(CUtensorMap* k, CUtensorMap* v, const AttendParams& p, int which, int row_bytes, int esz, int tile, bool whole_rows);

// few_rows.cuh
int launch_few_rows_f16(const AttendParams& p, int head_dim, bool i8, int device, cudaStream_t st);
int launch_few_rows_bf16(const AttendParams& p, int head_dim, bool i8, int device, cudaStream_t st);
uint64_t few_rows_workspace(int batch, int kv_heads, int rows, int head_dim);
// wide_rows.cuh
int launch_wide_rows_f16(const AttendParams& p, int head_dim, int device, cudaStream_t st);
int launch_wide_rows_bf16(const AttendParams& p, int head_dim, int device, cudaStream_t st);
uint64_t wide_rows_workspace(int batch, int kv_heads, int rows, int head_dim);

}  // namespace pk
