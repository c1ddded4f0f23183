// Attention of few query rows per key head (single tokens, chains and trees of drafted tokens, short
// prompts) over long keys: dense tensors or a paged cache, 16-bit or 8-bit with a scale per row.
// The formula is in pk_attend.cuh.
//
// What bounds it: every K and V row is read once for the few query rows that see it, 4 * rows / 2
// operations per byte, so device memory does.  The kernel is built to keep copies in flight:
//   - A producer warp fills a ring of three stages of 64 or 128 keys (K and V, up to 32 KB each) with
//     TMA, one copy per page; two CTAs per SM keep up to 192 KB on the way.
//   - The keys of all batch elements and heads form one list of such tiles; every CTA takes an
//     equal, contiguous share of it, whatever the lengths are (they are read on the device: nothing
//     about them is known to the host).  The ring runs on across the borders between sequences.
//   - A sequence that several CTAs share leaves pieces (un-normalised rows, maximum, sum) in the
//     workspace; a second small kernel joins them.
//   - Few and short units get a cluster of CTAs each, which joins its own pieces (`cluster_of`).
// The products use mma.sync: at up to 64 query rows the tensor work is far below the time of the
// copies, and its fragments can be filled straight from the rows as they lie in memory.  The
// contraction may visit features and keys in any order, as long as both operands use the same:
//   - K: a thread takes 16-byte pieces of one key's row as they are; four consecutive features feed
//     one 16-deep step (the query fragments use the same order).
//   - V: a thread takes 16-byte pieces of the two keys that share a register and interleaves them
//     with byte permutes, eight (or sixteen, 8-bit) output features at a time.
// An 8-bit row's V scale is folded into the exponent: p = 2^(s + log2(scale) - max), and the sum
// gets p / scale (the way the 8-bit attention of fused_attention.cu treats its key scales), so that
// p stays in the range of a 16-bit float whatever the scales are.  p is rounded to the query's
// 16-bit type for the product; maxima, sums and accumulators are 32-bit.
// Measured: 64 single tokens (32 / 8 heads of 128 features) over 1088 to 8192 bfloat16 rows, 1.22 GB: 197 us,
// 6.2 TB/s (0.95 of the measured copy).  48 tokens (40 / 8 heads) over 8-bit rows, window 4096, 417 MB: 126 us,
// 3.3 TB/s: there the conversions to 16 bits (about 170 of 560 instructions for 16 keys of a warp) and the
// latency of two warps per scheduler bound it, not memory.  One token over 1000 rows: 9.2 us.

#pragma once

#include "pk_attend.cuh"

namespace pk {
namespace {

constexpr int kStages = 3;
constexpr int kConsumers = 128;
constexpr int kThreads = kConsumers + 32;
constexpr int kJoinCols = 32;          // output columns that the warps of a CTA join at a time
constexpr float kRaise = 8.f;          // a row's reference exponent follows its maximum only beyond this
constexpr int kMaxWorkers = 2 * 148;   // two CTAs per SM
constexpr int kClusterWorkers = 256;   // CTAs of clusters of eight that the SMs hold at once
constexpr int kClusterTiles = 12;      // tiles of 16 rows for a CTA, at most, for a unit to get a cluster of its own

template <typename T, bool I8, int D, int WM>
struct Few {
  static constexpr int WN = 4 / WM;
  static constexpr int ROWS = 16 * WM;
  static constexpr int ESZ = I8 ? 1 : 2;
  static constexpr int ROW_BYTES = D * ESZ;
  // Keys per stage: 16 to 32 KB of K and V where the warps share them out; fewer where every warp takes all of
  // them for its own rows (a stage's time counts when there are few).
  static constexpr int TILE = ROW_BYTES > 128 || WM > 1 ? 64 : 128;
  static constexpr int LINE = ROW_BYTES > 128 ? 128 : ROW_BYTES;  // swizzled line
  static constexpr int HALVES = ROW_BYTES / LINE;
  static constexpr int KV_BYTES = TILE * ROW_BYTES;
  static constexpr int SCALE_BYTES = I8 ? 2 * TILE * 4 : 0;
  static constexpr int STAGE = 2 * KV_BYTES;
  static constexpr int KEYS = TILE / WN;  // keys of a tile per warp
  // In a 16-byte shared-memory access eight threads (two key columns x four pieces) are served at
  // once.  128-byte lines: neighbouring columns are mapped to keys four apart, whose pieces the
  // swizzle puts into the other half of the banks.  64-byte lines: neighbours are two halves of 128 bytes.
  static constexpr bool APART = LINE == 128;
  static constexpr int OFF_JOIN = kStages * STAGE;
  static constexpr int OFF_SCALE = OFF_JOIN + 4 * 16 * kJoinCols * 4;
  static constexpr int OFF_ML = OFF_SCALE + kStages * SCALE_BYTES;
  static constexpr int OFF_TREE = OFF_ML + 4 * 16 * 8;
  static constexpr int OFF_BAR = OFF_TREE + static_cast<int>(sizeof(TreeMasks));
  static constexpr int OFF_RED = OFF_BAR + 2 * kStages * 8;
  static constexpr int OFF_MISC = OFF_RED + 4 * 8 + 24;  // (sums, the group found, when rows were last evaluated one by one)
  static constexpr int OFF_THERE = OFF_MISC + 4;  // per stage: which of its pages exist, one bit each
  static constexpr int SMEM = OFF_THERE + kStages * 4;
};

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1, __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two signed bytes of `w` (the bytes that `sel` puts into the low byte of each half) as two 16-bit floats, exactly.
// f16: 1024 + (byte ^ 0x80) is a bit pattern; minus 1152.
__device__ __forceinline__ uint32_t two_bytes(uint32_t w, bool high, __half) {
  const uint32_t u = __byte_perm(w ^ 0x80808080u, 0x64646464u, high ? 0x4342 : 0x4140);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// bf16: 128 + (byte & 127) and 128 + (byte & 128) are bit patterns; their difference.
__device__ __forceinline__ uint32_t two_bytes(uint32_t w, bool high, __nv_bfloat16) {
  const uint32_t u = __byte_perm(w, 0u, high ? 0x4342 : 0x4140);
  const uint32_t lo = (u & 0x007F007Fu) | 0x43004300u, sg = (u & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lo), *reinterpret_cast<const __nv_bfloat162*>(&sg));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Plain loads (not inline assembly), so that the compiler may move them within what the waits allow.
__device__ __forceinline__ uint4 lds128(const uint8_t* smem, uint32_t at) { return *reinterpret_cast<const uint4*>(smem + at); }
__device__ __forceinline__ uint2 lds64(const uint8_t* smem, uint32_t at) { return *reinterpret_cast<const uint2*>(smem + at); }

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows of NaN and marked pieces for what a CTA leaves undone after a wait was given up: the tiles [w, w1) of its
// share, which began with w0.
template <typename T, bool I8, int D, int WM, bool TREE>
__device__ __noinline__ void leave_undone(const AttendParams& p, Walk<TREE, Few<T, I8, D, WM>::TILE, Few<T, I8, D, WM>::ROWS> walk, uint32_t w, uint32_t w0,
                                          uint32_t w1, uint32_t total) {
  using C = Few<T, I8, D, WM>;
  while (w < w1) {
    const Span& s = walk.s;
    const int from = walk.tile, n = static_cast<int>(min(static_cast<uint32_t>(s.n - from), w1 - w));
    const bool whole = from == 0 && n == s.n;
    const int slot = blockIdx.x * 2 + (from == 0 && w != w0 && !p.cluster ? 1 : 0);
    for (int r = threadIdx.x; r < C::ROWS; r += kConsumers) {
      if (s.rb * C::ROWS + r >= p.rows) continue;
      if (whole) nan_row<T, D, D>(p, s.b, walk.h, s.rb * C::ROWS + r, 0);
      else *reinterpret_cast<float2*>(p.partial + (static_cast<int64_t>(slot) * C::ROWS + r) * (D + 4) + D) = make_float2(-INFINITY, kUndone);
    }
    if (from == 0 && threadIdx.x == 0 && !p.cluster) {
      const int last = whole ? static_cast<int>(blockIdx.x) : static_cast<int>(owner_of(total, gridDim.x, w + s.n - 1));
      p.pieces[walk.g * p.kv_heads + walk.h] = Pieces{static_cast<int>(blockIdx.x), last, w != w0, 0};
    }
    w += n;
    walk.tile = from + n - 1;
    walk.next(p);
  }
}

template <typename T, bool I8, int D, int WM, bool TREE>
__device__ __forceinline__ void attend_share(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttendParams& p, uint8_t* smem) {
  using C = Few<T, I8, D, WM>;
  const uint32_t base = smem_u32(smem);
  uint32_t* red = reinterpret_cast<uint32_t*>(smem + C::OFF_RED);
  Found* found = reinterpret_cast<Found*>(smem + C::OFF_RED + 32);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC);
  volatile uint32_t* there = reinterpret_cast<volatile uint32_t*>(smem + C::OFF_THERE);
  volatile long long* busy = reinterpret_cast<volatile long long*>(smem + C::OFF_RED + 48);
  const uint32_t bars = base + C::OFF_BAR;  // full[kStages], empty[kStages]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid < 2 * kStages) {
    mbar_init(bars + 8 * tid, tid < kStages ? 1 : 4);
    fence_barrier_init();
  }
  if (tid == 0) *abort_flag = 0, *busy = 0;
  if (tid == kConsumers) { prefetch_tmap(&tm_k); prefetch_tmap(&tm_v); }
  cudaGridDependencySynchronize();
  __syncthreads();

  Walk<TREE, C::TILE, C::ROWS> walk;
  uint32_t total = 0, w0, w1;
  if (p.cluster) {  // an equal share of the cluster's unit
    const uint32_t unit = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
    walk.g = unit / p.kv_heads, walk.h = unit % p.kv_heads;
    walk.s = span_of<TREE, C::TILE, C::ROWS>(p, walk.g);
    w0 = share_begin(walk.s.n, p.cluster, rank), w1 = share_begin(walk.s.n, p.cluster, rank + 1);
    walk.tile = w0;
    if (w0 >= w1) return;
  } else {
    total = sum_tiles<TREE, C::TILE, C::ROWS>(p, 0, p.batch * p.row_blocks, red);
    w0 = share_begin(total, gridDim.x, blockIdx.x), w1 = share_begin(total, gridDim.x, blockIdx.x + 1);
    if (w0 >= w1) return;
    walk.start(p, find_group<TREE, C::TILE, C::ROWS>(p, 0, w0, red, found), w0);
  }

  if (warp == kConsumers / 32) {
    // ---------------------------------------------------------------- producer
    // Of a paged tile every page is a copy of its own, issued by a lane of its own; the pages of the next
    // tile are looked up while this one's stage is waited for.
    const int box = p.table ? min(p.page, C::TILE) : C::TILE, boxes = C::TILE / box;
    auto look_up = [&]() {
      const int j = walk.key() + lane * box;
      return p.table && lane < boxes && j < walk.s.len ? attend_page(p, walk.s.b, j) : -1;
    };
    int last = -1, page = look_up();
    for (uint32_t w = w0; w < w1; ++w) {
      const int i = static_cast<int>(w - w0), st = i % kStages, j0 = walk.key(), h = walk.h, b = walk.s.b;
      walk.next(p);
      const int next = w + 1 < w1 ? look_up() : -1;
      if (i >= kStages && !__all_sync(0xffffffffu, attend_wait(p, bars + 8 * (kStages + st), ((i / kStages) - 1) & 1, abort_flag, busy, 61))) break;
      const uint32_t full = bars + 8 * st, dst = base + st * C::STAGE;
      const uint32_t mask = p.table ? __ballot_sync(0xffffffffu, page >= 0) : 1u;
      if (lane == 0) {
        there[st] = mask;
        mbar_expect_tx(full, C::STAGE + (I8 ? __popc(mask) * 2 * box * 4 : 0));
      }
      __syncwarp();
      if (i == p.skip_copy) {  // drill
      } else if (!p.table) {
        if (lane == 0) {
          tma_load_5d(dst, &tm_k, full, 0, j0, 0, p.k_stride[1] ? h : 0, p.k_stride[0] ? b : 0);
          tma_load_5d(dst + C::KV_BYTES, &tm_v, full, 0, j0, 0, p.v_stride[1] ? h : 0, p.v_stride[0] ? b : 0);
        }
      } else if (lane < boxes) {
        // a page that is not there, or lies behind the sequence, reads as zeros (outside the map)
        const int row = (j0 + lane * box) & (p.page - 1), c4 = page >= 0 ? p.page_base + page : 0x7fffffff;
        tma_load_5d(dst + lane * box * C::ROW_BYTES, &tm_k, full, 0, row, 0, h, c4);
        tma_load_5d(dst + C::KV_BYTES + lane * box * C::ROW_BYTES, &tm_v, full, 0, row, 0, h, c4);
        if (I8 && page >= 0) {
          const int64_t at = (static_cast<int64_t>(page) * p.kv_heads + h) * p.page + row;
          const uint32_t sdst = base + C::OFF_SCALE + st * C::SCALE_BYTES + lane * box * 4;
          bulk_load(sdst, p.k_scale + at, box * 4, full);
          bulk_load(sdst + C::TILE * 4, p.v_scale + at, box * 4, full);
        }
      }
      page = next;
      last = i;
    }
    // The CTA may end early, when its other warps give up a wait: not before the copies that were issued have landed.
    for (int i = max(0, last - kStages + 1); i <= last; ++i) mbar_wait_quiet(bars + 8 * (i % kStages), (i / kStages) & 1, 100000);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int wm = warp % WM, wn = warp / WM;
  const int g8 = lane >> 2, c4 = lane & 3;
  TreeMasks* tm = reinterpret_cast<TreeMasks*>(smem + C::OFF_TREE);
  float* join = reinterpret_cast<float*>(smem + C::OFF_JOIN);
  float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  // key of column n of an 8-key step
  auto key_of = [](int n) { return C::APART ? ((n & 1) << 2) | (n >> 1) : n; };
  constexpr int OT = D / 8;  // output column tiles
  uint32_t qf[D / 16][4];
  float o[OT][4], m[2], l[2];
  RowView view[2];
  int tree_b = -1;
  bool ok = true;

  uint32_t w = w0;
  for (int i = 0; w < w1;) {
    // -------- a new unit: rows [rb * ROWS, ...) of key head h of batch element b
    const Span s = walk.s;
    const int h = walk.h, unit_from = walk.tile;
    if (TREE && s.b != tree_b) {
      asm volatile("bar.sync 1, 128;" ::: "memory");  // the previous masks have been read
      if (warp == 0) build_tree(p, s.b, s.off, lane, tm);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      tree_b = s.b;
    }
    const T* qrow[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = s.rb * C::ROWS + wm * 16 + g8 + 8 * x, t = token_of(p, r);
      view[x] = r < p.rows ? row_view(p, s.off, s.len, t, TREE ? tm : nullptr) : RowView{0, 0, 0};
      const bool there = r < p.rows;
      qrow[x] = there ? static_cast<const T*>(p.q) + s.b * p.q_stride[0] + (h * p.group + r - t * p.group) * p.q_stride[1] + t * p.q_stride[2] : nullptr;
      m[x] = -INFINITY;
      l[x] = 0.f;
    }
    // query fragments in the order in which K rows are read (16 bytes of a K row at a time)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      constexpr int PIECE = I8 ? 16 : 8;  // features per 16 bytes of K
#pragma unroll
      for (int j = 0; j < D / PIECE / 4; ++j) {
#pragma unroll
        for (int k = 0; k < PIECE / 8; ++k) {
          const int d = (j * 4 + c4) * PIECE + k * 8;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (qrow[x]) {
            if (p.q_vec) {
              v = *reinterpret_cast<const uint4*>(qrow[x] + d);
            } else {
              uint32_t e[8];
#pragma unroll
              for (int y = 0; y < 8; ++y) e[y] = *reinterpret_cast<const uint16_t*>(qrow[x] + d + y);
              v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
            }
          }
          const int step = (j * (PIECE / 8) + k) * 2;
          qf[step][x] = v.x, qf[step][2 + x] = v.y, qf[step + 1][x] = v.z, qf[step + 1][2 + x] = v.w;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < OT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;

    const int unit_tiles = static_cast<int>(min(static_cast<uint32_t>(s.n - walk.tile), w1 - w));
    const int box = p.table ? min(p.page, C::TILE) : C::TILE;
    for (int u = 0; u < unit_tiles; ++u, ++i) {
      const int st = i % kStages;
      ok = __all_sync(0xffffffffu, attend_wait(p, bars + 8 * st, (i / kStages) & 1, abort_flag, busy, 62));
      if (!ok) break;
      const int j0 = key_of_tile<C::TILE>(s, unit_from + u);
      // Keys on pages that are not there are masked like those that no row may see.
      const uint32_t held = there[st], all = (1u << (C::TILE / box)) - 1;
      const bool full = held == all && ((j0 >= s.full_lo && j0 + C::TILE <= s.full_hi) || (j0 + C::TILE <= min(p.sinks, s.full_hi)));
      const uint32_t kst = st * C::STAGE, vst = kst + C::KV_BYTES;  // offsets in shared memory
      const float* sc = reinterpret_cast<const float*>(smem + C::OFF_SCALE + st * C::SCALE_BYTES);
#pragma unroll(I8 ? 2 : 1)
      for (int step = 0; step < C::KEYS / 16; ++step) {
        const int k0 = wn * C::KEYS + step * 16;  // within the tile
        if (j0 + k0 >= s.len && !full) continue;  // behind the sequence (the same for the whole warp)
        const uint32_t off0 = C::HALVES == 2 ? (k0 / box) * (box * C::ROW_BYTES) + (k0 % box) * 128 : k0 * C::LINE;
        const uint32_t half = box * 128;
        // ---- scores of 16 keys: two 8-key columns of the fragment, each in two sums (a product that
        // accumulates waits for its predecessor; four chains are interleaved)
        float sv[2][4], sw[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int y = 0; y < 4; ++y) sv[nt][y] = sw[nt][y] = 0.f;
#pragma unroll
        for (int j = 0; j < C::ROW_BYTES / 64; ++j) {
          uint4 v[2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const int kk = nt * 8 + key_of(g8), chunk = j * 4 + c4;
            const int sw_ = C::LINE == 128 ? (kk & 7) : ((kk >> 1) & 3);
            v[nt] = lds128(smem, kst + off0 + kk * C::LINE + (C::HALVES == 2 ? (chunk >> 3) * half : 0) + (((chunk & (C::LINE / 16 - 1)) ^ sw_) << 4));
          }
          if (I8) {
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
              for (int nt = 0; nt < 2; ++nt) {
                const uint32_t w8 = y == 0 ? v[nt].x : y == 1 ? v[nt].y : y == 2 ? v[nt].z : v[nt].w;
                mma16816(y & 1 ? sw[nt] : sv[nt], qf[j * 4 + y], two_bytes(w8, false, T{}), two_bytes(w8, true, T{}), T{});
              }
          } else {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) mma16816(sv[nt], qf[j * 2], v[nt].x, v[nt].y, T{});
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) mma16816(sw[nt], qf[j * 2 + 1], v[nt].z, v[nt].w, T{});
          }
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int y = 0; y < 4; ++y) sv[nt][y] += sw[nt][y];
        // ---- to base-2 exponents; column n of the fragment is key key_of(n)
        float inv[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int kk = (y >> 1) * 8 + key_of(2 * c4 + (y & 1));
          float mul = p.scale_log2, add = 0.f;
          if (I8) {
            // A scale of zero makes a zero row, whose weight still counts: taken as 2^-60.
            float vs = sc[C::TILE + k0 + kk];
            vs = vs < 0x1p-60f ? 0x1p-60f : vs;
            mul *= sc[k0 + kk];
            add = __log2f(vs);
            inv[y] = rcp_approx(vs);
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float& e = sv[y >> 1][(y & 1) + 2 * x];
            e = I8 ? fmaf(e, mul, add) : e * mul;
          }
        }
        if (!full) {
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int j = j0 + k0 + (y >> 1) * 8 + key_of(2 * c4 + (y & 1));
            const bool in = j < s.len && ((held >> (k0 / box)) & 1);
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (!in || !sees<TREE>(view[x], j, s.off, p.sinks)) sv[y >> 1][(y & 1) + 2 * x] = -INFINITY;
          }
        }
        // ---- running maximum: the reference exponent moves only when a score exceeds it by more
        // than kRaise (2^kRaise fits every type); the quotient is the same for any reference
        float top[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) top[x] = fmaxf(fmaxf(sv[0][2 * x], sv[0][2 * x + 1]), fmaxf(sv[1][2 * x], sv[1][2 * x + 1]));
        const bool raise = top[0] > m[0] + kRaise || top[1] > m[1] + kRaise;
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float t = top[x];
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            const float mn = t > m[x] + kRaise ? t : m[x];
            const float keep = m[x] == mn ? 1.f : ex2_approx(m[x] - mn);
            m[x] = mn;
            l[x] *= keep;
#pragma unroll
            for (int t2 = 0; t2 < OT; ++t2) o[t2][2 * x] *= keep, o[t2][2 * x + 1] *= keep;
          }
        }
        uint32_t pf[4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float ref = m[x] == -INFINITY ? 0.f : m[x];
          float e[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            e[y] = ex2_approx(sv[y >> 1][(y & 1) + 2 * x] - ref);
            l[x] = I8 ? (e[y] != 0.f ? fmaf(e[y], inv[y], l[x]) : l[x]) : l[x] + e[y];
          }
          pf[x] = pack2<T>(e[0], e[1]);
          pf[2 + x] = pack2<T>(e[2], e[3]);
        }
        // ---- O += P V
        int kk[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) kk[y] = (y >> 1) * 8 + key_of(2 * c4 + (y & 1));
        // Rows behind the sequence are whatever an earlier owner of the page left (a NaN times the
        // weight 0 is a NaN): they are taken as zeros.
        const bool ragged = j0 + k0 + 16 > s.len;
        if (I8) {
          constexpr int W = D == 128 ? 4 : 2;  // words of a V row per thread
          uint32_t vw[4][4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t row = vst + off0 + kk[y] * C::LINE;
            if (D == 128) {
              const uint4 v = lds128(smem, row + ((key_of(g8) ^ (kk[y] & 7)) << 4));
              vw[y][0] = v.x, vw[y][1] = v.y, vw[y][2] = v.z, vw[y][3] = v.w;
            } else {
              const uint2 v = lds64(smem, row + (((g8 >> 1) ^ ((kk[y] >> 1) & 3)) << 4) + (g8 & 1) * 8);
              vw[y][0] = v.x, vw[y][1] = v.y, vw[y][2] = vw[y][3] = 0;
            }
          }
#pragma unroll
          for (int x = 0; x < W; ++x) {
            // bytes of two keys, alternating: a0 b0 a1 b1 / a2 b2 a3 b3
            const uint32_t lo01 = __byte_perm(vw[0][x], vw[1][x], 0x5140), lo23 = __byte_perm(vw[0][x], vw[1][x], 0x7362);
            const uint32_t hi01 = __byte_perm(vw[2][x], vw[3][x], 0x5140), hi23 = __byte_perm(vw[2][x], vw[3][x], 0x7362);
            mma16816(o[x * 4 + 0], pf, two_bytes(lo01, false, T{}), two_bytes(hi01, false, T{}), T{});
            mma16816(o[x * 4 + 1], pf, two_bytes(lo01, true, T{}), two_bytes(hi01, true, T{}), T{});
            mma16816(o[x * 4 + 2], pf, two_bytes(lo23, false, T{}), two_bytes(hi23, false, T{}), T{});
            mma16816(o[x * 4 + 3], pf, two_bytes(lo23, true, T{}), two_bytes(hi23, true, T{}), T{});
          }
        } else {
#pragma unroll
          for (int hf = 0; hf < D / 64; ++hf) {
            uint32_t vw[4][4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint4 v = lds128(smem, vst + off0 + hf * half + kk[y] * 128 + ((key_of(g8) ^ (kk[y] & 7)) << 4));
              vw[y][0] = v.x, vw[y][1] = v.y, vw[y][2] = v.z, vw[y][3] = v.w;
              if (ragged && j0 + k0 + kk[y] >= s.len) vw[y][0] = vw[y][1] = vw[y][2] = vw[y][3] = 0;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              mma16816(o[hf * 8 + 2 * x], pf, __byte_perm(vw[0][x], vw[1][x], 0x5410), __byte_perm(vw[2][x], vw[3][x], 0x5410), T{});
              mma16816(o[hf * 8 + 2 * x + 1], pf, __byte_perm(vw[0][x], vw[1][x], 0x7632), __byte_perm(vw[2][x], vw[3][x], 0x7632), T{});
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + 8 * (kStages + st));
    }

    // -------- join the warps that shared the unit's keys; write rows, or a piece for the join kernel
    const bool whole = unit_from == 0 && unit_tiles == s.n;
    if (unit_from == 0 && tid == 0 && !p.cluster) {
      const int last = whole ? static_cast<int>(blockIdx.x) : static_cast<int>(owner_of(total, gridDim.x, w + s.n - 1));
      p.pieces[walk.g * p.kv_heads + h] = Pieces{static_cast<int>(blockIdx.x), last, w != w0, 0};
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (c4 == 0) ml[warp * 16 + g8 + 8 * x] = make_float2(m[x], l[x]);
    }
    ok = vote_barrier(1, kConsumers, ok && *abort_flag == 0);  // the same answer in every warp: they leave together
    if (!ok) break;
    const int slot = blockIdx.x * 2 + (unit_from == 0 && w != w0 && !p.cluster ? 1 : 0);
    float* piece = p.partial + static_cast<int64_t>(slot) * C::ROWS * (D + 4);
    // thread -> (row, four consecutive columns) of the CTA's rows; a row's columns belong to 8 neighbouring threads
    bool bad[WM];
#pragma unroll
    for (int x = 0; x < WM; ++x) bad[x] = false;
#pragma unroll
    for (int pass = 0; pass < D / kJoinCols; ++pass) {
      // stage: [warp][16 rows][32 columns].  The fragment's columns are spread over the row (16-byte
      // pieces of V rows): this pass takes the output tiles whose features lie in its 32 columns.
#pragma unroll
      for (int t = 0; t < OT; ++t) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          int d;
          if (I8 && D == 128) d = (c4 + 4 * n) * 16 + t;
          else if (I8) d = (2 * c4 + n) * 8 + t;
          else d = (t >> 3) * 64 + (c4 + 4 * n) * 8 + (t & 7);
          if (d / kJoinCols == pass) {
#pragma unroll
            for (int x = 0; x < 2; ++x) join[(warp * 16 + g8 + 8 * x) * kJoinCols + (d % kJoinCols)] = o[t][n + 2 * x];
          }
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
      for (int it = 0; it < WM; ++it) {
        const int r16 = tid >> 3, col = (tid & 7) * 4;  // rows of warp row `it`
        const int row = s.rb * C::ROWS + it * 16 + r16;
        float mx = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < C::WN; ++n) mx = fmaxf(mx, ml[(n * WM + it) * 16 + r16].x);
#pragma unroll
        for (int n = 0; n < C::WN; ++n) {
          const float2 st = ml[(n * WM + it) * 16 + r16];
          const float wgt = st.x == mx ? 1.f : ex2_approx(st.x - mx);
          const float4 v = *reinterpret_cast<const float4*>(join + ((n * WM + it) * 16 + r16) * kJoinCols + col);
          sum = fmaf(st.y, wgt, sum);
          acc[0] = fmaf(v.x, wgt, acc[0]), acc[1] = fmaf(v.y, wgt, acc[1]), acc[2] = fmaf(v.z, wgt, acc[2]), acc[3] = fmaf(v.w, wgt, acc[3]);
        }
        if (row < p.rows) {
          if (!whole) {
            float* dst = piece + (it * 16 + r16) * (D + 4);
            *reinterpret_cast<float4*>(dst + pass * kJoinCols + col) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            if (pass == 0 && (tid & 7) == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mx, sum);
          } else {
            const int t = token_of(p, row), idx = s.off + t;
            const bool valid = idx >= 0 && idx < s.len;
            const float r = valid && sum != 0.f ? 1.f / sum : 0.f;
            float v[4];
            bad[it] |= valid && !(sum <= 3.0e38f);  // 1 / infinity would make zeros of a row of NaN
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              v[y] = r == 0.f ? 0.f : acc[y] * r;
              bad[it] |= !holds<T>(v[y]);
            }
            T* dst = static_cast<T*>(p.out) + ((static_cast<int64_t>(s.b) * p.heads + h * p.group + row - t * p.group) * p.tokens + t) * D + pass * kJoinCols + col;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
          }
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
    }
#pragma unroll
    for (int it = 0; it < WM; ++it) {
      // rows with a value that their type does not hold, evaluated again from their own keys
      const uint32_t vote = __ballot_sync(0xffffffffu, bad[it]);
      __syncwarp();
#pragma unroll 1
      for (int r = 0; vote && r < 4; ++r) {
        if (!(vote & (0xffu << (8 * r)))) continue;
        const int row = s.rb * C::ROWS + it * 16 + warp * 4 + r;
        plain_row<T, I8, D, true>(p, s.b, h, row, s.off, s.len, row_view(p, s.off, s.len, token_of(p, row), TREE ? tm : nullptr), TREE, busy);
      }
    }
    // the next unit
    w += unit_tiles;
    walk.tile = unit_from + unit_tiles - 1;
    walk.next(p);
  }
  if (w < w1) leave_undone<T, I8, D, WM, TREE>(p, walk, w, w0, w1, total);
  if (tid == 0 && *abort_flag != 0 && p.host_status != nullptr) atomicCAS_system(p.host_status, 0, *abort_flag);
}

template <typename T, bool I8, int D, int WM, bool TREE>
__device__ __noinline__ void join_cluster(const AttendParams& p, TreeMasks* tm) {
  using C = Few<T, I8, D, WM>;
  const int rank = blockIdx.x % p.cluster, first = blockIdx.x - rank, unit = blockIdx.x / p.cluster, g = unit / p.kv_heads;
  const int pieces = min(span_of<TREE, C::TILE, C::ROWS>(p, g).n, p.cluster), warps = kThreads / 32;
  if (pieces < 2) return;
  for (int r = rank * warps + (threadIdx.x >> 5); r < C::ROWS; r += p.cluster * warps)
    join_row<T, I8, D, TREE, C::ROWS>(p, Pieces{first, first + pieces - 1, 0, 0}, g, unit - g * p.kv_heads, r, tm);
}

template <typename T, bool I8, int D, int WM, bool TREE>
__global__ void __launch_bounds__(kThreads, 2)
few_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttendParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  attend_share<T, I8, D, WM, TREE>(tm_k, tm_v, p, smem);
  if (p.cluster < 2) return;
  // every thread of the cluster comes here, on every path; the barrier makes the pieces visible to all of them
  __syncwarp();
  cluster_barrier();
  join_cluster<T, I8, D, WM, TREE>(p, reinterpret_cast<TreeMasks*>(smem + Few<T, I8, D, WM>::OFF_TREE));
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
// Key tiles of a unit, at most.
inline int64_t few_tiles(const AttendParams& p, int tile, int rows) {
  const int64_t keys = p.table ? static_cast<int64_t>(p.width) * p.page : p.kv_len, span = p.tree ? p.tokens : rows / p.group + 1;
  const int64_t seen = p.window < keys - span ? p.window + span + p.key_align : keys, sinks = p.window < keys ? (p.sinks < keys ? p.sinks : keys) : 0;
  return (seen + tile - 1) / tile + (sinks + tile - 1) / tile;
}
// CTAs of the cluster that works on one unit and joins its pieces, or 0 to share all tiles out and join in a
// second kernel.  A cluster saves that kernel and finding the shares, and leaves few pieces, but its unit may be
// the longest by far and its CTAs copy 32 KB in 0.8 us (16 rows; 1.5 us at 32 rows, 2.6 us at 64) when few
// others do; the limit keeps that to some 10 us.  Above 16 rows it has warps enough to join all rows at once
// (16 tokens of 4 sequences, 64 rows, over 256: 18.8 us with eight CTAs each, 15.6 us shared); 16 CTAs take about
// 1 us more to start than eight, and only some eight such clusters are held at once (two sequences: 25 us).
// Cluster against shares, microseconds, 32 / 8 heads of 128 features, bfloat16: one token over 1024, 4096 and
// 16384 rows 8.9 / 11.4, 12.5 / 22.4, 24.0 / 25.2; 16 single tokens over 256, 512 and 1024 rows 10.4 / 11.9,
// 12.0 / 14.9, 15.9 / 18.9, over 128 to 1024 rows 15.3 / 19.0, one over 1024 beside 15 over 128 14.3 / 11.8;
// 16 tokens of one sequence (64 rows) over 1024 and 4096 rows 15.9 / 16.7, 26.2 / 31.4.
inline int cluster_of(int64_t units, int64_t tiles, int rows) {
  constexpr int WARPS = kThreads / 32;
  int n = tiles > 1 ? 16 : 1;
  while (n > 1 && (units * n > (n == 16 ? kClusterWorkers / 2 : kClusterWorkers) || ((n == 16 ? 2 * n : n / 2) >= tiles && n / 2 * WARPS >= rows))) n /= 2;
  if (units * n > kMaxWorkers || tiles * rows > static_cast<int64_t>(16 * kClusterTiles) * n) return 0;
  return tiles <= 1 || rows <= 16 || n * WARPS >= rows ? n : 0;
}

template <typename T, bool I8, int D, int WM, bool TREE>
int launch(AttendParams p, int device, cudaStream_t st) {
  using C = Few<T, I8, D, WM>;
  static_assert(C::SMEM <= 113 * 1024, "two CTAs share an SM");
  p.row_blocks = (p.rows + C::ROWS - 1) / C::ROWS;
  p.key_align = p.table ? (p.page < C::TILE ? p.page : C::TILE) : 8;
  CUtensorMap tk, tv;
  int rc;
  if ((rc = attend_maps(&tk, &tv, p, C::TILE == 64 ? 0 : 1, C::ROW_BYTES, C::ESZ, C::TILE, true))) return rc;
  if ((rc = allow_smem<few_rows_kernel<T, I8, D, WM, TREE>, true>(C::SMEM, device))) return rc;
  // No more CTAs than there can be tiles.
  const int64_t units = static_cast<int64_t>(p.batch) * p.row_blocks * p.kv_heads;
  const int64_t most = units * (((p.table ? p.width * p.page : p.kv_len) + C::TILE - 1) / C::TILE + 2);
  if (most >= (1ll << 31)) return fail(PK_ERR_BAD_ARG, "attention: too many keys and rows for one call; split it over the batch");
  p.workers = static_cast<int>(most < kMaxWorkers ? most : kMaxWorkers);
  p.cluster = cluster_of(units, few_tiles(p, C::TILE, C::ROWS), C::ROWS);
  if (p.cluster) p.workers = static_cast<int>(units) * p.cluster;
  p.first_unit = 0;
  p.pieces = reinterpret_cast<Pieces*>(p.partial);
  p.partial += (units * (sizeof(Pieces) / sizeof(float)) + 63) / 64 * 64;
  cudaError_t e = launch_clusters(p.cluster ? p.cluster : 1, few_rows_kernel<T, I8, D, WM, TREE>, dim3(p.workers), dim3(kThreads), C::SMEM, st, tk, tv, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return fail(PK_ERR_CUDA, "attention kernel launch failed: %s", cuda_err(e));
  if (p.cluster) return PK_OK;
  e = launch_chained(join_kernel<T, I8, D, TREE, C::TILE, C::ROWS>, dim3(static_cast<unsigned>(units) * (C::ROWS / kJoinRows)), dim3(32 * kJoinRows), 0, st, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return fail(PK_ERR_CUDA, "join kernel launch failed: %s", cuda_err(e));
  return PK_OK;
}

template <typename T, bool I8, int D, bool TREE>
int by_rows(const AttendParams& p, int device, cudaStream_t st) {
  if (p.rows <= 16) return launch<T, I8, D, 1, TREE>(p, device, st);
  if (p.rows <= 32) return launch<T, I8, D, 2, TREE>(p, device, st);
  return launch<T, I8, D, 4, TREE>(p, device, st);
}
template <typename T, bool I8, int D>
int by_tree(const AttendParams& p, int device, cudaStream_t st) {
  return p.tree ? by_rows<T, I8, D, true>(p, device, st) : by_rows<T, I8, D, false>(p, device, st);
}
template <typename T, bool I8>
int by_dim(const AttendParams& p, int head_dim, int device, cudaStream_t st) {
  return head_dim == 128 ? by_tree<T, I8, 128>(p, device, st) : by_tree<T, I8, 64>(p, device, st);
}

}  // namespace
}  // namespace pk
