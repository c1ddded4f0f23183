// Attention of many query rows per key head (prompts, large drafted trees), 16-bit keys and values,
// dense or paged, on the tensor cores.  The formula is in pk_attend.cuh.
//
// What bounds it: 4 D operations per visible pair against one exponential, so the tensor pipe and
// the exponential unit about equally (a 128 x 128 tile at D = 128 takes 1024 cycles of each).
//
// One CTA per SM works on 256 query rows of one key head (two 128-row tiles; row = token * group +
// query head of the group, so that a tile's rows stand close together and share their window) over
// 128-key tiles:
//   - four softmax warpgroups, two per row tile on 64 keys each, a thread per row: scores from tensor
//     memory, maximum, sum, probabilities back to tensor memory over the scores;
//   - an MMA warp: S = Q K^T from shared memory, O += P V with P from tensor memory; the row tiles take
//     turns, so that one's softmax runs beside the other's products;
//   - a copy warp: K and V tiles by TMA through one ring.
// Tensor memory holds one score tile of 128 columns and one accumulator per row tile, no more: a row
// tile's scores, softmax and products follow one another, and the time of this chain is the kernel's.
// So the softmax keeps it short:
//   - Probabilities are relative to a reference exponent that follows the running maximum only when the
//     probabilities have grown too far (their sum over 64 keys tells: no maximum is taken on the way).  The
//     exponentials start with the reference of the tile before; only when a row has to raise it (the first
//     tile, and rarely later) the maximum is taken, the accumulator rescaled and they are evaluated again.
//   - Tiles that every row sees whole take a path without branches.
//   - A few of the exponentials are evaluated on the FMA pipe beside the exponential unit.
// Measured: 4 prompts of 8192 tokens, 32 query and 8 key heads of 128 features, window 1024, float16:
// 697 us, 743 TFLOP/s of visible pairs (0.45 of the measured 1652); the last 2048 tokens of 32760, 40 / 8
// heads, window 4096, bfloat16: 184 us, 947 TFLOP/s (0.57); SM clock 1875 to 1965 MHz.  A tile's chain takes some 3600 cycles where the two
// row tiles' products fill 2048; two thirds of it are in the softmax, most of that latency (taking the
// exponentials out altogether makes the kernel 6 % faster), the rest in the products and the hand-overs.
// A unit's query rows in, first scores and rows out take about 9000 cycles, partly beside the other row tile.
// Tried and slower (one prompt of 8192, 32 / 8 heads, no window, 532 us): the maximum taken beside the
// exponentials, 543; narrower steps than 64 keys for a half, 575; one warpgroup per row tile, 595 us, and 670
// with the maximum first; 64-key tiles with two score buffers per row tile, with one or two warpgroups per
// row tile and one or two issuing warps, 660 to 870 us (half is in flight per buffer, and every hand-over
// costs the same); all of a half's scores in registers at once, 710 us (they spill).
// V is read as it lies in memory (keys in rows): the B operand is taken transposed.
#pragma once

#include "pk_attend.cuh"

namespace pk {
namespace {

constexpr int kWideTile = 128;
constexpr int kWideRows = 256;
constexpr int kWideThreads = 4 * 128 + 64;  // four softmax warpgroups, the MMA and the copy warp
// A row raises its reference exponent when its probabilities of 64 keys sum to more than this (2^12: the
// largest of them fits every type).
constexpr float kWideRaise = 4096.f;
constexpr int kThere = 8;  // a copy is issued at most STAGES / 2 + 1 key tiles ahead of a tile whose V is still in use
constexpr int kWideWorkers = 148;
// From four rounds of units on, the partial last round costs less than sharing it out (768 ragged units: 118
// against 135 us); below, sharing pays (320 units: 213 against 231 us).
constexpr int64_t kWideShareBelow = 4 * kWideWorkers;

#define WIDE_ALL(x) __all_sync(0xffffffffu, (x))

__device__ __forceinline__ float max3f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int D, bool TREE>
struct Wide {
  static constexpr int HALF = 128 * 128;                // 128 rows of 64 features
  static constexpr int TILE_BYTES = HALF * (D / 64);    // a K, V or Q tile
  static constexpr int STAGES = D == 128 ? (TREE ? 4 : 5) : 10;
  static_assert(STAGES / 2 + 1 < kThere, "entries of `there` outlive their tiles");
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_RING = 2 * TILE_BYTES;
  static constexpr int OFF_TOP = OFF_RING + STAGES * TILE_BYTES;  // [row tile][half][128]: maxima, then sums
  static constexpr int OFF_BAR = OFF_TOP + 2 * 2 * 128 * 4;
  static constexpr int BARS = 2 * STAGES + 9;  // ring full / empty; q_full, s_full, p_full, o_done per row tile; drained
  static constexpr int OFF_RED = OFF_BAR + (BARS + 1) / 2 * 16;
  static constexpr int OFF_THERE = OFF_RED + 64;
  static constexpr int OFF_MISC = OFF_THERE + kThere * 4;
  static constexpr int OFF_TREE = (OFF_MISC + 8 + 7) / 8 * 8;
  static constexpr int SMEM = OFF_TREE + (TREE ? 2 * static_cast<int>(sizeof(TreeMasks)) : 0);
  static constexpr uint32_t COL_S = 0, COL_O = 256;
};

// Both operands 16-bit, 32-bit accumulator.  B transposed: its rows lie along the contraction.
template <typename T>
__host__ __device__ constexpr uint32_t wide_idesc(int n, bool b_transposed) {  // M = 128
  const uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_transposed ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Transposed operand: 64 contiguous features per 128-byte line, one key per line; groups of eight
// keys 1024 bytes apart, the next 64 features HALF bytes further.
__device__ __forceinline__ uint64_t v_desc(uint32_t addr, int half) {
  return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(half >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}

// 2^x for two values on the FMA pipe beside the exponential unit (an eighth of them: without, a batch of four
// prompts of 8192 tokens, window 1024, takes 766 us instead of 700; more of them is slower): x = n + r with
// n the nearest integer and |r| <= 1/2; 2^r by a polynomial of degree 4, fitted here for the least
// largest relative error with value 1 at 0 (2.9e-6, measured over r in 32-bit arithmetic); n goes into
// the exponent, which holds [-127, 127]: x is limited to that.  Below, the result is 0 (r = 0 there).  Above, it
// is 2^127, like every x beyond kWideRaise a reason to raise the reference and evaluate again.  A NaN comes
// out as the largest finite number: the row's sum is then no smaller (the row is evaluated again).
constexpr int kPolyEvery = 8;
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  float a, b;
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC2FE0000;\n\tmin.NaN.f32 %0, t, 0f42FE0000;\n\t}" : "=f"(a) : "f"(x.x));  // [-127, 127]
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC2FE0000;\n\tmin.NaN.f32 %0, t, 0f42FE0000;\n\t}" : "=f"(b) : "f"(x.y));
  const float2 magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f), neg = make_float2(-1.f, -1.f);
  x = make_float2(a, b);
  const float2 u = __fadd2_rn(x, magic);             // 1.5 * 2^23 + n: n in the low bits
  const float2 r = __ffma2_rn(__fadd2_rn(u, minus), neg, x);
  float2 y = make_float2(0x1.3a007ap-7f, 0x1.3a007ap-7f);
  y = __ffma2_rn(y, r, make_float2(0x1.c9fd1ep-5f, 0x1.c9fd1ep-5f));
  y = __ffma2_rn(y, r, make_float2(0x1.ec0382p-3f, 0x1.ec0382p-3f));
  y = __ffma2_rn(y, r, make_float2(0x1.62e12ap-1f, 0x1.62e12ap-1f));
  y = __ffma2_rn(y, r, make_float2(1.f, 1.f));
  return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(u.x) << 23)), __int_as_float(__float_as_int(y.y) + (__float_as_int(u.y) << 23)));
}

// Sixteen bytes from global to shared memory, asynchronously; `bytes` 0: zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// What one CTA does next.  Every role walks the same list: first every gridDim.x-th of the whole units
// [0, first_unit), from the back (causal rows see the most keys there), then an equal, contiguous share
// of the tiles of the units from first_unit on.
template <bool TREE>
struct Segments {
  Walk<TREE, kWideTile, kWideRows> walk;
  int unit, units;           // next whole unit and how many there are
  uint32_t at, end;          // share of tiles
  Found found;               // group of the share's first tile
  __device__ __forceinline__ bool more() const { return unit < units || at < end; }
  __device__ __forceinline__ bool whole() const { return unit < units; }
  __device__ __forceinline__ int count() const { return whole() ? walk.s.n : static_cast<int>(min(static_cast<uint32_t>(walk.s.n - walk.tile), end - at)); }
  __device__ __forceinline__ void take(const AttendParams& p) {
    if (whole()) {
      const int u = units - 1 - unit;
      walk.g = u / p.kv_heads;
      walk.h = u - walk.g * p.kv_heads;
      walk.tile = 0;
      walk.s = span_of<TREE, kWideTile, kWideRows>(p, walk.g);
    } else if (at < end) {
      walk.start(p, found, at);
    }
  }
  __device__ __forceinline__ void advance(const AttendParams& p) {
    if (whole()) {
      unit += gridDim.x;
      take(p);
    } else {
      const int n = count();
      at += n;
      walk.tile += n - 1;
      walk.next(p);
    }
  }
};

// The keys that the rows of one 128-row tile see, for skipping key tiles that only the other needs.
struct Reach {
  int lo, hi;
};
template <bool TREE>
__device__ __forceinline__ Reach reach_of(const AttendParams& p, const Span& s, int tile) {
  const int r0 = s.rb * kWideRows + tile * 128, r1 = min(r0 + 128, p.rows) - 1;
  Reach r{0, 0};
  if (r0 >= p.rows) return r;
  const int t0 = token_of(p, r0), t1 = token_of(p, r1);
  if (s.off + t0 >= s.len) return r;
  r.hi = max(0, TREE ? min(s.len, s.off + p.tokens) : min(s.len, s.off + t1 + 1));
  r.lo = max(0, (TREE ? s.off : s.off + t0) - p.window + 1);
  return r;
}
// How many of a tile's keys, from its first on, a row tile has to look at (a multiple of 64; 0: none).
__device__ __forceinline__ int width_of(const Reach& r, int j0, int sinks) {
  const int end = j0 + kWideTile > r.lo ? r.hi : min(sinks, r.hi);
  return max(0, min((end - j0 + 63) & ~63, kWideTile));
}

__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }  // bits [0, n)

// Which of the keys [j, j + 32) a row sees.
template <bool TREE>
__device__ __forceinline__ uint32_t seen_bits(const RowView& v, int j, int off, int sinks) {
  uint32_t bits = below(v.lim - j) & (~below(v.low + 1 - j) | below(sinks - j));
  if (TREE) {
    const int a = off - j;  // bit of the first drafted token
    bits &= below(a);
    if (a < 32 && a > -64) bits |= a >= 0 ? static_cast<uint32_t>(v.mask << a) : static_cast<uint32_t>(v.mask >> -a);
  }
  return bits;
}

// Where a row tile's warps stopped, for what they leave undone after a wait was given up.
struct Stopped {
  int unit;
  uint32_t at;
};

// Rows of NaN and marked pieces for what the CTA has not finished; by the whole CTA, which finds its place in the
// list of units anew (carrying it to the end of the kernel cost the softmax registers and 2 % of the time).
template <typename T, int D, bool TREE>
__device__ __noinline__ void leave_undone(const AttendParams& p, const Stopped* stopped, uint32_t* red, Found* found) {
  const int tid = threadIdx.x, i = (tid >> 7) & 1, half = tid >> 8, row = i * 128 + (tid & 127);
  Segments<TREE> seg;
  seg.unit = stopped[i].unit;
  seg.units = p.first_unit;
  seg.at = seg.end = 0;
  uint32_t total = 0, share_from = 0;
  if (p.workers) {
    const int g0 = p.first_unit / p.kv_heads;
    total = sum_tiles<TREE, kWideTile, kWideRows>(p, g0, p.batch * p.row_blocks, red);
    share_from = share_begin(total, p.workers, blockIdx.x);
    seg.at = stopped[i].at;
    seg.end = share_begin(total, p.workers, blockIdx.x + 1);
    for (int x = 0; x < 2; ++x) {
      if (stopped[x].at >= seg.end) continue;  // the same for the whole CTA
      const Found f = find_group<TREE, kWideTile, kWideRows>(p, g0, stopped[x].at, red, found);
      if (x == i) seg.found = f;
      __syncthreads();
    }
  }
  if (tid >= 512) return;  // the other threads stand for a half row each
  for (seg.take(p); seg.more(); seg.advance(p)) {
    const Span& s = seg.walk.s;
    const int r = s.rb * kWideRows + row, slot = blockIdx.x * 2 + (!seg.whole() && seg.at != share_from ? 1 : 0);
    if (r < p.rows) {
      if (seg.whole() || (seg.walk.tile == 0 && seg.count() == s.n)) nan_row<T, D, D / 2>(p, s.b, seg.walk.h, r, half * (D / 2));
      else if (half == 0) *reinterpret_cast<float2*>(p.partial + (static_cast<int64_t>(slot) * kWideRows + row) * (D + 4) + D) = make_float2(-INFINITY, kUndone);
    }
    if (!seg.whole() && seg.walk.tile == 0 && tid == 0)
      p.pieces[seg.walk.g * p.kv_heads + seg.walk.h] = Pieces{static_cast<int>(blockIdx.x), static_cast<int>(owner_of(total, p.workers, seg.at + s.n - 1)), seg.at != share_from, 0};
  }
}

template <typename T, int D, bool TREE>
__global__ void __launch_bounds__(kWideThreads, 1)
wide_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttendParams p) {
  using C = Wide<D, TREE>;
  constexpr int ST = C::STAGES;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + C::OFF_MISC + 4);
  volatile uint32_t* there = reinterpret_cast<volatile uint32_t*>(smem + C::OFF_THERE);
  uint32_t* red = reinterpret_cast<uint32_t*>(smem + C::OFF_RED);
  Found* found = reinterpret_cast<Found*>(smem + C::OFF_RED + 32);
  volatile long long* busy = reinterpret_cast<volatile long long*>(smem + C::OFF_RED + 40);
  Stopped* stopped = reinterpret_cast<Stopped*>(smem + C::OFF_RED + 48);
  const uint32_t bars = base + C::OFF_BAR;
  auto full = [&](int i) { return bars + 8 * i; };
  auto empty = [&](int i) { return bars + 8 * (ST + i); };
  auto q_full = [&](int i) { return bars + 8 * (2 * ST + i); };
  auto s_full = [&](int i) { return bars + 8 * (2 * ST + 2 + i); };
  auto p_full = [&](int i) { return bars + 8 * (2 * ST + 4 + i); };
  auto o_done = [&](int i) { return bars + 8 * (2 * ST + 6 + i); };  // the products of a segment
  const uint32_t drained = bars + 8 * (2 * ST + 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int MMA_WARP = 16, COPY_WARP = 17;

  if (tid < C::BARS) {
    const int at = tid - 2 * ST;
    mbar_init(bars + 8 * tid, at < 0 || at == 2 || at == 3 || at >= 6 ? 1 : 256);  // q_full, p_full: two warpgroups
    fence_barrier_init();
  }
  if (tid == 0) *abort_flag = 0, *busy = 0;
  if (warp == MMA_WARP) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    tmem_relinquish();
    tc_fence_before();
  }
  if (warp == COPY_WARP && lane == 0) { prefetch_tmap(&tm_k); prefetch_tmap(&tm_v); }
  cudaGridDependencySynchronize();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  Segments<TREE> seg;
  seg.unit = blockIdx.x;
  seg.units = p.first_unit;
  seg.at = seg.end = 0;
  uint32_t total = 0, share_from = 0;
  if (p.workers) {
    const int g0 = p.first_unit / p.kv_heads;  // shared units begin with a group
    total = sum_tiles<TREE, kWideTile, kWideRows>(p, g0, p.batch * p.row_blocks, red);
    share_from = seg.at = share_begin(total, p.workers, blockIdx.x);
    seg.end = share_begin(total, p.workers, blockIdx.x + 1);
    if (seg.at < seg.end) seg.found = find_group<TREE, kWideTile, kWideRows>(p, g0, seg.at, red, found);
  }
  seg.take(p);

  if (warp == COPY_WARP) {
    // ---------------------------------------------------------------- copies
    // Of a paged tile every page and half of the features is a copy of its own, issued by a lane of its
    // own; the pages of the next tile are looked up while this one's stages are waited for.
    const int box = p.table ? min(p.page, kWideTile) : kWideTile, boxes = kWideTile / box;
    const int x = lane % 8, hf = lane / 8;
    const bool mine = x < boxes && hf < D / 64;
    uint32_t st = 0, ph = 1;
    int n = 0;  // K and V tiles issued
    bool ok = true;
    for (; ok && seg.more(); seg.advance(p)) {
      const Span& s = seg.walk.s;
      const int count = seg.count(), from = seg.walk.tile, h = seg.walk.h;
      auto look_up = [&](int u) {
        const int j = key_of_tile<kWideTile>(s, from + u) + x * box;
        return p.table && mine && u < count && j < s.len ? attend_page(p, s.b, j) : -1;
      };
      int page = look_up(0);
      for (int u = 0; ok && u < count; ++u) {
        const int j0 = key_of_tile<kWideTile>(s, from + u), next = look_up(u + 1);
        const uint32_t mask = p.table ? __ballot_sync(0xffffffffu, page >= 0) & 0xffu : 1u;
        if (lane == 0) there[(n / 2) % kThere] = mask;
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv, ++n) {
          if (n >= ST && !(ok = WIDE_ALL(attend_wait(p, empty(st), ph, abort_flag, busy, 71)))) break;
          const uint32_t dst = base + C::OFF_RING + st * C::TILE_BYTES;
          const CUtensorMap* tmap = kv ? &tm_v : &tm_k;
          if (lane == 0) mbar_expect_tx(full(st), C::TILE_BYTES);
          __syncwarp();
          if (n == p.skip_copy) {  // drill
          } else if (p.table) {
            // a page that is not there, or lies behind the sequence, reads as zeros (outside the map)
            if (mine)
              tma_load_5d(dst + hf * C::HALF + x * box * 128, tmap, full(st), 0, (j0 + x * box) & (p.page - 1), hf, h, page >= 0 ? p.page_base + page : 0x7fffffff);
          } else if (lane == 0) {
            const int64_t sh = kv ? p.v_stride[1] : p.k_stride[1], sb = kv ? p.v_stride[0] : p.k_stride[0];
            tma_load_5d(dst, tmap, full(st), 0, j0, 0, sh ? h : 0, sb ? s.b : 0);
          }
          if (++st == ST) st = 0, ph ^= 1;
        }
        page = next;
      }
    }
    // When the CTA gives up a wait it ends early: not before the copies that were issued have landed (nor, below, the
    // products that were issued).
    for (int i = max(0, n - ST); i < n; ++i) mbar_wait_quiet(full(i % ST), (i / ST) & 1, 100000);
  } else if (warp == MMA_WARP) {
    // ---------------------------------------------------------------- products
    // Scalars only, descriptors built once: this warp is in everybody's chain.
    constexpr uint32_t id_o = wide_idesc<T>(D, true), id_s0 = wide_idesc<T>(0, false);
    const uint64_t q_desc = umma_smem_desc(base + C::OFF_Q, 128), k_desc = umma_smem_desc(base + C::OFF_RING, 128);
    const uint64_t v_desc0 = v_desc(base + C::OFF_RING, C::HALF);
    uint32_t k_st = 0, k_ph = 0, v_st = 1, v_ph = 0;  // stages of K of tile u + 1 and of V of tile u
    uint32_t ph0 = 0, ph1 = 0, nq = 0;                // phases of the p_full barriers, segments so far
    auto scores = [&](int i, int width, uint64_t kd) {
      const uint32_t d = tmem + C::COL_S + i * 128, id = id_s0 | (static_cast<uint32_t>(width >> 3) << 17);
      const uint64_t qd = q_desc + i * (C::TILE_BYTES >> 4);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16_ss(d, qd + ((k >> 2) * (C::HALF >> 4) + 2 * (k & 3)), kd + ((k >> 2) * (C::HALF >> 4) + 2 * (k & 3)), id, k > 0);
        tc_commit(s_full(i));
      }
    };
    auto values = [&](int i, int width, uint64_t vd, bool more) {
      const uint32_t d = tmem + C::COL_O + i * 128, a = tmem + C::COL_S + i * 128;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kWideTile / 16; k += 2) {
          if (16 * k < width) {  // the second 64 keys' probabilities lie over their own scores
            umma_f16_ts(d, a + (k >> 2) * 64 + (k & 3) * 8, vd + k * (2048 >> 4), id_o, more || k > 0);
            umma_f16_ts(d, a + (k >> 2) * 64 + (k & 3) * 8 + 8, vd + (k + 1) * (2048 >> 4), id_o, 1);
          }
        }
      }
    };
    auto turn = [&](uint32_t& stage, uint32_t& phase) {
      stage += 2;
      if (stage >= ST) stage -= ST, phase ^= 1;
    };
    bool ok = true;
    for (; ok && seg.more(); seg.advance(p), ++nq) {
      const Span& s = seg.walk.s;
      const int count = seg.count(), from = seg.walk.tile;
      const Reach r0 = reach_of<TREE>(p, s, 0), r1 = reach_of<TREE>(p, s, 1);
      bool more0 = false, more1 = false;
      int w0 = 0, w1 = 0;  // widths of tile u for the two row tiles, 0: not needed
      for (int u = -1; ok && u < count; ++u) {
        int x0 = 0, x1 = 0;
        if (u + 1 < count) {
          const int j0 = key_of_tile<kWideTile>(s, from + u + 1);
          x0 = width_of(r0, j0, p.sinks), x1 = width_of(r1, j0, p.sinks);
          ok = WIDE_ALL(attend_wait(p, full(k_st), k_ph, abort_flag, busy, 73));
        }
        if (ok && u >= 0) ok = WIDE_ALL(attend_wait(p, full(v_st), v_ph, abort_flag, busy, 72));
        if (!ok) break;
        const uint64_t kd = k_desc + k_st * (C::TILE_BYTES >> 4), vd = v_desc0 + v_st * (C::TILE_BYTES >> 4);
        if (w0) {
          ok = WIDE_ALL(attend_wait(p, p_full(0), ph0, abort_flag, busy, 74));
          if (!ok) break;
          ph0 ^= 1;
          tc_fence_after();
          values(0, w0, vd, more0);
          more0 = true;
        }
        if (u + 1 == count && elect_one()) tc_commit(o_done(0));
        if (u < 0 && !(ok = WIDE_ALL(attend_wait(p, q_full(0), nq & 1, abort_flag, busy, 75)))) break;
        tc_fence_after();
        if (x0) scores(0, x0, kd);
        if (w1) {
          ok = WIDE_ALL(attend_wait(p, p_full(1), ph1, abort_flag, busy, 79));
          if (!ok) break;
          ph1 ^= 1;
          tc_fence_after();
          values(1, w1, vd, more1);
          more1 = true;
        }
        if (u < 0 && !(ok = WIDE_ALL(attend_wait(p, q_full(1), nq & 1, abort_flag, busy, 75)))) break;
        tc_fence_after();
        if (x1) scores(1, x1, kd);
        if (elect_one()) {  // complete with everything issued so far
          if (u >= 0) tc_commit(empty(v_st));
          if (u + 1 < count) tc_commit(empty(k_st));
          else tc_commit(o_done(1));
        }
        if (u >= 0) turn(v_st, v_ph);
        if (u + 1 < count) turn(k_st, k_ph);
        w0 = x0, w1 = x1;
      }
    }
    if (elect_one()) tc_commit(drained);
    mbar_wait_quiet(drained, 0, 100000);
  } else if (warp < 16) {
    // ---------------------------------------------------------------- softmax
    // Row tile i; of each key tile the 64 keys of half `half`, of its features (query rows in, output
    // rows out) likewise.
    const int i = (warp >> 2) & 1, half = warp >> 3, row = tid & 127, w4 = warp & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(w4 * 32) << 16);
    const uint32_t o_addr = lanes + C::COL_O + i * 128 + half * (D / 2), s_addr = lanes + C::COL_S + i * 128 + half * 64;
    constexpr int FEATURES = D / 2, PIECES = FEATURES / 8, PER = 32 / PIECES;  // 16-byte pieces of a row's half, rows per access
    uint8_t* q_tile = smem + C::OFF_Q + i * C::TILE_BYTES;
    auto q_piece = [&](int r, int piece) {  // of this half
      const int at = half * PIECES + piece;
      return q_tile + (at >> 3) * C::HALF + r * 128 + (((at & 7) ^ (r & 7)) << 4);
    };
    float* tops = reinterpret_cast<float*>(smem + C::OFF_TOP) + i * 256 + row;
    TreeMasks* tm = reinterpret_cast<TreeMasks*>(smem + C::OFF_TREE) + i;
    const int box = p.table ? min(p.page, kWideTile) : kWideTile;
    const uint32_t all = (1u << (kWideTile / box)) - 1;
    uint32_t nt = 0, ns = 0, nq = 0;  // key tiles, those that this row tile needed, and segments so far
    int tree_b = -1;
    bool ok = true;
    for (; ok && seg.more(); seg.advance(p)) {
      const Span& s = seg.walk.s;
      const int count = seg.count(), from = seg.walk.tile, h = seg.walk.h;
      const Reach reach = reach_of<TREE>(p, s, i);
      const int row0 = s.rb * kWideRows + i * 128;
      if (TREE && s.b != tree_b) {
        asm volatile("bar.sync %0, 256;" ::"r"(1 + i) : "memory");  // the previous masks have been used
        if (w4 == 0 && half == 0) build_tree(p, s.b, s.off, lane, tm);
        asm volatile("bar.sync %0, 256;" ::"r"(1 + i) : "memory");
        tree_b = s.b;
      }
      // ---- the query rows into shared memory
      {
        const int piece = lane % PIECES, rl0 = w4 * 32 + lane / PIECES;
        const T* q0 = static_cast<const T*>(p.q) + s.b * p.q_stride[0] + static_cast<int64_t>(h) * p.group * p.q_stride[1] + half * FEATURES + piece * 8;
#pragma unroll
        for (int a = 0; a < 32 / PER; ++a) {
          const int rl = rl0 + a * PER, r = row0 + rl, tq = token_of(p, r);
          const T* src = q0 + (r - tq * p.group) * p.q_stride[1] + tq * p.q_stride[2];
          uint8_t* dst = q_piece(rl, piece);
          if (p.q_vec) {
            copy16(smem_u32(dst), r < p.rows ? src : q0, r < p.rows ? 16 : 0);
          } else {
            uint32_t e[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) e[y] = r < p.rows ? *reinterpret_cast<const uint16_t*>(src + y) : 0;
            *reinterpret_cast<uint4*>(dst) = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full(i));

      const int r = row0 + row, t = token_of(p, r);
      const RowView view = r < p.rows ? row_view(p, s.off, s.len, t, TREE ? tm : nullptr) : RowView{0, 0, 0};
      // keys that every row of this row tile sees
      const int t_first = token_of(p, min(row0, p.rows - 1)), t_last = token_of(p, min(row0 + 127, p.rows - 1));
      const int full_hi = TREE ? s.full_hi : min(s.len, s.off + t_first + 1), full_lo = TREE ? s.full_lo : s.off + t_last - p.window + 1;
      // Reference exponent of the probabilities (none yet; a row that sees nothing needs none), sum of this half's.
      float ref = view.lim > 0 || view.mask != 0 ? -INFINITY : 0.f, l = 0.f;
      bool begun = false;
      for (int u = 0; u < count; ++u, ++nt) {
        const int j0 = key_of_tile<kWideTile>(s, from + u);
        const int width = width_of(reach, j0, p.sinks), mine = width - 64 * half;  // the same for the whole warpgroup
        if (width == 0) continue;
        ok = WIDE_ALL(attend_wait(p, s_full(i), ns & 1, abort_flag, busy, 76));
        ++ns;
        tc_fence_after();
        const uint32_t held = there[nt % kThere];
        const bool clear = held == all && ((j0 >= full_lo && j0 + width <= full_hi) || j0 + width <= min(p.sinks, full_hi));
        uint32_t sr[32], pk[32];
        float* sc = reinterpret_cast<float*>(sr);
        float shift;
        float2 l0, l1;
        const float2 mul2 = make_float2(p.scale_log2, p.scale_log2);
        // 32 keys in sr: those that this row does not see get -inf, where any row of the warp needs it
        auto mask32 = [&](int c) {
          const int at = 64 * half + 32 * c;
          uint32_t bits = seen_bits<TREE>(view, j0 + at, s.off, p.sinks);
          if (held != all) {
            if (!((held >> (at / box)) & 1)) bits &= 0xffff0000u;
            if (!((held >> ((at + 16) / box)) & 1)) bits &= 0x0000ffffu;
          }
          if (__all_sync(0xffffffffu, bits == 0xffffffffu)) return;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((bits >> e) & 1)) sc[e] = -INFINITY;
        };
        auto pass = [&](int c, auto masked) {  // exponentials relative to the reference
          tmem_ld32(s_addr + 32 * c, sr);
          tmem_wait_ld();
          if (masked.value) mask32(c);
          const float2 shift2 = make_float2(shift, shift);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = __ffma2_rn(make_float2(sc[2 * e], sc[2 * e + 1]), mul2, shift2);
            const float2 y = e % kPolyEvery == kPolyEvery - 1 ? exp2_poly(x) : make_float2(ex2_approx(x.x), ex2_approx(x.y));
            if (e & 1) l1 = __fadd2_rn(l1, y); else l0 = __fadd2_rn(l0, y);
            pk[16 * c + e] = pack2<T>(y.x, y.y);
          }
        };
        auto passes = [&]() {
          shift = ref == -INFINITY ? 0.f : -ref;
          l0 = l1 = make_float2(0.f, 0.f);
          if (mine > 0) {
            if (clear) {
              pass(0, std::false_type{});
              pass(1, std::false_type{});
            } else {
              pass(0, std::true_type{});
              pass(1, std::true_type{});
            }
          }
        };
        passes();
        // V rows behind the sequence may hold anything (0 * NaN is a NaN): they become zeros before this
        // thread's arrival, for which the product waits.  All warpgroups write the same zeros.
        if (j0 + width > s.len) {
          const uint32_t vn = 2 * nt + 1;
          ok = ok && WIDE_ALL(attend_wait(p, full(vn % ST), (vn / ST) & 1, abort_flag, busy, 80));
          uint8_t* vt = smem + C::OFF_RING + vn % ST * C::TILE_BYTES;
          if (ok && j0 + row >= s.len) {
#pragma unroll
            for (int x = 0; x < D / 8; ++x) *reinterpret_cast<uint4*>(vt + (x >> 3) * C::HALF + row * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        // Does a row of the row tile have to raise its reference, or does one have none yet (its first tile)?
        if (!vote_barrier(1 + i, 256, ok && ref != -INFINITY && !((l0.x + l0.y) + (l1.x + l1.y) > kWideRaise))) {
          float top = -INFINITY;
          for (int c = 0; c < 2 && mine > 0; ++c) {
            tmem_ld32(s_addr + 32 * c, sr);
            tmem_wait_ld();
            if (!clear) mask32(c);
#pragma unroll
            for (int e = 0; e < 32; e += 2) top = max3f(top, sc[e], sc[e + 1]);
          }
          tops[half * 128] = top * p.scale_log2;
          ok = vote_barrier(1 + i, 256, ok && *abort_flag == 0);
          if (!ok) break;  // the row tile's warps leave together when a wait was abandoned
          const float now = fmaxf(ref, fmaxf(tops[0], tops[128])), keep = now == ref ? 1.f : ex2_approx(ref - now);
          ref = now;
          l *= keep;
          if (begun) {
            // the products of the tiles before this one are complete: they were issued before its scores
#pragma unroll 1
            for (int c = 0; c < FEATURES; c += 16) {
              uint32_t o[16];
              tmem_ld16(o_addr + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmem_st16(o_addr + c, o);
            }
          }
          shift = ref == -INFINITY ? 0.f : -ref;
          l0 = l1 = make_float2(0.f, 0.f);
          if (mine > 0) {  // with the mask in any case: one copy of this code
            pass(0, std::true_type{});
            pass(1, std::true_type{});
          }
        }
        begun = true;
        l += (l0.x + l0.y) + (l1.x + l1.y);
        if (mine > 0) {
          tmem_st16(s_addr, pk);
          tmem_st16(s_addr + 16, pk + 16);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_full(i));
      }
      // ---- rows out; the two halves add their sums
      ok = vote_barrier(1 + i, 256, ok && *abort_flag == 0);  // and the maxima have been read
      if (!ok) break;
      tops[half * 128] = l;
      ok = vote_barrier(1 + i, 256, WIDE_ALL(attend_wait(p, o_done(i), nq & 1, abort_flag, busy, 78)));
      if (!ok) break;
      const float m = ref;
      l = tops[0] + tops[128];
      ++nq;
      tc_fence_after();
      const int idx = s.off + t;
      const bool valid = r < p.rows && idx >= 0 && idx < s.len;
      if (!seg.whole() && from == 0 && tid == 0)
        p.pieces[seg.walk.g * p.kv_heads + h] = Pieces{static_cast<int>(blockIdx.x), static_cast<int>(owner_of(total, p.workers, seg.at + s.n - 1)), seg.at != share_from, 0};
      if (!seg.whole() && (from != 0 || count != s.n)) {
        const int slot = blockIdx.x * 2 + (seg.at != share_from ? 1 : 0);
        float* dst = p.partial + (static_cast<int64_t>(slot) * kWideRows + i * 128) * (D + 4);
        // 32 features at a time through this warp's rows of the query tile, so that whole lines leave
        constexpr int STRIDE = FEATURES * 2;  // bytes of a row's half in the query tile: this half's 16-bit pieces
        static_assert(STRIDE >= 64, "eight lanes write 32 features of a row");
#pragma unroll 1
        for (int c = 0; c < FEATURES; c += STRIDE / 4) {
          uint32_t o[STRIDE / 4];
#pragma unroll
          for (int e = 0; e < STRIDE / 4; e += 16) tmem_ld16(o_addr + c + e, o + e);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < STRIDE / 16; ++e)
            *reinterpret_cast<uint4*>(q_piece(row, e)) = begun ? make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]) : make_uint4(0, 0, 0, 0);
          __syncwarp();
#pragma unroll
          for (int a = 0; a < 32 / PER; ++a) {
            const int piece = lane % PIECES, rl = w4 * 32 + a * PER + lane / PIECES;
            const uint4 x = *reinterpret_cast<const uint4*>(q_piece(rl, piece));
            if (row0 + rl < p.rows) *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(rl) * (D + 4) + half * FEATURES + c + piece * 4) = x;
          }
          __syncwarp();
        }
        if (r < p.rows && half == 0) *reinterpret_cast<float2*>(dst + static_cast<int64_t>(row) * (D + 4) + D) = make_float2(m, l);
        tc_fence_before();
        continue;
      }
      // The query tile has been read by every product: its place takes the output rows, from where
      // they leave as whole lines (a thread's own row would be written 16 bytes at a time).
      const float inv = valid && begun && l != 0.f ? 1.f / l : 0.f;
      bool bad = valid && !(l <= 3.0e38f);  // 1 / infinity would make zeros of a row of NaN
#pragma unroll
      for (int c = 0; c < FEATURES; c += 32) {
        uint32_t o[32];
        tmem_ld32(o_addr + c, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float x[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            x[y] = inv != 0.f ? __uint_as_float(o[e + y]) * inv : 0.f;
            bad |= !holds<T>(x[y]);
          }
          *reinterpret_cast<uint4*>(q_piece(row, (c + e) / 8)) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
        }
      }
      tc_fence_before();
      __syncwarp();
      {
        const int piece = lane % PIECES, rl0 = w4 * 32 + lane / PIECES;
        T* out0 = static_cast<T*>(p.out) + (static_cast<int64_t>(s.b) * p.heads + static_cast<int64_t>(h) * p.group) * p.tokens * D + half * FEATURES + piece * 8;
#pragma unroll
        for (int a = 0; a < 32 / PER; ++a) {
          const int rl = rl0 + a * PER, rr = row0 + rl, tq = token_of(p, rr);
          const uint4 x = *reinterpret_cast<const uint4*>(q_piece(rl, piece));
          if (rr < p.rows) *reinterpret_cast<uint4*>(out0 + (static_cast<int64_t>(rr - tq * p.group) * p.tokens + tq) * D) = x;
        }
      }
      uint32_t vote = __ballot_sync(0xffffffffu, bad);
      __syncwarp();
      while (vote) {  // rows with a value that their type does not hold, evaluated again from their own keys
        const int src = __ffs(vote) - 1, rr = row0 + w4 * 32 + src;
        vote &= vote - 1;
        plain_row<T, false, D, true>(p, s.b, h, rr, s.off, s.len, row_view(p, s.off, s.len, token_of(p, rr), TREE ? tm : nullptr), TREE, busy, half * FEATURES, half * FEATURES + FEATURES);
      }
    }
    if (half == 0 && row == 0) stopped[i] = Stopped{seg.unit, seg.at};
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) leave_undone<T, D, TREE>(p, stopped, red, found);
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (tid == 0 && *abort_flag != 0 && p.host_status != nullptr) atomicCAS_system(p.host_status, 0, *abort_flag);
}

// Whole rounds of units over the CTAs are worked on unit by unit.  What is left over (in groups: all key
// heads of some rows) is shared out by tiles where that shortens the last round by more than the sharing
// costs: starting, leaving pieces and joining them takes about as long as six key tiles (12 us).
struct WidePlan {
  int64_t units, whole;
};
inline WidePlan wide_plan(int batch, int kv_heads, int rows, int tiles) {
  const int64_t units = static_cast<int64_t>(batch) * kv_heads * ((rows + kWideRows - 1) / kWideRows), left = units % kWideWorkers;
  if (units >= kWideShareBelow || (kWideWorkers - left) * tiles <= 6 * kWideWorkers) return {units, units};
  return {units, (units - left) / kv_heads * kv_heads};
}
// Key tiles of a unit, at most.
inline int wide_tiles(const AttendParams& p) {
  const int keys = p.table ? p.width * p.page : p.kv_len, span = kWideRows / p.group + 1;
  const int seen = p.window < keys - span ? p.window + span : keys, sinks = p.window < keys ? (p.sinks < keys ? p.sinks : keys) : 0;
  return (seen + kWideTile - 1) / kWideTile + (sinks + kWideTile - 1) / kWideTile;
}

template <typename T, int D, bool TREE>
int launch_wide(AttendParams p, int device, cudaStream_t st) {
  using C = Wide<D, TREE>;
  static_assert(C::SMEM <= 227 * 1024, "shared memory of one CTA");
  p.row_blocks = (p.rows + kWideRows - 1) / kWideRows;
  p.key_align = p.table ? (p.page < kWideTile ? p.page : kWideTile) : 8;
  CUtensorMap tk, tv;
  int rc;
  if ((rc = attend_maps(&tk, &tv, p, 2, D * 2, 2, kWideTile, !p.table))) return rc;
  if ((rc = allow_smem<wide_rows_kernel<T, D, TREE>>(C::SMEM, device))) return rc;
  const WidePlan plan = wide_plan(p.batch, p.kv_heads, p.rows, wide_tiles(p));
  const int64_t most = plan.units * (((p.table ? p.width * p.page : p.kv_len) + kWideTile - 1) / kWideTile + 2);
  if (most >= (1ll << 31)) return fail(PK_ERR_BAD_ARG, "attention: too many keys and rows for one call; split it over the batch");
  p.first_unit = static_cast<int>(plan.whole);
  p.workers = plan.whole < plan.units ? kWideWorkers : 0;
  p.pieces = reinterpret_cast<Pieces*>(p.partial);
  p.partial += (plan.units * (sizeof(Pieces) / sizeof(float)) + 63) / 64 * 64;
  cudaError_t e = launch_chained(wide_rows_kernel<T, D, TREE>, dim3(p.workers || plan.units > kWideWorkers ? kWideWorkers : static_cast<unsigned>(plan.units)),
                                 dim3(kWideThreads), C::SMEM, st, tk, tv, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return fail(PK_ERR_CUDA, "attention kernel launch failed: %s", cuda_err(e));
  if (!p.workers) return PK_OK;
  e = launch_chained(join_kernel<T, false, D, TREE, kWideTile, kWideRows>, dim3(static_cast<unsigned>(plan.units - plan.whole) * (kWideRows / kJoinRows)),
                     dim3(32 * kJoinRows), 0, st, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return fail(PK_ERR_CUDA, "join kernel launch failed: %s", cuda_err(e));
  return PK_OK;
}

template <typename T>
int wide_by_dim(const AttendParams& p, int head_dim, int device, cudaStream_t st) {
  if (head_dim == 128) return p.tree ? launch_wide<T, 128, true>(p, device, st) : launch_wide<T, 128, false>(p, device, st);
  return p.tree ? launch_wide<T, 64, true>(p, device, st) : launch_wide<T, 64, false>(p, device, st);
}

}  // namespace
}  // namespace pk
