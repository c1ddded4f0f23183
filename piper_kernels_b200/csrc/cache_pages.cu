// Page work of the paged K/V cache (pk_cache in include/piper_b200.h): making room, storing and
// gathering rows, sharing, cutting and compacting sequences.  All of it runs on the device from
// device-side counts, so that a decoding step needs no host round trip and can be captured.
//
// What bounds it: extend, fork and truncate touch a few thousand words and are bound by launch and
// memory latency; write, read and compact move whole rows and are bound by device memory.
// Results do not depend on the order in which threads run: pages are chosen by rank (lowest free
// first, sequences in order), counts change by integer atomics only.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "pk_internal.h"
#include "pk_ptx.cuh"

namespace pk {
namespace {

constexpr int kMaxBatch = 4096;
constexpr int kPlan = 1024;  // threads of the planning CTA

struct Pages {
  int layers, pages, kv_heads, page, shift, dim, batch, width;
  uint8_t* keys;
  uint8_t* values;
  float* key_scales;
  float* value_scales;
  int32_t* table;
  int32_t* lengths;
  int32_t* starts;
  int32_t* uses;
  int32_t* refused;
  int32_t* scratch;
};

__device__ __forceinline__ int row_limit(const Pages& c) { return c.width << c.shift; }
__device__ __forceinline__ int length_of(const Pages& c, int b) { return max(0, min(c.lengths[b], row_limit(c))); }
__device__ __forceinline__ int pages_for(const Pages& c, int rows) { return (rows + c.page - 1) >> c.shift; }
__device__ __forceinline__ bool is_page(const Pages& c, int page) { return page >= 0 && page < c.pages; }
// First row of a (layer, page, head) block.
__device__ __forceinline__ int64_t block_row(const Pages& c, int layer, int page, int head) {
  return ((static_cast<int64_t>(layer) * c.pages + page) * c.kv_heads + head) << c.shift;
}

// Exclusive sum over the CTA's kPlan threads; `total` is the sum.
__device__ __forceinline__ int scan_plan(int mine, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const int before = (warp ? warp_sums[warp - 1] : 0) + incl - mine;
  *total = warp_sums[31];
  __syncthreads();
  return before;
}

// ---------------------------------------------------------------------------------------
// extend: one CTA plans, then copy_tails_kernel copies the shared last pages.
// scratch: [0] number of copies, then (source page, target page, rows) from word 4 on.
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kPlan) extend_kernel(const Pages c, const int32_t* __restrict__ counts) {
  extern __shared__ int plan[];
  int* tail = plan;                  // last, partly filled page of a sequence that grows; -1: none
  int* before = plan + c.batch;      // new pages of the sequences in front (batch + 1 entries)
  int* copies = before + c.batch + 1;  // whether the last page is replaced
  int* order = before;                 // until `before` is written: rows on the last page, the first sequence ahead among equals
  __shared__ int warp_sums[32];
  __shared__ int n_copies;
  const int tid = threadIdx.x;
  cudaGridDependencySynchronize();
  if (tid == 0) n_copies = 0;
  for (int b = tid; b < c.batch; b += kPlan) {
    const int len = length_of(c, b), add = max(counts[b], 0);
    int page = -1;
    if (add > 0 && add <= row_limit(c) - len && (len & (c.page - 1))) page = c.table[static_cast<int64_t>(b) * c.width + (len >> c.shift)];
    tail[b] = is_page(c, page) ? page : -1;
    order[b] = (len & (c.page - 1)) * kMaxBatch + kMaxBatch - 1 - b;
  }
  __syncthreads();
  // A last page that others name too is replaced; when all that name it grow, the longest of them keeps it (the
  // first of these): its new rows lie behind all rows of an owner that gets no page for its copy and stays.
  for (int b = tid; b < c.batch; b += kPlan) {
    bool copy = false;
    const int page = tail[b];
    if (page >= 0) {
      const int users = c.uses[page];
      if (users > 1) {
        int growing = 0, longest = 0;
        for (int o = 0; o < c.batch; ++o) {
          const int at = order[o];
          if (tail[o] == page) ++growing, longest = max(longest, at);
        }
        copy = growing < users || longest != order[b];
      }
    }
    copies[b] = copy;
  }
  int carry = 0;
  for (int b0 = 0; b0 < c.batch; b0 += kPlan) {
    const int b = b0 + tid;
    int need = 0;
    if (b < c.batch) {
      const int len = length_of(c, b), add = max(counts[b], 0);
      if (add <= row_limit(c) - len) need = pages_for(c, len + add) - pages_for(c, len) + copies[b];
    }
    int total;
    const int at = scan_plan(need, warp_sums, &total);
    if (b < c.batch) before[b] = carry + at;
    carry += total;
  }
  if (tid == 0) before[c.batch] = carry;
  __syncthreads();
  const int wanted = carry;
  // How many of the wanted pages exist: the free ones are counted until that many are found.
  int free_pages = 0;
  for (int p0 = 0; p0 < c.pages && free_pages < wanted; p0 += 4 * kPlan) {
    int mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int page = p0 + i * kPlan + tid;
      mine += page < c.pages && c.uses[page] == 0;
    }
    int total;
    scan_plan(mine, warp_sums, &total);
    free_pages += total;
  }
  const int granted = min(free_pages, wanted);
  // The free pages again, now each with its rank: page of rank r goes to the sequence b with
  // before[b] <= r < before[b + 1], unless that sequence does not get all it needs.
  int rank0 = 0;
  for (int p0 = 0; p0 < c.pages && rank0 < granted; p0 += kPlan) {
    const int page = p0 + tid;
    const int is_free = page < c.pages && c.uses[page] == 0;
    int total;
    const int r = rank0 + scan_plan(is_free, warp_sums, &total);
    if (is_free && r < granted) {
      int lo = 0, hi = c.batch - 1;  // the last b with before[b] <= r
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (before[mid] <= r) lo = mid; else hi = mid - 1;
      }
      if (before[lo + 1] <= granted) {
        const int b = lo, len = length_of(c, b), nth = r - before[b];
        // the copy of the last page comes first, the pages behind it after that
        const int column = copies[b] && nth == 0 ? len >> c.shift : pages_for(c, len) + nth - copies[b];
        c.table[static_cast<int64_t>(b) * c.width + column] = page;
        c.uses[page] = 1;
        if (copies[b] && nth == 0) {
          const int n = atomicAdd(&n_copies, 1);
          int32_t* e = c.scratch + 4 + 3 * n;
          e[0] = tail[b], e[1] = page, e[2] = len & (c.page - 1);
        }
      }
    }
    rank0 += total;
  }
  __syncthreads();
  for (int b = tid; b < c.batch; b += kPlan) {
    const int len = length_of(c, b), add = max(counts[b], 0);
    const bool fits = add <= row_limit(c) - len, served = before[b + 1] == before[b] || before[b + 1] <= granted;
    if (copies[b] && fits && served) atomicSub(&c.uses[tail[b]], 1);
    c.starts[b] = len;
    c.lengths[b] = fits && served ? len + add : len;
    c.refused[b] = !(fits && served);
  }
  if (tid == 0) c.scratch[0] = n_copies;
}

template <int ESZ>
__global__ void __launch_bounds__(256) copy_tails_kernel(const Pages c) {
  cudaGridDependencySynchronize();
  const int n = c.scratch[0], per = c.layers * c.kv_heads;
  const int row_bytes = c.dim * ESZ;
  for (int64_t item = blockIdx.x; item < static_cast<int64_t>(n) * per; item += gridDim.x) {
    const int32_t* e = c.scratch + 4 + 3 * (item / per);
    const int lh = static_cast<int>(item % per), layer = lh / c.kv_heads, head = lh % c.kv_heads;
    const int64_t from = block_row(c, layer, e[0], head), to = block_row(c, layer, e[1], head);
    const int pieces = e[2] * row_bytes / 16;
    const uint4* fk = reinterpret_cast<const uint4*>(c.keys + from * row_bytes);
    const uint4* fv = reinterpret_cast<const uint4*>(c.values + from * row_bytes);
    uint4* tk = reinterpret_cast<uint4*>(c.keys + to * row_bytes);
    uint4* tv = reinterpret_cast<uint4*>(c.values + to * row_bytes);
#pragma unroll 4
    for (int i = threadIdx.x; i < pieces; i += 256) {
      const uint4 a = fk[i], b = fv[i];
      tk[i] = a;
      tv[i] = b;
    }
    if (ESZ == 1) {
      for (int i = threadIdx.x; i < e[2]; i += 256) {
        c.key_scales[to + i] = c.key_scales[from + i];
        c.value_scales[to + i] = c.value_scales[from + i];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// write / read.  D / 8 neighbouring threads share a row, eight values (16 bytes of 16-bit input) each.
// ---------------------------------------------------------------------------------------
struct Source {
  const uint16_t* key;
  const uint16_t* value;
  int64_t ks[4], vs[4];  // layer, batch, head, token
  int tokens, layer0, layers, vec;
};

__device__ __forceinline__ uint4 load8(const uint16_t* s, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(s);
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = s[i];
  return make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
}
template <typename T>
__device__ __forceinline__ float2 two_floats(uint32_t w);
template <>
__device__ __forceinline__ float2 two_floats<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <>
__device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// Eight values of a row as 8-bit codes.  The row's maximum is taken over the bit patterns of the
// magnitudes (ordered like the values, NaN above infinity) by the row's D / 8 lanes.  Bound by
// instructions, hence the packed arithmetic.
template <typename T, int D>
__device__ __forceinline__ uint2 quantise8(uint4 raw, float* scale) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float2 x[4];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = two_floats<T>(w[i]);
    top = max(top, max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu));
  }
  constexpr uint32_t kLanes = D / 8, kMask = kLanes == 16 ? 0xffffu : 0xffu;
  top = __reduce_max_sync(kMask << (threadIdx.x & 31 & ~(kLanes - 1)), top);
  if (top >= 0x7f800000u) {
    *scale = __int_as_float(0x7fc00000);
    return make_uint2(0, 0);
  }
  const float s = __fadd_rn(__fdiv_rn(__uint_as_float(top), 127.f), 1e-7f);
  *scale = s;
  // rint(x / s): |x / s| <= 127, so no clamp, and 1.5 * 2^23 + integer has the code in its low byte.  x times
  // the approximate reciprocal lies within 127 * 2 * 2^-23 = 3.1e-5 of the quotient and rounds like it, unless
  // it is that near a half-integer: then (one value in some thousands) the quotient itself is rounded.
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float2 inv2 = make_float2(inv, inv), magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f), neg = make_float2(-1.f, -1.f);
  float2 m[4];
  float near = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = __fmul2_rn(x[i], inv2);
    m[i] = __fadd2_rn(q, magic);
    const float2 d = __ffma2_rn(__fadd2_rn(m[i], minus), neg, q);
    near = fmaxf(near, fmaxf(fabsf(d.x), fabsf(d.y)));
  }
  if (near > 0.4999f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = make_float2(__fadd_rn(__fdiv_rn(x[i].x, s), 12582912.f), __fadd_rn(__fdiv_rn(x[i].y, s), 12582912.f));
  }
  uint32_t two[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) two[i] = __byte_perm(__float_as_uint(m[i].x), __float_as_uint(m[i].y), 0x0040);
  return make_uint2(__byte_perm(two[0], two[1], 0x5410), __byte_perm(two[2], two[3], 0x5410));
}

// Rows per thread whose loads are issued together.  Storing: two (8-bit rows 31.8 us against 37.5 with one
// and 33.7 with four, 8 prompts of up to 2047 rows, 8 heads); gathering: one (36.0 / 37.5 / 49.0 us; its
// output alone, 134 MB, takes a fill kernel 39 us).
constexpr int kStoreDeep = 2, kGatherDeep = 1;

// blockIdx.x: (layer, sequence, head); blockIdx.y: a block of rows.
template <typename T, bool I8, int D>
__global__ void __launch_bounds__(256) write_kernel(const Pages c, const Source s) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES;
  const int sub = threadIdx.x % LANES, head = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads, b = rest % c.batch, layer = rest / c.batch;
  cudaGridDependencySynchronize();
  const int start = c.starts[b], added = min(length_of(c, b) - start, s.tokens);
  const uint16_t* key = s.key + layer * s.ks[0] + b * s.ks[1] + head * s.ks[2] + sub * 8;
  const uint16_t* value = s.value + layer * s.vs[0] + b * s.vs[1] + head * s.vs[2] + sub * 8;
  for (int t0 = blockIdx.y * ROWS * kStoreDeep; t0 < added && start >= 0; t0 += gridDim.y * ROWS * kStoreDeep) {
    int64_t row[kStoreDeep];
    uint4 k[kStoreDeep], v[kStoreDeep];
#pragma unroll
    for (int i = 0; i < kStoreDeep; ++i) {
      const int t = t0 + i * ROWS + threadIdx.x / LANES, at = start + t;
      row[i] = -1;
      k[i] = v[i] = make_uint4(0, 0, 0, 0);
      if (t >= added) continue;
      k[i] = load8(key + t * s.ks[3], s.vec);
      v[i] = load8(value + t * s.vs[3], s.vec);
      const int page = c.table[static_cast<int64_t>(b) * c.width + (at >> c.shift)];
      if (is_page(c, page)) row[i] = block_row(c, s.layer0 + layer, page, head) + (at & (c.page - 1));
    }
#pragma unroll
    for (int i = 0; i < kStoreDeep; ++i) {
      if (I8) {
        float ks, vs;
        const uint2 kc = quantise8<T, D>(k[i], &ks), vc = quantise8<T, D>(v[i], &vs);
        if (row[i] < 0) continue;
        *reinterpret_cast<uint2*>(c.keys + row[i] * D + sub * 8) = kc;
        *reinterpret_cast<uint2*>(c.values + row[i] * D + sub * 8) = vc;
        if (sub == 0) c.key_scales[row[i]] = ks, c.value_scales[row[i]] = vs;
      } else if (row[i] >= 0) {
        *reinterpret_cast<uint4*>(c.keys + row[i] * D * 2 + sub * 16) = k[i];
        *reinterpret_cast<uint4*>(c.values + row[i] * D * 2 + sub * 16) = v[i];
      }
    }
  }
}

template <typename T, bool I8>
__device__ __forceinline__ void fetch8(const uint8_t* base, const float* scales, int64_t row, int dim, int sub, float* x) {
  if (I8) {
    const uint2 w = *reinterpret_cast<const uint2*>(base + row * dim + sub * 8);
    const float s = scales[row];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)))) * s;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(base + (row * dim + sub * 8) * 2);
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = two_floats<T>(ww[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void store8(void* out, int dtype, int64_t at, const float* x) {
  if (dtype == PK_F32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == PK_F16) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, bool I8, int D>
__global__ void __launch_bounds__(256) read_kernel(const Pages c, int layer0, const int32_t* __restrict__ first, int count, void* key, void* value, int dtype) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES;
  const int sub = threadIdx.x % LANES, head = blockIdx.x % c.kv_heads, rest = blockIdx.x / c.kv_heads, b = rest % c.batch, layer = rest / c.batch;
  cudaGridDependencySynchronize();
  const int64_t first_row = first[b], out0 = static_cast<int64_t>(blockIdx.x) * count;
  const int len = length_of(c, b);
  for (int t0 = blockIdx.y * ROWS * kGatherDeep; t0 < count; t0 += gridDim.y * ROWS * kGatherDeep) {
    float k[kGatherDeep][8], v[kGatherDeep][8];
#pragma unroll
    for (int i = 0; i < kGatherDeep; ++i) {
      const int t = t0 + i * ROWS + threadIdx.x / LANES;
      const int64_t at = first_row + t;
#pragma unroll
      for (int x = 0; x < 8; ++x) k[i][x] = v[i][x] = 0.f;
      if (t >= count || at < 0 || at >= len) continue;
      const int page = c.table[static_cast<int64_t>(b) * c.width + (at >> c.shift)];
      if (!is_page(c, page)) continue;
      const int64_t row = block_row(c, layer0 + layer, page, head) + (at & (c.page - 1));
      fetch8<T, I8>(c.keys, c.key_scales, row, D, sub, k[i]);
      fetch8<T, I8>(c.values, c.value_scales, row, D, sub, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kGatherDeep; ++i) {
      const int t = t0 + i * ROWS + threadIdx.x / LANES;
      if (t >= count) continue;
      store8(key, dtype, (out0 + t) * D + sub * 8, k[i]);
      store8(value, dtype, (out0 + t) * D + sub * 8, v[i]);
    }
  }
}

// ---------------------------------------------------------------------------------------
// fork: a CTA owns some columns of the table for all sequences, so that every entry is read before
// any of these columns changes.
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) fork_kernel(const Pages c, const int32_t* __restrict__ parents, int columns) {
  extern __shared__ int fresh[];  // [batch][columns]
  cudaGridDependencySynchronize();
  const int c0 = blockIdx.x * columns, n = min(columns, c.width - c0);
  for (int i = threadIdx.x; i < c.batch * n; i += 256) {
    const int b = i / n, p = parents[b] < c.batch ? parents[b] : b;
    fresh[i] = p < 0 ? -1 : c.table[static_cast<int64_t>(p) * c.width + c0 + i % n];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < c.batch * n; i += 256) {
    int32_t* entry = c.table + static_cast<int64_t>(i / n) * c.width + c0 + i % n;
    const int was = *entry, is = fresh[i];
    if (was == is) continue;
    if (is_page(c, was)) atomicSub(&c.uses[was], 1);
    if (is_page(c, is)) atomicAdd(&c.uses[is], 1);
    *entry = is;
  }
  if (blockIdx.x) return;
  __syncthreads();
  for (int b = threadIdx.x; b < c.batch; b += 256) {
    const int p = parents[b] < c.batch ? parents[b] : b;
    fresh[b] = p < 0 ? 0 : c.lengths[p];
  }
  __syncthreads();
  for (int b = threadIdx.x; b < c.batch; b += 256) {
    c.lengths[b] = c.starts[b] = fresh[b];
    c.refused[b] = parents[b] >= c.batch;
  }
}

// Releases the pages of sequence b behind its first `keep` rows; one CTA.
__device__ __forceinline__ void cut(const Pages& c, int b, int keep) {
  int32_t* row = c.table + static_cast<int64_t>(b) * c.width;
  for (int i = pages_for(c, keep) + threadIdx.x; i < c.width; i += blockDim.x) {
    const int page = row[i];
    if (page == -1) continue;
    if (is_page(c, page)) atomicSub(&c.uses[page], 1);
    row[i] = -1;
  }
  if (threadIdx.x == 0) c.lengths[b] = c.starts[b] = keep;
}

__global__ void __launch_bounds__(128) truncate_kernel(const Pages c, const int32_t* __restrict__ lengths) {
  cudaGridDependencySynchronize();
  const int b = blockIdx.x, keep = min(length_of(c, b), max(lengths[b], 0));
  __syncthreads();  // everybody has read the length before thread 0 writes it
  cut(c, b, keep);
}

// ---------------------------------------------------------------------------------------
// compact: rows move first (a warp per layer and head of a sequence), then the sequences are cut.
// ---------------------------------------------------------------------------------------
struct Paths {
  const int32_t* paths;
  int64_t stride;
  const int32_t* counts;
  int most;
};

// Whether sequence b's path rises strictly within the rows added last; the whole warp.
__device__ __forceinline__ bool path_ok(const Pages& c, const Paths& p, int b, int lane, int* added) {
  const int n = length_of(c, b) - c.starts[b], count = p.counts[b];
  *added = n;
  if (count < 0 || count > p.most || count > n || c.starts[b] < 0) return false;
  bool good = true;
  for (int i = lane; i < count; i += 32) {
    const int at = p.paths[b * p.stride + i], prev = i ? p.paths[b * p.stride + i - 1] : -1;
    good = good && at > prev && at < n;
  }
  return __all_sync(0xffffffffu, good);
}

template <int ROW_BYTES, bool I8>
__global__ void __launch_bounds__(256) move_rows_kernel(const Pages c, const Paths p) {
  constexpr int LANES = ROW_BYTES / 16, ROWS = 32 / LANES, DEEP = 4;  // lanes per row, rows per access, accesses in flight
  cudaGridDependencySynchronize();
  const int lane = threadIdx.x & 31, per = c.layers * c.kv_heads;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= static_cast<int64_t>(per) * c.batch) return;
  const int b = static_cast<int>(item / per), lh = static_cast<int>(item % per), layer = lh / c.kv_heads, head = lh % c.kv_heads;
  int added;
  if (!path_ok(c, p, b, lane, &added)) return;
  const int count = p.counts[b], start = c.starts[b], sub = lane % LANES;
  const int32_t* table = c.table + static_cast<int64_t>(b) * c.width;
  auto row_of = [&](int at) -> int64_t {
    const int page = table[at >> c.shift];
    return is_page(c, page) ? block_row(c, layer, page, head) + (at & (c.page - 1)) : -1;
  };
  // A row's target is at or in front of its source and the path rises: a group of rows is read
  // before it is written, and later groups' sources lie behind every target written so far.
  for (int i0 = 0; i0 < count; i0 += ROWS * DEEP) {
    uint4 k[DEEP], v[DEEP];
    float ks[DEEP], vs[DEEP];
    int64_t to[DEEP];
#pragma unroll
    for (int x = 0; x < DEEP; ++x) {
      const int i = i0 + x * ROWS + lane / LANES;
      to[x] = -1;
      if (i >= count) continue;
      const int at = p.paths[b * p.stride + i];
      if (at == i) continue;  // already there
      const int64_t from = row_of(start + at);
      to[x] = row_of(start + i);
      if (from < 0) to[x] = -1;
      if (to[x] < 0) continue;
      k[x] = *reinterpret_cast<const uint4*>(c.keys + from * ROW_BYTES + sub * 16);
      v[x] = *reinterpret_cast<const uint4*>(c.values + from * ROW_BYTES + sub * 16);
      if (I8 && sub == 0) ks[x] = c.key_scales[from], vs[x] = c.value_scales[from];
    }
    __syncwarp();
#pragma unroll
    for (int x = 0; x < DEEP; ++x) {
      if (to[x] < 0) continue;
      *reinterpret_cast<uint4*>(c.keys + to[x] * ROW_BYTES + sub * 16) = k[x];
      *reinterpret_cast<uint4*>(c.values + to[x] * ROW_BYTES + sub * 16) = v[x];
      if (I8 && sub == 0) c.key_scales[to[x]] = ks[x], c.value_scales[to[x]] = vs[x];
    }
    __syncwarp();
  }
}

__global__ void __launch_bounds__(128) cut_paths_kernel(const Pages c, const Paths p) {
  cudaGridDependencySynchronize();
  const int b = blockIdx.x;
  int added;
  const bool good = path_ok(c, p, b, threadIdx.x & 31, &added);  // every warp comes to the same answer
  const int keep = c.starts[b] + p.counts[b];
  __syncthreads();
  if (threadIdx.x == 0) c.refused[b] = !good;
  if (good) cut(c, b, keep);
}

int pages_of(const pk_cache* c, Pages* p) {
  const int rc = validate_cache(c);
  if (rc) return rc;
  *p = Pages{c->layers, c->pages, c->kv_heads, c->page_size, __builtin_ctz(static_cast<unsigned>(c->page_size)), c->head_dim, c->batch, c->width,
             static_cast<uint8_t*>(c->keys), static_cast<uint8_t*>(c->values), c->key_scales, c->value_scales, c->table, c->lengths, c->starts,
             c->uses, c->refused, c->scratch};
  return PK_OK;
}

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? PK_OK : fail(PK_ERR_CUDA, "%s launch failed: %s", what, cuda_err(e));
}

// Checks shared by the entry points; makes the device current through `guard`.
#define PK_CACHE_ENTRY(c, p)                                                                                              \
  clear_error();                                                                                                          \
  Pages p;                                                                                                                \
  int rc = pages_of(c, &p);                                                                                               \
  if (rc) return rc;                                                                                                      \
  const DeviceGuard guard((c)->device);                                                                                   \
  if (guard.err != cudaSuccess) return fail(PK_ERR_CUDA, "cudaSetDevice(%d): %s", (c)->device, cuda_err(guard.err));      \
  if ((rc = check_arch((c)->device))) return rc;                                                                          \
  const cudaStream_t st = static_cast<cudaStream_t>((c)->stream)

unsigned copy_grid(int64_t items) { return static_cast<unsigned>(items < 148 * 8 ? (items > 0 ? items : 1) : 148 * 8); }

dim3 row_grid(const Pages& p, int layers, int rows, int deep) {
  const int per = 256 / (p.dim / 8) * deep, blocks = (rows + per - 1) / per;
  return dim3(static_cast<unsigned>(layers) * p.batch * p.kv_heads, blocks < 1024 ? blocks : 1024);
}

template <typename T, bool I8>
cudaError_t launch_write(const Pages& p, const Source& s, cudaStream_t st) {
  const dim3 grid = row_grid(p, s.layers, s.tokens, kStoreDeep);
  return p.dim == 128 ? launch_chained(write_kernel<T, I8, 128>, grid, dim3(256), 0, st, p, s)
                      : launch_chained(write_kernel<T, I8, 64>, grid, dim3(256), 0, st, p, s);
}
template <typename T, bool I8>
cudaError_t launch_read(const Pages& p, int layer0, int layers, const int32_t* first, int count, void* key, void* value, int dtype, cudaStream_t st) {
  const dim3 grid = row_grid(p, layers, count, kGatherDeep);
  return p.dim == 128 ? launch_chained(read_kernel<T, I8, 128>, grid, dim3(256), 0, st, p, layer0, first, count, key, value, dtype)
                      : launch_chained(read_kernel<T, I8, 64>, grid, dim3(256), 0, st, p, layer0, first, count, key, value, dtype);
}
template <int ROW_BYTES, bool I8>
cudaError_t launch_move(const Pages& p, const Paths& paths, cudaStream_t st) {
  const int64_t warps = static_cast<int64_t>(p.layers) * p.kv_heads * p.batch;
  return launch_chained(move_rows_kernel<ROW_BYTES, I8>, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256), 0, st, p, paths);
}

bool even_strides(const void* base, const int64_t* s) {
  return !(reinterpret_cast<uintptr_t>(base) & 15) && !((s[0] | s[1] | s[2] | s[3]) & 7);
}

}  // namespace

int validate_cache(const pk_cache* c) {
  if (!c) return fail(PK_ERR_BAD_ARG, "cache: null cache");
  if (c->layers <= 0 || c->pages <= 0 || c->kv_heads <= 0 || c->batch <= 0 || c->width <= 0) return fail(PK_ERR_BAD_ARG, "cache: sizes must be positive");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return fail(PK_ERR_BAD_ARG, "cache: page size must be 16, 32, 64, 128 or 256, got %d", c->page_size);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(PK_ERR_BAD_ARG, "cache supports head dimensions 64 and 128, got %d", c->head_dim);
  if (c->dtype != PK_F16 && c->dtype != PK_BF16 && c->dtype != PK_I8) return fail(PK_ERR_BAD_ARG, "cache dtype must be float16, bfloat16 or int8");
  if (c->batch > kMaxBatch) return fail(PK_ERR_BAD_ARG, "cache: at most %d sequences, got %d", kMaxBatch, c->batch);
  if (static_cast<int64_t>(c->width) * c->page_size >= (1 << 30)) return fail(PK_ERR_BAD_ARG, "cache: a sequence must stay below 2^30 rows");
  // `extend` sums the pages that all sequences want in 32 bits
  if (static_cast<int64_t>(c->batch) * c->width >= (1ll << 31)) return fail(PK_ERR_BAD_ARG, "cache: the table must have fewer than 2^31 entries");
  if (static_cast<int64_t>(c->layers) * c->pages >= (1ll << 31) - 1 || static_cast<int64_t>(c->layers) * c->kv_heads * c->batch >= (1ll << 31))
    return fail(PK_ERR_BAD_ARG, "cache: too many pages or heads");
  if (!c->keys || !c->values || !c->table || !c->lengths || !c->starts || !c->uses || !c->refused || !c->scratch) return fail(PK_ERR_BAD_ARG, "cache: null pointer");
  if (c->dtype == PK_I8 && (!c->key_scales || !c->value_scales)) return fail(PK_ERR_BAD_ARG, "an 8-bit cache needs key and value scales");
  if ((reinterpret_cast<uintptr_t>(c->keys) | reinterpret_cast<uintptr_t>(c->values)) & 15) return fail(PK_ERR_BAD_ARG, "cache: keys and values must be 16-byte aligned");
  if (c->dtype == PK_I8 && ((reinterpret_cast<uintptr_t>(c->key_scales) | reinterpret_cast<uintptr_t>(c->value_scales)) & 15))
    return fail(PK_ERR_BAD_ARG, "cache: scales must be 16-byte aligned");
  return PK_OK;
}

}  // namespace pk

using namespace pk;

extern "C" {

PK_API int pk_cache_extend(const pk_cache* c, const int32_t* counts) {
  PK_CACHE_ENTRY(c, p);
  if (!counts) return fail(PK_ERR_BAD_ARG, "cache extend: null counts");
  const int smem = (3 * p.batch + 1) * static_cast<int>(sizeof(int));
  // beside it the kernel has shared memory of fixed size, and the two must not pass 48 KB without leave
  if (smem > 40 * 1024 && (rc = allow_smem<extend_kernel>((3 * kMaxBatch + 1) * static_cast<int>(sizeof(int)), c->device))) return rc;
  if ((rc = launched(launch_chained(extend_kernel, dim3(1), dim3(kPlan), smem, st, p, counts), "extend"))) return rc;
  const int64_t items = static_cast<int64_t>(p.layers) * p.kv_heads * p.batch;
  const cudaError_t e = c->dtype == PK_I8 ? launch_chained(copy_tails_kernel<1>, dim3(copy_grid(items)), dim3(256), 0, st, p)
                                          : launch_chained(copy_tails_kernel<2>, dim3(copy_grid(items)), dim3(256), 0, st, p);
  return launched(e, "page copy");
}

PK_API int pk_cache_write(const pk_cache* c, int32_t layer, const void* key, const void* value, const int64_t key_stride[4],
                          const int64_t value_stride[4], int32_t dtype, int32_t tokens) {
  PK_CACHE_ENTRY(c, p);
  if (!key || !value || !key_stride || !value_stride) return fail(PK_ERR_BAD_ARG, "cache write: null pointer");
  if (layer < -1 || layer >= p.layers) return fail(PK_ERR_BAD_ARG, "cache write: layer %d of %d", layer, p.layers);
  if (tokens <= 0) return fail(PK_ERR_BAD_ARG, "cache write does not accept empty rows");
  if (dtype != PK_F16 && dtype != PK_BF16) return fail(PK_ERR_BAD_ARG, "cache write: rows must be float16 or bfloat16");
  if (c->dtype != PK_I8 && c->dtype != dtype) return fail(PK_ERR_BAD_ARG, "cache write: rows and cache must share a dtype");
  Source s{static_cast<const uint16_t*>(key), static_cast<const uint16_t*>(value), {}, {}, tokens, layer < 0 ? 0 : layer, layer < 0 ? p.layers : 1, 0};
  for (int i = 0; i < 4; ++i) s.ks[i] = key_stride[i], s.vs[i] = value_stride[i];
  if (layer >= 0) s.ks[0] = s.vs[0] = 0;
  s.vec = even_strides(key, s.ks) && even_strides(value, s.vs);
  cudaError_t e;
  if (dtype == PK_F16) e = c->dtype == PK_I8 ? launch_write<__half, true>(p, s, st) : launch_write<__half, false>(p, s, st);
  else e = c->dtype == PK_I8 ? launch_write<__nv_bfloat16, true>(p, s, st) : launch_write<__nv_bfloat16, false>(p, s, st);
  return launched(e, "cache write");
}

PK_API int pk_cache_read(const pk_cache* c, int32_t layer, const int32_t* first, int32_t count, void* key, void* value, int32_t dtype) {
  PK_CACHE_ENTRY(c, p);
  if (!first || !key || !value) return fail(PK_ERR_BAD_ARG, "cache read: null pointer");
  if (layer < -1 || layer >= p.layers) return fail(PK_ERR_BAD_ARG, "cache read: layer %d of %d", layer, p.layers);
  if (count <= 0) return fail(PK_ERR_BAD_ARG, "cache read does not accept an empty range");
  if (dtype != PK_F16 && dtype != PK_BF16 && dtype != PK_F32) return fail(PK_ERR_BAD_ARG, "cache read: output must be float16, bfloat16 or float32");
  if ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15) return fail(PK_ERR_BAD_ARG, "cache read: outputs must be 16-byte aligned");
  const int layer0 = layer < 0 ? 0 : layer, layers = layer < 0 ? p.layers : 1;
  cudaError_t e;
  if (c->dtype == PK_I8) e = launch_read<__half, true>(p, layer0, layers, first, count, key, value, dtype, st);
  else if (c->dtype == PK_F16) e = launch_read<__half, false>(p, layer0, layers, first, count, key, value, dtype, st);
  else e = launch_read<__nv_bfloat16, false>(p, layer0, layers, first, count, key, value, dtype, st);
  return launched(e, "cache read");
}

PK_API int pk_cache_fork(const pk_cache* c, const int32_t* parents) {
  PK_CACHE_ENTRY(c, p);
  if (!parents) return fail(PK_ERR_BAD_ARG, "cache fork: null parents");
  int columns = 8192 / p.batch;  // 32 KB of entries per CTA
  columns = columns < 1 ? 1 : columns > 32 ? 32 : columns;
  const size_t smem = static_cast<size_t>(p.batch) * columns * sizeof(int);
  return launched(launch_chained(fork_kernel, dim3((p.width + columns - 1) / columns), dim3(256), smem, st, p, parents, columns), "fork");
}

PK_API int pk_cache_truncate(const pk_cache* c, const int32_t* lengths) {
  PK_CACHE_ENTRY(c, p);
  if (!lengths) return fail(PK_ERR_BAD_ARG, "cache truncate: null lengths");
  return launched(launch_chained(truncate_kernel, dim3(p.batch), dim3(128), 0, st, p, lengths), "truncate");
}

PK_API int pk_cache_compact(const pk_cache* c, const int32_t* paths, int64_t path_stride, int32_t most, const int32_t* counts) {
  PK_CACHE_ENTRY(c, p);
  if (!paths || !counts) return fail(PK_ERR_BAD_ARG, "cache compact: null pointer");
  if (most <= 0) return fail(PK_ERR_BAD_ARG, "cache compact does not accept empty paths");
  const Paths paths_{paths, path_stride, counts, most};
  cudaError_t e;
  if (c->dtype == PK_I8) e = p.dim == 128 ? launch_move<128, true>(p, paths_, st) : launch_move<64, true>(p, paths_, st);
  else e = p.dim == 128 ? launch_move<256, false>(p, paths_, st) : launch_move<128, false>(p, paths_, st);
  if ((rc = launched(e, "row move"))) return rc;
  return launched(launch_chained(cut_paths_kernel, dim3(p.batch), dim3(128), 0, st, p, paths_), "cut");
}

}  // extern "C"
