// C entry points of the 16-bit attention operators: argument checks, and the choice of kernel.

#include <math.h>
#include <string.h>

#include "pk_attend.cuh"

namespace pk {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

int encode_map5(CUtensorMap* m, const void* base, const uint64_t dims[5], const uint64_t strides[4], const uint32_t box[5], int line, int esz) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(PK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], e[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < 5; ++i) d[i] = dims[i], b[i] = box[i];
  for (int i = 0; i < 4; ++i) s[i] = strides[i];
  const CUresult r = fn(m, esz == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, const_cast<void*>(base), d, s, b, e,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, line == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(PK_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
  return PK_OK;
}

int attend_map(CUtensorMap* m, const AttendParams& p, const void* base, const int64_t* stride, int line, int lines, int esz, int box, int box_lines) {
  const uint64_t row = static_cast<uint64_t>(line) * lines;  // bytes
  const uint32_t boxes[5] = {static_cast<uint32_t>(line / esz), static_cast<uint32_t>(box), static_cast<uint32_t>(box_lines), 1, 1};
  if (p.table) {
    // the whole pool, so that a page index outside it reads as zeros
    const uint64_t page = row * p.page;
    const uint64_t dims[5] = {static_cast<uint64_t>(line / esz), static_cast<uint64_t>(p.page), static_cast<uint64_t>(lines),
                              static_cast<uint64_t>(p.kv_heads), static_cast<uint64_t>(p.pool_pages)};
    const uint64_t strides[4] = {row, static_cast<uint64_t>(line), page, page * p.kv_heads};
    return encode_map5(m, base, dims, strides, boxes, line, esz);
  }
  // a broadcast (stride 0) axis is an axis of one
  const uint64_t dims[5] = {static_cast<uint64_t>(line / esz), static_cast<uint64_t>(p.kv_len), static_cast<uint64_t>(lines),
                            stride[1] ? static_cast<uint64_t>(p.kv_heads) : 1, stride[0] ? static_cast<uint64_t>(p.batch) : 1};
  const uint64_t strides[4] = {stride[2] ? static_cast<uint64_t>(stride[2]) * esz : row, static_cast<uint64_t>(line),
                               stride[1] ? static_cast<uint64_t>(stride[1]) * esz : row, stride[0] ? static_cast<uint64_t>(stride[0]) * esz : row};
  return encode_map5(m, base, dims, strides, boxes, line, esz);
}

int attend_maps(CUtensorMap* k, CUtensorMap* v, const AttendParams& p, int which, int row_bytes, int esz, int tile, bool whole_rows) {
  if (p.maps) {
    *k = p.maps[2 * which], *v = p.maps[2 * which + 1];
    return PK_OK;
  }
  const int line = row_bytes > 128 ? 128 : row_bytes, lines = row_bytes / line, box = p.table && p.page < tile ? p.page : tile;
  const int rc = attend_map(k, p, p.k, p.k_stride, line, lines, esz, box, whole_rows ? lines : 1);
  return rc ? rc : attend_map(v, p, p.v, p.v_stride, line, lines, esz, box, whole_rows ? lines : 1);
}

namespace {

// Rows of a tensor that no copy map can describe (odd strides or an odd address), made contiguous.
template <int D>
__global__ void __launch_bounds__(256) pack_rows_kernel(const uint16_t* src, int64_t sb, int64_t sh, int64_t sr, uint16_t* dst, int heads, int len, int64_t rows) {
  cudaGridDependencySynchronize();
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = at / (D / 8);
  if (row >= rows) return;
  const int d = static_cast<int>(at % (D / 8)) * 8;
  const int64_t r = row % len, h = row / len % heads, b = row / len / heads;
  const uint16_t* s = src + b * sb + h * sh + r * sr + d;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = s[i];
  *reinterpret_cast<uint4*>(dst + row * D + d) = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
}

// Whether a copy map can describe a [batch, heads, sequence, D] tensor of 16-bit values.
bool mappable(const void* base, const int64_t* stride, const int64_t* dims) {
  if (reinterpret_cast<uintptr_t>(base) & 15) return false;
  for (int i = 0; i < 3; ++i) {
    if (dims[i] == 1) continue;
    if (stride[i] & 7 || stride[i] < 0 || stride[i] >= (1ll << 38)) return false;
    if (i == 2 && stride[i] == 0) return false;
  }
  return true;
}
size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// Which kernel: the few-row one reads K and V at the speed of memory for up to 64 rows of a key head; more
// rows are worth the tensor cores' larger tiles.  8-bit caches have the few-row kernel only.
bool wide(int rows, bool i8) { return !i8 && rows > 64; }

uint64_t attend_workspace(int batch, int kv_heads, int rows, int head_dim, bool i8) {
  const uint64_t n = wide(rows, i8) ? wide_rows_workspace(batch, kv_heads, rows, head_dim) : few_rows_workspace(batch, kv_heads, rows, head_dim);
  return n ? n : 256;
}

int attend(const AttendParams& a, int head_dim, int dtype, bool i8, int device, cudaStream_t st) {
  if (wide(a.rows, i8)) return dtype == PK_F16 ? launch_wide_rows_f16(a, head_dim, device, st) : launch_wide_rows_bf16(a, head_dim, device, st);
  return dtype == PK_F16 ? launch_few_rows_f16(a, head_dim, i8, device, st) : launch_few_rows_bf16(a, head_dim, i8, device, st);
}

struct DenseLayout {
  size_t k, v, work, total;
  bool pack_k, pack_v;
};

DenseLayout dense_layout(const pk_window_problem& p) {
  DenseLayout l{};
  const int64_t dims[3] = {p.batch, p.kv_heads, p.kv_len};
  const size_t bytes = static_cast<size_t>(p.batch) * p.kv_heads * p.kv_len * p.head_dim * 2;
  l.pack_k = !mappable(p.k, p.k_stride, dims);
  l.pack_v = !mappable(p.v, p.v_stride, dims);
  size_t off = 0;
  l.k = off;
  if (l.pack_k) off += align256(bytes);
  l.v = off;
  if (l.pack_v) off += align256(bytes);
  l.work = off;
  off += attend_workspace(p.batch, p.kv_heads, p.heads / p.kv_heads * p.q_len, p.head_dim, false);
  l.total = off;
  return l;
}

int validate_window(const pk_window_problem* p, bool launching) {
  if (!p) return fail(PK_ERR_BAD_ARG, "window_attention: null problem");
  if (p->batch <= 0 || p->heads <= 0 || p->kv_heads <= 0) return fail(PK_ERR_BAD_ARG, "window_attention: batch and heads must be positive");
  if (p->heads % p->kv_heads) return fail(PK_ERR_BAD_ARG, "window_attention: heads must be a multiple of kv_heads, got %d/%d", p->heads, p->kv_heads);
  if (p->q_len <= 0 || p->kv_len <= 0) return fail(PK_ERR_BAD_ARG, "window_attention does not accept empty query or key sequences");
  if (p->head_dim != 64 && p->head_dim != 128) return fail(PK_ERR_BAD_ARG, "window_attention supports head dimensions 64 and 128, got %d", p->head_dim);
  if (p->dtype != PK_F16 && p->dtype != PK_BF16) return fail(PK_ERR_BAD_ARG, "window_attention inputs must be float16 or bfloat16");
  if (p->window < 1) return fail(PK_ERR_BAD_ARG, "window_attention: window must be at least 1, got %d", p->window);
  if (p->sinks < 0) return fail(PK_ERR_BAD_ARG, "window_attention: sinks must not be negative, got %d", p->sinks);
  if (!(p->scale > 0.f) || !isfinite(p->scale)) return fail(PK_ERR_BAD_ARG, "window_attention: scale must be finite and positive");
  if (static_cast<int64_t>(p->q_len) + p->kv_len >= (1 << 30)) return fail(PK_ERR_BAD_ARG, "window_attention: sequences must stay below 2^30 rows together");
  if (static_cast<int64_t>(p->heads / p->kv_heads) * p->q_len >= (1 << 30) ||
      static_cast<int64_t>(p->batch) * p->heads * ((p->q_len + 15) / 16) >= (1ll << 31))
    return fail(PK_ERR_BAD_ARG, "window_attention: too many query rows for one call; split it over the batch");
  if (!p->q || !p->k || !p->v) return fail(PK_ERR_BAD_ARG, "window_attention: null input pointer");
  if (launching) {
    if (!p->out || (reinterpret_cast<uintptr_t>(p->out) & 15)) return fail(PK_ERR_BAD_ARG, "window_attention: output must be a 16-byte aligned device pointer");
    if (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255))
      return fail(PK_ERR_WORKSPACE, "window_attention: workspace must be a 256-byte aligned device pointer");
    const size_t need = dense_layout(*p).total;
    if (p->workspace_bytes < need)
      return fail(PK_ERR_WORKSPACE, "window_attention: workspace too small: %llu bytes given, %llu needed",
                  static_cast<unsigned long long>(p->workspace_bytes), static_cast<unsigned long long>(need));
  }
  return PK_OK;
}

bool rows_aligned(const void* base, const int64_t* stride, const int64_t* dims) {
  if (reinterpret_cast<uintptr_t>(base) & 15) return false;
  for (int i = 0; i < 3; ++i)
    if (dims[i] > 1 && (stride[i] & 7)) return false;
  return true;
}

int pack(const pk_window_problem& p, const void* src, const int64_t* stride, void* dst, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.batch) * p.kv_heads * p.kv_len, threads = rows * (p.head_dim / 8);
  const unsigned blocks = static_cast<unsigned>((threads + 255) / 256);
  cudaError_t e;
  if (p.head_dim == 128)
    e = launch_chained(pack_rows_kernel<128>, dim3(blocks), dim3(256), 0, st, static_cast<const uint16_t*>(src), stride[0], stride[1], stride[2],
                       static_cast<uint16_t*>(dst), p.kv_heads, p.kv_len, rows);
  else
    e = launch_chained(pack_rows_kernel<64>, dim3(blocks), dim3(256), 0, st, static_cast<const uint16_t*>(src), stride[0], stride[1], stride[2],
                       static_cast<uint16_t*>(dst), p.kv_heads, p.kv_len, rows);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? PK_OK : fail(PK_ERR_CUDA, "row packing launch failed: %s", cuda_err(e));
}

int validate_query(const pk_cache* c, const pk_cache_query* q, bool launching) {
  int rc = validate_cache(c);
  if (rc) return rc;
  if (!q) return fail(PK_ERR_BAD_ARG, "cache_attention: null query");
  if (q->heads <= 0 || q->heads % c->kv_heads) return fail(PK_ERR_BAD_ARG, "cache_attention: heads must be a multiple of kv_heads, got %d/%d", q->heads, c->kv_heads);
  if (q->tokens <= 0) return fail(PK_ERR_BAD_ARG, "cache_attention does not accept empty queries");
  if (q->tree && q->tokens > kMaxTreeTokens) return fail(PK_ERR_BAD_ARG, "cache_attention: a tree has at most %d tokens, got %d", kMaxTreeTokens, q->tokens);
  if (q->layer < 0 || q->layer >= c->layers) return fail(PK_ERR_BAD_ARG, "cache_attention: layer %d of %d", q->layer, c->layers);
  if (q->dtype != PK_F16 && q->dtype != PK_BF16) return fail(PK_ERR_BAD_ARG, "cache_attention queries must be float16 or bfloat16");
  if (c->dtype != PK_I8 && c->dtype != q->dtype) return fail(PK_ERR_BAD_ARG, "cache_attention: query and cache must share a dtype");
  if (q->window < 0) return fail(PK_ERR_BAD_ARG, "cache_attention: window must not be negative, got %d", q->window);
  if (q->sinks < 0) return fail(PK_ERR_BAD_ARG, "cache_attention: sinks must not be negative, got %d", q->sinks);
  if (!(q->scale > 0.f) || !isfinite(q->scale)) return fail(PK_ERR_BAD_ARG, "cache_attention: scale must be finite and positive");
  if (static_cast<int64_t>(q->heads / c->kv_heads) * q->tokens >= (1 << 30) || static_cast<int64_t>(c->batch) * q->heads * ((q->tokens + 15) / 16) >= (1ll << 31))
    return fail(PK_ERR_BAD_ARG, "cache_attention: too many query rows for one call");
  if (!q->q) return fail(PK_ERR_BAD_ARG, "cache_attention: null query pointer");
  if (launching) {
    if (!q->out || (reinterpret_cast<uintptr_t>(q->out) & 15)) return fail(PK_ERR_BAD_ARG, "cache_attention: output must be a 16-byte aligned device pointer");
    if (!q->workspace || (reinterpret_cast<uintptr_t>(q->workspace) & 255))
      return fail(PK_ERR_WORKSPACE, "cache_attention: workspace must be a 256-byte aligned device pointer");
    const uint64_t need = attend_workspace(c->batch, c->kv_heads, q->heads / c->kv_heads * q->tokens, c->head_dim, c->dtype == PK_I8);
    if (q->workspace_bytes < need)
      return fail(PK_ERR_WORKSPACE, "cache_attention: workspace too small: %llu bytes given, %llu needed",
                  static_cast<unsigned long long>(q->workspace_bytes), static_cast<unsigned long long>(need));
  }
  return PK_OK;
}

struct Drill {  // the stalled-wait drill: see pk_debug_window_stall
  int64_t wait_cycles = 4 * kWaitCycleLimit;  // some seconds
  int skip_copy = -1;
};

int window_fwd(const pk_window_problem* pp, const Drill& drill) {
  int rc = validate_window(pp, true);
  if (rc) return rc;
  const pk_window_problem& p = *pp;
  const DeviceGuard g(p.device);
  if (g.err != cudaSuccess) return fail(PK_ERR_CUDA, "cudaSetDevice(%d): %s", p.device, cuda_err(g.err));
  if ((rc = check_arch(p.device))) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(p.stream);
  const DenseLayout l = dense_layout(p);
  char* ws = static_cast<char*>(p.workspace);
  AttendParams a{};
  a.wait_cycles = drill.wait_cycles, a.skip_copy = drill.skip_copy;
  a.q = p.q;
  a.out = p.out;
  a.batch = p.batch, a.heads = p.heads, a.kv_heads = p.kv_heads, a.group = p.heads / p.kv_heads, a.tokens = p.q_len;
  a.rows = a.group * a.tokens;
  a.group_inv = ~0ull / a.group + 1;  // not used for groups of one
  a.lengths = p.lengths;
  a.kv_len = p.kv_len, a.offset = p.kv_len - p.q_len;
  a.k = p.k, a.v = p.v;
  const int64_t packed[3] = {static_cast<int64_t>(p.kv_heads) * p.kv_len * p.head_dim, static_cast<int64_t>(p.kv_len) * p.head_dim, p.head_dim};
  memcpy(a.q_stride, p.q_stride, sizeof(a.q_stride));
  memcpy(a.k_stride, p.k_stride, sizeof(a.k_stride));
  memcpy(a.v_stride, p.v_stride, sizeof(a.v_stride));
  if (l.pack_k) {
    if ((rc = pack(p, p.k, p.k_stride, ws + l.k, st))) return rc;
    a.k = ws + l.k;
    memcpy(a.k_stride, packed, sizeof(packed));
  }
  if (l.pack_v) {
    if ((rc = pack(p, p.v, p.v_stride, ws + l.v, st))) return rc;
    a.v = ws + l.v;
    memcpy(a.v_stride, packed, sizeof(packed));
  }
  // the stride of an axis of one says nothing
  const int64_t dims[3] = {p.batch, p.kv_heads, p.kv_len};
  for (int i = 0; i < 2; ++i) {
    if (dims[i] == 1) a.k_stride[i] = a.v_stride[i] = 0;
  }
  if (p.kv_len == 1) a.k_stride[2] = a.v_stride[2] = 0;
  const int64_t qdims[3] = {p.batch, p.heads, p.q_len};
  a.q_vec = rows_aligned(p.q, p.q_stride, qdims);
  a.window = p.window < kNoWindow ? p.window : kNoWindow;
  a.sinks = p.sinks;
  a.scale_log2 = p.scale * kLog2e;
  a.partial = reinterpret_cast<float*>(ws + l.work);
  a.host_status = fault_word_device_ptr(p.device);
  return attend(a, p.head_dim, p.dtype, false, p.device, st);
}

int cache_fwd(const pk_cache* c, const pk_cache_query* q, const Drill& drill) {
  int rc = validate_query(c, q, true);
  if (rc) return rc;
  const DeviceGuard g(c->device);
  if (g.err != cudaSuccess) return fail(PK_ERR_CUDA, "cudaSetDevice(%d): %s", c->device, cuda_err(g.err));
  if ((rc = check_arch(c->device))) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(c->stream);
  const bool i8 = c->dtype == PK_I8;
  AttendParams a{};
  a.wait_cycles = drill.wait_cycles, a.skip_copy = drill.skip_copy;
  a.q = q->q;
  memcpy(a.q_stride, q->q_stride, sizeof(a.q_stride));
  const int64_t qdims[3] = {c->batch, q->heads, q->tokens};
  a.q_vec = rows_aligned(q->q, q->q_stride, qdims);
  a.out = q->out;
  a.batch = c->batch, a.heads = q->heads, a.kv_heads = c->kv_heads, a.group = q->heads / c->kv_heads, a.tokens = q->tokens;
  a.rows = a.group * a.tokens;
  a.group_inv = ~0ull / a.group + 1;  // not used for groups of one
  a.lengths = c->lengths, a.starts = c->starts;
  a.table = c->table, a.width = c->width, a.page = c->page_size, a.pages = c->pages, a.page_base = q->layer * c->pages;
  a.page_shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
  a.pool_pages = c->layers * c->pages;
  a.maps = static_cast<const CUtensorMap*>(c->maps);
  a.k = c->keys, a.v = c->values;
  const int64_t layer_rows = static_cast<int64_t>(c->pages) * c->kv_heads * c->page_size * q->layer;
  if (i8) a.k_scale = c->key_scales + layer_rows, a.v_scale = c->value_scales + layer_rows;
  a.tree = q->tree, a.tree_stride = q->tree_stride;
  a.window = q->window > 0 && q->window < kNoWindow ? q->window : kNoWindow;
  a.sinks = q->sinks;
  a.scale_log2 = q->scale * kLog2e;
  a.partial = static_cast<float*>(q->workspace);
  a.host_status = fault_word_device_ptr(c->device);
  return attend(a, c->head_dim, q->dtype, i8, c->device, st);
}

int check_drill(int64_t wait_cycles, int32_t copy) {
  if (wait_cycles <= 0 || wait_cycles > kWaitCycleLimit) return fail(PK_ERR_BAD_ARG, "stall: wait_cycles must be in [1, %lld], got %lld", kWaitCycleLimit, static_cast<long long>(wait_cycles));
  if (copy < -1) return fail(PK_ERR_BAD_ARG, "stall: copy must be -1 or more, got %d", copy);
  return PK_OK;
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" {

PK_API int pk_window_workspace_bytes(const pk_window_problem* p, uint64_t* bytes) {
  clear_error();
  if (!bytes) return fail(PK_ERR_BAD_ARG, "null size pointer");
  const int rc = validate_window(p, false);
  if (rc) return rc;
  *bytes = dense_layout(*p).total;
  return PK_OK;
}

PK_API int pk_window_attention_fwd(const pk_window_problem* p) {
  clear_error();
  return window_fwd(p, Drill{});
}

PK_API int pk_debug_window_stall(const pk_window_problem* p, int64_t wait_cycles, int32_t copy) {
  clear_error();
  const int rc = check_drill(wait_cycles, copy);
  return rc ? rc : window_fwd(p, Drill{wait_cycles, copy});
}

PK_API int pk_cache_maps(const pk_cache* c, void* maps) {
  clear_error();
  int rc = validate_cache(c);
  if (rc) return rc;
  if (!maps || (reinterpret_cast<uintptr_t>(maps) & 63)) return fail(PK_ERR_BAD_ARG, "cache maps: the maps need host memory aligned to 64 bytes");
  static_assert(6 * sizeof(CUtensorMap) == PK_CACHE_MAP_BYTES, "three pairs of maps");
  AttendParams a{};
  a.table = c->table, a.page = c->page_size, a.kv_heads = c->kv_heads, a.pool_pages = c->layers * c->pages;
  a.k = c->keys, a.v = c->values;
  const int esz = c->dtype == PK_I8 ? 1 : 2;
  CUtensorMap* m = static_cast<CUtensorMap*>(maps);
  if ((rc = attend_maps(m, m + 1, a, 0, c->head_dim * esz, esz, 64, true))) return rc;
  if ((rc = attend_maps(m + 2, m + 3, a, 1, c->head_dim * esz, esz, 128, true))) return rc;
  if (esz == 1) return PK_OK;  // 8-bit rows have no kernel for many rows
  return attend_maps(m + 4, m + 5, a, 2, c->head_dim * esz, esz, 128, false);
}

PK_API int pk_cache_attention_workspace_bytes(const pk_cache* c, const pk_cache_query* q, uint64_t* bytes) {
  clear_error();
  if (!bytes) return fail(PK_ERR_BAD_ARG, "null size pointer");
  const int rc = validate_query(c, q, false);
  if (rc) return rc;
  *bytes = attend_workspace(c->batch, c->kv_heads, q->heads / c->kv_heads * q->tokens, c->head_dim, c->dtype == PK_I8);
  return PK_OK;
}

PK_API int pk_cache_attention_fwd(const pk_cache* c, const pk_cache_query* q) {
  clear_error();
  return cache_fwd(c, q, Drill{});
}

PK_API int pk_debug_cache_stall(const pk_cache* c, const pk_cache_query* q, int64_t wait_cycles, int32_t copy) {
  clear_error();
  const int rc = check_drill(wait_cycles, copy);
  return rc ? rc : cache_fwd(c, q, Drill{wait_cycles, copy});
}

}  // extern "C"
