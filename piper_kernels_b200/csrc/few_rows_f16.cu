// Few-row attention (few_rows.cuh) for float16 queries.
#include "few_rows.cuh"

namespace pk {

uint64_t few_rows_workspace(int batch, int kv_heads, int rows, int head_dim) {
  const int64_t block = rows <= 16 ? 16 : rows <= 32 ? 32 : 64, units = static_cast<int64_t>(batch) * kv_heads * ((rows + block - 1) / block);
  return (units * sizeof(Pieces) + 255) / 256 * 256 + static_cast<uint64_t>(kMaxWorkers) * 2 * block * (head_dim + 4) * sizeof(float);
}

int launch_few_rows_f16(const AttendParams& p, int head_dim, bool i8, int device, cudaStream_t st) {
  return i8 ? by_dim<__half, true>(p, head_dim, device, st) : by_dim<__half, false>(p, head_dim, device, st);
}

}  // namespace pk
