// Wide-row attention (wide_rows.cuh) for float16.
#include "wide_rows.cuh"

namespace pk {

uint64_t wide_rows_workspace(int batch, int kv_heads, int rows, int head_dim) {
  const WidePlan plan = wide_plan(batch, kv_heads, rows, 1 << 30);  // as if there were keys enough to share any rest
  if (plan.whole == plan.units) return 0;
  return (plan.units * sizeof(Pieces) + 255) / 256 * 256 + static_cast<uint64_t>(kWideWorkers) * 2 * kWideRows * (head_dim + 4) * sizeof(float);
}

int launch_wide_rows_f16(const AttendParams& p, int head_dim, int device, cudaStream_t st) {
  return wide_by_dim<__half>(p, head_dim, device, st);
}

}  // namespace pk
