// Wide-row attention (wide_rows.cuh) for bfloat16.
#include "wide_rows.cuh"

namespace pk {

int launch_wide_rows_bf16(const AttendParams& p, int head_dim, int device, cudaStream_t st) {
  return wide_by_dim<__nv_bfloat16>(p, head_dim, device, st);
}

}  // namespace pk
