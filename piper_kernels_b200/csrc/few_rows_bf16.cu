// Few-row attention (few_rows.cuh) for bfloat16 queries.
#include "few_rows.cuh"

namespace pk {

int launch_few_rows_bf16(const AttendParams& p, int head_dim, bool i8, int device, cudaStream_t st) {
  return i8 ? by_dim<__nv_bfloat16, true>(p, head_dim, device, st) : by_dim<__nv_bfloat16, false>(p, head_dim, device, st);
}

}  // namespace pk
