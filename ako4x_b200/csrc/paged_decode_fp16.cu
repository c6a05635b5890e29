// Paged decode: the kernels for fp16 queries.
#include "paged_decode.cuh"

int ako::paged::run_fp16(const Params& p, const Plan& pl, int64_t dim, bool fp8, cudaStream_t st) {
  return fp8 ? launch_dim<__half, true>(p, pl, dim, st) : launch_dim<__half, false>(p, pl, dim, st);
}
