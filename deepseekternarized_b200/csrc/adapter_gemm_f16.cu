// The low-rank adapters' kernels for f16 activations.
#include "adapter_gemm.cuh"

int dst::adapter_launch_f16(const AdapterCall& c, int rank_padded, int64_t max_tiles, cudaStream_t st) {
  return launch_for<__half>(c, rank_padded, max_tiles, st);
}
