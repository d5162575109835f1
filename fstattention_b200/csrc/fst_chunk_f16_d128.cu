// Chunk attention kernels for __half, head_dim 128.
#include "fst_chunk_body.cuh"
namespace fst {
cudaError_t launch_chunk_f16_d128(const ChunkArgs &a, int n_ctas, cudaStream_t stream) { return launch_chunk_t<__half, 128>(a, n_ctas, stream); }
}  // namespace fst
