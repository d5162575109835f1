// Chunk attention kernels for __half, head_dim 64.
#include "fst_chunk_body.cuh"
namespace fst {
cudaError_t launch_chunk_f16_d64(const ChunkArgs &a, int n_ctas, cudaStream_t stream) { return launch_chunk_t<__half, 64>(a, n_ctas, stream); }
}  // namespace fst
