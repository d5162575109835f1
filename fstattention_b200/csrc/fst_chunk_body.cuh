// Dispatch of a chunk attention call for one type and head dimension (the .cu files instantiate it).
#pragma once

#include "fst_chunk_mma.cuh"
#include "fst_chunk_token.cuh"
#include "fst_chunk_umma.cuh"

namespace fst {

template <typename T, int D>
cudaError_t launch_chunk_t(const ChunkArgs &a, int n_ctas, cudaStream_t stream) {
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    alignas(64) CUtensorMap tk, tv;
    if (chunk_many_rows(a)) {
        if (!make_pool_maps(&tk, &tv, a.c, bf16, D, a.H_kv, 1 << a.c.page_shift)) return cudaErrorNotSupported;
        ChunkArgs b = a;
        alignas(64) CUtensorMap tq = tk;
        b.q_boxes = 128 % a.group == 0 && a.qs_z > 0 && a.qs_h > 0 && a.qs_n > 0;       // (broadcast queries: by plain loads)
        if (b.q_boxes && !make_pool_map(&tq, PoolKey{a.q, a.qs_z, a.qs_h, a.qs_n, bf16 ? POOL_BF16 : POOL_F16, D, a.H, a.n_q, a.Z, a.group, 128 / a.group}))
            return cudaErrorNotSupported;
        return a.c.k_scale != nullptr ? launch_chunk_umma<T, D, true>(b, tq, tk, tv, n_ctas, stream) : launch_chunk_umma<T, D, false>(b, tq, tk, tv, n_ctas, stream);
    }
    if (!make_pool_maps(&tk, &tv, a.c, bf16, D, a.H_kv, 1 << a.c.page_shift)) return cudaErrorNotSupported;
    if (chunk_row_tile(a) == 8)
        return a.c.k_scale != nullptr ? launch_chunk_token<T, D, true>(a, tk, tv, n_ctas, stream) : launch_chunk_token<T, D, false>(a, tk, tv, n_ctas, stream);
    const bool one = chunk_row_tile(a) == 16;
    if (a.c.k_scale != nullptr)
        return one ? launch_chunk_mma<T, D, true, 1>(a, tk, tv, n_ctas, stream) : launch_chunk_mma<T, D, true, 2>(a, tk, tv, n_ctas, stream);
    return one ? launch_chunk_mma<T, D, false, 1>(a, tk, tv, n_ctas, stream) : launch_chunk_mma<T, D, false, 2>(a, tk, tv, n_ctas, stream);
}

}  // namespace fst
