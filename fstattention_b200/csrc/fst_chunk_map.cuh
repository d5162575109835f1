// Tensor maps over a page pool for the chunk kernels, encoded by every call: a table of them by address, as make_map has, gained nothing that
// could be measured (5.3 us of host time for a small call either way).
#pragma once

#include "fst_attention_tma.cuh"
#include "fst_cache.cuh"

namespace fst {

enum PoolType { POOL_F16 = 0, POOL_BF16 = 1, POOL_E4M3 = 2 };

struct PoolKey {
    const void *base;
    int64_t stride_page, stride_row, stride_head;
    int32_t type, D, page, H, n_pages, box_rows, box_heads;
};

// Rank 4: columns, rows of a page, K/V heads, pages; boxes of 64 columns of 16 bits, or a whole row of e4m3, by box_rows rows by
// box_heads heads.
// 128 bytes of a row are swizzled over 128 bytes, the 64 bytes of an e4m3 row at D 64 over 64.
inline bool make_pool_map(CUtensorMap *map, const PoolKey &key) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return false;
    const bool bytes = key.type == POOL_E4M3;
    const cuuint64_t size = bytes ? 1 : 2;
    const cuuint64_t dims[4] = {cuuint64_t(key.D), cuuint64_t(key.page), cuuint64_t(key.H), cuuint64_t(key.n_pages)};
    const cuuint64_t strides[3] = {cuuint64_t(key.stride_row) * size, cuuint64_t(key.stride_head) * size, cuuint64_t(key.stride_page) * size};
    const cuuint32_t box[4] = {cuuint32_t(bytes ? key.D : 64), cuuint32_t(key.box_rows), cuuint32_t(key.box_heads), 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                           : key.type == POOL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    // What L2 is asked to bring along: a row (it is the neighbouring head's that lies next to it, and nobody needs that soon), or as much as
    // goes where a head's rows lie together.  (Two sequences of 115000 e4m3 rows, heads inside rows: 100 us with 256 bytes, 87 with 128.)
    const int64_t row_bytes = key.stride_row == key.D ? 256 : int64_t(key.D * size);
    const CUtensorMapL2promotion along = row_bytes >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                                         : row_bytes >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
    return fn(map, type, 4, const_cast<void *>(key.base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              bytes && key.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, along,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// K's and V's maps of a cache (e4m3 where it has scales, else 16 bits as `bf16` says)
inline bool make_pool_maps(CUtensorMap *tk, CUtensorMap *tv, const CacheArgs &c, bool bf16, int D, int H_kv, int box_rows) {
    PoolKey key{c.k_pool, c.stride_page, c.stride_row, c.stride_head, c.k_scale != nullptr ? POOL_E4M3 : bf16 ? POOL_BF16 : POOL_F16,
                D, 1 << c.page_shift, H_kv, c.n_pages, box_rows, 1};
    if (!make_pool_map(tk, key)) return false;
    key.base = c.v_pool;
    return make_pool_map(tv, key);
}

}  // namespace fst
