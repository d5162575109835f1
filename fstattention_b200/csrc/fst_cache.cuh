// A paged K/V cache as the kernels see it, and the arithmetic of its 8-bit form.
//
// A row x of one head is held as D e4m3 values and one exponent: with a = max |x_i|, e is the smallest integer in
// [-117, 119] with a <= 448 * 2^e, element i is e4m3(x_i * 2^-e) and the row stands for e4m3 * 2^e.  A power of two
// costs a floating-point format no precision (only one binade of its range, which starts 2^-16 below the row's largest
// value), and it makes both directions exact but for the one rounding to e4m3: x_i * 2^-e is exact in fp32, and so is
// e4m3 * 2^e in bf16 and fp32.  The bounds of e keep every product a normal fp32 number.  A row with an element that is not
// finite is held as zeros with the scale NaN, so that the kernels need not look for NaN among the bytes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fst_common.cuh"

namespace fst {

struct CacheArgs {
    void *k_pool, *v_pool;
    uint8_t *k_scale, *v_scale;            // [n_pages][H_kv][page_size] biased exponents (e8m0), null: rows in 16 bits
    const int32_t *table;                  // [Z][width] page numbers
    int width, page_shift, n_pages;
    int64_t stride_page, stride_row, stride_head;
};

// These kernels become resident while the launch ahead of them still writes their tables, lengths and rows, and wait for it before their first
// access: loads for data that is read-only for a kernel's whole life (__ldg) would not have to see that.
template <typename T>
__device__ __forceinline__ T load(const T *p) {
    __builtin_assume(__isGlobal(p));
    return *p;
}

// e of a row whose largest magnitude is a (finite)
__device__ __forceinline__ int e4m3_exponent(float a) {
    const uint32_t bits = __float_as_uint(a);
    const int e = int(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);   // 448 = 1.75 * 2^8
    return min(max(e, -117), 119);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
// 2^(b - 127) of the two bytes of b, NaN for 255; exact in bf16 and fp32, also for b = 0, where it is not a normal number (a comparison for
// that byte took the kernels of 9 to 32 rows 5 to 10 % of their time, the instruction takes none)
__device__ __forceinline__ float2 e8m0_values(uint32_t b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;\n" : "=r"(r) : "h"(uint16_t(b)));
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}
__device__ __forceinline__ float e8m0_value(uint32_t b) { return e8m0_values(b).x; }

// two e4m3 values of two fp32 ones (saturating, nearest even)
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// the two values of the low 16 bits
__device__ __forceinline__ float2 e4m3_values(uint32_t pair) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(uint16_t(pair)));
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
// rounded to T; fp16 saturates (a row of fp16 values may round past 65504: 448 * 2^7 < 65504 < 256 * 2^8)
template <typename T>
__device__ __forceinline__ uint32_t pack_cache(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack_cache<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_cache<__half>(float x, float y) {
    x = x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;      // (a NaN stays one)
    y = y > 65504.f ? 65504.f : y < -65504.f ? -65504.f : y;
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

struct AppendArgs {
    CacheArgs c;
    const void *k, *v;                     // [Z][H_kv][N][D]
    int64_t ks_z, ks_h, ks_n, vs_z, vs_h, vs_n;
    const int32_t *start, *lens, *rows;    // [Z], [Z] or null, [Z][M] or null
    int Z, H_kv, N, M;
    int32_t *status;
};
struct ReadArgs {
    CacheArgs c;
    void *k, *v;                           // [Z][H_kv][M][D]
    int64_t ks_z, ks_h, ks_n, vs_z, vs_h, vs_n;
    const int32_t *lens;
    int Z, H_kv, M;
    int32_t *status;
};
// An 8-bit cache as a 16-bit one of the same pages' rows: page i of sequence z is page z * width + i of the pools k, v, contiguous
// [Z * width][H_kv][page_size][D], as table says, [Z][width].  Only pages with rows are written.
struct ExpandArgs {
    CacheArgs c;
    void *k, *v;
    int32_t *table;
    const int32_t *lens, *q_lens;          // [Z], [Z] or null: a sequence without queries has no rows
    int Z, H_kv;
    int32_t *status;
};
cudaError_t launch_cache_expand(const ExpandArgs &a, int dtype, int D, cudaStream_t stream);
cudaError_t launch_cache_append(const AppendArgs &a, int dtype, int D, cudaStream_t stream);
cudaError_t launch_cache_read(const ReadArgs &a, int dtype, int D, cudaStream_t stream);

}  // namespace fst
