// Rows into and out of a paged K/V cache (fst_cache_append, fst_cache_read).
//
// Both move each row of a head once and compute next to nothing: HBM bounds the large calls, the launch and a chain of
// three memory latencies (length, page number, row) the small ones.  A row of D 16-bit values is D / 8 lanes of 16 bytes, K and V by
// the same lanes, so that a warp moves 512 bytes of either at a time and the lookups serve both.
#include <type_traits>

#include "fst_cache.cuh"

namespace fst {

constexpr int CACHE_THREADS = 256;

template <typename T>
__device__ __forceinline__ float2 two_floats(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}

// Eight values of a row that D / 8 neighbouring lanes hold: the row's largest magnitude is taken over them.
template <typename T, int D>
__device__ __forceinline__ uint2 quantise8(uint4 in, uint32_t &biased) {
    const uint32_t w[4] = {in.x, in.y, in.z, in.w};
    float x[8], a = 0.f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = two_floats<T>(w[i]);
        x[2 * i] = p.x;
        x[2 * i + 1] = p.y;
        a = fmaxf(a, fmaxf(fabsf(p.x), fabsf(p.y)));
        finite = finite && !isnan(p.x) && !isnan(p.y);    // (a maximum passes over them)
    }
    if (!finite) a = INFINITY;
#pragma unroll
    for (int s = 1; s < D / 8; s *= 2) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, s));
    if (a == INFINITY) {
        biased = 255u;
        return make_uint2(0u, 0u);
    }
    const int e = e4m3_exponent(a);
    const float f = pow2f(-e);
    biased = uint32_t(e + 127);
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = e4m3_pair(x[2 * i] * f, x[2 * i + 1] * f);
    return make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
}

template <typename T, int D, bool QUANT>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_append_kernel(const AppendArgs a) {
    constexpr int LPR = D / 8, RPB = CACHE_THREADS / LPR;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    // unit: row j of head h of sequence z, j fastest (neighbouring rows of the source, and of a page)
    const unsigned unit = blockIdx.x * RPB + threadIdx.x / LPR, col = (threadIdx.x % LPR) * 8;
    const unsigned zh = unit / unsigned(a.M), j = unit - zh * unsigned(a.M), z = zh / unsigned(a.H_kv), h = zh - z * unsigned(a.H_kv);
    bool live = z < unsigned(a.Z);
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    int64_t pos = 0;
    if (live) {
        int row = a.rows != nullptr ? __ldg(a.rows + size_t(z) * a.M + j) : int(j);
        const int count = a.lens != nullptr ? __ldg(a.lens + z) : a.M;
        pos = int64_t(__ldg(a.start + z)) + j;
        live = int(j) < count;
        if (live && (row < 0 || row >= a.N || pos < 0 || (pos >> a.c.page_shift) >= a.c.width)) {
            if (col == 0) report(a.status, FST_DEV_INDEX_RANGE, int(z), int(j));
            live = false;
        }
        if (live) {
            k = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.k) + z * a.ks_z + h * a.ks_h + row * a.ks_n + col));
            v = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.v) + z * a.vs_z + h * a.vs_h + row * a.vs_n + col));
        }
    }
    int page = 0;
    if (live) {
        page = __ldg(a.c.table + size_t(z) * a.c.width + (pos >> a.c.page_shift));
        if (unsigned(page) >= unsigned(a.c.n_pages)) {
            if (col == 0) report(a.status, FST_DEV_INDEX_RANGE, int(z), int(j));
            live = false;
        }
    }
    const int off = int(pos) & ((1 << a.c.page_shift) - 1);
    const int64_t to = page * a.c.stride_page + off * a.c.stride_row + h * a.c.stride_head + col;
    if constexpr (QUANT) {
        uint32_t ek, ev;                                  // (all lanes take part in the maximum)
        const uint2 qk = quantise8<T, D>(k, ek), qv = quantise8<T, D>(v, ev);
        if (!live) return;
        *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(a.c.k_pool) + to) = qk;
        *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(a.c.v_pool) + to) = qv;
        if (col == 0) {
            const size_t at = ((size_t(page) * a.H_kv + h) << a.c.page_shift) + off;
            a.c.k_scale[at] = uint8_t(ek);
            a.c.v_scale[at] = uint8_t(ev);
        }
    } else if (live) {
        *reinterpret_cast<uint4 *>(static_cast<T *>(a.c.k_pool) + to) = k;
        *reinterpret_cast<uint4 *>(static_cast<T *>(a.c.v_pool) + to) = v;
    }
}

// eight values of a quantised row
template <typename T>
__device__ __forceinline__ uint4 expand8(uint2 b, float scale) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = e4m3_values((i < 2 ? b.x : b.y) >> (i & 1) * 16);
        r[i] = pack_cache<T>(x.x * scale, x.y * scale);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

template <typename T, int D, bool QUANT>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_read_kernel(const ReadArgs a) {
    constexpr int LPR = D / 8, RPB = CACHE_THREADS / LPR;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const unsigned unit = blockIdx.x * RPB + threadIdx.x / LPR, col = (threadIdx.x % LPR) * 8;
    const unsigned zh = unit / unsigned(a.M), r = unit - zh * unsigned(a.M), z = zh / unsigned(a.H_kv), h = zh - z * unsigned(a.H_kv);
    if (z >= unsigned(a.Z)) return;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (int(r) < __ldg(a.lens + z)) {                     // (rows behind a sequence's end are zeros)
        const int idx = int(r >> a.c.page_shift), page = idx < a.c.width ? __ldg(a.c.table + size_t(z) * a.c.width + idx) : -1;
        if (unsigned(page) >= unsigned(a.c.n_pages)) {
            if (col == 0) report(a.status, FST_DEV_INDEX_RANGE, int(z), int(r));
        } else {
            const int off = int(r) & ((1 << a.c.page_shift) - 1);
            const int64_t from = page * a.c.stride_page + off * a.c.stride_row + h * a.c.stride_head + col;
            if constexpr (QUANT) {
                const size_t at = ((size_t(page) * a.H_kv + h) << a.c.page_shift) + off;
                const uint2 bk = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.c.k_pool) + from));
                const uint2 bv = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.c.v_pool) + from));
                const float ek = e8m0_value(__ldg(a.c.k_scale + at)), ev = e8m0_value(__ldg(a.c.v_scale + at));
                k = expand8<T>(bk, ek);
                v = expand8<T>(bv, ev);
            } else {
                k = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.c.k_pool) + from));
                v = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.c.v_pool) + from));
            }
        }
    }
    *reinterpret_cast<uint4 *>(static_cast<T *>(a.k) + z * a.ks_z + h * a.ks_h + r * a.ks_n + col) = k;
    *reinterpret_cast<uint4 *>(static_cast<T *>(a.v) + z * a.vs_z + h * a.vs_h + r * a.vs_n + col) = v;
}

// A block takes pages of one head, every gridDim.x-th of all that hold rows; the lengths are read once per 256 sequences.
template <typename T, int D>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_expand_kernel(const ExpandArgs a) {
    constexpr int LPR = D / 8, RPB = CACHE_THREADS / LPR;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    __shared__ int pages[256];
    const int col = (threadIdx.x % LPR) * 8, ps = 1 << a.c.page_shift;
    unsigned skip = blockIdx.x;                           // units ahead of my next one
#pragma unroll 1
    for (int z0 = 0; z0 < a.Z; z0 += 256) {
        __syncthreads();
        if (z0 + int(threadIdx.x) < a.Z) pages[threadIdx.x] = min((max(__ldg(a.lens + z0 + threadIdx.x), 0) + ps - 1) >> a.c.page_shift, a.c.width);
        __syncthreads();
#pragma unroll 1
        for (int z = z0; z < min(a.Z, z0 + 256); ++z) {
            const unsigned n = unsigned(pages[z - z0]) * unsigned(a.H_kv);
#pragma unroll 1
            for (; skip < n; skip += gridDim.x) {
                const int idx = int(skip / unsigned(a.H_kv)), h = int(skip - unsigned(idx) * unsigned(a.H_kv));
                const size_t to_page = size_t(z) * a.c.width + idx;
                const int page = __ldg(a.c.table + to_page);
                const bool bad = unsigned(page) >= unsigned(a.c.n_pages);        // its rows read as zeros: no page of the new pool either
                if (h == 0 && threadIdx.x == 0) {
                    if (bad) report(a.status, FST_DEV_INDEX_RANGE, z, idx << a.c.page_shift);
                    a.table[to_page] = bad ? -1 : int(to_page);
                }
                if (bad) continue;
#pragma unroll 2
                for (int r = threadIdx.x / LPR; r < ps; r += RPB) {
                    const int64_t from = page * a.c.stride_page + r * a.c.stride_row + h * a.c.stride_head + col;
                    const size_t at = ((size_t(page) * a.H_kv + h) << a.c.page_shift) + r, to = (((to_page * a.H_kv + h) << a.c.page_shift) + r) * D + col;
                    const uint2 bk = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.c.k_pool) + from));
                    const uint2 bv = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.c.v_pool) + from));
                    const float ek = e8m0_value(__ldg(a.c.k_scale + at)), ev = e8m0_value(__ldg(a.c.v_scale + at));
                    *reinterpret_cast<uint4 *>(static_cast<T *>(a.k) + to) = expand8<T>(bk, ek);
                    *reinterpret_cast<uint4 *>(static_cast<T *>(a.v) + to) = expand8<T>(bv, ev);
                }
            }
            skip -= n;
        }
    }
}

template <typename T, int D>
static cudaError_t launch_expand_t(const ExpandArgs &a, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(8 * sm_count());
    cfg.blockDim = dim3(CACHE_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, cache_expand_kernel<T, D>, a);
}
cudaError_t launch_cache_expand(const ExpandArgs &a, int dtype, int D, cudaStream_t stream) {
    if (dtype == FST_F16) return D == 128 ? launch_expand_t<__half, 128>(a, stream) : launch_expand_t<__half, 64>(a, stream);
    return D == 128 ? launch_expand_t<__nv_bfloat16, 128>(a, stream) : launch_expand_t<__nv_bfloat16, 64>(a, stream);
}

// One lane group per row; launched so that the grid may become resident while the one ahead of it drains.
template <int D, typename K, typename A>
static cudaError_t launch_rows(K kernel, const A &a, cudaStream_t stream) {
    constexpr int RPB = CACHE_THREADS / (D / 8);
    const long long units = (long long)a.Z * a.H_kv * a.M;
    if (units > 0x7fffffffLL - RPB) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned((units + RPB - 1) / RPB));
    cfg.blockDim = dim3(CACHE_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, int D>
static cudaError_t launch_append_t(const AppendArgs &a, cudaStream_t stream) {
    return a.c.k_scale != nullptr ? launch_rows<D>(cache_append_kernel<T, D, true>, a, stream)
                                  : launch_rows<D>(cache_append_kernel<T, D, false>, a, stream);
}
template <typename T, int D>
static cudaError_t launch_read_t(const ReadArgs &a, cudaStream_t stream) {
    return a.c.k_scale != nullptr ? launch_rows<D>(cache_read_kernel<T, D, true>, a, stream)
                                  : launch_rows<D>(cache_read_kernel<T, D, false>, a, stream);
}

cudaError_t launch_cache_append(const AppendArgs &a, int dtype, int D, cudaStream_t stream) {
    if (dtype == FST_F16) return D == 128 ? launch_append_t<__half, 128>(a, stream) : launch_append_t<__half, 64>(a, stream);
    return D == 128 ? launch_append_t<__nv_bfloat16, 128>(a, stream) : launch_append_t<__nv_bfloat16, 64>(a, stream);
}
cudaError_t launch_cache_read(const ReadArgs &a, int dtype, int D, cudaStream_t stream) {
    if (dtype == FST_F16) return D == 128 ? launch_read_t<__half, 128>(a, stream) : launch_read_t<__half, 64>(a, stream);
    return D == 128 ? launch_read_t<__nv_bfloat16, 128>(a, stream) : launch_read_t<__nv_bfloat16, 64>(a, stream);
}

}  // namespace fst
