// Rows into and out of a paged K/V cache (fst_cache_append, fst_cache_read).
//
// Both move each row of a head once and compute next to nothing: HBM bounds the large calls, the launch and a chain of
// three memory latencies (length, page number, row) the small ones.  A row of D 16-bit values is D / 8 lanes of 16 bytes, K and V by
// the same lanes, so that a warp moves 512 bytes of either at a time and the lookups serve both.
#include <type_traits>

#include "fst_cache.cuh"

namespace fst {

constexpr int CACHE_THREADS = 256;
constexpr int CACHE_ROWS = 2;          // rows of a thread that reads many: 30011 rows of 8 heads out of e4m3 with 1: 36.8 us, 2: 33.2, 4: 37.1

template <typename T>
__device__ __forceinline__ float2 two_floats(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}

// Sixteen values of a row that D / 16 neighbouring lanes hold: the row's largest magnitude is taken over them.  Magnitudes are compared as
// integers, two at a time, where NaN and infinity are the largest (instructions bound large appends: 12.9 us with floats, 11.2 so).
template <typename T, int D>
__device__ __forceinline__ uint4 quantise16(const uint4 (&in)[2], uint32_t &biased) {
    constexpr bool HALF = std::is_same<T, __half>::value;
    const uint32_t w[8] = {in[0].x, in[0].y, in[0].z, in[0].w, in[1].x, in[1].y, in[1].z, in[1].w};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
#pragma unroll
    for (int s = 1; s < D / 16; s *= 2) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, s));
    top = max(top & 0xffffu, top >> 16);
    if (top >= (HALF ? 0x7c00u : 0x7f80u)) {
        biased = 255u;
        return make_uint4(0u, 0u, 0u, 0u);
    }
    const int e = e4m3_exponent(two_floats<T>(top).x);
    const float f = pow2f(-e);
    biased = uint32_t(e + 127);
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 x = two_floats<T>(w[i]);
        b[i] = e4m3_pair(x.x * f, x.y * f);
    }
    return make_uint4(b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16);
}

// New row j of head h of sequence z, all (z, h, j) in one line; neighbours in the source and in a page by neighbouring threads, 16 bytes a lane
// into a page.  (Quantising, 8 bytes a lane and two rows a thread took 10.6 us for 8192 rows of 8 heads, this 8.6; two rows a thread then gain
// nothing.)
template <typename T, int D, bool QUANT>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_append_kernel(const AppendArgs a) {
    constexpr int C = QUANT ? 2 : 1, LPR = D / (8 * C), RPB = CACHE_THREADS / LPR;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const unsigned r = blockIdx.x * RPB + threadIdx.x / LPR, col = (threadIdx.x % LPR) * (8 * C);
    const unsigned zh = r / unsigned(a.M), j = r - zh * unsigned(a.M), z = zh / unsigned(a.H_kv), h = zh - z * unsigned(a.H_kv);
    uint4 k[C], v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) k[c] = v[c] = make_uint4(0, 0, 0, 0);
    int64_t pos = 0;
    int page = 0;
    bool live = z < unsigned(a.Z);
    if (live) {
        const int row = a.rows != nullptr ? load(a.rows + size_t(z) * a.M + j) : int(j);
        const int count = a.lens != nullptr ? load(a.lens + z) : a.M;
        pos = int64_t(load(a.start + z)) + j;
        live = int(j) < count;
        if (count > a.M && j == 0 && h == 0 && col == 0) report(a.status, FST_DEV_INDEX_RANGE, int(z), count);
        if (live && (row < 0 || row >= a.N || pos < 0 || (pos >> a.c.page_shift) >= a.c.width)) {
            if (col == 0) report(a.status, FST_DEV_INDEX_RANGE, int(z), int(j));
            live = false;
        }
        if (live) {
            const T *from_k = static_cast<const T *>(a.k) + z * a.ks_z + h * a.ks_h + row * a.ks_n + col;
            const T *from_v = static_cast<const T *>(a.v) + z * a.vs_z + h * a.vs_h + row * a.vs_n + col;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                k[c] = load(reinterpret_cast<const uint4 *>(from_k) + c);
                v[c] = load(reinterpret_cast<const uint4 *>(from_v) + c);
            }
            page = load(a.c.table + size_t(z) * a.c.width + (pos >> a.c.page_shift));
            if (unsigned(page) >= unsigned(a.c.n_pages)) {
                if (col == 0) report(a.status, FST_DEV_INDEX_RANGE, int(z), int(j));
                live = false;
            }
        }
    }
    const int off = int(pos) & ((1 << a.c.page_shift) - 1);
    const int64_t to = page * a.c.stride_page + off * a.c.stride_row + h * a.c.stride_head + col;
    if constexpr (QUANT) {
        uint32_t ek, ev;                                  // (all lanes take part in the maximum)
        const uint4 qk = quantise16<T, D>(k, ek), qv = quantise16<T, D>(v, ev);
        if (!live) return;
        *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(a.c.k_pool) + to) = qk;
        *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(a.c.v_pool) + to) = qv;
        if (col == 0) {
            const size_t at = ((size_t(page) * a.H_kv + h) << a.c.page_shift) + off;
            a.c.k_scale[at] = uint8_t(ek);
            a.c.v_scale[at] = uint8_t(ev);
        }
    } else if (live) {
        *reinterpret_cast<uint4 *>(static_cast<T *>(a.c.k_pool) + to) = k[0];
        *reinterpret_cast<uint4 *>(static_cast<T *>(a.c.v_pool) + to) = v[0];
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

// Eight values a lane, so that the lanes of a row write it as a whole.  R = 1: all (z, h, row) in one line.  R > 1: a block has R * RPB rows of one
// head, so that nothing is divided and a thread has R rows on their way.  Rows behind a sequence's end are only written.
template <typename T, int D, bool QUANT, int R>
__global__ void __launch_bounds__(CACHE_THREADS)
cache_read_kernel(const ReadArgs a) {
    constexpr int LPR = D / 8, RPB = CACHE_THREADS / LPR;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const unsigned first = blockIdx.x * (RPB * R) + threadIdx.x / LPR, col = (threadIdx.x % LPR) * 8;
    uint4 k[R], v[R];
    float ek[R], ev[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        unsigned r = first + i * RPB, z = blockIdx.z, h = blockIdx.y;
        if constexpr (R == 1) {
            const unsigned zh = r / unsigned(a.M);
            r -= zh * unsigned(a.M);
            z = zh / unsigned(a.H_kv);
            h = zh - z * unsigned(a.H_kv);
        }
        k[i] = v[i] = make_uint4(0, 0, 0, 0);             // (rows behind a sequence's end are zeros)
        ek[i] = ev[i] = 0.f;
        if ((R == 1 ? z >= unsigned(a.Z) : r >= unsigned(a.M)) || int(r) >= load(a.lens + z)) continue;
        const int idx = int(r >> a.c.page_shift), page = idx < a.c.width ? load(a.c.table + size_t(z) * a.c.width + idx) : -1;
        if (unsigned(page) >= unsigned(a.c.n_pages)) {
            if (col == 0) report(a.status, FST_DEV_INDEX_RANGE, int(z), int(r));
            continue;
        }
        const int off = int(r) & ((1 << a.c.page_shift) - 1);
        const int64_t from = page * a.c.stride_page + off * a.c.stride_row + h * a.c.stride_head + col;
        if constexpr (QUANT) {
            const size_t at = ((size_t(page) * a.H_kv + h) << a.c.page_shift) + off;
            const uint2 bk = load(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.c.k_pool) + from));
            const uint2 bv = load(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.c.v_pool) + from));
            k[i] = make_uint4(bk.x, bk.y, 0, 0);
            v[i] = make_uint4(bv.x, bv.y, 0, 0);
            ek[i] = e8m0_value(load(a.c.k_scale + at));
            ev[i] = e8m0_value(load(a.c.v_scale + at));
        } else {
            k[i] = load(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.c.k_pool) + from));
            v[i] = load(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.c.v_pool) + from));
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        unsigned r = first + i * RPB, z = blockIdx.z, h = blockIdx.y;
        if constexpr (R == 1) {
            const unsigned zh = r / unsigned(a.M);
            r -= zh * unsigned(a.M);
            z = zh / unsigned(a.H_kv);
            h = zh - z * unsigned(a.H_kv);
        }
        if (R == 1 ? z >= unsigned(a.Z) : r >= unsigned(a.M)) continue;
        if constexpr (QUANT) {
            k[i] = expand8<T>(make_uint2(k[i].x, k[i].y), ek[i]);
            v[i] = expand8<T>(make_uint2(v[i].x, v[i].y), ev[i]);
        }
        *reinterpret_cast<uint4 *>(static_cast<T *>(a.k) + z * a.ks_z + h * a.ks_h + r * a.ks_n + col) = k[i];
        *reinterpret_cast<uint4 *>(static_cast<T *>(a.v) + z * a.vs_z + h * a.vs_h + r * a.vs_n + col) = v[i];
    }
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
        if (z0 + int(threadIdx.x) < a.Z) {                 // (cut to the table first: the rounding up must not leave 31 bits)
            const int rows = min(max(load(a.lens + z0 + threadIdx.x), 0), a.c.width << a.c.page_shift);
            const bool idle = a.q_lens != nullptr && load(a.q_lens + z0 + threadIdx.x) <= 0;
            pages[threadIdx.x] = idle ? 0 : (rows + ps - 1) >> a.c.page_shift;
        }
        __syncthreads();
#pragma unroll 1
        for (int z = z0; z < min(a.Z, z0 + 256); ++z) {
            const unsigned n = unsigned(pages[z - z0]) * unsigned(a.H_kv);
#pragma unroll 1
            for (; skip < n; skip += gridDim.x) {
                const int idx = int(skip / unsigned(a.H_kv)), h = int(skip - unsigned(idx) * unsigned(a.H_kv));
                const size_t to_page = size_t(z) * a.c.width + idx;
                const int page = load(a.c.table + to_page);
                const bool bad = unsigned(page) >= unsigned(a.c.n_pages);        // its rows read as zeros: no page of the new pool either
                if (h == 0 && threadIdx.x == 0) {
                    if (bad) report(a.status, FST_DEV_INDEX_RANGE, z, idx << a.c.page_shift);
                    a.table[to_page] = bad ? -1 : int(to_page);
                }
                if (bad) continue;
#pragma unroll 1
                for (int r0 = threadIdx.x / LPR; r0 < ps; r0 += 2 * RPB) {       // two rows on their way
                    uint2 bk[2], bv[2];
                    float ek[2], ev[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = r0 + i * RPB;
                        if (r >= ps) continue;
                        const int64_t from = page * a.c.stride_page + r * a.c.stride_row + h * a.c.stride_head + col;
                        const size_t at = ((size_t(page) * a.H_kv + h) << a.c.page_shift) + r;
                        bk[i] = load(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.c.k_pool) + from));
                        bv[i] = load(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.c.v_pool) + from));
                        ek[i] = e8m0_value(load(a.c.k_scale + at));
                        ev[i] = e8m0_value(load(a.c.v_scale + at));
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = r0 + i * RPB;
                        if (r >= ps) continue;
                        const size_t to = (((to_page * a.H_kv + h) << a.c.page_shift) + r) * D + col;
                        *reinterpret_cast<uint4 *>(static_cast<T *>(a.k) + to) = expand8<T>(bk[i], ek[i]);
                        *reinterpret_cast<uint4 *>(static_cast<T *>(a.v) + to) = expand8<T>(bv[i], ev[i]);
                    }
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

// Launched so that the grid may become resident while the one ahead of it drains.
template <typename K, typename A>
static cudaError_t launch_rows(K kernel, const A &a, dim3 grid, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(CACHE_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}
// The one-row kernel where rows are few or would not fill blocks of R * RPB of one head, else the R-row one.
template <int R, int RPB, typename K1, typename KR, typename A>
static cudaError_t launch_rows(K1 one, KR several, const A &a, cudaStream_t stream) {
    const long long units = (long long)a.Z * a.H_kv * a.M;
    if (a.M >= 2 * R * RPB && units >= 8LL * R * RPB * sm_count() && a.H_kv <= 65535 && a.Z <= 65535)
        return launch_rows(several, a, dim3((a.M + R * RPB - 1) / (R * RPB), a.H_kv, a.Z), stream);
    if (units > 0x7fffffffLL - RPB) return cudaErrorInvalidConfiguration;
    return launch_rows(one, a, dim3(unsigned((units + RPB - 1) / RPB)), stream);
}

template <typename T, int D, bool QUANT>
static cudaError_t launch_append_t(const AppendArgs &a, cudaStream_t stream) {
    constexpr int RPB = CACHE_THREADS / (D / (QUANT ? 16 : 8));
    const long long units = (long long)a.Z * a.H_kv * a.M;
    if (units > 0x7fffffffLL - RPB) return cudaErrorInvalidConfiguration;
    return launch_rows(cache_append_kernel<T, D, QUANT>, a, dim3(unsigned((units + RPB - 1) / RPB)), stream);
}
template <typename T, int D, bool QUANT>
static cudaError_t launch_read_t(const ReadArgs &a, cudaStream_t stream) {
    return launch_rows<CACHE_ROWS, CACHE_THREADS / (D / 8)>(cache_read_kernel<T, D, QUANT, 1>, cache_read_kernel<T, D, QUANT, CACHE_ROWS>, a, stream);
}
template <typename T, int D>
static cudaError_t launch_append_t(const AppendArgs &a, cudaStream_t stream) {
    return a.c.k_scale != nullptr ? launch_append_t<T, D, true>(a, stream) : launch_append_t<T, D, false>(a, stream);
}
template <typename T, int D>
static cudaError_t launch_read_t(const ReadArgs &a, cudaStream_t stream) {
    return a.c.k_scale != nullptr ? launch_read_t<T, D, true>(a, stream) : launch_read_t<T, D, false>(a, stream);
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
