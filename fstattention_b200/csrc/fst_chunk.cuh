// Attention of a chunk of new tokens over a paged K/V cache: what its kernels share.
//
// The cache holds kv_lens[z] rows of sequence z, the chunk's own q_lens[z] among them as the last ones; query i stands
// at position kv_len - q_len + i and attends to the rows up to it (causal) or to all of them:
//     o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),   s_j = sm_scale log2(e) q . k_j,   m = max_j s_j
// A query that sees no row has o = 0 and a log-sum-exp of -inf.
//
// The rows (query i, head g of the group) of a sequence and K/V head, r = i * group + g, are cut into row tiles, the keys
// that a row tile sees into key tiles.  Lengths live on the device, so the work is divided there: all (z, K/V
// head, row tile) items stand in one line, each as long as its key tiles, and every CTA of a grid that fills the GPU once
// takes an equal piece of the line.  Any mix of lengths is balanced that way without the host knowing
// them, a captured graph stays valid while sequences grow, and a CTA has at most two pieces that are not whole items:
// the first and the last.  Those leave their rows in a workspace of fixed size; chunk_combine_kernel merges them
// in the order of the CTAs, so the result does not depend on timing.
#pragma once

#include <algorithm>
#include <type_traits>

#include "fst_attention_mma.cuh"
#include "fst_cache.cuh"

namespace fst {

struct ChunkArgs {
    CacheArgs c;
    const void *q;
    void *o;
    float *lse;
    const int32_t *kv_lens, *q_lens;       // [Z], q_lens null: n_q everywhere
    int Z, H, H_kv, group, n_q;
    int64_t qs_z, qs_h, qs_n, os_z, os_h, os_n;
    uint32_t group_mul;                    // x / group = x * group_mul >> group_shift for x in [0, 2^31): see set_group
    int group_shift;
    uint64_t cta_mul;                      // x / n = the high half of x * cta_mul for x < 2^64 / n, n the CTAs of a call: see set_ctas
    float scale_log2;                      // sm_scale * log2(e), positive
    int causal;
    int q_boxes;                           // Q comes as boxes of `group` heads by 128 / group tokens
    float *part;                           // pieces: [2 CTAs][rows][D] sums, [2 CTAs][rows] (exponent, sum), [CTAs] ChunkCut
    int32_t *status;
};

// With s the smallest number of bits for which 2^s >= d and m = ceil(2^(31 + s) / d), which is below 2^32, m d exceeds 2^(31 + s) by less
// than 2^s, so x m / 2^(31 + s) exceeds x / d by less than 1 / d for x < 2^31: the same integer.
inline void set_group(ChunkArgs &a, int group) {
    a.group = group;
    int s = 0;
    while ((1u << s) < unsigned(group)) ++s;
    a.group_mul = uint32_t(((1ull << (31 + s)) + unsigned(group) - 1) / unsigned(group));
    a.group_shift = 31 + s;
}
__device__ __forceinline__ int by_group(const ChunkArgs &a, int x) { return int(uint64_t(uint32_t(x)) * a.group_mul >> a.group_shift); }

// With m = floor(2^64 / n) + 1, m n exceeds 2^64 by at most n, so x m / 2^64 exceeds x / n by at most x / 2^64: less than 1 / n for x < 2^64 / n.
// (n is at least 2.)
inline void set_ctas(ChunkArgs &a, int n) { a.cta_mul = ~uint64_t(0) / uint64_t(n) + 1; }

// The line of work for row tiles of ROWS and key tiles of KEYS.  An item is OVER units longer than it has key tiles: its own start and end
// cost a CTA as much as that many tiles (a CTA that got seven items of two tiles each ended at 51 us, the others at 30).  They lie
// before its first tile; a place among them means that tile.
template <int ROWS, int KEYS, int OVER>
struct ChunkLine {
    const ChunkArgs &a;
    __device__ __forceinline__ explicit ChunkLine(const ChunkArgs &args) : a(args) {}

    __device__ __forceinline__ int kv_len(int z) const {
        const int n = load(a.kv_lens + z), most = a.c.width << a.c.page_shift;
        return min(max(n, 0), most);
    }
    __device__ __forceinline__ int q_len(int z) const { return a.q_lens == nullptr ? a.n_q : min(max(load(a.q_lens + z), 0), a.n_q); }
    __device__ __forceinline__ int row_tiles(int ql) const { return (ql * a.group + ROWS - 1) / ROWS; }
    // keys that the last row of a row tile sees
    __device__ __forceinline__ int keys(int kv, int ql, int qt) const {
        if (!a.causal) return kv;
        const int last = min(by_group(a, (qt + 1) * ROWS - 1), ql - 1);
        return max(0, min(kv, kv - ql + last + 1));
    }
    // at least one key tile, so that rows which see nothing are written too
    __device__ __forceinline__ static int tiles_of(int keys) { return max(1, (keys + KEYS - 1) / KEYS); }
    // Units of one K/V head of a sequence: by one lane, or by a whole warp where the row tiles are many (64 row tiles one after
    // the other take a lane 2 us).
    __device__ __forceinline__ bool wide() const { return a.causal && row_tiles(a.n_q) > 8; }
    __device__ __forceinline__ long long head_units(int kv, int ql) const {
        const int n = row_tiles(ql);
        if (!a.causal) return (long long)n * (tiles_of(kv) + OVER);
        long long s = 0;
#pragma unroll 1
        for (int qt = 0; qt < n; ++qt) s += tiles_of(keys(kv, ql, qt)) + OVER;
        return s;
    }
    __device__ __forceinline__ long long head_units_by_warp(int kv, int ql) const {
        long long s = 0;
#pragma unroll 1
        for (int qt = threadIdx.x & 31, n = row_tiles(ql); qt < n; qt += 32) s += tiles_of(keys(kv, ql, qt)) + OVER;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
        return s;
    }
};

// A place in the line; the same in all lanes of a warp.
template <int ROWS, int KEYS, int OVER>
struct ChunkCursor {
    using Line = ChunkLine<ROWS, KEYS, OVER>;
    int z, h, qt, tile, tiles, keys, kv, ql, n_qt;

    __device__ __forceinline__ void at_row_tile(const Line &line) {
        keys = line.keys(kv, ql, qt);
        tiles = line.tiles_of(keys);
    }
    __device__ __forceinline__ void open(const Line &line) {
        kv = line.kv_len(z);
        ql = line.q_len(z);
        n_qt = line.row_tiles(ql);
    }
    // by a whole warp: length of the line
    __device__ __forceinline__ static long long total(const Line &line) {
        const int lane = threadIdx.x & 31;
        long long sum = 0;
        if (line.wide()) {
#pragma unroll 1
            for (int z = 0; z < line.a.Z; ++z) sum += line.head_units_by_warp(line.kv_len(z), line.q_len(z));
            return sum * line.a.H_kv;
        }
#pragma unroll 1
        for (int z = lane; z < line.a.Z; z += 32) sum += line.head_units(line.kv_len(z), line.q_len(z));
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        return sum * line.a.H_kv;
    }
    // running sums over the lanes
    __device__ __forceinline__ static long long scan(long long v) {
#pragma unroll
        for (int s = 1; s < 32; s *= 2) {
            const long long below = __shfl_up_sync(0xffffffffu, v, s);
            if (int(threadIdx.x & 31) >= s) v += below;
        }
        return v;
    }
    // by a whole warp: to the tile at or behind unit `pos` of the line, which has to be in it; the tiles of the line ahead of that one
    __device__ __forceinline__ long long seek(const Line &line, long long pos) {
        const int lane = threadIdx.x & 31;
        const long long at = pos;
        long long head = 1, items = 0;                    // of the sequences ahead
        z = 0;
        if (line.wide()) {
#pragma unroll 1
            for (;; ++z) {
                head = line.head_units_by_warp(line.kv_len(z), line.q_len(z));
                if (pos < head * line.a.H_kv || z + 1 == line.a.Z) break;
                pos -= head * line.a.H_kv;
                items += line.row_tiles(line.q_len(z));
            }
        } else {
#pragma unroll 1
            for (int z0 = 0; z0 < line.a.Z; z0 += 32) {
                const bool real = z0 + lane < line.a.Z;
                const int mine_q = real ? line.q_len(z0 + lane) : 0;
                const long long mine = real ? line.head_units(line.kv_len(z0 + lane), mine_q) : 0;
                const long long upto = scan(mine * line.a.H_kv);
                const unsigned past = __ballot_sync(0xffffffffu, pos < upto);
                const int f = past != 0u ? __ffs(past) - 1 : 32;
                long long n = lane < f ? line.row_tiles(mine_q) : 0;
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) n += __shfl_xor_sync(0xffffffffu, n, s);
                items += n;
                if (past != 0u) {
                    z = z0 + f;
                    head = __shfl_sync(0xffffffffu, mine, f);
                    pos -= __shfl_sync(0xffffffffu, upto, f) - head * line.a.H_kv;
                    break;
                }
                pos -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        open(line);
        h = int(__fdividef(float(pos), float(head)));     // (a division of 64 bits is a hundred instructions to fetch; the estimate is off by one at most, or little more)
        while (h > 0 && h * head > pos) --h;
        while ((h + 1) * head <= pos) ++h;
        pos -= h * head;
        qt = 0;
        if (n_qt > 1) {
#pragma unroll 1
            for (int q0 = 0; q0 < n_qt; q0 += 32) {
                const long long mine = q0 + lane < n_qt ? line.tiles_of(line.keys(kv, ql, q0 + lane)) + OVER : 0, upto = scan(mine);
                const unsigned past = __ballot_sync(0xffffffffu, pos < upto);
                if (past != 0u) {
                    const int f = __ffs(past) - 1;
                    qt = q0 + f;
                    pos -= __shfl_sync(0xffffffffu, upto - mine, f);
                    break;
                }
                pos -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        at_row_tile(line);
        tile = max(0, int(pos) - OVER);
        return at - pos - OVER * (items * line.a.H_kv + (long long)h * n_qt + qt) + tile;
    }
    // to the next tile; the last tile of the line has none
    __device__ __forceinline__ void next(const Line &line) {
        if (++tile < tiles) return;
        tile = 0;
        if (++qt == n_qt) {
            qt = 0;
            if (++h == line.a.H_kv) {
                h = 0;
                do {
                    if (++z == line.a.Z) {
                        z = line.a.Z - 1;
                        return;
                    }
                    open(line);
                } while (n_qt == 0);
            }
        }
        at_row_tile(line);
    }
};


// CTA i of n takes the tiles of units [first(i), first(i + 1)) of the line
__device__ __forceinline__ long long chunk_share(const ChunkArgs &a, long long total) { return (long long)__umul64hi(uint64_t(total), a.cta_mul); }
__device__ __forceinline__ long long chunk_first(const ChunkArgs &a, long long total, int i, int n) {
    const long long each = chunk_share(a, total);
    return each * i + min((long long)i, total - each * n);
}

// A CTA's piece of the line, found by two of its warps for all (in shared memory).
template <int ROWS, int KEYS, int OVER>
struct ChunkPiece {
    ChunkCursor<ROWS, KEYS, OVER> from;
    long long total, before, upto;         // units of the line; tiles ahead of my first one, ahead of the next CTA's
    __device__ __forceinline__ int tiles() const { return int(upto - before); }
    // by the CTA's first two warps, ahead of a barrier
    __device__ __forceinline__ void find(const ChunkLine<ROWS, KEYS, OVER> &line) {
        const int warp = threadIdx.x >> 5;
        if (warp > 1) return;
        ChunkCursor<ROWS, KEYS, OVER> c;
        const long long all = c.total(line), lo = chunk_first(line.a, all, blockIdx.x, gridDim.x), hi = chunk_first(line.a, all, blockIdx.x + 1, gridDim.x);
        long long n = 0;
        if (hi > lo) n = c.seek(line, warp == 0 ? lo : min(hi, all - 1)) + (warp == 1 && hi == all ? 1 : 0);         // (the line ends with a tile)
        if ((threadIdx.x & 31) != 0) return;
        if (warp == 0) {
            from = c;
            before = n;
            total = all;
        } else {
            upto = n;
        }
    }
};

// What the merge has to know of the item that CTA i's last piece begins: its pieces are CTA i's last one and the first ones of the
// CTAs behind it.
struct ChunkCut {
    int z, h, qt, ql, pieces;              // 1 (or 0, a CTA without work): nothing to merge
    int pad[3];
};

// Probabilities that are rounded to fp16 for the second product are taken 2^15 times too large (against a reference that is 15 below
// the maximum), so that they fill its range: at most 2^15, and those below 2^-14 are rounded to steps of 2^-24, by 2^-40 of the largest one.  At
// most 1 they would lose what lies 2^24 below the largest one, which many keys together can make the larger part of the result.  Where the
// reference may lag by 2^8 (chunk_umma_kernel) the factor is 2^7 and that step's half 2^-32 of the largest: equal probabilities of
// 2^-25.5 of it all become 45 steps where they are 45.25, and what 60000 of them make of a result comes out half a percent low.
constexpr float kLift = 15.f;

// ---- values that are not finite where not every row of a tile attends to them.  The second product multiplies a masked
// key's V by a probability of zero, and zero times NaN or infinity is NaN.  In key groups that some row does not see, such elements
// are taken out of V, and what they do to the rows that see them is added at the end: a kernel that met none never looks again.

// Of two 16-bit values only those that are finite and among the first n; whether one among the first n was not finite.
template <typename T>
__device__ __forceinline__ bool keep_finite(uint32_t &w, int n) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    if (n < 2) w = n < 1 ? 0u : w & 0xffffu;
    bool met = false;
    if ((w & E) == E) {
        w &= 0xffff0000u;
        met = true;
    }
    if ((w >> 16 & E) == E) {
        w &= 0xffffu;
        met = true;
    }
    return met;
}
// out[k] += the elements c0 + k of V in rows [from, to) of a sequence that are not finite (of an 8-bit cache: all of a row, as NaN)
template <typename T, int N, bool QUANT>
__device__ __forceinline__ void add_not_finite(const ChunkArgs &a, int z, int h, int from, int to, int c0, float (&out)[N]) {
#pragma unroll 1
    for (int key = from; key < to; ++key) {
        const int idx = key >> a.c.page_shift, off = key & ((1 << a.c.page_shift) - 1);
        const int page = load(a.c.table + size_t(z) * a.c.width + idx);
        if (unsigned(page) >= unsigned(a.c.n_pages)) continue;
        if constexpr (QUANT) {
            const bool odd = load(a.c.v_scale + ((size_t(page) * a.H_kv + h) << a.c.page_shift) + off) == 255;
#pragma unroll
            for (int k = 0; k < N; ++k) out[k] = odd ? NAN : out[k];
        } else {
            const T *v = static_cast<const T *>(a.c.v_pool) + page * a.c.stride_page + off * a.c.stride_row + h * a.c.stride_head + c0;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const float x = float(v[k]);
                out[k] += isfinite(x) ? 0.f : x;
            }
        }
    }
}

// A launch that may become resident while the kernel ahead of it drains; the kernel waits before its first access.
template <typename... P, typename... A>
cudaError_t launch_serialised(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

__host__ __device__ inline size_t chunk_stats_at(int n_ctas, int rows, int D) { return size_t(2) * n_ctas * rows * D; }
__host__ __device__ inline size_t chunk_cuts_at(int n_ctas, int rows, int D) { return chunk_stats_at(n_ctas, rows, D) + size_t(4) * n_ctas * rows; }
inline size_t chunk_part_bytes(int n_ctas, int rows, int D) { return chunk_cuts_at(n_ctas, rows, D) * sizeof(float) + n_ctas * sizeof(ChunkCut); }

// CTA i's note for the merge, by one thread, `last` being its last tile.  (Every CTA behind it takes `per` tiles or one more, so
// that the count is a division and at most a step or two.)
template <int D, int ROWS, int KEYS, int OVER>
__device__ __forceinline__ void leave_cut(const ChunkArgs &a, const ChunkCursor<ROWS, KEYS, OVER> &last, long long total, int n_tiles) {
    ChunkCut cut = {};
    if (n_tiles > 0) {
        cut.z = last.z;
        cut.h = last.h;
        cut.qt = last.qt;
        cut.ql = last.ql;
        cut.pieces = 1;
        const int behind = last.tiles - last.tile - 1;
        if (behind > 0 && n_tiles > last.tile) {          // it goes on (then its next tile is the next CTA's first unit), and began here
            const int me = blockIdx.x, n = gridDim.x;
            const long long end = chunk_first(a, total, me + 1, n) + behind;
            int c = me + 1 + (behind - 1) / int(min(chunk_share(a, total) + 1, 0x7fffffffLL));
            while (c + 1 < n && chunk_first(a, total, c + 1, n) < end) ++c;
            cut.pieces = c - me + 1;
        }
    }
    reinterpret_cast<ChunkCut *>(a.part + chunk_cuts_at(gridDim.x, ROWS, D))[blockIdx.x] = cut;
}

// The pieces of the item that CTA x's last piece begins, merged in their order: a warp for RPW rows at a time, eight warps a block.
// The factors of up to 32 pieces are taken by a lane each, so that nothing but the additions is a chain.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256)
chunk_combine_kernel(const ChunkArgs a, int n_ctas) {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    constexpr int C = D / 32, RPW = ROWS >= 32 ? 4 : ROWS / 8;   // columns of a lane, rows of a warp
    const ChunkCut it = reinterpret_cast<const ChunkCut *>(a.part + chunk_cuts_at(n_ctas, ROWS, D))[blockIdx.x];
    const int row0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * RPW, lane = threadIdx.x & 31;
    if (it.pieces <= 1 || it.qt * ROWS + row0 >= it.ql * a.group) return;
    const float2 *stats = reinterpret_cast<const float2 *>(a.part + chunk_stats_at(n_ctas, ROWS, D));
    auto slot = [&](int piece) { return (size_t(2) * (blockIdx.x + piece) + (piece == 0 ? 1 : 0)) * ROWS + row0; };
    float acc[RPW][C] = {}, top[RPW], sum[RPW];
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
        top[i] = -INFINITY;
        sum[i] = 0.f;
    }
#pragma unroll 1
    for (int p0 = 0; p0 < it.pieces; p0 += 32) {
        const int n = min(32, it.pieces - p0);
        float2 st[RPW];
        float w[RPW];
#pragma unroll
        for (int i = 0; i < RPW; ++i) st[i] = lane < n ? stats[slot(p0 + lane) + i] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int i = 0; i < RPW; ++i) {
            float now = st[i].x;
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, s));
            now = fmaxf(now, top[i]);
            // a piece that saw nothing has no part in it; one whose scores were all NaN has no exponent, but a sum
            w[i] = st[i].x == -INFINITY ? (st[i].y == 0.f ? 0.f : 1.f) : fast_exp2(st[i].x - now);
            const float w_old = top[i] == -INFINITY ? 1.f : fast_exp2(top[i] - now);
            float part = st[i].y * w[i];
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) part += __shfl_xor_sync(0xffffffffu, part, s);
            sum[i] = sum[i] * w_old + part;
            top[i] = now;
#pragma unroll
            for (int k = 0; k < C; ++k) acc[i][k] *= w_old;
        }
#pragma unroll 4
        for (int p = 0; p < n; ++p) {
            const float *from = a.part + slot(p0 + p) * D + lane * C;
#pragma unroll
            for (int i = 0; i < RPW; ++i) {
                const float f = __shfl_sync(0xffffffffu, w[i], p);
                float v[C];
                if constexpr (C == 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(from + i * D);
                    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                } else {
                    const float2 x = *reinterpret_cast<const float2 *>(from + i * D);
                    v[0] = x.x; v[1] = x.y;
                }
#pragma unroll
                for (int k = 0; k < C; ++k) acc[i][k] = f == 0.f ? acc[i][k] : fmaf(v[k], f, acc[i][k]);      // (not written where f is zero)
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
        const int r = it.qt * ROWS + row0 + i, tok = by_group(a, r), head = it.h * a.group + (r - tok * a.group);
        if (tok >= it.ql) continue;
        const float inv = sum[i] == 0.f ? 0.f : 1.f / sum[i];
        T *dst = static_cast<T *>(a.o) + it.z * a.os_z + head * a.os_h + tok * a.os_n + lane * C;
        if constexpr (C == 4)
            *reinterpret_cast<uint2 *>(dst) = make_uint2(MmaTraits<T>::pack(acc[i][0] * inv, acc[i][1] * inv), MmaTraits<T>::pack(acc[i][2] * inv, acc[i][3] * inv));
        else
            *reinterpret_cast<uint32_t *>(dst) = MmaTraits<T>::pack(acc[i][0] * inv, acc[i][1] * inv);
        if (a.lse != nullptr && lane == 0) a.lse[(size_t(it.z) * a.H + head) * a.n_q + tok] = sum[i] == 0.f ? -INFINITY : top[i] + log2f(sum[i]);
    }
}

template <typename T, int D, int ROWS>
cudaError_t launch_chunk_combine(const ChunkArgs &a, int n_ctas, cudaStream_t stream) {
    constexpr int PER_BLOCK = 8 * (ROWS >= 32 ? 4 : ROWS / 8);
    return launch_serialised(chunk_combine_kernel<T, D, ROWS>, dim3(n_ctas, ROWS / PER_BLOCK), dim3(256), 0, stream, a, n_ctas);
}

// CTAs of a call's line: one per SM (a workspace holds two pieces for each).
inline int chunk_ctas() { return std::max(sm_count(), 2); }
// Which kernel: up to 32 rows those on mma.sync, which read a key for little more than its bytes; up to 8 the one that has them as columns.  Measured
// with 8 sequences of 16000 rows, us at bf16 D 128 / e4m3 D 128 / fp16 D 64 / e4m3 D 64: 24 rows on mma.sync 102 / 109 / 58 / 73, on
// tcgen05 105 / 128 / 92 / 101; 36 rows on tcgen05 106 / 130 / 93 / 99, in two tiles on mma.sync 177 / 164 (before bf16 weights had exponents
// of their own) / 100 / 134; 8 rows as columns 86 / 54 / 53 / 43, as a tile of 16 rows 88 / 62 / 53 / 48.
inline bool chunk_many_rows(const ChunkArgs &a) { return (long long)a.n_q * a.group > 32; }
inline int chunk_row_tile(const ChunkArgs &a) {
    const long long rows = (long long)a.n_q * a.group;
    return chunk_many_rows(a) ? 256 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
}
// An 8-bit cache under many queries is expanded once, ahead of the call, rather than by every row tile on its way, but only as long as the copy
// of all that the tables can hold stays below 2 GB.  What it costs goes with the keys, what it saves with keys and rows, so rows decide:
// 8 heads, D 128 / 64, expanded and on the way, us: 512 rows over 16384 71 and 55 / 51 and 44; 2048 rows over 16384 146 and 148 / 123
// and 120; 8192 rows over 8192 220 and 251 / 196 and 201.  (The rows are those of n_q: a call of a prompt and 63 single tokens expands all 64.)
constexpr long long kExpandRows = 2048;
constexpr long long kMostExpanded = 2LL << 30;
inline long long chunk_expanded_bytes(const ChunkArgs &a, int D) { return 4LL * a.Z * a.c.width * a.H_kv * D << a.c.page_shift; }
inline bool chunk_expands(const ChunkArgs &a, int D) {
    const long long pages = (long long)a.Z * a.c.width;   // (times the heads it is below 2^62, times the bytes of a page it need not be)
    return a.c.k_scale != nullptr && (long long)a.n_q * a.group >= kExpandRows && pages < 0x7fffffffLL && pages * a.H_kv <= kMostExpanded / (4LL * D << a.c.page_shift);
}
// Whether any piece can be less than an item: not if all that the table can hold is one key tile.
inline bool chunk_splits(const ChunkArgs &a, int keys) { return ((long long)a.c.width << a.c.page_shift) > keys; }

cudaError_t launch_chunk_f16_d64(const ChunkArgs &, int, cudaStream_t);
cudaError_t launch_chunk_f16_d128(const ChunkArgs &, int, cudaStream_t);
cudaError_t launch_chunk_bf16_d64(const ChunkArgs &, int, cudaStream_t);
cudaError_t launch_chunk_bf16_d128(const ChunkArgs &, int, cudaStream_t);

}  // namespace fst
