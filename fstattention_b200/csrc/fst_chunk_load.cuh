// Loads of the chunk kernels on mma.sync: one warp keeps a ring of K and V tiles filled for the computing ones.
#pragma once

#include "fst_chunk.cuh"
#include "fst_chunk_map.cuh"
#include "fst_umma.cuh"

namespace fst {

// A wait with a limit: a million tries, which took 4.2 seconds of a barrier that nobody arrived at (a try is held back for 4 us at a hint of one).  The
// longest waits are for an item, or for several that do not concern the waiting role, at some 1.6 us a tile: 2.6 million tiles.  Short, and without the
// report that mbar_wait makes, because it stands in two dozen places of a kernel that instruction fetches bound: the roles report at their ends.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (int it = 0; it < (1 << 20); ++it) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                     : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000u) : "memory");
        if (ok != 0u) return true;
    }
    return false;
}

// Sums of weights against m_w become sums against m when multiplied by `by` and `then`: halves of the factor, since 2^(m_w - m) itself may be below
// what an exponential returns as a normal number (rows of V around 2^-110).  `unlift` takes back what the sums are too large by.
__device__ __forceinline__ void weights_back(float m, float m_w, float unlift, float &by, float &then) {
    by = m == -INFINITY ? 1.f : fast_exp2(0.5f * (m_w - m));
    then = by * unlift;
}
static_assert(kLift == 15.f, "fp16 weights are 2^15 times too large");

// two e4m3 bytes (the low ones, the high ones) -> a pair of fp16
__device__ __forceinline__ uint32_t e4m3_halves(uint32_t w, bool high) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"(uint16_t(high ? w >> 16 : w)));
    return r;
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
// By one warp: the tiles of a CTA's piece of the line, K and V in turn, into G::STAGES stages of G::TILE bytes at s_base (KEYS rows: 64-column
// halves of 16 bits, or bytes), an 8-bit tile's scales at G::OFF_SCALES; full[stage] says that it has landed, empty[stage] that it may go.
template <typename G, int D, bool QUANT, typename Line, typename Cursor>
__device__ __forceinline__ void load_tiles(const ChunkArgs &a, const Line &line, Cursor me, int n_tiles, const CUtensorMap &tm_k, const CUtensorMap &tm_v, uint32_t s_base,
                                           unsigned char *smem, uint32_t bar_full, uint32_t bar_empty) {
    const int lane = threadIdx.x & 31;
    // ====== loads: a box per page and 64 columns, by one lane; the page numbers are looked up a tile ahead ======
    // (While each warp fetched its own 16 rows, asking for them took it as long as computing with them.)
    const int ps = 1 << a.c.page_shift;
    int st = 0, page = 0;
    uint32_t use = 0;
    bool alive = true;
    auto look_up = [&]() {
        const int key = me.tile * G::KEYS + lane * ps;
        page = lane * ps < G::KEYS && key < me.keys ? load(a.c.table + size_t(me.z) * a.c.width + (key >> a.c.page_shift)) : 0;
    };
    look_up();
#pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
        const int here = page, key0 = me.tile * G::KEYS, h = me.h, z = me.z;
        const int pages = (min(G::KEYS, me.keys - key0) + ps - 1) >> a.c.page_shift;         // 0: an item that sees nothing
        me.next(line);
        if (i + 1 < n_tiles) look_up();
        if (pages <= 0) continue;
        const bool bad = lane < pages && unsigned(here) >= unsigned(a.c.n_pages);            // the boxes then read as zeros
        if (bad) report(a.status, FST_DEV_INDEX_RANGE, z, key0 + lane * ps);
#pragma unroll 1
        for (int v = 0; v < 2; ++v) {
            if (use > 0 && alive) alive = __all_sync(0xffffffffu, wait_for(bar_empty + st * 8, (use - 1) & 1));
            if (!alive) break;
            const CUtensorMap *map = v ? &tm_v : &tm_k;
            const uint32_t bar = bar_full + st * 8, to = s_base + st * G::TILE;
            unsigned char *scales = smem + G::OFF_SCALES + st * G::KEYS;
            if constexpr (QUANT) {                        // sixteen rows' scales a lane, zeros for a bad page
                static_assert(G::KEYS <= 512, "a lane each");
                const int p = lane >> (a.c.page_shift - 4), pg = __shfl_sync(0xffffffffu, here, p);
                if (p < pages && lane * 16 < G::KEYS) {
                    const uint8_t *from = v ? a.c.v_scale : a.c.k_scale;
                    const bool there = unsigned(pg) < unsigned(a.c.n_pages);
                    cp_async16(smem_u32(scales + lane * 16), there ? from + ((size_t(pg) * a.H_kv + h) << a.c.page_shift) + (lane * 16 & (ps - 1)) : from, there);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
            }
            if (lane == 0) mbar_arrive_expect_tx(bar, (pages << a.c.page_shift) * D * (QUANT ? 1 : 2));
            __syncwarp();
            // Who asks for the pages, measured in us.  An 8-bit cache: a lane each, or one lane one after the other: 98 and 112 (two sequences of 115000
            // rows) where pages have 16 rows, 90 and 87 where they have 64.  16 bits (64 sequences of 4500 rows): a lane each 187, one lane four
            // at a time 183.
            if constexpr (QUANT) {
                if (ps <= 32) {
                    if (lane < pages) tma_load_4d(to + lane * ps * D, map, 0, 0, h, here, bar);
                } else {
#pragma unroll 1
                    for (int p = 0; p < pages; ++p) {
                        const int pg = __shfl_sync(0xffffffffu, here, p);
                        if (umma::elect_one()) tma_load_4d(to + p * ps * D, map, 0, 0, h, pg, bar);
                    }
                }
            } else {
#pragma unroll 1
                for (int p = 0; p < pages; p += 4) {
                    int pg[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) pg[k] = __shfl_sync(0xffffffffu, here, p + k);
                    if (!umma::elect_one()) continue;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (p + k >= pages) break;
#pragma unroll
                        for (int hf = 0; hf < D / 64; ++hf) tma_load_4d(to + hf * (G::KEYS * 128) + (p + k) * ps * 128, map, hf * 64, 0, h, pg[k], bar);
                    }
                }
            }
            if (++st == G::STAGES) {
                st = 0;
                ++use;
            }
        }
        if (!alive) break;
    }
    // nothing may land after the CTA has left, also when a wait ran out: the last fill of every stage
#pragma unroll 1
    for (int s = 0; s < G::STAGES; ++s) {
        const uint32_t fills = use + (s < st ? 1u : 0u);
        if (fills > 0) alive = wait_for(bar_full + s * 8, (fills - 1) & 1) && alive;
    }
    if (!alive && lane == 0) report(a.status, FST_DEV_TIMEOUT, blockIdx.x, G::WARPS);
}

}  // namespace fst
