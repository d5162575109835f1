// Chunk attention of many rows on tcgen05: pieces of prompts.
//
// An item is 256 rows of one sequence and K/V head in two groups of 128 (one if there are no more), its tiles are 128 keys:
//     S = Q K^T    tcgen05.mma M=128 N=128, both operands in shared memory
//     P            one thread per row: the row of S in registers, probabilities against a lazily moved reference, back to tensor memory
//     O += P V     tcgen05.mma, A = P in tensor memory, B = V (its rows are the summed index)
// A K/V tile comes in once for both groups, and while one group's products run the other group's warps take exponentials.
//
// What bounds a tile: the tensor cores need 2048 cycles for it at D 128 (1024 at D 64) and the 16 exponentials a clock of an SM 2048, so the
// hand-overs between the two have to stay short; it takes 3100 at either D.  Instructions come next: the roles' code is more than the
// instruction cache holds, so what runs in turn is kept small (one copy of the issuing code for both groups and short waits: 4096 tokens over 16400
// rows of 8 heads 929 -> 776 us, four prompts of 1024 tokens at D 64 69.5 -> 58.5).  The first is 1.05 - 1.25 PFLOP/s, as the power limit
// lets clocks be; the second has 3.5 items of 2 to 8 tiles a CTA, and their starts and ends are half of it.
// ptxas spills 432 bytes a thread in every instance, the softmax's most likely: its 128 scores, packed halves and sums.
// Tried and not kept: an issuing lane per group (263 -> 299 us at D 128: the groups fall into step; nothing at D 64, with S of the next tile
// ahead), 4 or 8 of 32 exponentials by a polynomial (0 to 4 %, slower for short items), two threads a row, steps of 64 keys, no exponentials for
// the parts of a tile that a warp does not see (branches among them: 56.7 -> 59.4 us for the prompts).
//
// Sixteen warps: 0-3 and 4-7 are the softmax groups; 8 loads K and V, lane j page j of a tile; one lane of 9 issues the products;
// 10 (and 11, where rows come one by one) bring the items' rows of Q; 12-15 look through the V tiles that not every row attends to all of (the diagonal, the
// sequence's end): rows past the end become zeros, elements that are not finite are taken out and noted, see fst_chunk.cuh.
// All hand-offs are mbarriers, the CTA's items follow one another without a break: Q of the next item arrives while the last
// tile of the one before is in the softmax.  Every wait is bounded; on expiry FST_DEV_TIMEOUT is recorded and
// all roles run out.
#pragma once

#include "fst_chunk.cuh"
#include "fst_chunk_map.cuh"
#include "fst_chunk_load.cuh"
#include "fst_umma.cuh"

namespace fst {

template <int D, bool QUANT>
struct ChunkUmmaGeo {
    static constexpr int ROWS = 256, KEYS = 128, THREADS = 512, OVER = 3;
    static constexpr int TILE = (D / 64) * umma::HALF;              // 128 rows
    static constexpr int QBUF = D == 128 ? 1 : 2;                   // items whose Q is there at a time
    static constexpr int RING = QUANT ? (D == 128 ? 3 : 6) : (D == 128 ? 4 : 8);
    static constexpr int RAW = QUANT ? (D == 128 ? 2 : 4) : 0;      // stages of 8-bit tiles: 128 rows of D bytes
    static constexpr int OFF_RING = QBUF * 2 * TILE, OFF_RAW = OFF_RING + RING * TILE;
    static constexpr int OFF_OUT = OFF_RAW + RAW * 128 * D;         // [softmax warp] 32 rows of 128 bytes on their way out
    static constexpr int OFF_BAR = OFF_OUT + 8 * 4096;
    static constexpr int BARS = 3 * RING + 2 * RAW + 4 * QBUF + 9;
    static constexpr int OFF_NOTE = (OFF_BAR + BARS * 8 + 15) & ~15;             // first item that held values that are not finite; tensor memory's address
    static constexpr int OFF_SCALES = OFF_NOTE + 16;                // [raw stage] 128 bytes
    static constexpr int OFF_PLAN = OFF_SCALES + RAW * 128;         // [stage] what a tile is to the issuing lane, see there
    static constexpr int OFF_RAW_PLAN = OFF_PLAN + RING * 4;        // [raw stage] the same
    static constexpr int OFF_PIECE = (OFF_RAW_PLAN + RAW * 4 + 15) & ~15;       // ChunkPiece
    static constexpr int BYTES = OFF_PIECE + 96 + 1024;             // + alignment
    // of 65536 registers a launch of 512 threads gets 128 each; the softmax warps take 192 and leave 64 to the others
    static constexpr int REGS_SOFTMAX = 192, REGS_OTHERS = 64;
};
static_assert(256 * 192 + 256 * 64 <= 512 * 128, "the split draws on what the launch was given");

__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
// whether one of the pairs of 16-bit values has an exponent of ones: the top bit of a half that overflows into it
template <typename T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u, U = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
    return ((w & E) + U) & 0x80008000u;
}
// Row r of an 8-bit tile (128 rows of D bytes, swizzled as TMA leaves them) times 2^(b - 127) into row r of a tile of T; zeros if `none`.
template <typename T, int D>
__device__ __forceinline__ void widen_row(uint32_t from, uint32_t to, int r, uint32_t b, bool none) {
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    // fp16: the conversion instruction and a multiplication by 2^e.  bf16: the value's bits under bf16's exponent are value * 2^-120, and one
    // multiplication by 2^(e + 120) gives the value.  The factor has to be one that T holds as a normal number, and no product may
    // leave T's range.  (fp16 by the bits as well: 406 us for 2048 tokens over 8192 rows, 322 by the instruction.)
    const int e = int(b) - 127;
    const bool quick = BF16 ? e <= 7 : e <= 7 && e >= -14;
    const uint32_t f = BF16 ? uint32_t(e + 247) << 7 : uint32_t(e + 15) << 10, ff = f | f << 16;
    const float scale = e8m0_value(b);
    const uint32_t src = from + r * D;
    auto put = [&](int chunk, const uint32_t *v) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(to + (chunk >> 3) * umma::HALF + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)),
                     "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]));
    };
    auto chunk_at = [&](int c) { return src + ((D == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4); };
    if (__all_sync(0xffffffffu, quick)) {                 // (one branch for the warp's rows: one for every 16 bytes cost 2000 cycles a tile)
        constexpr int AHEAD = 4;                          // loads ahead of their use
#pragma unroll
        for (int c0 = 0; c0 < D / 16; c0 += AHEAD) {
            uint32_t in[AHEAD][4];
#pragma unroll
            for (int c = 0; c < AHEAD; ++c) {
                const uint4 w = lds128(chunk_at(c0 + c));
                in[c][0] = none ? 0u : w.x; in[c][1] = none ? 0u : w.y; in[c][2] = none ? 0u : w.z; in[c][3] = none ? 0u : w.w;
            }
#pragma unroll
            for (int c = 0; c < AHEAD; ++c) {
                uint32_t out[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if constexpr (BF16) {                 // bytes 2 k, 2 k + 1 at the tops of 16-bit halves
                        const uint32_t x = __byte_perm(in[c][k >> 1], 0, k & 1 ? 0x3424 : 0x1404);
                        out[k] = (x & 0x80008000u) | ((x >> 4) & 0x07f007f0u);
                        asm("mul.rn.bf16x2 %0, %0, %1;\n" : "+r"(out[k]) : "r"(ff));
                    } else {
                        asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(out[k]) : "h"(uint16_t(in[c][k >> 1] >> (k & 1) * 16)));
                        asm("mul.rn.f16x2 %0, %0, %1;\n" : "+r"(out[k]) : "r"(ff));
                    }
                }
                put(2 * (c0 + c), out);
                put(2 * (c0 + c) + 1, out + 4);
            }
        }
    } else {
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
            const uint4 w = lds128(chunk_at(c));
            const uint32_t in[4] = {w.x, w.y, w.z, w.w};
            uint32_t out[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float2 x = e4m3_values(in[k >> 1] >> (k & 1) * 16);
                out[k] = none ? 0u : pack_cache<T>(x.x * scale, x.y * scale);
            }
            put(2 * c, out);
            put(2 * c + 1, out + 4);
        }
    }
}

template <typename T, int D, bool QUANT>
__global__ void __launch_bounds__(512, 1)
chunk_umma_kernel(const ChunkArgs a, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
    using namespace umma;
    using G = ChunkUmmaGeo<D, QUANT>;
    using MT = MmaTraits<T>;
    using Line = ChunkLine<G::ROWS, G::KEYS, G::OVER>;
    using Cursor = ChunkCursor<G::ROWS, G::KEYS, G::OVER>;
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    constexpr int DH = D / 64, TILE = G::TILE, RING = G::RING, QBUF = G::QBUF, RAW = G::RAW;

    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    extern __shared__ unsigned char smem_raw[];
    const uint32_t s_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char *smem = smem_raw + (s_base - smem_u32(smem_raw));
    // (the warp's number by a shuffle: so that its roles are known to be the same for its lanes; without, issuing the products took longer than they do:
    // 257 instead of 241 us for 2000 tokens over 9001 rows)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t s_ring = s_base + G::OFF_RING;
    // full / raw (landed, to be looked through) / empty of every stage; Q there / done with, [buffer][group]; S landed, halves of P written,
    // O complete of either group
    const uint32_t bar_full = s_base + G::OFF_BAR, bar_raw = bar_full + RING * 8, bar_empty = bar_raw + RING * 8, bar_q = bar_empty + RING * 8,
                   bar_qfree = bar_q + QBUF * 16, bar_s = bar_qfree + QBUF * 16, bar_p = bar_s + 16, bar_o = bar_p + 32, bar_end = bar_o + 16,
                   bar_in = bar_end + 8, bar_out = bar_in + RAW * 8;      // 8-bit tiles: landed, widened
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + G::OFF_NOTE + 8);
    volatile uint32_t *plan = reinterpret_cast<volatile uint32_t *>(smem + G::OFF_PLAN);
    volatile uint32_t *raw_plan = reinterpret_cast<volatile uint32_t *>(smem + G::OFF_RAW_PLAN);
    volatile int *note = reinterpret_cast<volatile int *>(smem + G::OFF_NOTE);
    if (warp == 8) {
        if (lane == 0) {
            for (int i = 0; i < 3 * RING; ++i) mbar_init(bar_full + i * 8, 1);
            for (int i = 0; i < 2 * QBUF; ++i) {
                mbar_init(bar_q + i * 8, a.q_boxes ? 1 : 64);
                mbar_init(bar_qfree + i * 8, 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(bar_s + i * 8, 1);
                mbar_init(bar_p + i * 16, 128);
                mbar_init(bar_p + i * 16 + 8, 128);
                mbar_init(bar_o + i * 8, 1);
            }
            mbar_init(bar_end, 1);
            for (int i = 0; i < 2 * RAW; ++i) mbar_init(bar_in + i * 8, i < RAW ? 33 : 1);
            *note = 0x7fffffff;
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
    } else if (warp == 9) {
        tmem_alloc_all(smem_u32(tmem_slot));
        fence_before_sync();
    }
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const Line line(a);
    using Piece = ChunkPiece<G::ROWS, G::KEYS, G::OVER>;
    static_assert(sizeof(Piece) <= 96, "its place");
    Piece &piece = *reinterpret_cast<Piece *>(smem + G::OFF_PIECE);
    piece.find(line);
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    Cursor me = piece.from;
    const int n_tiles = piece.tiles();
    const int where = blockIdx.x;
    // key tiles of the item that group g takes part in: none where it has no rows, and the first group sees less than the second
    auto group_tiles = [&](int g) {
        if (me.keys == 0 || (g == 1 && me.ql * a.group - me.qt * G::ROWS <= 128)) return 0;
        if (g == 1 || !a.causal) return me.tiles;
        return line.tiles_of(max(0, min(me.kv, me.kv - me.ql + min(by_group(a, me.qt * G::ROWS + 127), me.ql - 1) + 1)));
    };
    // keys that the item's first row (that of its group g) sees: tiles past it are not seen whole by every row
    auto first_limit = [&](int g = 0) { return a.causal ? min(me.kv, me.kv - me.ql + by_group(a, me.qt * G::ROWS + g * 128) + 1) : me.kv; };
    auto gave_up = [&]() { report(a.status, FST_DEV_TIMEOUT, where, warp); };

    // (Each side asks for its share inside its own branch, since code that both reach gets the lower count; and no function is called
    // there, wait_slow for instance: ptxas then finds no allocation.)
    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(G::REGS_OTHERS));
    if (warp == 8) {
        // ====== K and V, tile by tile; the page numbers of a tile are asked for a tile ahead ======
        const int ps = 1 << a.c.page_shift, npt = G::KEYS >> a.c.page_shift;
        int st = 0, page = 0;
        uint32_t use = 0, to_raw = 0, raw_fills = 0;      // fills of the current stage; bit s: stage s was last filled to be looked through, parity of such fills
        bool alive = true;
        auto look_up = [&]() {
            const int idx = me.tile * npt + lane;
            page = 0;
            if (lane < npt && idx * ps < me.keys)
                page = load(a.c.table + size_t(me.z) * a.c.width + idx);
        };
        // The plan of a tile goes into the word of its K's stage: 16-key steps with keys in them (bits 0-3), and of either group whether it
        // takes part (4, 5), whether the tile is its piece's first (6, 7) or last (8, 9), which buffer holds Q (10); 0: no more tiles.
        // The issuing lane has to hand over a product every 64 cycles and did not come to it (4400 instead of 2048 cycles a
        // tile) while it kept the place in the line itself.
        int tiles0 = 0, tiles1 = 0, item = 0;
        if (n_tiles > 0) look_up();
#pragma unroll 1
        for (int i = 0; i <= n_tiles && alive; ++i) {
            const int here = page, key0 = me.tile * G::KEYS, h = me.h, z = me.z;
            int pages = 0;                                // 0: an item that sees nothing
            bool edge = false;
            uint32_t word = 0;
            if (i < n_tiles) {
                const bool begins = i == 0 || me.tile == 0;
                if (begins) {
                    if (i > 0) ++item;
                    tiles0 = group_tiles(0);
                    tiles1 = group_tiles(1);
                }
                pages = (min(G::KEYS, me.keys - key0) + ps - 1) >> a.c.page_shift;
                edge = key0 + G::KEYS > first_limit();
                const uint32_t on = (me.tile < tiles0 ? 1u : 0u) | (me.tile < tiles1 ? 2u : 0u);
                const uint32_t ends = on & (i + 1 == n_tiles ? 3u : (me.tile + 1 == tiles0 ? 1u : 0u) | (me.tile + 1 == tiles1 ? 2u : 0u));
                word = uint32_t(min(8, (me.keys - key0 + 15) >> 4)) | on << 4 | (begins ? on << 6 : 0u) | ends << 8 | uint32_t(QBUF == 1 ? 0 : item & 1) << 10;
                me.next(line);
                if (i + 1 < n_tiles) look_up();
                if (pages <= 0) continue;
            }
            if constexpr (QUANT) {
#pragma unroll 1
                for (int v = 0; v < (i < n_tiles ? 2 : 1); ++v) {
                    const uint32_t bar = bar_in + st * 8;
                    if (use > 0) alive = __all_sync(0xffffffffu, wait_for(bar_out + st * 8, (use - 1) & 1));
                    if (!alive) break;
                    if (v == 0 && lane < pages && unsigned(here) >= unsigned(a.c.n_pages)) report(a.status, FST_DEV_INDEX_RANGE, z, key0 + lane * ps);
                    // sixteen rows' scales a lane, zeros for a bad page, as its rows are (see load_tiles)
                    const int p = lane >> (a.c.page_shift - 4), pg = __shfl_sync(0xffffffffu, here, p);
                    if (p < pages && lane < G::KEYS / 16) {
                        const uint8_t *from = v ? a.c.v_scale : a.c.k_scale;
                        const bool there = unsigned(pg) < unsigned(a.c.n_pages);
                        cp_async16(smem_u32(smem + G::OFF_SCALES + st * 128 + lane * 16), there ? from + ((size_t(pg) * a.H_kv + h) << a.c.page_shift) + (lane * 16 & (ps - 1)) : from, there);
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
                    if (lane == 0) {
                        if (v == 0) raw_plan[st] = word;
                        mbar_arrive_expect_tx(bar, (pages * D) << a.c.page_shift);
                    }
                    __syncwarp();
                    if (lane < pages) tma_load_4d(s_base + G::OFF_RAW + st * 128 * D + lane * ps * D, v ? &tm_v : &tm_k, 0, 0, h, here, bar);
                    if (++st == RAW) {
                        st = 0;
                        ++use;
                    }
                }
            } else {
#pragma unroll 1
            for (int v = 0; v < (i < n_tiles ? 2 : 1); ++v) {
                const uint32_t dst = s_ring + st * TILE, bar = (v && edge ? bar_raw : bar_full) + st * 8;
                if (use > 0) alive = __all_sync(0xffffffffu, wait_for(bar_empty + st * 8, (use - 1) & 1));
                if (!alive) break;
                to_raw = (to_raw & ~(1u << st)) | uint32_t(v && edge) << st;
                raw_fills ^= uint32_t(v && edge) << st;
                if (lane == 0) {
                    if (v == 0) plan[st] = word;
                    mbar_arrive_expect_tx(bar, (pages << a.c.page_shift) * D * 2);
                }
                __syncwarp();
                if (lane < pages) {
                    if (unsigned(here) >= unsigned(a.c.n_pages) && v == 0) report(a.status, FST_DEV_INDEX_RANGE, z, key0 + lane * ps);
#pragma unroll
                    for (int hf = 0; hf < DH; ++hf) tma_load_4d(dst + hf * HALF + lane * ps * 128, v ? &tm_v : &tm_k, hf * 64, 0, h, here, bar);
                }
                if (++st == RING) {
                    st = 0;
                    ++use;
                }
            }
            }
        }
        // nothing may land after the CTA has left, also when a wait ran out: the last fill of every stage
#pragma unroll 1
        for (int s = 0; s < (QUANT ? RAW : RING); ++s) {
            const uint32_t fills = use + (s < st ? 1u : 0u);
            if (QUANT && fills > 0) alive = wait_for(bar_in + s * 8, (fills - 1) & 1) && alive;
            else if (fills > 0) alive = wait_for((to_raw >> s & 1 ? bar_raw : bar_full) + s * 8, to_raw >> s & 1 ? (raw_fills >> s & 1) ^ 1u : (fills - 1) & 1) && alive;
        }
        if (!alive && lane == 0) gave_up();
    } else if (warp == 9) {
        // ====== products: for either group O += P V of the tile before, then S of this one ======
        if (elect_one()) {
            const uint32_t idesc_s = instr_desc(BF16, false, G::KEYS), idesc_pv = instr_desc(BF16, true, D);
            const uint64_t dq = smem_desc(s_base, 16), dk = smem_desc(s_ring, 16), dv = smem_desc(s_ring, HALF);
            int k_st = 0, v_st = 1;                       // stages of the next K and V
            uint32_t k_ph = 0, v_ph = 0, p_ph = 0, q_ph = 0;      // (bits: group, or Q's buffer and group)
            auto step2 = [&](int &st, uint32_t &ph) {
                st += 2;
                if (st >= RING) {
                    st -= RING;
                    ph ^= 1u;
                }
            };
            bool alive = true;
            uint32_t before = 0, now = 0;                 // the plan's words of the tile before and of this one
            // O += P V of the tile before, without a branch among the products where all of its 128 keys count
            auto second_product = [&](int g) {
                const uint32_t tmem_o = tmem + 256 + g * D, tmem_p = D == 128 ? tmem + g * 128 : tmem + 384 + g * 64;
                const uint64_t dvs = dv + uint64_t(v_st * (TILE >> 4));
                const int steps = before & 15u;
                const bool fresh = before >> (6 + g) & 1u;
                alive = wait_for(bar_p + g * 16, p_ph >> g & 1);
                if (!alive) return;
                fence_after_sync();
                if (steps == 8) {
                    mma_f16_ts(tmem_o, tmem_p, dvs, idesc_pv, !fresh);
#pragma unroll
                    for (int ks = 1; ks < 4; ++ks) mma_f16_ts(tmem_o, tmem_p + ks * 8, dvs + uint64_t((ks * 16 * 128) >> 4), idesc_pv, true);
                    alive = wait_for(bar_p + g * 16 + 8, p_ph >> g & 1);
                    fence_after_sync();
#pragma unroll
                    for (int ks = 4; ks < 8; ++ks) mma_f16_ts(tmem_o, tmem_p + ks * 8, dvs + uint64_t((ks * 16 * 128) >> 4), idesc_pv, true);
                } else {
                    alive = wait_for(bar_p + g * 16 + 8, p_ph >> g & 1);
                    fence_after_sync();
#pragma unroll 1
                    for (int ks = 0; ks < steps; ++ks) mma_f16_ts(tmem_o, tmem_p + ks * 8, dvs + uint64_t((ks * 16 * 128) >> 4), idesc_pv, ks > 0 || !fresh);
                }
                p_ph ^= 1u << g;
                if (before >> (8 + g) & 1u) mma_commit(bar_o + g * 8);
                if ((before >> 4 & 3u) >> g == 1u) {      // the last group to read this V
                    mma_commit(bar_empty + v_st * 8);
                    step2(v_st, v_ph);
                }
            };
            auto first_product = [&](int g) {
                const uint32_t tmem_s = tmem + g * 128, at = (now >> 10 & 1u) * 2 + g;
                if (now >> (6 + g) & 1u) {
                    alive = wait_for(bar_q + at * 8, q_ph >> at & 1);
                    q_ph ^= 1u << at;
                    if (!alive) return;
                    fence_after_sync();
                }
                const uint64_t dqs = dq + uint64_t(at * (TILE >> 4)), dks = dk + uint64_t(k_st * (TILE >> 4));
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint64_t koff = ((ks >> 2) * HALF + (ks & 3) * 32) >> 4;
                    mma_f16(tmem_s, dqs + koff, dks + koff, idesc_s, ks > 0);
                }
                mma_commit(bar_s + g * 8);
                if (now >> (8 + g) & 1u) mma_commit(bar_qfree + at * 8);
                if ((now >> 4 & 3u) >> g == 1u) {
                    mma_commit(bar_empty + k_st * 8);
                    step2(k_st, k_ph);
                }
            };
#pragma unroll 1
            while (alive) {
                alive = wait_for(bar_full + k_st * 8, k_ph);
                if (!alive) break;
                fence_after_sync();
                now = plan[k_st];
                if (before != 0u) {
                    alive = wait_for(bar_full + v_st * 8, v_ph);
                    fence_after_sync();
                }
#pragma unroll 1
                for (int g = 0; g < 2; ++g) {             // (one copy of the code for both groups: see the note on instructions above)
                    if (alive && (before >> (4 + g) & 1u)) second_product(g);
                    if (alive && (now >> (4 + g) & 1u)) first_product(g);
                }
                before = now;
                if (now == 0u) break;
            }
            mma_commit(bar_end);                          // all products are done before tensor memory is given back
            if (!(wait_for(bar_end, 0) && alive)) gave_up();
        }
    } else if (warp == 10 || warp == 11) {
        // ====== rows of Q, an item (D 128) or two ahead of its products' end: one box where whole tokens fit a tile (3 us sooner) ======
        // With boxes this is warp 10's role, which waits for a buffer as a whole before it fills that.  (Threads that wait and hold up no fill by it may
        // miss a phase and the one behind it; then they wait for a third, which need not come.)
        const int t64 = tid - 320;
        if (!a.q_boxes || warp == 10) {
        uint32_t qfree_ph = 0, used = 0;                  // bit: buffer and group
        bool alive = true;
        int item = 0, len;
#pragma unroll 1
        for (int i = 0; i < n_tiles; i += len, ++item) {
            len = min(me.tiles - me.tile, n_tiles - i);
            if (t64 == 0 && me.h == 0 && me.qt == 0 && (me.kv != load(a.kv_lens + me.z) || (a.q_lens != nullptr && me.ql != load(a.q_lens + me.z))))
                report(a.status, FST_DEV_INDEX_RANGE, me.z, load(a.kv_lens + me.z));
#pragma unroll 1
            for (int g = 0; g < 2; ++g) {
                if (group_tiles(g) <= me.tile) continue;      // (a piece may begin behind the first group's last tile)
                const int at = (QBUF == 1 ? 0 : (item & 1) * 2) + g;
                if (used >> at & 1) {                 // the products that read what is there
                    if (alive) alive = __all_sync(0xffffffffu, wait_for(bar_qfree + at * 8, qfree_ph >> at & 1));
                    qfree_ph ^= 1u << at;
                }
                used |= 1u << at;
                const int row0 = me.qt * G::ROWS + g * 128, bar = bar_q + at * 8;
                if (a.q_boxes) {                          // heads of a token side by side, tokens behind the tensor's end as zeros
                    if (t64 == 0) {
                        mbar_arrive_expect_tx(bar, TILE);
#pragma unroll
                        for (int hf = 0; hf < DH; ++hf) tma_load_4d(s_base + at * TILE + hf * HALF, &tm_q, hf * 64, me.h * a.group, by_group(a, row0), me.z, bar);
                    }
                    continue;
                }
                constexpr int CH = D / 8, STEP = 64 / CH;
                const int c = t64 % CH;
                const uint32_t dst = s_base + at * TILE + (c >> 3) * HALF;
                int tok = by_group(a, row0 + t64 / CH), sub = row0 + t64 / CH - tok * a.group;
#pragma unroll 4
                for (int r = t64 / CH; r < 128; r += STEP) {
                    const bool there = tok < me.ql;
                    const T *src = static_cast<const T *>(a.q) + me.z * a.qs_z + (me.h * a.group + sub) * a.qs_h + tok * a.qs_n + c * 8;
                    cp_async16(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4), there ? src : static_cast<const T *>(a.q), there);
#pragma unroll 1
                    for (sub += STEP; sub >= a.group; sub -= a.group) ++tok;
                }
                cp_async_commit();
                cp_async_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
            }
            me.tile += len - 1;
            if (i + len < n_tiles) me.next(line);
        }
        if (!alive && lane == 0) gave_up();
        }
    } else {
        const int t128 = tid - 384;
        bool alive = true;
        if constexpr (QUANT) {
            // ====== 8-bit tiles into 16-bit ones, a thread per row: a scale each, and rows of a swizzled tile are free of conflicts ======
            int st = 0, rs = 0, item = 0;
            uint32_t use = 0, turn = 0;
#pragma unroll 1
            for (int i = 0; i <= n_tiles; ++i) {
                if (i > 0 && i < n_tiles && me.tile == 0) ++item;
                const int key0 = me.tile * G::KEYS;
                if (i == n_tiles || me.keys > 0) {
                    const bool edge = key0 + G::KEYS > first_limit();
                    const int have = me.kv - key0;        // V rows behind the sequence's end become zeros
#pragma unroll 1
                    for (int v = 0; v < (i < n_tiles ? 2 : 1); ++v) {
                        if (alive) alive = wait_for(bar_in + rs * 8, turn & 1);
                        if (alive && use > 0) alive = wait_for(bar_empty + st * 8, (use - 1) & 1);
                        if (i < n_tiles) {
                            const uint32_t b = smem[G::OFF_SCALES + rs * 128 + t128];
                            bool none = false;            // a V row that is left out
                            if (v) {
                                none = t128 >= have;
                                if (edge && !none && b == 255u && t128 < ((me.keys - key0 + 15) & ~15)) {
                                    none = true;
                                    atomicMin_block(const_cast<int *>(note), item);
                                }
                            }
                            widen_row<T, D>(s_base + G::OFF_RAW + rs * 128 * D, s_ring + st * TILE, t128, b, none);
                            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                        }
                        asm volatile("bar.sync 2, 128;\n" ::: "memory");
                        if (t128 == 0) {
                            if (v == 0) plan[st] = raw_plan[rs];
                            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar_full + st * 8) : "memory");
                            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar_out + rs * 8) : "memory");
                        }
                        if (++st == RING) {
                            st = 0;
                            ++use;
                        }
                        if (++rs == RAW) {
                            rs = 0;
                            ++turn;
                        }
                    }
                }
                if (i + 1 < n_tiles) me.next(line);
            }
        } else {
        // ====== V tiles that not every row attends to all of ======
        int st = 1, item = 0;                             // stage of the tile's V
        uint32_t raw_ph = 0;
#pragma unroll 1
        for (int i = 0; i < n_tiles; ++i) {
            if (i > 0 && me.tile == 0) ++item;
            const int key0 = me.tile * G::KEYS;
            if (me.keys > 0) {
                if (key0 + G::KEYS > first_limit()) {
                    if (alive) alive = wait_for(bar_raw + st * 8, raw_ph >> st & 1);
                    raw_ph ^= 1u << st;
                    // Rows that take part, whole 16-key steps of them (what lies behind may be anything, and a look there would find it), and
                    // rows of the sequence: those behind become zeros.  Neighbouring threads have neighbouring chunks of 16 bytes.
                    const int rows = (min(G::KEYS, me.keys - key0) + 15) & ~15, have = me.kv - key0;
                    constexpr int PER = D / 8;            // chunks of a thread
                    unsigned char *tile = smem + G::OFF_RING + st * TILE;
                    uint32_t odd = have < rows;
#pragma unroll
                    for (int k = 0; k < PER; ++k) {
                        const int at = (k * 128 + t128) * 16;
                        const uint4 w = *reinterpret_cast<const uint4 *>(tile + at);
                        const uint32_t bits = odd_bits<T>(w.x) | odd_bits<T>(w.y) | odd_bits<T>(w.z) | odd_bits<T>(w.w);
                        odd |= at % HALF / 128 < rows ? bits : 0u;
                    }
                    if (odd != 0u) {                      // (the order of a row's chunks does not matter)
                        bool met = false;
#pragma unroll 1
                        for (int k = 0; k < PER; ++k) {
                            const int at = (k * 128 + t128) * 16, r = at % HALF / 128;
                            if (r >= rows) continue;
                            uint4 w = *reinterpret_cast<const uint4 *>(tile + at);
                            if (r >= have) {
                                w = make_uint4(0, 0, 0, 0);
                            } else {
                                met = keep_finite<T>(w.x, 2) || met;
                                met = keep_finite<T>(w.y, 2) || met;
                                met = keep_finite<T>(w.z, 2) || met;
                                met = keep_finite<T>(w.w, 2) || met;
                            }
                            *reinterpret_cast<uint4 *>(tile + at) = w;
                        }
                        if (met) atomicMin_block(const_cast<int *>(note), item);
                        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    }
                    asm volatile("bar.sync 2, 128;\n" ::: "memory");
                    if (t128 == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar_full + st * 8) : "memory");
                }
                st += 2;
                if (st >= RING) st -= RING;
            }
            if (i + 1 < n_tiles) me.next(line);
        }
        }
        if (!alive && t128 == 0) gave_up();
        if (t128 == 0 && a.part != nullptr) leave_cut<D>(a, me, piece.total, n_tiles);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(G::REGS_SOFTMAX));
        // ====== softmax: two groups of 128 threads, one thread per row ======
        const int r = tid & 127, g = tid >> 7;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + g * 128 + lanes, tmem_o = tmem + 256 + g * D + lanes, tmem_p = D == 128 ? tmem_s : tmem + 384 + g * 64 + lanes;
        const uint32_t my_s = bar_s + g * 8, my_p = bar_p + g * 16;
        const float c2 = a.scale_log2;
        constexpr float LIFT = BF16 ? 0.f : kLift - 8.f;  // (a reference may be passed by 2^8, see below)
        uint32_t s_ph = 0, o_ph = 0;
        int item = 0, len;
        bool alive = true;
        auto announce = [&](uint32_t bar) {
            tmem_st_wait();
            fence_before_sync();
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
        };
        // probabilities of two scores, into the row's sum and as a pair of 16-bit values
        auto exp2_pair = [&](uint64_t x, uint64_t &sum, uint32_t &out) {
            float p0, p1;
            unpair(x, p0, p1);
            p0 = fast_exp2(p0);
            p1 = fast_exp2(p1);
            sum = add2(sum, pair(p0, p1));
            out = MT::pack(p0, p1);
        };
#pragma unroll 1
        for (int i = 0; i < n_tiles; i += len, ++item) {
            len = min(me.tiles - me.tile, n_tiles - i);
            const int mine = min(max(group_tiles(g) - me.tile, 0), len);         // tiles of the piece that my group takes
            const int row = me.qt * G::ROWS + g * 128 + r, tok = by_group(a, row);
            const int limit = tok >= me.ql ? 0 : a.causal ? min(me.kv, me.kv - me.ql + tok + 1) : me.kv;
            float m_ref = -INFINITY, l = 0.f;
            // keys of the tile that I see, and that every row of my group sees
            int n = limit - me.tile * G::KEYS, n_all = first_limit(g) - me.tile * G::KEYS;
#pragma unroll 1
            for (int j = 0; j < mine; ++j, n -= G::KEYS, n_all -= G::KEYS) {
                if (alive) alive = __all_sync(0xffffffffu, wait_for(my_s, s_ph));
                s_ph ^= 1u;
                fence_after_sync();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s[c], tmem_s + c * 32);
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_wait(s[c]);
                if (n_all < G::KEYS) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (c * 32 + k >= n) s[c][k] = 0xff800000u;
                }
                // The exponentials of the first half are taken against the reference that the tiles before left, and the row's maximum in
                // between (an exponential keeps its unit for 8 cycles, a maximum fits in).  Where a row has outgrown the reference by more
                // than 2^8 it moves, what was summed so far with it, and they are taken again.  On a piece's first tile the maximum comes first.
                uint64_t l2[2], scale2 = pair(c2, c2), shift2;
                if (j == 0) {
                    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 32; k += 4) {
                            m0 = max3(m0, __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
                            m1 = max3(m1, __uint_as_float(s[c][k + 2]), __uint_as_float(s[c][k + 3]));
                        }
                    m_ref = fmaxf(m0, m1);
                }
#pragma unroll 1
                for (int again = 0;; ++again) {
                    const float mu = m_ref == -INFINITY ? 0.f : m_ref * c2 - LIFT;
                    shift2 = pair(-mu, -mu);
                    float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
                    l2[0] = l2[1] = 0;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t packed[16];
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            const float x0 = __uint_as_float(s[c][k]), x1 = __uint_as_float(s[c][k + 1]);
                            exp2_pair(fma2(pair(x0, x1), scale2, shift2), l2[(k >> 1) & 1], packed[k >> 1]);
                            if ((k >> 1) & 1) {
                                m0 = max3(m0, x0, x1);
                                m1 = max3(m1, __uint_as_float(s[c + 2][k]), __uint_as_float(s[c + 2][k + 1]));
                            } else {
                                m2 = max3(m2, x0, x1);
                                m3 = max3(m3, __uint_as_float(s[c + 2][k]), __uint_as_float(s[c + 2][k + 1]));
                            }
                        }
                        tmem_st16(tmem_p + c * 16, packed);       // (nobody reads it before it is announced)
                    }
                    const float mx = max3(fmaxf(m0, m1), m2, m3);
                    const bool up = (mx - m_ref) * c2 > 8.f;
                    if (again > 0 || j == 0 || !__any_sync(0xffffffffu, up)) break;
                    // (S of this tile has landed: O += P V of the one before is done)
                    const float alpha = up ? fast_exp2((m_ref - mx) * c2) : 1.f;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t o[16];
                        tmem_ld16(o, tmem_o + c0);
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                        tmem_st16(tmem_o + c0, o);
                    }
                    tmem_st_wait();
                    l *= alpha;
                    if (up) m_ref = mx;
                }
                announce(my_p);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t packed[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 2)
                        exp2_pair(fma2(pair(__uint_as_float(s[c + 2][k]), __uint_as_float(s[c + 2][k + 1])), scale2, shift2), l2[(k >> 1) & 1], packed[k >> 1]);
                    tmem_st16(tmem_p + 32 + c * 16, packed);
                }
                announce(my_p + 8);
                float la, lb;
                unpair(add2(l2[0], l2[1]), la, lb);
                l += la + lb;
            }

            // ---- the piece's rows: the output where it is the whole item, else sums for the merge
            if (mine > 0) {
                if (alive) alive = __all_sync(0xffffffffu, wait_for(bar_o + g * 8, o_ph));
                o_ph ^= 1u;
                fence_after_sync();
            }
            const bool bad = mine > 0 && *note <= item;   // (then also for the items behind: a look in vain)
            const bool whole = len == me.tiles, there = tok < me.ql;
            const int look_from = max(max(first_limit(), 0) & ~(G::KEYS - 1), me.tile * G::KEYS), look_to = min(limit, (me.tile + len) * G::KEYS);
            const float f = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l, mu = m_ref == -INFINITY ? -INFINITY : m_ref * c2 - LIFT;
            const int head = me.h * a.group + (row - tok * a.group);
            const size_t slot = (size_t(2) * blockIdx.x + (me.tile == 0 ? 1 : 0)) * G::ROWS + g * 128 + r;
            // The rows leave through shared memory, four whole lines of 128 bytes a store: by 16 or 32 bytes of 32 rows at a time a piece took
            // 5 us to write, by lines 3.3.
            const uint32_t out_at = s_base + G::OFF_OUT + warp * 4096;
            const unsigned long long to = reinterpret_cast<unsigned long long>(
                whole ? static_cast<void *>(static_cast<T *>(a.o) + me.z * a.os_z + head * a.os_h + tok * a.os_n) : static_cast<void *>(a.part + slot * D));
            const unsigned rows_there = __ballot_sync(0xffffffffu, there);
            const int width = whole ? 64 : 32;            // columns in 128 bytes
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += width) {
#pragma unroll 1
                for (int c1 = 0; c1 < width; c1 += 32) {
                    float o[32];
                    if (mine > 0) {
                        uint32_t w[32];
                        tmem_ld32(w, tmem_o + c0 + c1);
                        tmem_ld_wait(w);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __uint_as_float(w[k]);
                        if (bad) add_not_finite<T, 32, QUANT>(a, me.z, me.h, look_from, look_to, c0 + c1, o);
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = 0.f;
                    }
                    auto put = [&](int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(out_at + lane * 128 + ((chunk ^ (lane & 7)) << 4)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
                    };
                    if (whole) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8)
                            put((c1 + k) >> 3, MT::pack(o[k] * f, o[k + 1] * f), MT::pack(o[k + 2] * f, o[k + 3] * f), MT::pack(o[k + 4] * f, o[k + 5] * f),
                                MT::pack(o[k + 6] * f, o[k + 7] * f));
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            put(k >> 2, __float_as_uint(o[k]), __float_as_uint(o[k + 1]), __float_as_uint(o[k + 2]), __float_as_uint(o[k + 3]));
                    }
                }
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int from = k * 4 + (lane >> 3), chunk = lane & 7;
                    const uint4 v = lds128(out_at + from * 128 + ((chunk ^ (from & 7)) << 4));
                    unsigned char *dst = reinterpret_cast<unsigned char *>(__shfl_sync(0xffffffffu, to, from));
                    if (rows_there >> from & 1u) *reinterpret_cast<uint4 *>(dst + c0 * (whole ? 2 : 4) + chunk * 16) = v;
                }
                __syncwarp();
            }
            if (there) {
                if (!whole) reinterpret_cast<float2 *>(a.part + chunk_stats_at(gridDim.x, G::ROWS, D))[slot] = make_float2(mu, l);
                else if (a.lse != nullptr) a.lse[(size_t(me.z) * a.H + head) * a.n_q + tok] = l == 0.f ? -INFINITY : mu + log2f(l);
            }
            fence_before_sync();                          // (O has been read before the next item's P is announced)
            me.tile += len - 1;
            if (i + len < n_tiles) me.next(line);
        }
        if (!alive && lane == 0) gave_up();
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    if (warp == 9) {
        fence_after_sync();
        tmem_free_all(tmem);
    }
}

template <typename T, int D, bool QUANT>
static cudaError_t launch_chunk_umma(const ChunkArgs &a, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, int n_ctas, cudaStream_t stream) {
    using G = ChunkUmmaGeo<D, QUANT>;
    static_assert(G::BYTES <= 227 * 1024, "one CTA's shared memory");
    static DeviceOnce configured;
    const cudaError_t ce = configured.run([&] {
        return cudaFuncSetAttribute(chunk_umma_kernel<T, D, QUANT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::BYTES);
    });
    if (ce != cudaSuccess) return ce;
    const cudaError_t e = launch_serialised(chunk_umma_kernel<T, D, QUANT>, dim3(n_ctas), dim3(G::THREADS), G::BYTES, stream, a, tq, tk, tv);
    if (e != cudaSuccess || !chunk_splits(a, G::KEYS)) return e;
    return launch_chunk_combine<T, D, G::ROWS>(a, n_ctas, stream);
}

}  // namespace fst
