// Chunk attention of many rows on tcgen05: pieces of prompts.
//
// An item is 256 rows of one sequence and K/V head in two groups of 128 (one if there are no more), its tiles are 128 keys:
//     S = Q K^T    tcgen05.mma M=128 N=128, both operands in shared memory
//     P            one thread per row: the row of S in registers, probabilities against a lazily moved reference, back to tensor memory
//     O += P V     tcgen05.mma, A = P in tensor memory, B = V (its rows are the summed index)
// A K/V tile comes in once for both groups, and while one group's products run the other group's warps take exponentials.
//
// What bounds a tile at D 128: the tensor cores need 4 x 512 cycles for it and the 16 exponentials a clock of an SM
// just as many, so the hand-overs between the two have to stay short.
//
// Sixteen warps: 0-3 and 4-7 are the softmax groups; 8 loads K and V, lane j page j of a tile; one lane of 9 issues the products;
// 10 and 11 bring the items' rows of Q; 12-15 look through the V tiles that not every row attends to all of (the diagonal, the
// sequence's end): rows past the end become zeros, elements that are not finite are taken out and noted, see fst_chunk.cuh.
// All hand-offs are mbarriers, the CTA's items follow one another without a break: Q of the next item arrives while the last
// tile of the one before is in the softmax.  Every wait is bounded; on expiry FST_DEV_TIMEOUT is recorded and
// all roles run out.
#pragma once

#include "fst_chunk.cuh"
#include "fst_chunk_map.cuh"
#include "fst_umma.cuh"

namespace fst {

template <int D>
struct ChunkUmmaGeo {
    static constexpr int ROWS = 256, KEYS = 128, THREADS = 512;
    static constexpr int TILE = (D / 64) * umma::HALF;              // 128 rows
    static constexpr int QBUF = D == 128 ? 1 : 2;                   // items whose Q is there at a time
    static constexpr int RING = D == 128 ? 5 : 8;
    static constexpr int OFF_RING = QBUF * 2 * TILE, OFF_BAR = OFF_RING + RING * TILE;
    static constexpr int BARS = 3 * RING + 4 * QBUF + 9;
    static constexpr int OFF_NOTE = OFF_BAR + BARS * 8;             // first item that held values that are not finite; tensor memory's address
    static constexpr int BYTES = OFF_NOTE + 16 + 1024;              // + alignment
    // of 65536 registers a launch of 512 threads gets 128 each; the softmax warps take 192 and leave 64 to the others
    static constexpr int REGS_SOFTMAX = 192, REGS_OTHERS = 64;
};
static_assert(256 * 192 + 256 * 64 <= 512 * 128, "the split draws on what the launch was given");

// 2^x for x up to 127, zero from -127 down: Cody and Waite's split x = n + f, f in [-1/2, 1/2], and the polynomial of degree 4 with the smallest
// relative error on it (Remez' exchange; 2.6e-6), two at a time.
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void exp2_poly(uint64_t x, float &p0, float &p1) {
    using namespace umma;
    const float kRound = 12582912.f;                      // 1.5 * 2^23: adding it leaves round(x) in the low bits
    float a, b;
    unpair(x, a, b);
    x = pair(fmaxf(a, -127.f), fmaxf(b, -127.f));
    const uint64_t t = add2(x, pair(kRound, kRound)), f = add2(x, fma2(t, pair(-1.f, -1.f), pair(kRound, kRound)));
    uint64_t r = fma2(f, pair(0.009570102207362652f, 0.009570102207362652f), pair(0.05591785907745361f, 0.05591785907745361f));
    r = fma2(r, f, pair(0.240247443318367f, 0.240247443318367f));
    r = fma2(r, f, pair(0.6931217908859253f, 0.6931217908859253f));
    r = fma2(r, f, pair(0.9999992847442627f, 0.9999992847442627f));
    float t0, t1;
    unpair(t, t0, t1);                                    // 2^n by its exponent; that of -127 is zero, and so is the result
    r = mul2(r, pair(__uint_as_float((__float_as_uint(t0) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(t1) << 23) + 0x3f800000u)));
    unpair(r, p0, p1);
}
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
template <typename T, int D>
__global__ void __launch_bounds__(512, 1)
chunk_umma_kernel(const ChunkArgs a, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
    using namespace umma;
    using G = ChunkUmmaGeo<D>;
    using MT = MmaTraits<T>;
    using Line = ChunkLine<G::ROWS, G::KEYS>;
    using Cursor = ChunkCursor<G::ROWS, G::KEYS>;
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    constexpr int DH = D / 64, TILE = G::TILE, RING = G::RING, QBUF = G::QBUF;

    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    extern __shared__ unsigned char smem_raw[];
    const uint32_t s_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char *smem = smem_raw + (s_base - smem_u32(smem_raw));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t s_ring = s_base + G::OFF_RING;
    // full / raw (landed, to be looked through) / empty of every stage; Q there / done with, [buffer][group]; S landed, halves of P written,
    // O complete of either group
    const uint32_t bar_full = s_base + G::OFF_BAR, bar_raw = bar_full + RING * 8, bar_empty = bar_raw + RING * 8, bar_q = bar_empty + RING * 8,
                   bar_qfree = bar_q + QBUF * 16, bar_s = bar_qfree + QBUF * 16, bar_p = bar_s + 16, bar_o = bar_p + 32, bar_end = bar_o + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + G::OFF_NOTE + 8);
    volatile int *note = reinterpret_cast<volatile int *>(smem + G::OFF_NOTE);
    if (warp == 8) {
        if (lane == 0) {
            for (int i = 0; i < 3 * RING; ++i) mbar_init(bar_full + i * 8, 1);
            for (int i = 0; i < 2 * QBUF; ++i) {
                mbar_init(bar_q + i * 8, 64);
                mbar_init(bar_qfree + i * 8, 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(bar_s + i * 8, 1);
                mbar_init(bar_p + i * 16, 128);
                mbar_init(bar_p + i * 16 + 8, 128);
                mbar_init(bar_o + i * 8, 1);
            }
            mbar_init(bar_end, 1);
            *note = 0x7fffffff;
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
    } else if (warp == 9) {
        tmem_alloc_all(smem_u32(tmem_slot));
        fence_before_sync();
    }
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    const Line line(a);
    const long long total = Cursor::total(line), first = chunk_first(total, blockIdx.x, gridDim.x);
    const int n_tiles = int(chunk_first(total, blockIdx.x + 1, gridDim.x) - first);
    Cursor me;
    if (n_tiles > 0) me.seek(line, first);
    const int where = blockIdx.x;
    // key tiles of the item that group g takes part in: none where it has no rows, and the first group sees less than the second
    auto group_tiles = [&](int g) {
        if (me.keys == 0 || (g == 1 && me.ql * a.group - me.qt * G::ROWS <= 128)) return 0;
        if (g == 1 || !a.causal) return me.tiles;
        return line.tiles_of(max(0, min(me.kv, me.kv - me.ql + min((me.qt * G::ROWS + 127) / a.group, me.ql - 1) + 1)));
    };
    // keys that the item's first row sees: tiles past it are not seen whole by every row
    auto first_limit = [&]() { return a.causal ? min(me.kv, me.kv - me.ql + me.qt * G::ROWS / a.group + 1) : me.kv; };

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
                page = a.c.table == nullptr ? me.z * a.c.width + idx : __ldg(a.c.table + size_t(me.z) * a.c.width + idx);
        };
        if (n_tiles > 0) look_up();
#pragma unroll 1
        for (int i = 0; i < n_tiles && alive; ++i) {
            const int here = page, key0 = me.tile * G::KEYS, h = me.h, z = me.z;
            const int pages = (min(G::KEYS, me.keys - key0) + ps - 1) >> a.c.page_shift;      // 0: an item that sees nothing
            const bool edge = key0 + G::KEYS > first_limit();
            me.next(line);
            if (i + 1 < n_tiles) look_up();
            if (pages <= 0) continue;
#pragma unroll 1
            for (int v = 0; v < 2; ++v) {
                const uint32_t dst = s_ring + st * TILE, bar = (v && edge ? bar_raw : bar_full) + st * 8;
                if (use > 0) alive = __all_sync(0xffffffffu, mbar_wait(bar_empty + st * 8, (use - 1) & 1, a.status, where));
                if (!alive) break;
                to_raw = (to_raw & ~(1u << st)) | uint32_t(v && edge) << st;
                raw_fills ^= uint32_t(v && edge) << st;
                if (lane == 0) mbar_arrive_expect_tx(bar, (pages << a.c.page_shift) * D * 2);
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
        // nothing may land after the CTA has left, also when a wait ran out: the last fill of every stage
#pragma unroll 1
        for (int s = 0; s < RING; ++s) {
            const uint32_t fills = use + (s < st ? 1u : 0u);
            if (fills > 0) mbar_wait((to_raw >> s & 1 ? bar_raw : bar_full) + s * 8, to_raw >> s & 1 ? (raw_fills >> s & 1) ^ 1u : (fills - 1) & 1, a.status, where);
        }
    } else if (warp == 9) {
        // ====== products: for either group O += P V of the tile before, then S of this one ======
        if (elect_one() && n_tiles > 0) {
            const uint32_t idesc_s = instr_desc(BF16, false, G::KEYS), idesc_pv = instr_desc(BF16, true, D);
            const uint64_t dq = smem_desc(s_base, 16), dk = smem_desc(s_ring, 16), dv = smem_desc(s_ring, HALF);
            int k_st = 0, v_st = 1;                       // stages of the next K and V
            uint32_t k_ph = 0, v_ph = 0, p_ph = 0, q_ph = 0;                                  // (bit g: group g)
            auto step2 = [&](int &st, uint32_t &ph) {
                st += 2;
                if (st >= RING) {
                    st -= RING;
                    ph ^= 1u;
                }
            };
            bool alive = true;
            int item = 0;
            // of the tile before: 16-key steps with keys in them, and of either group whether it takes part (bit g), whether this was its
            // piece's first or last tile
            int steps_b = 0;
            uint32_t on_b = 0, first_b = 0, last_b = 0;
            int tiles_g[2] = {0, 0};
#pragma unroll 1
            for (int i = 0; i <= n_tiles && alive; ++i) {
                const bool real = i < n_tiles && me.keys > 0;
                if (real && (i == 0 || me.tile == 0)) {
                    tiles_g[0] = group_tiles(0);
                    tiles_g[1] = group_tiles(1);
                }
                if (i > 0 && i < n_tiles && me.tile == 0) ++item;
                const int qbuf = QBUF == 1 ? 0 : item & 1;
                const int steps = real ? min(8, (me.keys - me.tile * G::KEYS + 15) >> 4) : 0;
                uint32_t on = 0, first_here = 0, last_here = 0;
                if (real) {
#pragma unroll
                    for (int g = 0; g < 2; ++g)
                        if (me.tile < tiles_g[g]) {
                            on |= 1u << g;
                            if (i == 0 || me.tile == 0) first_here |= 1u << g;
                            if (me.tile + 1 == tiles_g[g] || i + 1 == n_tiles) last_here |= 1u << g;
                        }
                }
#pragma unroll 1
                for (int g = 0; g < 2 && alive; ++g) {
                    const uint32_t tmem_s = tmem + g * 128, tmem_o = tmem + 256 + g * D, tmem_p = D == 128 ? tmem_s : tmem + 384 + g * 64;
                    if (on_b >> g & 1) {
                        if (g == 0 || on_b == 2) alive = mbar_wait(bar_full + v_st * 8, v_ph, a.status, where);
                        alive = alive && mbar_wait(bar_p + g * 16, p_ph >> g & 1, a.status, where);
                        if (!alive) break;
                        fence_after_sync();
                        const uint64_t dvs = dv + uint64_t(v_st * (TILE >> 4));
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            if (ks == 4) {
                                alive = mbar_wait(bar_p + g * 16 + 8, p_ph >> g & 1, a.status, where);
                                fence_after_sync();
                            }
                            if (ks < steps_b) mma_f16_ts(tmem_o, tmem_p + ks * 8, dvs + uint64_t((ks * 16 * 128) >> 4), idesc_pv, ks > 0 || !(first_b >> g & 1));
                        }
                        p_ph ^= 1u << g;
                        if (last_b >> g & 1) mma_commit(bar_o + g * 8);
                        if (on_b >> g == 1) {             // the last group to read this V
                            mma_commit(bar_empty + v_st * 8);
                            step2(v_st, v_ph);
                        }
                    }
                    if ((on >> g & 1) && alive) {
                        if (g == 0 || on == 2) alive = mbar_wait(bar_full + k_st * 8, k_ph, a.status, where);
                        if (first_here >> g & 1) {
                            alive = alive && mbar_wait(bar_q + (qbuf * 2 + g) * 8, q_ph >> (qbuf * 2 + g) & 1, a.status, where);
                            q_ph ^= 1u << (qbuf * 2 + g);
                        }
                        if (!alive) break;
                        fence_after_sync();
                        const uint64_t dqs = dq + uint64_t((qbuf * 2 + g) * (TILE >> 4)), dks = dk + uint64_t(k_st * (TILE >> 4));
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks) {
                            const uint64_t koff = ((ks >> 2) * HALF + (ks & 3) * 32) >> 4;
                            mma_f16(tmem_s, dqs + koff, dks + koff, idesc_s, ks > 0);
                        }
                        mma_commit(bar_s + g * 8);
                        if (last_here >> g & 1) mma_commit(bar_qfree + (qbuf * 2 + g) * 8);
                        if (on >> g == 1) {
                            mma_commit(bar_empty + k_st * 8);
                            step2(k_st, k_ph);
                        }
                    }
                }
                steps_b = steps;
                on_b = on;
                first_b = first_here;
                last_b = last_here;
                if (i + 1 < n_tiles) me.next(line);
            }
            mma_commit(bar_end);                          // all products are done before tensor memory is given back
            mbar_wait(bar_end, 0, a.status, where);
        }
    } else if (warp == 10 || warp == 11) {
        // ====== rows of Q, an item (D 128) or two ahead of its products' end ======
        const int t64 = tid - 320;
        uint32_t qfree_ph = 0, used = 0;                  // bit: buffer and group
        bool alive = true;
        int item = 0, len;
#pragma unroll 1
        for (int i = 0; i < n_tiles; i += len, ++item) {
            len = min(me.tiles - me.tile, n_tiles - i);
            if (t64 == 0 && me.h == 0 && me.qt == 0 && (me.kv != __ldg(a.kv_lens + me.z) || (a.q_lens != nullptr && me.ql != __ldg(a.q_lens + me.z))))
                report(a.status, FST_DEV_INDEX_RANGE, me.z, __ldg(a.kv_lens + me.z));
#pragma unroll 1
            for (int g = 0; g < 2; ++g) {
                if (group_tiles(g) <= me.tile) continue;      // (a piece may begin behind the first group's last tile)
                const int at = (QBUF == 1 ? 0 : (item & 1) * 2) + g;
                if (used >> at & 1) {                 // the products that read what is there
                    if (alive) alive = mbar_wait(bar_qfree + at * 8, qfree_ph >> at & 1, a.status, where);
                    qfree_ph ^= 1u << at;
                }
                used |= 1u << at;
                constexpr int CH = D / 8;
                const int c = t64 % CH;
                const uint32_t dst = s_base + at * TILE + (c >> 3) * HALF;
#pragma unroll 4
                for (int r = t64 / CH; r < 128; r += 64 / CH) {
                    const int row = me.qt * G::ROWS + g * 128 + r, tok = row / a.group;
                    const bool there = tok < me.ql;
                    const T *src = static_cast<const T *>(a.q) + me.z * a.qs_z + (me.h * a.group + (row - tok * a.group)) * a.qs_h + tok * a.qs_n + c * 8;
                    cp_async16(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4), there ? src : static_cast<const T *>(a.q), there);
                }
                cp_async_commit();
                cp_async_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar_q + at * 8) : "memory");
            }
            me.tile += len - 1;
            if (i + len < n_tiles) me.next(line);
        }
    } else {
        // ====== V tiles that not every row attends to all of ======
        const int t128 = tid - 384;
        int st = 1, item = 0;                             // stage of the tile's V
        uint32_t raw_ph = 0;
        bool alive = true;
#pragma unroll 1
        for (int i = 0; i < n_tiles; ++i) {
            if (i > 0 && me.tile == 0) ++item;
            const int key0 = me.tile * G::KEYS;
            if (me.keys > 0) {
                if (key0 + G::KEYS > first_limit()) {
                    if (alive) alive = mbar_wait(bar_raw + st * 8, raw_ph >> st & 1, a.status, where);
                    raw_ph ^= 1u << st;
                    // thread: a row's half at D 64, a whole row at D 128; chunks in an order that spreads the rows over the banks
                    const int have = me.kv - key0;        // rows behind the sequence's end become zeros
                    constexpr int PER = D / 8;            // chunks of 16 bytes: 128 rows of D / 8 over 128 threads
                    unsigned char *tile = smem + G::OFF_RING + st * TILE;
                    uint32_t odd = 0;
                    if (have >= G::KEYS) {
#pragma unroll
                        for (int k = 0; k < PER; ++k) {
                            const uint4 w = *reinterpret_cast<const uint4 *>(tile + (k * 128 + t128) * 16);
                            odd |= odd_bits<T>(w.x) | odd_bits<T>(w.y) | odd_bits<T>(w.z) | odd_bits<T>(w.w);
                        }
                    } else {
                        odd = 1u;
                    }
                    if (odd != 0u) {                      // (the order of a row's chunks does not matter)
                        bool met = false;
#pragma unroll 1
                        for (int k = 0; k < PER; ++k) {
                            const int at = (k * 128 + t128) * 16, r = at % HALF / 128;
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
        if (t128 == 0 && a.part != nullptr) leave_cut<G::ROWS, D>(a, me, total, n_tiles);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(G::REGS_SOFTMAX));
        // ====== softmax: two groups of 128 threads, one thread per row ======
        const int r = tid & 127, g = tid >> 7;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + g * 128 + lanes, tmem_o = tmem + 256 + g * D + lanes, tmem_p = D == 128 ? tmem_s : tmem + 384 + g * 64 + lanes;
        const uint32_t my_s = bar_s + g * 8, my_p = bar_p + g * 16;
        const float c2 = a.scale_log2;
        uint32_t s_ph = 0, o_ph = 0;
        int item = 0, len;
        bool alive = true;
#pragma unroll 1
        for (int i = 0; i < n_tiles; i += len, ++item) {
            len = min(me.tiles - me.tile, n_tiles - i);
            const int mine = min(max(group_tiles(g) - me.tile, 0), len);         // tiles of the piece that my group takes
            const int row = me.qt * G::ROWS + g * 128 + r, tok = row / a.group;
            const int limit = tok >= me.ql ? 0 : a.causal ? min(me.kv, me.kv - me.ql + tok + 1) : me.kv;
            float m_ref = -INFINITY, l = 0.f;
            // keys of the tile that I see, and that every row sees
            int n = limit - me.tile * G::KEYS, n_all = first_limit() - me.tile * G::KEYS;
#pragma unroll 1
            for (int j = 0; j < mine; ++j, n -= G::KEYS, n_all -= G::KEYS) {
                if (alive) alive = __all_sync(0xffffffffu, mbar_wait(my_s, s_ph, a.status, where));
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
                float mx4[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    mx4[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
                    for (int k = 2; k < 32; k += 2) mx4[c] = max3(mx4[c], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
                }
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                // the reference moves when a row has outgrown it by more than 2^8 (always on its first live tile)
                const bool up = (mx - m_ref) * c2 > 8.f;
                if (__any_sync(0xffffffffu, up)) {
                    if (j > 0) {                          // (S of this tile has landed: O += P V of the one before is done)
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
                    }
                    if (up) m_ref = mx;
                }
                const float mu = m_ref == -INFINITY ? 0.f : m_ref * c2;
                const uint64_t scale2 = pair(c2, c2), shift2 = pair(-mu, -mu);
                uint64_t l2[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t packed[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const uint64_t x = fma2(pair(__uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1])), scale2, shift2);
                        float p0, p1;
                        if ((k >> 1) % 4 == 3) {
                            exp2_poly(x, p0, p1);
                        } else {
                            unpair(x, p0, p1);
                            p0 = fast_exp2(p0);
                            p1 = fast_exp2(p1);
                        }
                        l2[(k >> 1) & 1] = add2(l2[(k >> 1) & 1], pair(p0, p1));
                        packed[k >> 1] = MT::pack(p0, p1);
                    }
                    tmem_st16(tmem_p + c * 16, packed);
                    if (c & 1) {
                        tmem_st_wait();
                        fence_before_sync();
                        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(my_p + (c >> 1) * 8) : "memory");
                    }
                }
                float la, lb;
                unpair(add2(l2[0], l2[1]), la, lb);
                l += la + lb;
            }

            // ---- the piece's rows: the output where it is the whole item, else sums for the merge
            if (mine > 0) {
                if (alive) alive = __all_sync(0xffffffffu, mbar_wait(bar_o + g * 8, o_ph, a.status, where));
                o_ph ^= 1u;
                fence_after_sync();
            }
            const bool bad = mine > 0 && *note <= item;   // (then also for the items behind: a look in vain)
            const bool whole = len == me.tiles, there = tok < me.ql;
            const int look_from = max(max(first_limit(), 0) & ~(G::KEYS - 1), me.tile * G::KEYS), look_to = min(limit, (me.tile + len) * G::KEYS);
            const float f = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l, mu = m_ref == -INFINITY ? -INFINITY : m_ref * c2;
            const int head = me.h * a.group + (row - tok * a.group);
            const size_t slot = (size_t(2) * blockIdx.x + (me.tile == 0 ? 1 : 0)) * G::ROWS + g * 128 + r;
            T *dst = static_cast<T *>(a.o) + me.z * a.os_z + head * a.os_h + tok * a.os_n;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                float o[32];
                if (mine > 0) {
                    uint32_t w[32];
                    tmem_ld32(w, tmem_o + c0);
                    tmem_ld_wait(w);
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __uint_as_float(w[k]);
                    if (bad) add_not_finite<T, 32>(a, me.z, me.h, look_from, look_to, c0, o);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = 0.f;
                }
                if (!there) continue;
                if (whole) {
#pragma unroll
                    for (int k = 0; k < 32; k += 8)
                        *reinterpret_cast<uint4 *>(dst + c0 + k) = make_uint4(MT::pack(o[k] * f, o[k + 1] * f), MT::pack(o[k + 2] * f, o[k + 3] * f),
                                                                              MT::pack(o[k + 4] * f, o[k + 5] * f), MT::pack(o[k + 6] * f, o[k + 7] * f));
                } else {
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<float4 *>(a.part + slot * D + c0 + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
            }
            if (there) {
                if (!whole) reinterpret_cast<float2 *>(a.part + chunk_stats_at(gridDim.x, G::ROWS, D))[slot] = make_float2(mu, l);
                else if (a.lse != nullptr) a.lse[(size_t(me.z) * a.H + head) * a.n_q + tok] = l == 0.f ? -INFINITY : mu + log2f(l);
            }
            fence_before_sync();                          // (O has been read before the next item's P is announced)
            me.tile += len - 1;
            if (i + len < n_tiles) me.next(line);
        }
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    if (warp == 9) {
        fence_after_sync();
        tmem_free_all(tmem);
    }
}

template <typename T, int D>
static cudaError_t launch_chunk_umma(const ChunkArgs &a, const CUtensorMap &tk, const CUtensorMap &tv, int n_ctas, cudaStream_t stream) {
    using G = ChunkUmmaGeo<D>;
    static_assert(G::BYTES <= 227 * 1024, "one CTA's shared memory");
    static DeviceOnce configured;
    const cudaError_t ce = configured.run([&] {
        return cudaFuncSetAttribute(chunk_umma_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::BYTES);
    });
    if (ce != cudaSuccess) return ce;
    const cudaError_t e = launch_serialised(chunk_umma_kernel<T, D>, dim3(n_ctas), dim3(G::THREADS), G::BYTES, stream, a, tk, tv);
    if (e != cudaSuccess || !chunk_splits(a, G::KEYS)) return e;
    return launch_chunk_combine<T, D, G::ROWS>(a, n_ctas, stream);
}

}  // namespace fst
