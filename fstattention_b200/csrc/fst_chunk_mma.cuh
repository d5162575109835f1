// Chunk attention of few rows on mma.sync: decode steps and drafted tokens.
//
// A tile is 16 or 32 rows and 128 or 256 keys; a call like that reads each key and value once for a handful of products, so HBM bounds it
// and the tensor cores' rate does not matter.  What matters is bytes in flight and that the warps seldom wait: a ninth warp has TMA
// fill a ring of tiles, each of the eight others takes 16 or 32 keys of a tile and has an accumulator of its own for all rows, so
// that nothing but the ring's barriers lies between them.  They meet once per item, to add up.
//
// 8-bit rows become matrix fragments in registers, without their scales.  The order of the summed index is free as long as both operands
// agree, so lane (g, t) of a K fragment takes the contiguous bytes D/4 t .. of key g, and Q is loaded in the same order; of V it
// takes bytes D/8 g .. of its four keys, which only permutes the columns of the result.  K is fp16, by the conversion instruction.  A
// key's scale multiplies its score; bf16 queries become fp16 times a power of two per row, with the row's largest value next to 2^15:
// what fp16 loses then is 2^-39 of that.  V's scales go into the exponents of weights of their own, as in chunk_token_kernel: no single
// factor brings all of their range, 2^-117 to 2^119, through a 16-bit probability and an fp32 sum.  Under fp16 queries weights and V are fp16.  Under
// bf16 queries they are bf16, whose range keeps rows of V apart that are more than 2^39 smaller than others: a byte's seven low bits
// moved under bf16's exponent are its value * 2^-120, and weights are taken 2^120 times too large.
//
// 7 draft tokens of 4 heads behind 24 x 8 heads of 2300 e4m3 rows at D 64: 45 us (58 MB, 9 us of HBM): a fixed 20, of them 4 for the merge and as many for
// the warps' meetings at every item's end, and 2.1 us a tile of 256 keys: some 1300 instructions a warp for it, most of them conversions and
// the softmax, from two warps to a scheduler.
#pragma once

#include "fst_chunk_load.cuh"

namespace fst {

template <int D, bool QUANT, int MT>
struct ChunkMmaGeo {
    static constexpr int WARPS = 8, KW = !QUANT && D == 128 ? 16 : 32, KEYS = WARPS * KW, ROWS = 16 * MT, OVER = 2;
    static constexpr int THREADS = WARPS * 32 + 128;                // and a loading warp, in a warpgroup that gives its registers away
    static constexpr int REGS = 224, REGS_LOADS = 56;
    static_assert(256 * REGS + 128 * REGS_LOADS <= THREADS * 168, "the split draws on what the launch was given");
    static constexpr int TILE = KEYS * D * (QUANT ? 1 : 2);         // bytes of a tile of K or V: 64-column halves of KEYS rows, or rows of bytes
    static constexpr int STAGES = QUANT && D == 64 ? 8 : 4;         // of a tile of K or of V, which take turns
    static constexpr bool Q_SHARED = D == 128 && MT == 2;           // fragments of Q in shared memory: registers would not hold them
    static constexpr int OFF_MERGE = STAGES * TILE;             // [warp][16 rows][D + 4] fp32
    static constexpr int OFF_STATS = OFF_MERGE + WARPS * 16 * (D + 4) * 4;      // [warp][ROWS] (exponent, sum)
    static constexpr int OFF_SCALES = OFF_STATS + WARPS * ROWS * 8; // [stage] KEYS bytes
    static constexpr int OFF_Q = OFF_SCALES + (QUANT ? STAGES * KEYS : 0);  // [row tile][step][lane] 16 bytes
    static constexpr int OFF_BAR = OFF_Q + (Q_SHARED ? MT * D / 16 * 512 : 0);
    static constexpr int BYTES = OFF_BAR + 2 * STAGES * 8 + 1024;   // + alignment
};

// four e4m3 bytes -> two pairs of bf16 (bytes 0 and 2, bytes 1 and 3), smaller by 2^120
__device__ __forceinline__ void e4m3_bits(uint32_t w, uint32_t &even, uint32_t &odd) {
    odd = (w & 0x80008000u) | ((w >> 4) & 0x07f007f0u);
    const uint32_t u = w << 8;
    even = (u & 0x80008000u) | ((u >> 4) & 0x07f007f0u);
}
template <typename T, int D, bool QUANT, int MT>
__global__ void __launch_bounds__(384, 1)
chunk_mma_kernel(const ChunkArgs a, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
    using G = ChunkMmaGeo<D, QUANT, MT>;
    using MT_ = MmaTraits<T>;
    using MK = MmaTraits<typename std::conditional<QUANT, __half, T>::type>;     // of the first product
    using Line = ChunkLine<G::ROWS, G::KEYS, G::OVER>;
    using Cursor = ChunkCursor<G::ROWS, G::KEYS, G::OVER>;
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    constexpr float LIFT = !QUANT && !BF16 ? kLift : 0.f, LIFT_W = BF16 ? 120.f : kLift;      // of probabilities, of weights
    constexpr int KS = D / 16, ND = D / 8;               // steps of the first product, column tiles of the second
    constexpr int KW = G::KW, NK = KW / 8, SUBS = KW / 16;
    constexpr int HALF_BYTES = G::KEYS * 128, SUB_BYTES = 16 * (QUANT ? D : 128);         // a tile's half of 64 columns of 16 bits, 16 rows in it

    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    extern __shared__ unsigned char smem_raw[];
    const uint32_t s_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char *smem = smem_raw + (s_base - smem_u32(smem_raw));
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t bar_full = s_base + G::OFF_BAR, bar_empty = bar_full + G::STAGES * 8;
    if (tid == 0) {
        for (int i = 0; i < G::STAGES; ++i) {
            mbar_init(bar_full + i * 8, QUANT ? 33 : 1);      // (the lanes' scales, see load_tiles)
            mbar_init(bar_empty + i * 8, G::WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const Line line(a);
    __shared__ ChunkPiece<G::ROWS, G::KEYS, G::OVER> piece;
    piece.find(line);
    __syncthreads();
    Cursor me = piece.from;
    const long long total = piece.total;
    const int n_tiles = piece.tiles();
    if (n_tiles == 0) {
        if (tid == 0 && a.part != nullptr) leave_cut<D>(a, me, total, 0);
        return;
    }

    // (each side asks inside its own branch, see chunk_umma_kernel)
    if (warp >= G::WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(G::REGS_LOADS));
        if (warp > G::WARPS) return;
        load_tiles<G, D, QUANT>(a, line, me, n_tiles, tm_k, tm_v, s_base, smem, bar_full, bar_empty);
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(G::REGS));
    auto meet = [&]() { asm volatile("bar.sync 1, 256;\n" ::: "memory"); };     // the computing warps
    auto group_of = [&](const Cursor &c) { return c.tile * G::KEYS + warp * KW; };

    // ---- products
    const float c2 = a.scale_log2;
    uint32_t qf[G::Q_SHARED ? 1 : MT][G::Q_SHARED ? 1 : KS][4];
    const uint32_t q_at = s_base + G::OFF_Q + lane * 16;
    // fragment of step st of row tile x
    auto q_frag = [&](int x, int st, uint32_t (&f)[4]) {
        if constexpr (G::Q_SHARED) {
            const uint4 v = lds128(q_at + (x * KS + st) * 512);
            f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = qf[x][st][k];
        }
    };
    float acc[MT][ND][4], m[MT][2], l[MT][2];
    float row_c2[QUANT ? MT : 1][2];                      // an 8-bit cache: c2 over the row's factor
    float m_w[QUANT ? MT : 1][2];                       // running maximum of score and V's exponent
    int limit[MT][2], lim_first = 0, slot = 0;
    uint32_t parity = 0;
    bool poisoned = false, alive = true;                  // a V that is not finite was met where not every row attends to it

#pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
        if (i == 0 || me.tile == 0) {                     // a new item: its rows of Q
            if (tid == 0 && me.h == 0 && me.qt == 0 && (me.kv != load(a.kv_lens + me.z) || (a.q_lens != nullptr && me.ql != load(a.q_lens + me.z))))
                report(a.status, FST_DEV_INDEX_RANGE, me.z, load(a.kv_lens + me.z));
            poisoned = false;
            lim_first = a.causal ? min(me.kv, me.kv - me.ql + by_group(a, me.qt * G::ROWS) + 1) : me.kv;
#pragma unroll
            for (int x = 0; x < MT; ++x) {
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    const int r = me.qt * G::ROWS + x * 16 + hh * 8 + g, tok = by_group(a, r);
                    const bool real = tok < me.ql;
                    limit[x][hh] = !real ? 0 : a.causal ? min(me.kv, me.kv - me.ql + tok + 1) : me.kv;
                    m[x][hh] = -INFINITY;
                    l[x][hh] = 0.f;
                    const T *src = static_cast<const T *>(a.q) + me.z * a.qs_z + (me.h * a.group + (r - tok * a.group)) * a.qs_h + tok * a.qs_n;
                    // two of the four registers of a row tile's fragments: the row's part of two steps in an 8-bit cache's order, or of one
                    float by = 1.f;                       // the row's factor
                    if constexpr (QUANT) m_w[x][hh] = -INFINITY;
                    if constexpr (QUANT) {
                        if constexpr (BF16) {
                            uint32_t top = 0;
#pragma unroll
                            for (int s2 = 0; s2 < KS / 2; ++s2) {
                                const uint4 w = real ? load(reinterpret_cast<const uint4 *>(src + t * (D / 4) + s2 * 8)) : make_uint4(0, 0, 0, 0);
                                top = __vmaxu2(top, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
                            }
                            top = max(top & 0xffffu, top >> 16);
                            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                            // exponent of the largest magnitude to 14; rows of zeros, and of what is not finite, as they are
                            if (top >= 0x80u && top < 0x7f80u) by = pow2f(min(141 - int(top >> 7), 126));
                        }
                        row_c2[x][hh] = c2 / by;
                    }
                    auto two_steps = [&](int s2, uint32_t (&f)[4]) {         // steps 2 s2 and 2 s2 + 1: D / 4 contiguous values
                        const uint4 w = real ? load(reinterpret_cast<const uint4 *>(src + t * (D / 4) + s2 * 8)) : make_uint4(0, 0, 0, 0);
                        f[0] = w.x; f[1] = w.y; f[2] = w.z; f[3] = w.w;
                        if constexpr (BF16) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) f[k] = MK::pack(__uint_as_float(f[k] << 16) * by, __uint_as_float(f[k] & 0xffff0000u) * by);
                        }
                    };
                    auto one_step = [&](int st, uint32_t &lo, uint32_t &hi) {
                        lo = real ? load(reinterpret_cast<const uint32_t *>(src + st * 16 + 2 * t)) : 0u;
                        hi = real ? load(reinterpret_cast<const uint32_t *>(src + st * 16 + 8 + 2 * t)) : 0u;
                    };
                    if constexpr (G::Q_SHARED) {          // every warp brings a step (KS = 8 warps)
                        uint32_t lo, hi;
                        if constexpr (QUANT) {
                            uint32_t f[4];
                            two_steps(warp >> 1, f);
                            lo = warp & 1 ? f[2] : f[0];
                            hi = warp & 1 ? f[3] : f[1];
                        } else {
                            one_step(warp, lo, hi);
                        }
                        asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(q_at + (x * KS + warp) * 512 + hh * 4), "r"(lo) : "memory");
                        asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(q_at + (x * KS + warp) * 512 + 8 + hh * 4), "r"(hi) : "memory");
                    } else if constexpr (QUANT) {
#pragma unroll
                        for (int s2 = 0; s2 < KS / 2; ++s2) {
                            uint32_t f[4];
                            two_steps(s2, f);
                            qf[x][2 * s2][hh] = f[0];
                            qf[x][2 * s2][2 + hh] = f[1];
                            qf[x][2 * s2 + 1][hh] = f[2];
                            qf[x][2 * s2 + 1][2 + hh] = f[3];
                        }
                    } else {
#pragma unroll
                        for (int st = 0; st < KS; ++st) one_step(st, qf[x][st][hh], qf[x][st][2 + hh]);
                    }
                }
#pragma unroll
                for (int n = 0; n < ND; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[x][n][k] = 0.f;
            }
            if constexpr (G::Q_SHARED) meet();
        }

        const int key0 = group_of(me);
        if (me.keys > 0 && alive) alive = __all_sync(0xffffffffu, wait_for(bar_full + slot * 8, parity));
        bool k_held = me.keys > 0;
        auto done_with = [&](int stage) {
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar_empty + stage * 8) : "memory");
        };
        if (key0 < me.keys && alive) {
            const uint32_t k_at = s_base + slot * G::TILE + warp * SUBS * SUB_BYTES, v_at = k_at + G::TILE;          // my rows
            const unsigned char *scales = smem + G::OFF_SCALES + slot * G::KEYS + warp * KW;
            const bool edge = key0 + KW > lim_first;      // not every row attends to all of the group
            float s[MT][NK][4];
#pragma unroll
            for (int x = 0; x < MT; ++x)
#pragma unroll
                for (int n = 0; n < NK; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[x][n][k] = 0.f;
            if constexpr (QUANT) {
                // K: key 8 n + g, bytes D/4 t ..
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {        // 16 bytes: four steps
                    uint4 b[NK];
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
                        const int row = 8 * n + g, chunk = D == 128 ? ((2 * t + c) ^ (row & 7)) : (t ^ ((row >> 1) & 3));
                        b[n] = lds128(k_at + row * D + chunk * 16);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t q[MT][4];
#pragma unroll
                        for (int x = 0; x < MT; ++x) q_frag(x, c * 4 + k, q[x]);
#pragma unroll
                        for (int n = 0; n < NK; ++n) {
                            const uint32_t w = k == 0 ? b[n].x : k == 1 ? b[n].y : k == 2 ? b[n].z : b[n].w;
                            const uint32_t b0 = e4m3_halves(w, false), b1 = e4m3_halves(w, true);
#pragma unroll
                            for (int x = 0; x < MT; ++x) MK::mma(s[x][n], q[x], b0, b1);
                        }
                    }
                }
            } else {
                const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    const int chunk = 2 * st + ((lane >> 3) & 1);
                    uint32_t q[MT][4];
#pragma unroll
                    for (int x = 0; x < MT; ++x) q_frag(x, st, q[x]);
#pragma unroll
                    for (int sub = 0; sub < SUBS; ++sub) {
                        uint32_t b[4];
                        ldmatrix_x4(b, k_at + sub * SUB_BYTES + (chunk >> 3) * HALF_BYTES + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
#pragma unroll
                        for (int x = 0; x < MT; ++x) {
                            MT_::mma(s[x][2 * sub], q[x], b[0], b[1]);
                            MT_::mma(s[x][2 * sub + 1], q[x], b[2], b[3]);
                        }
                    }
                }
            }
            if constexpr (!QUANT) {                       // (an 8-bit tile's scales are still to be read)
                done_with(slot);
                k_held = false;
            }
            // ---- softmax of the group: scores in base-2 units against the row's running maximum
            uint32_t pf[MT][SUBS][4];
            float mx[MT][2];
#pragma unroll
            for (int x = 0; x < MT; ++x) mx[x][0] = mx[x][1] = -INFINITY;
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                float ks[2] = {1.f, 1.f};                 // of my keys 8 n + 2 t + k
                if constexpr (QUANT) {
                    const float2 both = e8m0_values(*reinterpret_cast<const uint16_t *>(scales + 8 * n + 2 * t));
                    ks[0] = both.x;
                    ks[1] = both.y;
                }
#pragma unroll
                for (int x = 0; x < MT; ++x)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float v = s[x][n][k] * (QUANT ? ks[k & 1] * row_c2[x][k >> 1] : c2);
                        if (edge && key0 + 8 * n + 2 * t + (k & 1) >= limit[x][k >> 1]) v = -INFINITY;
                        s[x][n][k] = v;
                        mx[x][k >> 1] = fmaxf(mx[x][k >> 1], v);
                    }
            }
            if constexpr (QUANT) {
                done_with(slot);
                k_held = false;
            }
            alive = __all_sync(0xffffffffu, wait_for(bar_full + (slot + 1) * 8, parity));     // V
            float mw[QUANT ? MT : 1][2], e_v[QUANT ? NK : 1][2];
            if constexpr (QUANT) {
#pragma unroll
                for (int x = 0; x < MT; ++x) mw[x][0] = mw[x][1] = -INFINITY;
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    const int b = *reinterpret_cast<const uint16_t *>(scales + G::KEYS + 8 * n + 2 * t);
                    e_v[n][0] = (b & 255) == 255 ? NAN : float((b & 255) - 127);
                    e_v[n][1] = b >> 8 == 255 ? NAN : float((b >> 8) - 127);
#pragma unroll
                    for (int x = 0; x < MT; ++x)
#pragma unroll
                        for (int k = 0; k < 4; ++k) mw[x][k >> 1] = fmaxf(mw[x][k >> 1], s[x][n][k] + e_v[n][k & 1]);        // (a maximum passes over a NaN)
                }
            }
#pragma unroll
            for (int x = 0; x < MT; ++x) {
                bool up = false;
                float alpha[2], alpha_w[2];
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    auto move = [&](float &had, float &seen, float &by, float lift) {    // the running maximum, as a reference, and what it takes what was summed by
                        seen = fmaxf(seen, __shfl_xor_sync(0xffffffffu, seen, 1));
                        seen = fmaxf(seen, __shfl_xor_sync(0xffffffffu, seen, 2));
                        const float now = fmaxf(had, seen);
                        up = up || now > had;
                        by = now == -INFINITY ? 1.f : fast_exp2(had - now);
                        had = now;
                        seen = now == -INFINITY ? 0.f : now - lift;
                    };
                    move(m[x][hh], mx[x][hh], alpha[hh], LIFT);
                    alpha_w[hh] = alpha[hh];
                    if constexpr (QUANT) move(m_w[x][hh], mw[x][hh], alpha_w[hh], LIFT_W);
                }
                if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                    for (int n = 0; n < ND; ++n) {
                        acc[x][n][0] *= alpha_w[0];
                        acc[x][n][1] *= alpha_w[0];
                        acc[x][n][2] *= alpha_w[1];
                        acc[x][n][3] *= alpha_w[1];
                    }
                    l[x][0] *= alpha[0];
                    l[x][1] *= alpha[1];
                }
            }
#pragma unroll
            for (int n = 0; n < NK; ++n) {
#pragma unroll
                for (int x = 0; x < MT; ++x) {
                    float p[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float v = s[x][n][k];
                        p[k] = fast_exp2(v - mx[x][k >> 1]);
                        l[x][k >> 1] += p[k];
                        // (what a masked key holds, NaN too, stays out)
                        if constexpr (QUANT) p[k] = v == -INFINITY ? 0.f : fast_exp2(v + e_v[n][k & 1] - mw[x][k >> 1]);
                    }
                    pf[x][n >> 1][(n & 1) * 2] = MT_::pack(p[0], p[1]);
                    pf[x][n >> 1][(n & 1) * 2 + 1] = MT_::pack(p[2], p[3]);
                }
            }
            // ---- second product
            const int here = min(me.kv, (me.keys + 15) & ~15) - key0;     // rows of V that were fetched and are the sequence's
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub) {
                if constexpr (QUANT) {
                    // V: keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9, bytes D/8 g ..: column tile j holds columns D/8 n + j
                    uint32_t w[4][D / 32];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int row = sub * 16 + 2 * t + (k & 1) + (k >> 1) * 8;
                        if constexpr (D == 128) {
                            const uint4 b = lds128(v_at + row * 128 + ((g ^ (row & 7)) << 4));
                            w[k][0] = b.x; w[k][1] = b.y; w[k][2] = b.z; w[k][3] = b.w;
                        } else {
                            const uint2 b = lds64(v_at + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8);
                            w[k][0] = b.x; w[k][1] = b.y;
                        }
                        if (!BF16 && edge && row >= here) {           // zero times a NaN byte would be NaN
#pragma unroll
                            for (int c = 0; c < D / 32; ++c) w[k][c] = 0u;
                        }
                    }
#pragma unroll
                    for (int c = 0; c < D / 32; ++c)
#pragma unroll
                        for (int hl = 0; hl < 2; ++hl) {  // two column tiles from bytes 2 hl, 2 hl + 1 of either key
                            uint32_t b0[2], b1[2];
                            if constexpr (BF16) {
                                e4m3_bits(__byte_perm(w[0][c], w[1][c], hl ? 0x7632 : 0x5410), b0[0], b0[1]);
                                e4m3_bits(__byte_perm(w[2][c], w[3][c], hl ? 0x7632 : 0x5410), b1[0], b1[1]);
                            } else {
                                const uint32_t y0 = __byte_perm(w[0][c], w[1][c], hl ? 0x7362 : 0x5140), y1 = __byte_perm(w[2][c], w[3][c], hl ? 0x7362 : 0x5140);
                                b0[0] = e4m3_halves(y0, false);
                                b0[1] = e4m3_halves(y0, true);
                                b1[0] = e4m3_halves(y1, false);
                                b1[1] = e4m3_halves(y1, true);
                            }
#pragma unroll
                            for (int k = 0; k < 2; ++k)
#pragma unroll
                                for (int x = 0; x < MT; ++x) MT_::mma(acc[x][c * 4 + hl * 2 + k], pf[x][sub], b0[k], b1[k]);
                        }
                } else {
                    const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
                    for (int j = 0; j < ND / 2; ++j) {
                        const int chunk = 2 * j + (lane >> 4);
                        uint32_t b[4];
                        ldmatrix_x4_trans(b, v_at + sub * SUB_BYTES + (chunk >> 3) * HALF_BYTES + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
                        if (edge) {                       // zero times what is not finite would be NaN
#pragma unroll
                            for (int k = 0; k < 4; ++k) poisoned = keep_finite<T>(b[k], here - sub * 16 - (k & 1) * 8 - 2 * t) || poisoned;
                        }
#pragma unroll
                        for (int x = 0; x < MT; ++x) {
                            MT_::mma(acc[x][2 * j], pf[x][sub], b[0], b[1]);
                            MT_::mma(acc[x][2 * j + 1], pf[x][sub], b[2], b[3]);
                        }
                    }
                }
            }
        } else if (me.keys > 0 && alive) {
            // No key of this tile is mine.  V's stage is given back only once it has been filled: that is what says that every warp has
            // given back its last filling, which an arrival ahead of that would have stood in for a warp that still reads it.
            alive = __all_sync(0xffffffffu, wait_for(bar_full + (slot + 1) * 8, parity));
        }
        if (me.keys > 0) {
            if (k_held) done_with(slot);
            done_with(slot + 1);
            slot += 2;
            if (slot == G::STAGES) {
                slot = 0;
                parity ^= 1u;
            }
        }

        if (me.tile + 1 == me.tiles || i + 1 == n_tiles) {
            // ---- the warps' results of this piece: 16 rows at a time through shared memory
            const bool from_start = i >= me.tile, whole = from_start && me.tile + 1 == me.tiles;
            uint32_t bad;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, 1, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                         : "=r"(bad) : "r"(uint32_t(poisoned)) : "memory");
            float2 *stats = reinterpret_cast<float2 *>(smem + G::OFF_STATS);
            float *rows = reinterpret_cast<float *>(smem + G::OFF_MERGE);
#pragma unroll
            for (int x = 0; x < MT; ++x) {
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    float sum = l[x][hh];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    if (t == 0) stats[warp * G::ROWS + x * 16 + hh * 8 + g] = make_float2(m[x][hh] - LIFT, sum);
                    float *to = rows + (warp * 16 + hh * 8 + g) * (D + 4);
                    if constexpr (QUANT) {                // weights back to the probabilities' reference
                        float by, then;
                        weights_back(m[x][hh], m_w[x][hh], BF16 ? 1.f : 1.f / 32768.f, by, then);
#pragma unroll
                        for (int j = 0; j < ND; ++j)
#pragma unroll
                            for (int k = 0; k < 2; ++k) acc[x][j][2 * hh + k] = acc[x][j][2 * hh + k] * by * then;
                    }
                    if constexpr (QUANT) {
#pragma unroll
                        for (int j = 0; j < ND; j += 4)
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                *reinterpret_cast<float4 *>(to + (2 * t + k) * (D / 8) + j) =
                                    make_float4(acc[x][j][2 * hh + k], acc[x][j + 1][2 * hh + k], acc[x][j + 2][2 * hh + k], acc[x][j + 3][2 * hh + k]);
                    } else {
#pragma unroll
                        for (int n = 0; n < ND; ++n)
                            *reinterpret_cast<float2 *>(to + n * 8 + 2 * t) = make_float2(acc[x][n][2 * hh], acc[x][n][2 * hh + 1]);
                    }
                }
                meet();
                // sixteen threads a row, D / 16 columns each
                const int row = tid >> 4, c0 = (tid & 15) * (D / 16);
                float top = -INFINITY, sum = 0.f, out[D / 16];
#pragma unroll
                for (int w = 0; w < G::WARPS; ++w) top = fmaxf(top, stats[w * G::ROWS + x * 16 + row].x);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) out[k] = 0.f;
#pragma unroll
                for (int w = 0; w < G::WARPS; ++w) {
                    const float2 st = stats[w * G::ROWS + x * 16 + row];
                    if (st.x == -INFINITY && st.y == 0.f) continue;              // saw nothing
                    const float f = top == -INFINITY ? 1.f : fast_exp2(st.x - top);
                    sum += st.y * f;
#pragma unroll
                    for (int k = 0; k < D / 16; k += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(rows + (w * 16 + row) * (D + 4) + c0 + k);
                        out[k] += v.x * f;
                        out[k + 1] += v.y * f;
                        out[k + 2] += v.z * f;
                        out[k + 3] += v.w * f;
                    }
                }
                const int r = me.qt * G::ROWS + x * 16 + row, tok = by_group(a, r), head = me.h * a.group + (r - tok * a.group);
                if (bad != 0u && tok < me.ql) {
                    // keys of this piece whose groups were looked through, as far as my row sees them
                    const int keys = a.causal ? min(me.kv, me.kv - me.ql + tok + 1) : me.kv;
                    add_not_finite<T, D / 16, QUANT>(a, me.z, me.h, max(max(lim_first, 0) & ~(KW - 1), max(0, me.tile - i) * G::KEYS),
                                              min(keys, (me.tile + 1) * G::KEYS), c0, out);
                }
                if (whole) {
                    if (tok < me.ql) {
                        const float inv = sum == 0.f ? 0.f : 1.f / sum;
                        T *dst = static_cast<T *>(a.o) + me.z * a.os_z + head * a.os_h + tok * a.os_n + c0;
                        uint32_t w[D / 32];
#pragma unroll
                        for (int k = 0; k < D / 32; ++k) w[k] = MT_::pack(out[2 * k] * inv, out[2 * k + 1] * inv);
                        if constexpr (D == 128) *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
                        else *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
                        if (a.lse != nullptr && c0 == 0) a.lse[(size_t(me.z) * a.H + head) * a.n_q + tok] = sum == 0.f ? -INFINITY : top + log2f(sum);
                    }
                } else {
                    const size_t at = (size_t(2) * blockIdx.x + (from_start ? 1 : 0)) * G::ROWS + x * 16 + row;
#pragma unroll
                    for (int k = 0; k < D / 16; k += 4)
                        *reinterpret_cast<float4 *>(a.part + at * D + c0 + k) = make_float4(out[k], out[k + 1], out[k + 2], out[k + 3]);
                    if (c0 == 0) reinterpret_cast<float2 *>(a.part + chunk_stats_at(gridDim.x, G::ROWS, D))[at] = make_float2(top, sum);
                }
                meet();
            }
        }
        if (i + 1 < n_tiles) me.next(line);
    }
    if (!alive && lane == 0) report(a.status, FST_DEV_TIMEOUT, blockIdx.x, warp);
    if (tid == 0 && a.part != nullptr) leave_cut<D>(a, me, total, n_tiles);
}

template <typename T, int D, bool QUANT, int MT>
static cudaError_t launch_chunk_mma(const ChunkArgs &a, const CUtensorMap &tk, const CUtensorMap &tv, int n_ctas, cudaStream_t stream) {
    using G = ChunkMmaGeo<D, QUANT, MT>;
    static_assert(G::BYTES <= 227 * 1024, "one CTA's shared memory");
    static DeviceOnce configured;
    const cudaError_t ce = configured.run([&] {
        return cudaFuncSetAttribute(chunk_mma_kernel<T, D, QUANT, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::BYTES);
    });
    if (ce != cudaSuccess) return ce;
    const cudaError_t e = launch_serialised(chunk_mma_kernel<T, D, QUANT, MT>, dim3(n_ctas), dim3(G::THREADS), G::BYTES, stream, a, tk, tv);
    if (e != cudaSuccess || !chunk_splits(a, G::KEYS)) return e;
    return launch_chunk_combine<T, D, G::ROWS>(a, n_ctas, stream);
}

}  // namespace fst
