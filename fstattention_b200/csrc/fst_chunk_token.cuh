// Chunk attention of at most eight rows on mma.sync: the single tokens of decode steps.
//
// As chunk_mma_kernel (fst_chunk_mma.cuh), with the products the other way round: S^T = K Q^T and O^T = V^T P^T, keys and columns as the 16 rows
// of a product and the rows as its 8 columns.  The fragments of K and V are the same registers; half as many products, scores
// and sums are left where sixteen rows would have been half empty.  A thread has the scores of two rows and, of every 16
// keys, keys g and g + 8; movmatrix turns the probabilities into the second product's operand.
//
// An 8-bit cache: K and V are fp16 fragments by the conversion instruction, without their scales.  A key's scale multiplies its score.  A value's
// scale 2^e goes into the exponent of its weight: beside p = 2^(s - m), which the sum l is made of, there is w = 2^(s + e - m'), m' the
// maximum of s + e, which multiplies V; neither leaves its format, whatever the scales are, and the result is sum w v / l * 2^(m' - m).  Weights are
// fp16 under bf16 queries too, for three more bits (errors of 0.0017 of a result instead of 0.0022), taken 2^15 times too large: what a row of V
// adds is rounded by 2^-40 of what the largest scale times its probability stands for, which shows where that row has zeros.
// bf16 queries become fp16 as in chunk_mma_kernel.
//
// Two sequences of 115000 e4m3 rows under 8 rows: 89 us where heads lie inside rows (5.3 TB/s; a copy has 6.55), 81 where a head's rows lie
// together; chunk_mma_kernel took 108 when this took 101.  64 sequences of 4500 bf16 rows: 185 us, 6.5 TB/s.  What bounds it: HBM in 16 bits; in 8 bits
// requests of 128 bytes, and the chain of a warp's dependent instructions (two warps to a scheduler issue in 37 % of the cycles; 12 or 16 warps were
// slower, so were half tiles in more stages: 117 us, and a reference for the maximum that moves less often made no difference).
#pragma once

#include "fst_chunk_load.cuh"

namespace fst {

template <int D, bool QUANT>
struct ChunkTokenGeo {
    static constexpr int WARPS = 8, KW = !QUANT && D == 128 ? 16 : 32, KEYS = WARPS * KW, ROWS = 8, OVER = 2;
    static constexpr int THREADS = WARPS * 32 + 32;                 // and a loading warp
    static constexpr int TILE = KEYS * D * (QUANT ? 1 : 2);
    static constexpr int STAGES = QUANT && D == 64 ? 8 : 4;
    static constexpr int OFF_MERGE = STAGES * TILE;                 // [warp][8 rows][D + 4] fp32
    static constexpr int OFF_STATS = OFF_MERGE + WARPS * 8 * (D + 4) * 4;       // [warp][8 rows] (exponent, sum)
    static constexpr int OFF_SCALES = OFF_STATS + WARPS * 8 * 8;    // [stage] KEYS bytes
    static constexpr int OFF_BAR = OFF_SCALES + (QUANT ? STAGES * KEYS : 0);
    static constexpr int BYTES = OFF_BAR + 2 * STAGES * 8 + 1024;   // + alignment
};

// an 8 x 8 matrix of 16-bit values, a pair of a row's a thread, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
    return r;
}

template <typename T, int D, bool QUANT>
__global__ void __launch_bounds__(ChunkTokenGeo<D, QUANT>::THREADS, 1)
chunk_token_kernel(const ChunkArgs a, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
    using G = ChunkTokenGeo<D, QUANT>;
    using MP = MmaTraits<typename std::conditional<QUANT, __half, T>::type>;
    using Line = ChunkLine<G::ROWS, G::KEYS, G::OVER>;
    using Cursor = ChunkCursor<G::ROWS, G::KEYS, G::OVER>;
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    constexpr float LIFT = !QUANT && !BF16 ? kLift : 0.f;
    constexpr int KS = D / 16, NP = D / 16;               // steps of the first product, 16-column tiles of the second
    constexpr int KW = G::KW, SUBS = KW / 16;
    constexpr int HALF_BYTES = G::KEYS * 128, SUB_BYTES = 16 * (QUANT ? D : 128);

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
    if (warp == G::WARPS) {
        load_tiles<G, D, QUANT>(a, line, me, n_tiles, tm_k, tm_v, s_base, smem, bar_full, bar_empty);
        return;
    }
    auto meet = [&]() { asm volatile("bar.sync 1, %0;\n" ::"n"(G::WARPS * 32) : "memory"); };      // the computing warps
    auto done_with = [&](int stage) {
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar_empty + stage * 8) : "memory");
    };

    // rows 2 t and 2 t + 1 are mine in scores and sums, row g in Q's fragments
    uint32_t qf[KS][2];
    float acc[NP][4], m[2], l[2], m_w[2], row_c2[2];
    int limit[2], lim_first = 0, slot = 0;
    uint32_t parity = 0;
    bool poisoned = false, alive = true;                  // a V that is not finite was met where not every row attends to it

#pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
        if (i == 0 || me.tile == 0) {                     // a new item
            if (tid == 0 && me.h == 0 && me.qt == 0 && (me.kv != load(a.kv_lens + me.z) || (a.q_lens != nullptr && me.ql != load(a.q_lens + me.z))))
                report(a.status, FST_DEV_INDEX_RANGE, me.z, load(a.kv_lens + me.z));
            poisoned = false;
            lim_first = a.causal ? min(me.kv, me.kv - me.ql + by_group(a, me.qt * G::ROWS) + 1) : me.kv;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int tok = by_group(a, me.qt * G::ROWS + 2 * t + q);
                limit[q] = tok >= me.ql ? 0 : a.causal ? min(me.kv, me.kv - me.ql + tok + 1) : me.kv;
                m[q] = m_w[q] = -INFINITY;
                l[q] = 0.f;
                row_c2[q] = a.scale_log2;
            }
#pragma unroll
            for (int n = 0; n < NP; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[n][k] = 0.f;
            const int r = me.qt * G::ROWS + g, tok = by_group(a, r);
            const bool real = tok < me.ql;
            const T *src = static_cast<const T *>(a.q) + me.z * a.qs_z + (me.h * a.group + (r - tok * a.group)) * a.qs_h + tok * a.qs_n;
            if constexpr (QUANT) {                        // D / 4 contiguous values of the row, in the order of K's bytes
                uint4 w[KS / 2];
                uint32_t top = 0;
#pragma unroll
                for (int s2 = 0; s2 < KS / 2; ++s2) {
                    w[s2] = real ? load(reinterpret_cast<const uint4 *>(src + t * (D / 4) + s2 * 8)) : make_uint4(0, 0, 0, 0);
                    top = __vmaxu2(top, __vmaxu2(__vmaxu2(w[s2].x & 0x7fff7fffu, w[s2].y & 0x7fff7fffu), __vmaxu2(w[s2].z & 0x7fff7fffu, w[s2].w & 0x7fff7fffu)));
                }
                float by = 1.f;                           // the row's factor: its largest magnitude's exponent to 14
                if constexpr (BF16) {
                    top = max(top & 0xffffu, top >> 16);
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (top >= 0x80u && top < 0x7f80u) by = pow2f(min(141 - int(top >> 7), 126));        // (zeros, and what is not finite, as they are)
                }
#pragma unroll
                for (int s2 = 0; s2 < KS / 2; ++s2) {
                    uint32_t f[4] = {w[s2].x, w[s2].y, w[s2].z, w[s2].w};
                    if constexpr (BF16) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) f[k] = MP::pack(__uint_as_float(f[k] << 16) * by, __uint_as_float(f[k] & 0xffff0000u) * by);
                    }
                    qf[2 * s2][0] = f[0];
                    qf[2 * s2][1] = f[1];
                    qf[2 * s2 + 1][0] = f[2];
                    qf[2 * s2 + 1][1] = f[3];
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) row_c2[q] = a.scale_log2 / __shfl_sync(0xffffffffu, by, (2 * t + q) * 4);
            } else {
#pragma unroll
                for (int st = 0; st < KS; ++st)
#pragma unroll
                    for (int k = 0; k < 2; ++k) qf[st][k] = real ? load(reinterpret_cast<const uint32_t *>(src + st * 16 + k * 8 + 2 * t)) : 0u;
            }
        }

        const int key0 = me.tile * G::KEYS + warp * KW;
        if (me.keys > 0 && alive) alive = __all_sync(0xffffffffu, wait_for(bar_full + slot * 8, parity));
        bool k_held = me.keys > 0;
        if (key0 < me.keys && alive) {
            const uint32_t k_at = s_base + slot * G::TILE + warp * SUBS * SUB_BYTES, v_at = k_at + G::TILE;          // my rows
            const unsigned char *scales = smem + G::OFF_SCALES + slot * G::KEYS + warp * KW;
            const bool edge = key0 + KW > lim_first;      // not every row attends to all of the group
            float s[SUBS][4];
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[sub][k] = 0.f;
            if constexpr (QUANT) {
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {        // 16 bytes: four steps
                    uint4 b[2 * SUBS];
#pragma unroll
                    for (int n = 0; n < 2 * SUBS; ++n) {
                        const int row = 8 * n + g, chunk = D == 128 ? ((2 * t + c) ^ (row & 7)) : (t ^ ((row >> 1) & 3));
                        b[n] = lds128(k_at + row * D + chunk * 16);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int sub = 0; sub < SUBS; ++sub) {
                            const uint4 lo = b[2 * sub], hi = b[2 * sub + 1];
                            const uint32_t x = k == 0 ? lo.x : k == 1 ? lo.y : k == 2 ? lo.z : lo.w, y = k == 0 ? hi.x : k == 1 ? hi.y : k == 2 ? hi.z : hi.w;
                            const uint32_t f[4] = {e4m3_halves(x, false), e4m3_halves(y, false), e4m3_halves(x, true), e4m3_halves(y, true)};
                            MP::mma(s[sub], f, qf[c * 4 + k][0], qf[c * 4 + k][1]);
                        }
                }
            } else {
                const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    const int chunk = 2 * st + ((lane >> 3) & 1);
#pragma unroll
                    for (int sub = 0; sub < SUBS; ++sub) {
                        uint32_t b[4];
                        ldmatrix_x4(b, k_at + sub * SUB_BYTES + (chunk >> 3) * HALF_BYTES + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
                        const uint32_t f[4] = {b[0], b[2], b[1], b[3]};
                        MP::mma(s[sub], f, qf[st][0], qf[st][1]);
                    }
                }
                done_with(slot);
                k_held = false;
            }
            // ---- softmax of the group: key sub * 16 + kk * 8 + g and row 2 t + q at s[sub][2 kk + q]
            float mx[2] = {-INFINITY, -INFINITY}, mw[2] = {-INFINITY, -INFINITY}, e_v[SUBS][2];
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const int key = sub * 16 + kk * 8 + g;
                    const float ks = QUANT ? e8m0_value(scales[key]) : 1.f;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float v = s[sub][2 * kk + q] * (QUANT ? ks * row_c2[q] : a.scale_log2);
                        if (edge && key0 + key >= limit[q]) v = -INFINITY;
                        s[sub][2 * kk + q] = v;
                        mx[q] = fmaxf(mx[q], v);
                    }
                }
            if constexpr (QUANT) {
                done_with(slot);
                k_held = false;
            }
            alive = __all_sync(0xffffffffu, wait_for(bar_full + (slot + 1) * 8, parity));     // V
            if constexpr (QUANT) {
#pragma unroll
                for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk) {
                        const int b = scales[G::KEYS + sub * 16 + kk * 8 + g];
                        e_v[sub][kk] = b == 255 ? NAN : float(b - 127);
#pragma unroll
                        for (int q = 0; q < 2; ++q) mw[q] = fmaxf(mw[q], s[sub][2 * kk + q] + e_v[sub][kk]);         // (a maximum passes over a NaN)
                    }
            }
            bool up = false;
            float alpha[2], alpha_w[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                auto move = [&](float &had, float &seen, float &by, float lift) {        // the running maximum, as a reference, and what it takes what was summed by
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) seen = fmaxf(seen, __shfl_xor_sync(0xffffffffu, seen, x));
                    const float now = fmaxf(had, seen);
                    up = up || now > had;
                    by = now == -INFINITY ? 1.f : fast_exp2(had - now);
                    had = now;
                    seen = now == -INFINITY ? 0.f : now - lift;
                };
                move(m[q], mx[q], alpha[q], LIFT);
                alpha_w[q] = alpha[q];
                if constexpr (QUANT) move(m_w[q], mw[q], alpha_w[q], kLift);
            }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int n = 0; n < NP; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[n][k] *= alpha_w[k & 1];
                l[0] *= alpha[0];
                l[1] *= alpha[1];
            }
            uint32_t pf[SUBS][2];
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    float p[2];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const float v = s[sub][2 * kk + q];
                        p[q] = fast_exp2(v - mx[q]);
                        l[q] += p[q];
                        // (what a masked key holds, NaN too, stays out)
                        if constexpr (QUANT) p[q] = v == -INFINITY ? 0.f : fast_exp2(v + e_v[sub][kk] - mw[q]);
                    }
                    pf[sub][kk] = transposed(MP::pack(p[0], p[1]));
                }
            // ---- second product
            const int here = min(me.kv, (me.keys + 15) & ~15) - key0;     // rows of V that were fetched and are the sequence's
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub) {
                if constexpr (QUANT) {
                    // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9, bytes D/8 g ..: columns D/8 n + j in tile j of eight
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
                        if (edge && row >= here) {        // zero times a NaN byte would be NaN
#pragma unroll
                            for (int c = 0; c < D / 32; ++c) w[k][c] = 0u;
                        }
                    }
#pragma unroll
                    for (int c = 0; c < D / 32; ++c)
#pragma unroll
                        for (int hl = 0; hl < 2; ++hl) {  // column tiles from bytes 2 hl, 2 hl + 1 of the keys
                            const uint32_t x = __byte_perm(w[0][c], w[1][c], hl ? 0x7362 : 0x5140), y = __byte_perm(w[2][c], w[3][c], hl ? 0x7362 : 0x5140);
                            const uint32_t f[4] = {e4m3_halves(x, false), e4m3_halves(x, true), e4m3_halves(y, false), e4m3_halves(y, true)};
                            MP::mma(acc[c * 2 + hl], f, pf[sub][0], pf[sub][1]);
                        }
                } else {
                    const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
                    for (int j = 0; j < NP; ++j) {
                        const int chunk = 2 * j + (lane >> 4);
                        uint32_t b[4];
                        ldmatrix_x4_trans(b, v_at + sub * SUB_BYTES + (chunk >> 3) * HALF_BYTES + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
                        if (edge) {                       // zero times what is not finite would be NaN
#pragma unroll
                            for (int k = 0; k < 4; ++k) poisoned = keep_finite<T>(b[k], here - sub * 16 - (k & 1) * 8 - 2 * t) || poisoned;
                        }
                        const uint32_t f[4] = {b[0], b[2], b[1], b[3]};
                        MP::mma(acc[j], f, pf[sub][0], pf[sub][1]);
                    }
                }
            }
        } else if (me.keys > 0 && alive) {
            // No key of this tile is mine: V's stage goes back once it is full, see chunk_mma_kernel.
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
            // ---- the warps' results of this piece, through shared memory
            const bool from_start = i >= me.tile, whole = from_start && me.tile + 1 == me.tiles;
            uint32_t bad;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, 1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                         : "=r"(bad) : "r"(uint32_t(poisoned)), "n"(G::WARPS * 32) : "memory");
            float2 *stats = reinterpret_cast<float2 *>(smem + G::OFF_STATS);
            float *rows = reinterpret_cast<float *>(smem + G::OFF_MERGE);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float sum = l[q];
#pragma unroll
                for (int x = 4; x < 32; x *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                if (g == 0) stats[warp * 8 + 2 * t + q] = make_float2(m[q] - LIFT, sum);
                float *to = rows + (warp * 8 + 2 * t + q) * (D + 4);
                if constexpr (QUANT) {
                    float by, then;                       // weights back to the probabilities' reference
                    weights_back(m[q], m_w[q], 1.f / 32768.f, by, then);
#pragma unroll
                    for (int n = 0; n < NP; n += 2)
                        *reinterpret_cast<float4 *>(to + g * (D / 8) + 2 * n) =
                            make_float4(acc[n][q] * by * then, acc[n][2 + q] * by * then, acc[n + 1][q] * by * then, acc[n + 1][2 + q] * by * then);
                } else {
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        to[n * 16 + g] = acc[n][q];
                        to[n * 16 + 8 + g] = acc[n][2 + q];
                    }
                }
            }
            meet();
            if (G::WARPS == 8 || warp < 8) {              // a warp per row
                constexpr int C = D / 32;
                float top = -INFINITY, sum = 0.f, out[C];
#pragma unroll
                for (int w = 0; w < G::WARPS; ++w) top = fmaxf(top, stats[w * 8 + warp].x);
#pragma unroll
                for (int k = 0; k < C; ++k) out[k] = 0.f;
#pragma unroll
                for (int w = 0; w < G::WARPS; ++w) {
                    const float2 st = stats[w * 8 + warp];
                    if (st.x == -INFINITY && st.y == 0.f) continue;              // saw nothing
                    const float f = top == -INFINITY ? 1.f : st.x == -INFINITY ? 1.f : fast_exp2(st.x - top);
                    sum += st.y * f;
#pragma unroll
                    for (int k = 0; k < C; ++k) out[k] += rows[(w * 8 + warp) * (D + 4) + lane * C + k] * f;
                }
                const int r = me.qt * G::ROWS + warp, tok = by_group(a, r), head = me.h * a.group + (r - tok * a.group);
                if (bad != 0u && tok < me.ql) {
                    // keys of this piece whose groups were looked through, as far as my row sees them
                    const int keys = a.causal ? min(me.kv, me.kv - me.ql + tok + 1) : me.kv;
                    add_not_finite<T, C, QUANT>(a, me.z, me.h, max(max(lim_first, 0) & ~(KW - 1), max(0, me.tile - i) * G::KEYS),
                                                min(keys, (me.tile + 1) * G::KEYS), lane * C, out);
                }
                if (whole) {
                    if (tok < me.ql) {
                        const float inv = sum == 0.f ? 0.f : 1.f / sum;
                        T *dst = static_cast<T *>(a.o) + me.z * a.os_z + head * a.os_h + tok * a.os_n + lane * C;
                        if constexpr (C == 4)
                            *reinterpret_cast<uint2 *>(dst) = make_uint2(MmaTraits<T>::pack(out[0] * inv, out[1] * inv), MmaTraits<T>::pack(out[2] * inv, out[3] * inv));
                        else
                            *reinterpret_cast<uint32_t *>(dst) = MmaTraits<T>::pack(out[0] * inv, out[1] * inv);
                        if (a.lse != nullptr && lane == 0) a.lse[(size_t(me.z) * a.H + head) * a.n_q + tok] = sum == 0.f ? -INFINITY : top + log2f(sum);
                    }
                } else {
                    const size_t at = (size_t(2) * blockIdx.x + (from_start ? 1 : 0)) * G::ROWS + warp;
#pragma unroll
                    for (int k = 0; k < C; ++k) a.part[at * D + lane * C + k] = out[k];
                    if (lane == 0) reinterpret_cast<float2 *>(a.part + chunk_stats_at(gridDim.x, G::ROWS, D))[at] = make_float2(top, sum);
                }
            }
            meet();
        }
        if (i + 1 < n_tiles) me.next(line);
    }
    if (!alive && lane == 0) report(a.status, FST_DEV_TIMEOUT, blockIdx.x, warp);
    if (tid == 0 && a.part != nullptr) leave_cut<D>(a, me, total, n_tiles);
}

template <typename T, int D, bool QUANT>
static cudaError_t launch_chunk_token(const ChunkArgs &a, const CUtensorMap &tk, const CUtensorMap &tv, int n_ctas, cudaStream_t stream) {
    using G = ChunkTokenGeo<D, QUANT>;
    static_assert(G::BYTES <= 227 * 1024, "one CTA's shared memory");
    static DeviceOnce configured;
    const cudaError_t ce = configured.run([&] {
        return cudaFuncSetAttribute(chunk_token_kernel<T, D, QUANT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::BYTES);
    });
    if (ce != cudaSuccess) return ce;
    const cudaError_t e = launch_serialised(chunk_token_kernel<T, D, QUANT>, dim3(n_ctas), dim3(G::THREADS), G::BYTES, stream, a, tk, tv);
    if (e != cudaSuccess || !chunk_splits(a, G::KEYS)) return e;
    return launch_chunk_combine<T, D, G::ROWS>(a, n_ctas, stream);
}

}  // namespace fst
