// Dense 4-bit matrix-vector products for the decode batch:
//   y[m, n] = bf16( sum_g s[g, n] * sum_{k in group g} q[k, n] * x[m, k] )
// with q the int4pack words of the artifact, read unchanged (int32 [K, N/8], nibble t of word j of a
// row = q[k, 8j+t], two's complement; tools/repack_w4a16.py:64-70), s bf16 [G, N], x bf16 [M, K].
// The products of one scale group are sums of small integers times bf16 values, exact in fp32 up to
// the accumulation; the group sum is then multiplied by its scale in fp32.  No weight is rounded:
// bf16(q * s), what the grouped GEMM multiplies with, would cost a rounding per weight and an
// instruction more.
//
// Bound: the weight stream, K * N / 2 bytes read once, at long streams the issue of its conversion (8192 x
// 28672, groups of 128, one token: 33.8 us, 3.6 TB/s of weights and scales; 4096 x 28672, groups of 32,
// 16 tokens: 28.0 us), at short ones a launch and the cluster's sum (2048 x 5120, one token: 5.8 us).
// The products run on mma.sync m16n8k16, which is far from its rate at this traffic (21 % busy): weights
// are the 16-row operand straight from registers, the tokens the 8-column one.  A byte permute brings
// the same byte of two rows' words into the two halves of a register, whose nibbles are then the (k, k+1)
// pairs that the fragments want (nib_lo, nib_hi).
// Split: the warps of a CTA split its 256 features (224: see QUAD) and K; the CTAs of a cluster split K
// again and add their parts through distributed shared memory in a fixed order (deterministic).
//
// w4_dense_kernel, short streams: a lane loads one or two words of four consecutive rows k, rows 4t ..
// 4t+3 of a 16-row step (the order of k inside a fragment is free as long as the tokens use the same
// one), so its tokens are one 8-byte load.
#pragma once
#include "fnx_common.cuh"

namespace fnx {

constexpr int W4D_THREADS = 256;
constexpr int W4D_FEATS = 256;                  // features of a CTA

// The signed nibbles of both halves of v, times 2^-6, exact in bf16.  v holds one byte of row k's word
// in the low byte of its low half and the same byte of row k+1's in its high half (other bits are
// masked).  The masked nibble, its sign bit flipped, is read as a bf16 subnormal (or, from 8 on, the
// first normal binade, which has the same spacing): n * 2^-133 for the low nibble, n * 2^-129 for the
// high one, with no shift; one multiply-add takes it to (n - 8) * 2^-6.  Against the mantissa of 128.0
// and a subtraction this saves every shift: 12 integer instructions for 16 weights instead of 16, on
// the half-rate pipe that bounds the kernel.  The sums carry the 2^-6 (a power of two) to the end.
FNX_DEV uint32_t nib_lo(uint32_t v) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(v), "r"(0x000f000fu), "r"(0x00080008u));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(r), "r"(0x7f007f00u), "r"(0xbe00be00u));
    return r;
}
FNX_DEV uint32_t nib_hi(uint32_t v) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(v), "r"(0x00f000f0u), "r"(0x00800080u));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(r), "r"(0x7d007d00u), "r"(0xbe00be00u));
    return r;
}
// Fragment registers of four MMAs (features i and i + 4 of a word, i < 4) from the words of rows k, k+1
// and k+8, k+9.
FNX_DEV void nib_fragments(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&a)[4][4]) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const uint32_t sel = 0x4400u + 0x1111u * b, sel2 = sel + 0x2222u;
        const uint32_t p0 = __byte_perm(w0, w1, sel), p1 = __byte_perm(w0, w1, sel2);
        const uint32_t q0 = __byte_perm(w2, w3, sel), q1 = __byte_perm(w2, w3, sel2);
        a[2 * b][0] = nib_lo(p0); a[2 * b][1] = nib_lo(p1); a[2 * b][2] = nib_lo(q0); a[2 * b][3] = nib_lo(q1);
        a[2 * b + 1][0] = nib_hi(p0); a[2 * b + 1][1] = nib_hi(p1);
        a[2 * b + 1][2] = nib_hi(q0); a[2 * b + 1][3] = nib_hi(q1);
    }
}

struct W4DenseParams {
    const bf16* x;
    const uint32_t* w;
    const bf16* s;
    bf16* y;
    long long ld_x;
    int M, K, N, gs;
};

// Adds the parts of the CTA's warps, then of the cluster's CTAs, in order, and writes y.  red: [WK][mt][W4D_FEATS].
template <int WPL, int NT, int FEATS>
FNX_DEV void w4_dense_finish(const W4DenseParams& p, const float (&tot)[WPL][4][NT][4], float* red, int wn, int wk, int g,
                             int t, uint32_t rank, int CL, int m0, int mt) {
    constexpr int WF = 64 * WPL, WN = W4D_FEATS / WF, WK = 8 / WN;
    constexpr int WW = FEATS / 8 / WN;          // words of a warp (lanes beyond them hold nothing)
    pdl_launch_dependents();
#pragma unroll
    for (int a = 0; a < WPL; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int tok = n * 8 + 2 * t + c;
                if (tok < mt && g * WPL + a < WW) {
                    float* o = red + ((size_t)wk * mt + tok) * FEATS + (wn * WW + g * WPL + a) * 8;
                    *reinterpret_cast<float4*>(o) = make_float4(tot[a][0][n][c], tot[a][1][n][c], tot[a][2][n][c],
                                                                tot[a][3][n][c]);
                    *reinterpret_cast<float4*>(o + 4) = make_float4(tot[a][0][n][2 + c], tot[a][1][n][2 + c],
                                                                    tot[a][2][n][2 + c], tot[a][3][n][2 + c]);
                }
            }
    __syncthreads();
    const int cells = mt * FEATS;
    for (int i = threadIdx.x; i < cells; i += blockDim.x) {
        float v = red[i];
#pragma unroll
        for (int k = 1; k < WK; ++k) v += red[k * cells + i];
        red[i] = v;
    }
    if (CL > 1) cluster_sync_all(); else __syncthreads();
    const int per = (cells / 2 + CL - 1) / CL;                  // pairs of features of this CTA
    for (int i = (int)rank * per + threadIdx.x; i < min(cells / 2, (int)(rank + 1) * per); i += blockDim.x) {
        const int tok = 2 * i / FEATS, f = blockIdx.x * FEATS + 2 * i % FEATS;
        if (f >= p.N) continue;
        float2 v = *reinterpret_cast<const float2*>(red + 2 * i);
        if (CL > 1) {
            float2 q[8];                                        // all requested before the first is added
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < CL)
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                                 : "=f"(q[r].x), "=f"(q[r].y) : "r"(mapa_rank(red + 2 * i, r)) : "memory");
            v = q[0];
#pragma unroll
            for (int r = 1; r < 8; ++r)
                if (r < CL) {
                    v.x += q[r].x;
                    v.y += q[r].y;
                }
        }
        *reinterpret_cast<uint32_t*>(p.y + (long long)(m0 + tok) * p.N + f) = pack_bf2(v.x * 64.f, v.y * 64.f);
    }
    if (CL > 1) cluster_sync_all();                             // every part stays until all have read it
}

// WPL words of a row per lane (two need N % 16 == 0), NT tiles of 8 tokens.
template <int WPL, int NT>
__global__ void __launch_bounds__(W4D_THREADS, 2) w4_dense_kernel(const W4DenseParams p) {
    constexpr int WF = 64 * WPL;                // features of a warp
    constexpr int WN = W4D_FEATS / WF;          // warps over features
    constexpr int WK = 8 / WN;                  // warps over K
    constexpr int U = 2;                        // 16-row steps per load batch
    extern __shared__ __align__(16) float red[];     // [WK][tokens][W4D_FEATS]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int wn = warp % WN, wk = warp / WN;
    const int m0 = blockIdx.z * 8 * NT;
    const int mt = min(p.M - m0, 8 * NT);
    const uint32_t rank = cluster_rank();
    const int CL = gridDim.y;

    // this warp's 16-row steps
    const int steps = (p.K + 15) / 16, parts = CL * WK, part = (int)rank * WK + wk;
    const int st0 = (int)((long long)steps * part / parts), st1 = (int)((long long)steps * (part + 1) / parts);
    const int words = p.N / 8;
    const int wc = blockIdx.x * (W4D_FEATS / 8) + wn * (WF / 8) + g * WPL;       // first word of this lane
    const bool col_ok = wc < words;
    const uint32_t* wp = p.w + wc;

    pdl_wait();
    float tot[WPL][4][NT][4], acc[WPL][4][NT][4];
#pragma unroll
    for (int a = 0; a < WPL; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) tot[a][i][n][e] = acc[a][i][n][e] = 0.f;

    uint32_t wv[2][U][4][WPL];
    uint2 xv[2][U][NT];
    auto load = [&](int buf, int st) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (st + u) * 16 + 4 * t;
            const bool k_ok = st + u < st1 && k < p.K;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (WPL == 2) {
                    uint2 v = make_uint2(0, 0);
                    if (k_ok && col_ok) v = __ldcs(reinterpret_cast<const uint2*>(wp + (long long)(k + r) * words));
                    wv[buf][u][r][0] = v.x;
                    wv[buf][u][r][WPL - 1] = v.y;
                } else {
                    wv[buf][u][r][0] = k_ok && col_ok ? __ldcs(wp + (long long)(k + r) * words) : 0u;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                xv[buf][u][n] = make_uint2(0, 0);
                if (k_ok && n * 8 + g < mt)
                    xv[buf][u][n] = *reinterpret_cast<const uint2*>(p.x + (long long)(m0 + n * 8 + g) * p.ld_x + k);
            }
        }
    };
    auto scale = [&](int grp) {
        float sc[8];
#pragma unroll
        for (int a = 0; a < WPL; ++a) {
            uint4 u4 = make_uint4(0, 0, 0, 0);
            if (col_ok) u4 = *reinterpret_cast<const uint4*>(p.s + (long long)grp * p.N + (wc + a) * 8);
            sc[0] = bf_lo(u4.x); sc[1] = bf_hi(u4.x); sc[2] = bf_lo(u4.y); sc[3] = bf_hi(u4.y);
            sc[4] = bf_lo(u4.z); sc[5] = bf_hi(u4.z); sc[6] = bf_lo(u4.w); sc[7] = bf_hi(u4.w);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        tot[a][i][n][e] = fmaf(sc[i + (e >= 2 ? 4 : 0)], acc[a][i][n][e], tot[a][i][n][e]);
                        acc[a][i][n][e] = 0.f;
                    }
        }
    };

    const int gsteps = p.gs / 16;
    int grp = st0 / gsteps, left = gsteps - st0 % gsteps;       // steps to the end of the group
    auto compute = [&](int buf, int st) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (st + u >= st1) break;
#pragma unroll
            for (int a = 0; a < WPL; ++a) {
                uint32_t f[4][4];
                nib_fragments(wv[buf][u][0][a], wv[buf][u][1][a], wv[buf][u][2][a], wv[buf][u][3][a], f);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma_16816_bf16(acc[a][i][n], f[i][0], f[i][1], f[i][2], f[i][3], xv[buf][u][n].x, xv[buf][u][n].y);
            }
            if (--left == 0) {
                scale(grp);
                ++grp;
                left = gsteps;
            }
        }
    };
    if (st0 < st1) {
        load(0, st0);
        int st = st0;
        while (true) {
            if (st + U < st1) load(1, st + U);
            compute(0, st);
            st += U;
            if (st >= st1) break;
            if (st + U < st1) load(0, st + U);
            compute(1, st);
            st += U;
            if (st >= st1) break;
        }
        if (left != gsteps) scale(grp);
    }

    w4_dense_finish<WPL, NT, W4D_FEATS>(p, tot, red, wn, wk, g, t, rank, CL, m0, mt);
}

template <int WPL, int NT>
inline size_t w4_dense_smem(int M) {
    constexpr int WK = 8 / (W4D_FEATS / (64 * WPL));
    return (size_t)WK * (M < 8 * NT ? M : 8 * NT) * W4D_FEATS * sizeof(float);
}

// The same sums for long weight streams: a ring of two or three stages of 256 rows x 256
// features kept in flight by TMA, with the tokens' 256 columns and the stage's scale rows, so neither
// the stream's depth nor a scale's latency is the warps' concern.  With the 128-byte swizzle the
// fragment loads are free of bank conflicts for the natural order of k (lane t: rows 2t, 2t+1, 2t+8,
// 2t+9 of a 16-row step).  A warp takes 64 features and half of the steps of a stage, and scales its
// sums at the end of each group or stage.  Bound by issue: the exact conversion alone is 1.25
// instructions a weight, 0.75 of them on the half-rate integer pipe.
constexpr int W4T_ROWS = 256;
constexpr int W4T_MAX_STAGES = 3;
constexpr int W4T_W_BYTES = W4T_ROWS * 128;

struct W4TmaParams {
    CUtensorMap tw, tx, ts;          // words, box {32, 256}; x, box {64, 8 NT}; scales, box {256, srows}
    W4DenseParams d;
    int stages, srows;               // of the ring; scale rows of a stage
    int gshift;                      // log2 of the steps of a group, or -1
};

__host__ __device__ inline int w4_tma_stage_bytes(int nt, int srows) {
    return W4T_W_BYTES + W4T_ROWS / 64 * nt * 1024 + (srows * 512 + 1023) / 1024 * 1024;      // x's boxes: 1 KB per 8 tokens and 64 k
}

// SEG: steps between two scalings where groups end at multiples of it in every warp's half of a stage
// (gs 32, 64, or a multiple of 128: 2, 4, 8), so that the eight steps are one straight piece of code;
// 0: wherever the group ends.
// QUAD: where N % 32 != 0 a row does not start on the 16 bytes that a copy needs.  Four rows together do,
// so the copies see K / 4 rows of four, one box for each row j of the four, from the 16 bytes below its
// first word (d_j = j * N / 8 mod 4 words further down); 28 words of a box's 32 are then the tile's,
// whichever d_j.  What a box holds beyond a row's end belongs to features that are not stored.
template <int NT, int SEG, int QUAD>
__global__ void __launch_bounds__(W4D_THREADS, 2) w4_dense_tma_kernel(const __grid_constant__ W4TmaParams q) {
    constexpr int WN = 4, WK = 2, STEPS = W4T_ROWS / 16 / WK;
    constexpr int TW = QUAD ? 28 : 32, WW = TW / WN;     // words of a tile and of a warp
    const W4DenseParams& p = q.d;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = align1024(smem_raw);
    __shared__ uint64_t full[W4T_MAX_STAGES], empty[W4T_MAX_STAGES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int wn = warp % WN, wk = warp / WN;
    const int m0 = blockIdx.z * 8 * NT, mt = min(p.M - m0, 8 * NT);
    const uint32_t rank = cluster_rank();
    const int CL = gridDim.y;
    const int stage_bytes = w4_tma_stage_bytes(NT, q.srows);
    const int total = (p.K + W4T_ROWS - 1) / W4T_ROWS;
    const int s0 = (int)((long long)total * rank / CL), ns = (int)((long long)total * (rank + 1) / CL) - s0;
    const int gsteps = p.gs / 16;
    auto group_of = [&](int step) { return q.gshift >= 0 ? step >> q.gshift : step / gsteps; };

    if (threadIdx.x == 0) {
        for (int i = 0; i < W4T_MAX_STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 8);
        }
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    const int NS = q.stages;
    auto fetch = [&](int j, int s) {                     // stage j of this CTA into slot s, by one thread
        const int row = (s0 + j) * W4T_ROWS;
        const uint32_t w = smem_u32(base + s * stage_bytes);
        mbar_arrive_expect_tx(&full[s], W4T_W_BYTES + W4T_ROWS / 64 * NT * 1024 + q.srows * 512);
        if (QUAD) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                tma_load_2d(w + i * (W4T_W_BYTES / 4), &q.tw, &full[s], (i * (p.N / 8) + (int)blockIdx.x * TW) & ~3, row / 4);
        } else {
            tma_load_2d(w, &q.tw, &full[s], blockIdx.x * TW, row);
        }
#pragma unroll
        for (int i = 0; i < W4T_ROWS / 64; ++i)
            tma_load_2d(w + W4T_W_BYTES + i * NT * 1024, &q.tx, &full[s], row + 64 * i, m0);
        tma_load_2d(w + W4T_W_BYTES + W4T_ROWS / 64 * NT * 1024, &q.ts, &full[s], blockIdx.x * (TW * 8),
                    group_of((s0 + j) * (W4T_ROWS / 16)));
    };
    if (warp == 0) {
        if (elect_one())
            for (int j = 0; j < min(ns, NS); ++j) fetch(j, j);
        __syncwarp();
    }

    float tot[1][4][NT][4], acc[4][NT][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) tot[0][i][n][e] = acc[i][n][e] = 0.f;
    // offsets in a stage: the words of rows 2t and 2t+1 of this warp's first step (rows 8 further are
    // 1024 bytes on, steps 2048), the tokens' words of its first eight k (eight k further: another
    // 16-byte chunk, its index exchanged with the row's by the swizzle)
    const int word = wn * WW + min(g, WW - 1);
    uint32_t w0, w1;
    if (QUAD) {                                          // row r of a step: box r % 4, its row 4 step + r / 4
        auto at = [&](int r) {
            const int d = word + (((r & 3) * (p.N / 8)) & 3);
            return (r & 3) * (W4T_W_BYTES / 4) + (wk * STEPS * 4 + (r >> 2)) * 128 + (((d >> 2) ^ (r >> 2)) << 4) + (d & 3) * 4;
        };
        w0 = at(2 * t);
        w1 = at(2 * t + 1);
    } else {
        auto at = [&](int r) {
            return wk * STEPS * 2048 + r * 128 + (((word >> 2) ^ r) << 4) + (word & 3) * 4;
        };
        w0 = at(2 * t);
        w1 = at(2 * t + 1);
    }
    // word i (row 2t, 2t+1, 2t+8, 2t+9) of step u
    auto word_at = [&](int u, int i) {
        const uint32_t o = i & 1 ? w1 : w0;
        return QUAD ? (o ^ (((4 * u + (i & 2)) & 7) << 4)) + u * 512 + (i & 2) * 128 : o + u * 2048 + (i & 2) * 512;
    };
    const uint32_t x0 = W4T_W_BYTES + wk * (STEPS / 4) * NT * 1024 + g * 128 + (g << 4) + t * 4;
    const uint32_t c0 = W4T_W_BYTES + W4T_ROWS / 64 * NT * 1024 + word * 16;

    bool alive = true;                                   // no wait has expired
    for (int j = 0, s = 0, ph = 0; j < ns; ++j) {
        // the slot of the stage before is refilled once its warps are done (the phase the other slots had)
        if (warp == 0 && j >= 1 && j - 1 + NS < ns) {
            const int sp = s ? s - 1 : NS - 1;
            alive = __all_sync(0xffffffffu, mbar_wait(&empty[sp], s ? ph : ph ^ 1));
            if (!alive) break;
            if (elect_one()) fetch(j - 1 + NS, sp);
            __syncwarp();
        }
        alive = __all_sync(0xffffffffu, mbar_wait(&full[s], ph));
        if (!alive) break;
        const uint8_t* S = base + s * stage_bytes;
        const int first = (s0 + j) * (W4T_ROWS / 16), mine = first + wk * STEPS;
        int left = 0;                                    // steps to the end of the group
        const int grp = group_of(mine);
        if (SEG == 0) left = (grp + 1) * gsteps - mine;
        const uint8_t* sc = S + c0 + (grp - group_of(first)) * 512;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            uint32_t wv[4], b[NT][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) wv[i] = *reinterpret_cast<const uint32_t*>(S + word_at(u, i));
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    b[n][h] = *reinterpret_cast<const uint32_t*>(S + (x0 ^ (((2 * u + h) & 7) << 4)) + (u / 4 * NT + n) * 1024);
            uint32_t f[4][4];
            nib_fragments(wv[0], wv[1], wv[2], wv[3], f);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_16816_bf16(acc[i][n], f[i][0], f[i][1], f[i][2], f[i][3], b[n][0], b[n][1]);
            if (SEG ? u % (SEG ? SEG : 1) == SEG - 1 : (--left == 0 || u == STEPS - 1)) {
                const uint4 u4 = *reinterpret_cast<const uint4*>(sc);
                const float v[8] = {bf_lo(u4.x), bf_hi(u4.x), bf_lo(u4.y), bf_hi(u4.y),
                                    bf_lo(u4.z), bf_hi(u4.z), bf_lo(u4.w), bf_hi(u4.w)};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            tot[0][i][n][e] = fmaf(v[i + (e >= 2 ? 4 : 0)], acc[i][n][e], tot[0][i][n][e]);
                            acc[i][n][e] = 0.f;
                        }
                sc += 512;
                left = gsteps;
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        if (++s == NS) s = 0, ph ^= 1;
    }
    if (!alive)                                          // time for the copies in flight to end
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();                                     // every stage is read: the sums reuse the ring
    w4_dense_finish<1, NT, TW * 8>(p, tot, reinterpret_cast<float*>(base), wn, wk, g, t, rank, CL, m0, mt);
}

// Stages of the ring: as many as leave room for two CTAs on an SM, at least two.
static_assert(1024 + 2 * (W4T_W_BYTES + W4T_ROWS / 64 * 2 * 1024 + ((W4T_ROWS - 1) / 16 + 2) * 512 + 1024) <= 113 * 1024 &&
                  1024 + 2 * 16 * W4D_FEATS * 4 <= 113 * 1024, "ring and sums");
inline int w4_tma_stages(int nt, int srows) {
    const int n = (int)(111 * 1024 / w4_tma_stage_bytes(nt, srows));
    return n < 2 ? 2 : n > W4T_MAX_STAGES ? W4T_MAX_STAGES : n;
}
template <int NT>
inline size_t w4_dense_tma_smem(int M, int srows) {
    const size_t ring = (size_t)w4_tma_stages(NT, srows) * w4_tma_stage_bytes(NT, srows);
    const size_t sums = w4_dense_smem<1, NT>(M);
    return 1024 + (ring > sums ? ring : sums);
}

}  // namespace fnx
