// Dense 4-bit matrix-vector products for the decode batch:
//   y[m, n] = bf16( sum_g s[g, n] * sum_{k in group g} q[k, n] * x[m, k] )
// with q the int4pack words of the artifact, read unchanged (int32 [K, N/8], nibble t of word j of a
// row = q[k, 8j+t], two's complement; tools/repack_w4a16.py:64-70), s bf16 [G, N], x bf16 [M, K].
// The products of one scale group are sums of small integers times bf16 values, exact in fp32 up to
// the accumulation; the group sum is then multiplied by its scale in fp32.  No weight is rounded:
// bf16(q * s), what the grouped GEMM multiplies with, would cost a rounding per weight and an
// instruction more.
//
// Bound: the weight stream, K * N / 2 bytes read once.  The products run on mma.sync m16n8k16, which
// is far from its rate at this traffic: weights are the 16-row operand straight from registers, the
// tokens the 8-column one.  A lane loads one or two words of four consecutive rows k; two rows'
// words interleaved by byte permutes hold the (k, k+1) pairs the fragments want: nibble i of both in
// one word, extracted with one and-or into the mantissa of 128.0 and one subtraction (exact).  The
// order of k inside a fragment is free as long as the tokens use the same one: lane t of a fragment
// group takes rows 4t .. 4t+3 of a 16-row step, so its tokens are one 8-byte load.
// Split: a warp takes 64 * WPL features; eight warps of a CTA split 4 / 2 over K and the rest over
// features; the CTAs of a cluster split K again and add their parts through distributed shared
// memory in a fixed order (deterministic).
#pragma once
#include "fnx_common.cuh"

namespace fnx {

constexpr int W4D_THREADS = 256;
constexpr int W4D_FEATS = 256;                  // features of a CTA

// (a & 0xf of both halves) ^ 0x4308 - 136: the signed nibbles of both 16-bit halves, exact in bf16
FNX_DEV uint32_t nib_pair(uint32_t v) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(v), "r"(0x000f000fu), "r"(0x43084308u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0x43084308u));
    return r;
}

struct W4DenseParams {
    const bf16* x;
    const uint32_t* w;
    const bf16* s;
    bf16* y;
    long long ld_x;
    int M, K, N, gs;
};

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
                uint32_t lo0 = __byte_perm(wv[buf][u][0][a], wv[buf][u][1][a], 0x5410);
                uint32_t hi0 = __byte_perm(wv[buf][u][0][a], wv[buf][u][1][a], 0x7632);
                uint32_t lo1 = __byte_perm(wv[buf][u][2][a], wv[buf][u][3][a], 0x5410);
                uint32_t hi1 = __byte_perm(wv[buf][u][2][a], wv[buf][u][3][a], 0x7632);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t a0 = nib_pair(lo0 >> (4 * i)), a1 = nib_pair(hi0 >> (4 * i));
                    const uint32_t a2 = nib_pair(lo1 >> (4 * i)), a3 = nib_pair(hi1 >> (4 * i));
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma_16816_bf16(acc[a][i][n], a0, a1, a2, a3, xv[buf][u][n].x, xv[buf][u][n].y);
                }
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

    // parts of the CTA's warps, then of the cluster's CTAs, in order
#pragma unroll
    for (int a = 0; a < WPL; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int tok = n * 8 + 2 * t + c;
                if (tok < mt) {
                    float* o = red + ((size_t)wk * mt + tok) * W4D_FEATS + wn * WF + (g * WPL + a) * 8;
                    *reinterpret_cast<float4*>(o) = make_float4(tot[a][0][n][c], tot[a][1][n][c], tot[a][2][n][c],
                                                                tot[a][3][n][c]);
                    *reinterpret_cast<float4*>(o + 4) = make_float4(tot[a][0][n][2 + c], tot[a][1][n][2 + c],
                                                                    tot[a][2][n][2 + c], tot[a][3][n][2 + c]);
                }
            }
    __syncthreads();
    const int cells = mt * W4D_FEATS;
    for (int i = threadIdx.x; i < cells; i += W4D_THREADS) {
        float v = red[i];
#pragma unroll
        for (int k = 1; k < WK; ++k) v += red[k * cells + i];
        red[i] = v;
    }
    if (CL > 1) cluster_sync_all(); else __syncthreads();
    const int per = (cells / 2 + CL - 1) / CL;                  // pairs of features of this CTA
    for (int i = (int)rank * per + threadIdx.x; i < min(cells / 2, (int)(rank + 1) * per); i += W4D_THREADS) {
        const int tok = 2 * i / W4D_FEATS, f = blockIdx.x * W4D_FEATS + 2 * i % W4D_FEATS;
        if (f >= p.N) continue;
        float2 v = make_float2(0.f, 0.f);
        for (int r = 0; r < CL; ++r) {
            float2 q;
            if (CL > 1) {
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                             : "=f"(q.x), "=f"(q.y) : "r"(mapa_rank(red + 2 * i, r)) : "memory");
            } else {
                q = *reinterpret_cast<const float2*>(red + 2 * i);
            }
            v.x += q.x;
            v.y += q.y;
        }
        *reinterpret_cast<uint32_t*>(p.y + (long long)(m0 + tok) * p.N + f) = pack_bf2(v.x, v.y);
    }
    if (CL > 1) cluster_sync_all();                             // every part stays until all have read it
}

template <int WPL, int NT>
inline size_t w4_dense_smem(int M) {
    constexpr int WK = 8 / (W4D_FEATS / (64 * WPL));
    return (size_t)WK * (M < 8 * NT ? M : 8 * NT) * W4D_FEATS * sizeof(float);
}

}  // namespace fnx
