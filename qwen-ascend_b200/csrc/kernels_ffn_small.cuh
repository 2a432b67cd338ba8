// The products of the gated feed-forward block (kernels_ffn.cuh) where the 256 x 256 tiles of a CTA
// pair are too few for the 148 SMs: decode batches, short training batches, narrow blocks.  One CTA
// takes a 128 x BN tile and one part of K; the CTAs of a cluster hold the parts of one tile and add
// their fp32 accumulators through distributed shared memory in rank order (deterministic, no
// workspace) before the epilogue, which the ranks share.
//
// Bound: at few rows the weights' bytes (BN rows of 128 bytes per k-block and CTA through a ring of TMA
// copies as deep as shared memory allows: 16 rows of 4096 x 11008 take 50.3 us, 5.4 TB/s); at more rows
// or narrow blocks the latency of the chain of copies, products and the cluster's sum, 4 to 6 us a
// launch (one token of 2560 x 640: 9.8 us, a training step of 509 rows of 2048 x 512: 35.5 us).  Rows of A that do not exist are not loaded: the box holds p.a_rows (a power
// of two >= M) and the tensor core multiplies whatever lies behind it into rows that are not stored.
// A launch is a programmatic dependent of the kernel before it on the stream.  Behind another product
// of the chain its weights (operands that no kernel of the chain writes, b_early) stream in while that
// one finishes, the rest waits.  The last product of a chain lets its successor start when its own
// products are done (9.9 against 10.3 us for one token when it did so at once).
#pragma once
#include <type_traits>

#include "kernels_ffn.cuh"

namespace fnx {

constexpr int FS_THREADS = 256;      // warp 0 copies, 1 products, 2-5 drain the accumulator, all add the parts
constexpr int FS_MAX_STAGES = 16;
constexpr int FS_MAX_CL = 8;

struct FfnSmallProduct {
    CUtensorMap ta, tb;              // box {64, a_rows} / {64, BN/2} K-major, {64, 64} MN-major
    bf16 *c, *c2;                    // C; h; dg and du
    long long ldc;
    int M, N, K, amn, bmn, b_early;
    int nt, tiles;                   // column tiles, all tiles
};
struct FfnSmallParams {
    FfnSmallProduct q[FF_MAX_PRODUCTS];
    float* gu;
    int count, a_rows, stages, CL;   // a_rows: rows of a K-major A's box
    int followed;                    // another product of the chain follows: let it start at once
};

struct FfnSmallSmem {
    uint64_t full[FS_MAX_STAGES], empty[FS_MAX_STAGES], done;
    uint32_t tmem_base;
    volatile int abort;
};

FNX_DEV float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
FNX_DEV void st_bf16x4(bf16* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf2(a, b), pack_bf2(c, d));
}

// shared memory: the ring (the sums reuse it), 16 KB that the products may read behind the last stage
__host__ __device__ inline size_t ffn_small_ring(int bn, int a_rows, int stages) {
    return (size_t)stages * (a_rows * 128 + bn * 128);
}
__host__ __device__ inline size_t ffn_small_body(int bn, int a_rows, int stages) {
    const size_t ring = ffn_small_ring(bn, a_rows, stages) + 16384, sums = (size_t)128 * (bn + 4) * 4;
    return ring > sums ? ring : sums;
}

template <int EPI, int BN>
__global__ void __launch_bounds__(FS_THREADS) ffn_small_kernel(const __grid_constant__ FfnSmallParams p) {
    constexpr int COLS = EPI == FF_GATED ? BN / 2 : BN;      // columns of the output per tile
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = align1024(smem_raw);
    FfnSmallSmem& S = *reinterpret_cast<FfnSmallSmem*>(base + ffn_small_body(BN, p.a_rows, p.stages));
    float* sums = reinterpret_cast<float*>(base);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int CL = p.CL, rank = blockIdx.x % CL;             // clusters of CL consecutive CTAs
    int tile = blockIdx.x / CL, pi = 0;
    while (pi + 1 < p.count && tile >= p.q[pi].tiles) tile -= p.q[pi++].tiles;
    const FfnSmallProduct& q = p.q[pi];
    const int n = tile % q.nt, m0 = tile / q.nt * 128;
    const int rows = min(128, q.M - m0);
    const int KB = (q.K + FF_BK - 1) / FF_BK;
    const int kb0 = KB * rank / CL, nkb = KB * (rank + 1) / CL - kb0;
    const int a_bytes = p.a_rows * 128, stage_bytes = a_bytes + BN * 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        mbar_init(&S.done, 1);
        S.abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&S.tmem_base, BN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = S.tmem_base;

    if (warp == 0) {
        // ------------------------------------------------ TMA copies (a whole warp electing the issuer)
        auto load_b = [&](int s, int kb) {
            const uint32_t b = smem_u32(base + s * stage_bytes + a_bytes);
            const int k = kb * FF_BK;
            if (q.bmn) {
#pragma unroll
                for (int i = 0; i < BN / 64; ++i) tma_load_2d(b + i * 8192, &q.tb, &S.full[s], n * BN + i * 64, k);
            } else {
                const int r0 = EPI == FF_GATED ? n * COLS : n * BN;
                tma_load_2d(b, &q.tb, &S.full[s], k, r0);
                tma_load_2d(b + BN * 64, &q.tb, &S.full[s], k, EPI == FF_GATED ? q.N + r0 : r0 + BN / 2);
            }
        };
        auto load_a = [&](int s, int kb) {
            const uint32_t a = smem_u32(base + s * stage_bytes);
            const int k = kb * FF_BK;
            if (q.amn) {
                tma_load_2d(a, &q.ta, &S.full[s], m0, k);
                tma_load_2d(a + 8192, &q.ta, &S.full[s], m0 + 64, k);
            } else {
                tma_load_2d(a, &q.ta, &S.full[s], k, m0);
            }
        };
        if (!q.b_early) pdl_wait();
        // a successor of the chain reads its weights before its own wait: it may start once every CTA
        // here has seen the kernels before this one complete (followed only without b_early)
        if (p.followed) pdl_launch_dependents();
        const int first = min(nkb, p.stages);
        if (elect_one())
            for (int j = 0; j < first; ++j) {
                mbar_arrive_expect_tx(&S.full[j], stage_bytes);
                load_b(j, kb0 + j);
                if (!q.b_early) load_a(j, kb0 + j);
            }
        __syncwarp();
        if (q.b_early) {
            pdl_wait();
            if (elect_one())
                for (int j = 0; j < first; ++j) load_a(j, kb0 + j);
            __syncwarp();
        }
        for (int j = first; j < nkb; ++j) {
            const int s = j % p.stages;
            if (!__all_sync(0xffffffffu, mbar_spin(&S.empty[s], ((j / p.stages) & 1) ^ 1))) { S.abort = 1; break; }
            if (elect_one()) {
                mbar_arrive_expect_tx(&S.full[s], stage_bytes);
                load_b(s, kb0 + j);
                load_a(s, kb0 + j);
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issue
        pdl_wait();                                          // the bounded waits count from here
        auto multiply = [&](auto amn, auto bmn) {
            constexpr int AMN = decltype(amn)::value, BMN = decltype(bmn)::value;
            const uint32_t idesc = idesc_bf16_f32(128, BN) | ((uint32_t)AMN << 15) | ((uint32_t)BMN << 16);
            for (int j = 0; j < nkb; ++j) {
                const int s = j % p.stages;
                if (!__all_sync(0xffffffffu, mbar_spin(&S.full[s], (j / p.stages) & 1))) { S.abort = 1; break; }
                tc_fence_after();
                const uint32_t a0 = smem_u32(base + s * stage_bytes), b0 = a0 + a_bytes;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < FF_BK / 16; ++kk)
                        umma_bf16(tmem, sdesc_at(sdesc_sw128_base(AMN), a0 + kk * kstep_bytes(AMN)),
                                  sdesc_at(sdesc_sw128_base(BMN), b0 + kk * kstep_bytes(BMN)), idesc, (j | kk) ? 1u : 0u);
                    umma_commit(&S.empty[s]);
                }
                __syncwarp();
            }
        };
        using zero = std::integral_constant<int, 0>;
        using one = std::integral_constant<int, 1>;
        if (q.amn) multiply(one{}, one{});
        else if (q.bmn) multiply(zero{}, one{});
        else multiply(zero{}, zero{});
        if (elect_one()) umma_commit(&S.done);
        __syncwarp();
    } else if (warp < 6) {
        // ------------------------------------------------ this part's accumulators -> shared memory
        pdl_wait();
        const bool ok = mbar_wait(&S.done, 0);
        if (!__all_sync(0xffffffffu, ok)) S.abort = 1;
        tc_fence_after();
        const int lq = warp & 3, row = lq * 32 + lane;
        if (lq * 32 < rows) {
            float* o = sums + (size_t)row * (BN + 4);
#pragma unroll
            for (int c0 = 0; c0 < BN; c0 += 32) {
                uint32_t v[32];
                tmem_ld32(tmem + ((uint32_t)(lq * 32) << 16) + c0, v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    *reinterpret_cast<uint4*>(o + c0 + 4 * e) =
                        nkb ? make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]) : make_uint4(0, 0, 0, 0);
            }
        }
        tc_fence_before();
    }
    // after a wait that expired: time for the copies and products in flight to end
    if (S.abort)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();
    if (CL > 1) cluster_sync_all();
    pdl_wait();
    if (!p.followed) pdl_launch_dependents();

    // ---------------------------------------------------- the ranks' shares of the tile
    constexpr int C4 = COLS / 4;
    const int cells = rows * C4, per = (cells + CL - 1) / CL;
    const int cols4 = 2 * q.N / 4;
    for (int i = rank * per + threadIdx.x; i < min(cells, (rank + 1) * per); i += FS_THREADS) {
        const int r = i / C4, c = (i - r * C4) * 4, col = n * COLS + c;
        if (col >= q.N) continue;
        const float* src = sums + (size_t)r * (BN + 4) + c;
        float4 v = *reinterpret_cast<const float4*>(src), w = make_float4(0.f, 0.f, 0.f, 0.f);
        if (EPI == FF_GATED) w = *reinterpret_cast<const float4*>(src + COLS);
        if (CL > 1) {
            float4 a[FS_MAX_CL], b[FS_MAX_CL];               // all requested before the first is added
#pragma unroll
            for (int k = 0; k < FS_MAX_CL; ++k)
                if (k < CL) {
                    a[k] = ld_cluster_f4(mapa_rank(src, k));
                    if (EPI == FF_GATED) b[k] = ld_cluster_f4(mapa_rank(src + COLS, k));
                }
            v = a[0];
            if (EPI == FF_GATED) w = b[0];
#pragma unroll
            for (int k = 1; k < FS_MAX_CL; ++k)
                if (k < CL) {
                    v.x += a[k].x; v.y += a[k].y; v.z += a[k].z; v.w += a[k].w;
                    if (EPI == FF_GATED) { w.x += b[k].x; w.y += b[k].y; w.z += b[k].z; w.w += b[k].w; }
                }
        }
        const long long row = m0 + r;
        if (EPI == FF_PLAIN) {
            st_bf16x4(q.c + row * q.ldc + col, v.x, v.y, v.z, v.w);
        } else if (EPI == FF_GATED) {
            if (p.gu) {
                reinterpret_cast<float4*>(p.gu)[ffn_gu_index((int)row, col / 4, cols4)] = v;
                reinterpret_cast<float4*>(p.gu)[ffn_gu_index((int)row, cols4 / 2 + col / 4, cols4)] = w;
            }
            st_bf16x4(q.c + row * q.ldc + col, v.x * fast_sigmoid(v.x) * w.x, v.y * fast_sigmoid(v.y) * w.y,
                      v.z * fast_sigmoid(v.z) * w.z, v.w * fast_sigmoid(v.w) * w.w);
        } else {
            const float4 g4 = reinterpret_cast<const float4*>(p.gu)[ffn_gu_index((int)row, col / 4, cols4)];
            const float4 u4 = reinterpret_cast<const float4*>(p.gu)[ffn_gu_index((int)row, cols4 / 2 + col / 4, cols4)];
            const float g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w}, dh[4] = {v.x, v.y, v.z, v.w};
            float dg[4], du[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float s = fast_sigmoid(g[e]);
                dg[e] = dh[e] * u[e] * s * (1.0f + g[e] * (1.0f - s));
                du[e] = dh[e] * g[e] * s;
            }
            st_bf16x4(q.c + row * q.ldc + col, dg[0], dg[1], dg[2], dg[3]);
            st_bf16x4(q.c2 + row * q.ldc + col, du[0], du[1], du[2], du[3]);
        }
    }
    if (CL > 1) cluster_sync_all();                          // every part stays until all ranks have read it
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, BN);
    }
}

}  // namespace fnx
