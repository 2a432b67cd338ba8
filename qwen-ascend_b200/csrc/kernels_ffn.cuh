// The bf16 gated feed-forward block and its gradients on the 5th-generation tensor cores:
//   g = x Wg^T, u = x Wu^T, h = silu(g) u, y = h Wd^T                                       (forward)
//   dh = dy Wd, s = sigmoid(g): dg = dh u s (1 + g (1 - s)), du = dh g s,
//   dx = dg Wg + du Wu, dWgu = [dg du]^T x, dWd = dy^T h                                   (backward)
// (the always-on expert of the reference's deployment, fnx/engine.py:1786-1790: one concatenated
// gate/up GEMM, silu(gate) * up, down).  Six products, one kernel: C[m, n] = sum_k A(m, k) B(n, k) with
// each operand K-major (rows of k) or MN-major (rows of m / n, read transposed by the tensor core), so
// no operand is ever transposed in memory.  The activation runs in the epilogue of the gate/up
// product on the unrounded accumulators, and its derivative in the epilogue of dh, which is never
// stored; for that the forward of a training step keeps g and u in fp32 (8 bytes per element of h
// against four for bf16: rounding them would put two more roundings, 2^-9 each, into every gradient).
// What is rounded to bf16 between the products: h and [dg du], the operands of the next ones.
//
// A cluster of two CTAs (cta_group::2) takes a 256 x 256 tile: each CTA loads its half of the rows of
// A and of B by TMA (128-byte swizzle) into a ring of FF_STAGES 64-deep k-blocks; rank 0 issues
// M = 256, N = 256, K = 16 MMAs that read both CTAs' halves; every CTA holds 128 rows x 256 columns of
// fp32 in tensor memory, twice, so that one tile's epilogue runs under the next one's products.
// Both CTAs' copies complete on rank 0's `full` barrier; rank 0's commits release the stage and hand
// over the accumulator in both CTAs.  Edges read the tensor maps' zero fill and are clipped by the
// stores.  Roles:  warp 0 TMA copies (one thread), warp 1 MMA issue (rank 0), warps 2-5 epilogue.
#pragma once
#include "fnx_common.cuh"

namespace fnx {

constexpr int FF_BM = 256, FF_BN = 256, FF_BK = 64;
constexpr int FF_STAGES = 6;
constexpr int FF_A_BYTES = 128 * FF_BK * 2, FF_B_BYTES = 128 * FF_BK * 2;      // per CTA
constexpr int FF_STAGE = FF_A_BYTES + FF_B_BYTES;
constexpr int FF_EPI_BUF = 32 * 128;                                           // 32 rows x 64 bf16
constexpr int FF_THREADS = 192;

enum { FF_PLAIN = 0, FF_GATED = 1, FF_DGATE = 2 };

struct FfnParams {
    CUtensorMap ta, tb;              // operands: box {64, 128} K-major, {64, 64} MN-major
    CUtensorMap tc, tc2;             // outputs, box {64, 32}: C; h; or dg and du
    float* gu;                       // g and u, blocked (see ffn_gu_index); NULL: not kept
    int M, N, K;                     // N: columns of C (of h for FF_GATED, of dh for FF_DGATE)
};

struct FfnSmem {
    uint64_t full[FF_STAGES], empty[FF_STAGES], acc_full[2], acc_empty[2];
    uint32_t tmem_base;
    volatile int abort;
};

// g and u [rows, 2I] as float4s of four columns, blocks of 128 rows: consecutive lanes (rows) are
// consecutive 16-byte words, for the epilogue that writes them and the one that reads them.
FNX_DEV size_t ffn_gu_index(int row, int col4, int cols4) {
    return ((size_t)(row >> 7) * cols4 + col4) * 128 + (row & 127);
}

FNX_DEV void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar_cluster), "r"(x), "r"(y) : "memory");
}
FNX_DEV void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(map), "r"(src), "r"(x), "r"(y) : "memory");
}
FNX_DEV void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
FNX_DEV void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
template <int N>
FNX_DEV void bulk_wait() { asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory"); }

FNX_DEV void umma_bf16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 lanes x 32 consecutive 32-bit columns -> 32 registers per thread.
FNX_DEV void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// Shared-memory matrix descriptor, MN-major with the 128-byte swizzle: 64 m (or n) of one k are a
// 128-byte row, 8 k a 1024-byte group; groups of 8 k are 1024 B apart (SBO), the next 64 m (n) 8192 B
// further (LBO; a 64 x 64 box of the copy).
FNX_DEV uint64_t sdesc_mnmajor_sw128(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(8192 >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// sigmoid(g) for the activation: exponential and reciprocal are the fast forms (2^-21 relative), whose
// error is far below the bf16 rounding of every result
FNX_DEV float fast_sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

// Tile t of the schedule: groups of 8 row tiles, columns outside, rows inside, so the tiles in flight
// share rows of A and columns of B in L2.
FNX_DEV void ffn_tile(int t, int mt, int nt, int& m, int& n) {
    const int per = 8 * nt, g = t / per, r = t - g * per;
    const int rows = min(8, mt - 8 * g);
    n = r / rows;
    m = 8 * g + r - n * rows;
}

template <int AMN, int BMN, int EPI>
__global__ void __launch_bounds__(FF_THREADS, 1) ffn_gemm_kernel(const __grid_constant__ FfnParams p) {
    constexpr int COLS = EPI == FF_GATED ? 128 : 256;        // columns of the output (h, dh) per tile
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* epi_buf = base + FF_STAGES * FF_STAGE;
    FfnSmem& S = *reinterpret_cast<FfnSmem*>(epi_buf + 8 * FF_EPI_BUF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int cid = (int)cluster_id_x(), ncl = (int)num_clusters_x();
    const int mt = (p.M + FF_BM - 1) / FF_BM, nt = (p.N + COLS - 1) / COLS;
    const int total = mt * nt, KB = (p.K + FF_BK - 1) / FF_BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < FF_STAGES; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], 8);                   // four epilogue warps in each CTA
        }
        S.abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(&S.tmem_base, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = S.tmem_base;

    if (warp == 0) {
        // ------------------------------------------------ TMA copies of this CTA's halves
        if (lane == 0) {
            tma_prefetch_desc(&p.ta);
            tma_prefetch_desc(&p.tb);
            int j = 0;
            for (int t = cid; t < total && !S.abort; t += ncl) {
                int m, n;
                ffn_tile(t, mt, nt, m, n);
                const int ra = m * FF_BM + (int)rank * 128;
                // the gate/up product: rank 0 holds the gate rows of W, rank 1 the up rows
                const int rb = EPI == FF_GATED ? n * 128 + (int)rank * p.N : n * FF_BN + (int)rank * 128;
                for (int kb = 0; kb < KB; ++kb, ++j) {
                    const int s = j % FF_STAGES;
                    if (!mbar_wait_cluster(&S.empty[s], ((j / FF_STAGES) & 1) ^ 1)) { S.abort = 1; break; }
                    if (rank == 0) mbar_arrive_expect_tx(&S.full[s], 2 * FF_STAGE);
                    const uint32_t bar = mapa_rank(&S.full[s], 0);
                    const uint32_t a = smem_u32(base + s * FF_STAGE), b = a + FF_A_BYTES;
                    const int k = kb * FF_BK;
                    if (AMN) {
                        tma_load_2d_pair(a, &p.ta, bar, ra, k);
                        tma_load_2d_pair(a + 8192, &p.ta, bar, ra + 64, k);
                    } else {
                        tma_load_2d_pair(a, &p.ta, bar, k, ra);
                    }
                    if (BMN) {
                        tma_load_2d_pair(b, &p.tb, bar, rb, k);
                        tma_load_2d_pair(b + 8192, &p.tb, bar, rb + 64, k);
                    } else {
                        tma_load_2d_pair(b, &p.tb, bar, k, rb);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issue
        if (rank == 0 && lane == 0) {
            const uint32_t idesc = idesc_bf16_f32(FF_BM, FF_BN) | ((uint32_t)AMN << 15) | ((uint32_t)BMN << 16);
            int j = 0, i = 0;
            for (int t = cid; t < total && !S.abort; t += ncl, ++i) {
                const int ab = i & 1;
                if (!mbar_wait_cluster(&S.acc_empty[ab], ((i >> 1) & 1) ^ 1)) { S.abort = 1; break; }
                tc_fence_after();
                const uint32_t d = tmem + ab * FF_BN;
                for (int kb = 0; kb < KB; ++kb, ++j) {
                    const int s = j % FF_STAGES;
                    if (!mbar_wait_cluster(&S.full[s], (j / FF_STAGES) & 1)) { S.abort = 1; break; }
                    tc_fence_after();
                    const uint32_t a0 = smem_u32(base + s * FF_STAGE), b0 = a0 + FF_A_BYTES;
#pragma unroll
                    for (int kk = 0; kk < FF_BK / 16; ++kk)
                        umma_bf16_pair(d, AMN ? sdesc_mnmajor_sw128(a0 + kk * 2048) : sdesc_kmajor_sw128(a0 + kk * 32),
                                       BMN ? sdesc_mnmajor_sw128(b0 + kk * 2048) : sdesc_kmajor_sw128(b0 + kk * 32),
                                       idesc, (kb | kk) ? 1u : 0u);
                    umma_commit_pair(&S.empty[s], 3);
                }
                umma_commit_pair(&S.acc_full[ab], 3);
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ epilogue (lane quarter warp % 4)
        const int q = warp & 3;
        uint8_t* buf = epi_buf + (warp - 2) * 2 * FF_EPI_BUF;
        const int cols4 = 2 * p.N / 4;                       // float4 columns of g and u
        auto put = [&](int which, int half, const uint32_t (&o)[16]) {     // 32 columns of a 64-wide row
            uint8_t* b = buf + which * FF_EPI_BUF;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<uint4*>(b + sw128_offset(lane, half * 4 + c)) =
                    make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        };
        int i = 0, chunk = 0;
        for (int t = cid; t < total; t += ncl, ++i) {
            const int ab = i & 1;
            int m, n;
            ffn_tile(t, mt, nt, m, n);
            const bool ok = !S.abort && mbar_wait_cluster(&S.acc_full[ab], (i >> 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) { S.abort = 1; break; }
            tc_fence_after();
            const int row0 = m * FF_BM + (int)rank * 128 + q * 32;
            const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + ab * FF_BN;
            const int row = row0 + lane;
            const bool kept = row0 < ((p.M + 127) & ~127);
#pragma unroll 1
            for (int c0 = 0; c0 < COLS; c0 += 64, ++chunk) {
                const int col = n * COLS + c0;
                if (col >= p.N) break;
                const int bsel = EPI == FF_DGATE ? 0 : chunk & 1;
                // the store issued from this buffer before has read it
                if (lane == 0) { if (EPI == FF_DGATE) bulk_wait_read<0>(); else bulk_wait_read<1>(); }
                __syncwarp();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t v[32], o[16];
                    tmem_ld32(acc + c0 + half * 32, v);
                    if (EPI == FF_PLAIN) {
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = pack_bf2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
                        put(bsel, half, o);
                    } else if (EPI == FF_GATED) {
                        uint32_t w[32];
                        tmem_ld32(acc + 128 + c0 + half * 32, w);
                        tmem_ld_wait();
                        const int i4 = (col + half * 32) / 4;
                        if (p.gu && kept) {
                            float4* gu = reinterpret_cast<float4*>(p.gu);
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if ((i4 + e) * 4 < p.N) {
                                    gu[ffn_gu_index(row, i4 + e, cols4)] =
                                        make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                                    __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
                                    gu[ffn_gu_index(row, cols4 / 2 + i4 + e, cols4)] =
                                        make_float4(__uint_as_float(w[4 * e]), __uint_as_float(w[4 * e + 1]),
                                                    __uint_as_float(w[4 * e + 2]), __uint_as_float(w[4 * e + 3]));
                                }
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float g = __uint_as_float(v[e]);
                            v[e] = __float_as_uint(g * fast_sigmoid(g) * __uint_as_float(w[e]));
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = pack_bf2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
                        put(bsel, half, o);
                    } else {
                        const int i4 = (col + half * 32) / 4;
                        const float4* gu = reinterpret_cast<const float4*>(p.gu);
                        float dg[32];
                        float4 g4[8], u4[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const bool in = kept && (i4 + e) * 4 < p.N;
                            g4[e] = in ? gu[ffn_gu_index(row, i4 + e, cols4)] : make_float4(0, 0, 0, 0);
                            u4[e] = in ? gu[ffn_gu_index(row, cols4 / 2 + i4 + e, cols4)] : make_float4(0, 0, 0, 0);
                        }
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float g = reinterpret_cast<const float*>(g4)[e], u = reinterpret_cast<const float*>(u4)[e];
                            const float s = fast_sigmoid(g), dh = __uint_as_float(v[e]);
                            dg[e] = dh * u * s * (1.0f + g * (1.0f - s));
                            v[e] = __float_as_uint(dh * g * s);
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = pack_bf2(dg[2 * e], dg[2 * e + 1]);
                        put(0, half, o);
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = pack_bf2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
                        put(1, half, o);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (row0 < p.M) {
                        tma_store_2d(&p.tc, smem_u32(buf + bsel * FF_EPI_BUF), col, row0);
                        if (EPI == FF_DGATE) tma_store_2d(&p.tc2, smem_u32(buf + FF_EPI_BUF), col, row0);
                    }
                    bulk_commit();
                }
            }
            tc_fence_before();
            __syncwarp();
            // the accumulator reads completed (tcgen05.wait::ld): a relaxed arrival suffices
            if (lane == 0) {
                if (rank == 0) mbar_arrive(&S.acc_empty[ab]);
                else mbar_arrive_remote_relaxed(mapa_rank(&S.acc_empty[ab], 0));
            }
        }
        if (lane == 0) bulk_wait<0>();
        __syncwarp();
    }

    // after a wait that expired: time for the copies and products in flight to end
    if (S.abort)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

inline size_t ffn_gemm_smem() { return 1024 + (size_t)FF_STAGES * FF_STAGE + 8 * FF_EPI_BUF + sizeof(FfnSmem); }

}  // namespace fnx
