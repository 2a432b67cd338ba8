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
// A cluster of two CTAs (cta_group::2) takes a 256 x bn tile (bn <= 256, chosen on the host so that the
// tiles fill the waves of 74 pairs): each CTA loads its half of the rows of A and of B by TMA (128-byte
// swizzle) into a ring of 5 or 6 64-deep k-blocks; rank 0 issues M = 256, N = bn, K = 16 MMAs that
// read both CTAs' halves; every CTA holds 128 rows x bn columns of fp32 in tensor memory, twice, so
// that one tile's epilogue runs under the next one's products.  Both CTAs' copies complete on rank 0's
// `full` barrier; rank 0's commits release the stage and hand over the accumulator in both CTAs.
// Edges read the tensor maps' zero fill and are clipped by the stores.  One launch takes up to three
// products (the three that follow dh), so that they share one tail.
// Roles:  warp 0 TMA copies, warp 1 MMA issue (rank 0), warps 2-9 epilogue (lane quarter warp % 4, every
// other 64 columns).  The issuing loops run in whole warps that elect a thread around each issue: a loop
// of one thread (lane == 0) took 560 cycles a k-block whatever its width; the elected form takes 519 at
// bn = 256, where the products alone are 512, and 383 at 128, where the copies (64 bytes a cycle and SM)
// bound it, which is why narrow tiles are worth (256 + bn) / 512 of a wide one and not bn / 256.
//
// Bound: the tensor cores, and over long calls the board's power: 8191 rows of 4096 x 8192 take 1178 us
// (1400 TFLOP/s; cuBLAS sustains 1390 on the same card at its power cap), a training step of 4096 rows
// 1.95 to 2.0 ms (1238 to 1270; the launch after dh keeps the tensor pipe 97 % busy at 1.27 GHz).  Short
// calls pay about 9,000 cycles a launch for its start, first copies and last epilogue: 4096 rows of
// 2560 x 640 take 40.5 us, 25 of them products.
#pragma once
#include "fnx_common.cuh"

namespace fnx {

constexpr int FF_BM = 256, FF_BN = 256, FF_BK = 64;
constexpr int FF_A_BYTES = 128 * FF_BK * 2, FF_B_BYTES = 128 * FF_BK * 2;      // per CTA
constexpr int FF_STAGE = FF_A_BYTES + FF_B_BYTES;
constexpr int FF_EPI_BUF = 32 * 128;                                           // 32 rows x 64 bf16
constexpr int FF_EPI_WARPS = 8;                                                // two per lane quarter
constexpr int FF_THREADS = 32 * (2 + FF_EPI_WARPS);
constexpr int FF_MAX_PRODUCTS = 3;

enum { FF_PLAIN = 0, FF_GATED = 1, FF_DGATE = 2 };
// dh's epilogue stages two outputs, so its ring is one k-block shorter
__host__ __device__ constexpr int ff_stages(int epi) { return epi == FF_DGATE ? 5 : 6; }
__host__ __device__ constexpr int ff_epi_bufs(int epi) { return epi == FF_DGATE ? 2 : 1; }

struct FfnProduct {
    CUtensorMap ta, tb;              // operands: box {64, 128} / {64, bn/2} K-major, {64, 64} MN-major
    CUtensorMap tc, tc2;             // outputs, box {64, 32}: C; h; or dg and du
    bf16 *c, *c2;
    long long ldc;
    int M, N, K;                     // N: columns of C (of h for FF_GATED, of dh for FF_DGATE)
    int bn, amn, bmn;                // tile width (with both halves of FF_GATED), MN-major operands
    int mt, nt;                      // tiles
};
struct FfnParams {
    FfnProduct q[FF_MAX_PRODUCTS];
    float* gu;                       // g and u, blocked (see ffn_gu_index); NULL: not kept
    int count, total;
    int followed;                    // another product of the chain follows: let it start at once
};

struct FfnSmem {
    uint64_t full[6], empty[6], acc_full[2], acc_empty[2];
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

// Shared-memory matrix descriptors but for the start address (see sdesc_kmajor_sw128); MN-major with
// the 128-byte swizzle: 64 m (or n) of one k are a 128-byte row, 8 k a 1024-byte group; groups of 8 k
// are 1024 B apart (SBO), the next 64 m (n) 8192 B further (LBO; a 64 x 64 box of the copy).
FNX_DEV uint64_t sdesc_sw128_base(int mn_major) {
    return ((uint64_t)(mn_major ? 8192 >> 4 : 1) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
FNX_DEV uint64_t sdesc_at(uint64_t base, uint32_t saddr) { return base | ((saddr & 0x3FFFFu) >> 4); }
// bytes from one K = 16 step of a k-block to the next
FNX_DEV uint32_t kstep_bytes(int mn_major) { return mn_major ? 2048u : 32u; }

// Bounded wait of a single thread without back-off: the copy and the product threads are the chain that
// the tensor core waits for.  What these barriers order are asynchronous copies and products, whose
// completion the barrier itself carries, so the wait needs no acquire of cluster scope.
FNX_DEV bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
                 " selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
FNX_DEV bool mbar_spin(uint64_t* bar, uint32_t parity) {
    if (mbar_test_wait(bar, parity)) return true;
    const uint64_t t0 = fnx_globaltimer();
    while (true) {
#pragma unroll 1
        for (int i = 0; i < 256; ++i)
            if (mbar_test_wait(bar, parity)) return true;
        if (fnx_globaltimer() - t0 > FNX_WAIT_NS) {
            fnx_flag_error(FNX_DEVERR_TIMEOUT);
            return false;
        }
    }
}

// sigmoid(g) for the activation: exponential and reciprocal are the fast forms.  The exponential's error
// grows with |g| (2 + 1.173 |g| units of its last place), so towards negative g, where the sigmoid is that
// exponential's inverse, the result is good to 2^-21 at g = -2, 2^-18 at -20 and 2^-16 at -87: far below
// the bf16 rounding of every result.  Below -87.3 the sigmoid is 0 (it is smaller than 2^-126).
FNX_DEV float fast_sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

// Tile t of the launch: its product, and within it groups of 8 row tiles, columns outside, rows
// inside, so the tiles in flight share rows of A and columns of B in L2.
FNX_DEV const FfnProduct& ffn_tile(const FfnParams& p, int t, int& m, int& n) {
    int i = 0;
    while (i + 1 < p.count && t >= p.q[i].mt * p.q[i].nt) t -= p.q[i].mt * p.q[i].nt, ++i;
    const FfnProduct& q = p.q[i];
    const int per = 8 * q.nt, g = t / per, r = t - g * per;
    const int rows = min(8, q.mt - 8 * g);
    n = r / rows;
    m = 8 * g + r - n * rows;
    return q;
}

// The copies and the products of one tile (stages j, j + 1, ... of the ring), by a whole warp that
// elects the issuing thread; false when a wait expired.
template <int AMN, int BMN, int STAGES>
FNX_DEV bool ffn_copy_tile(FfnSmem& S, uint8_t* base, const FfnProduct& q, int KB, int ra, int rb, uint32_t rank, int& j) {
    const CUtensorMap *ta = &q.ta, *tb = &q.tb;
    const bool two = !BMN || q.bn > 128;                     // MN-major: boxes of 64 columns
    const uint32_t bytes = 2 * (FF_A_BYTES + (BMN ? (two ? 16384 : 8192) : q.bn * 64));
    for (int kb = 0; kb < KB; ++kb, ++j) {
        const int s = j % STAGES;
        if (!__all_sync(0xffffffffu, mbar_spin(&S.empty[s], ((j / STAGES) & 1) ^ 1))) return false;
        if (elect_one()) {
            if (rank == 0) mbar_arrive_expect_tx(&S.full[s], bytes);
            const uint32_t bar = mapa_rank(&S.full[s], 0);
            const uint32_t a = smem_u32(base + s * FF_STAGE), b = a + FF_A_BYTES;
            const int k = kb * FF_BK;
            if (AMN) {
                tma_load_2d_pair(a, ta, bar, ra, k);
                tma_load_2d_pair(a + 8192, ta, bar, ra + 64, k);
            } else {
                tma_load_2d_pair(a, ta, bar, k, ra);
            }
            if (BMN) {
                tma_load_2d_pair(b, tb, bar, rb, k);
                if (two) tma_load_2d_pair(b + 8192, tb, bar, rb + 64, k);
            } else {
                tma_load_2d_pair(b, tb, bar, k, rb);
            }
        }
        __syncwarp();
    }
    return true;
}
template <int AMN, int BMN, int STAGES>
FNX_DEV bool ffn_multiply_tile(FfnSmem& S, uint8_t* base, int bn, int KB, uint32_t d, uint64_t* acc_full, int& j) {
    const uint32_t idesc = idesc_bf16_f32(FF_BM, bn) | ((uint32_t)AMN << 15) | ((uint32_t)BMN << 16);
    for (int kb = 0; kb < KB; ++kb, ++j) {
        const int s = j % STAGES;
        if (!__all_sync(0xffffffffu, mbar_spin(&S.full[s], (j / STAGES) & 1))) return false;
        tc_fence_after();
        const uint32_t a0 = smem_u32(base + s * FF_STAGE), b0 = a0 + FF_A_BYTES;
        if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < FF_BK / 16; ++kk)
                umma_bf16_pair(d, sdesc_at(sdesc_sw128_base(AMN), a0 + kk * kstep_bytes(AMN)),
                               sdesc_at(sdesc_sw128_base(BMN), b0 + kk * kstep_bytes(BMN)), idesc, (kb | kk) ? 1u : 0u);
            umma_commit_pair(&S.empty[s], 3);
            if (kb == KB - 1) umma_commit_pair(acc_full, 3);
        }
        __syncwarp();
    }
    return true;
}

// dg and du of 32 columns from dh (v) and the kept g and u, packed to bf16 pairs.
FNX_DEV void ffn_dgate32(const uint32_t (&v)[32], const float4 (&g4)[8], const float4 (&u4)[8], uint32_t (&og)[16],
                         uint32_t (&ou)[16]) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float dg[2], du[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = 2 * e + k;
            const float g = reinterpret_cast<const float*>(g4)[i], u = reinterpret_cast<const float*>(u4)[i];
            const float s = fast_sigmoid(g), dh = __uint_as_float(v[i]);
            dg[k] = dh * u * s * (1.0f + g * (1.0f - s));
            du[k] = dh * g * s;
        }
        og[e] = pack_bf2(dg[0], dg[1]);
        ou[e] = pack_bf2(du[0], du[1]);
    }
}

template <int EPI>
__global__ void __launch_bounds__(FF_THREADS, 1) ffn_gemm_kernel(const __grid_constant__ FfnParams p) {
    constexpr int STAGES = ff_stages(EPI), BUFS = ff_epi_bufs(EPI);
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* base = align1024(smem_raw);
    uint8_t* epi_buf = base + STAGES * FF_STAGE;
    FfnSmem& S = *reinterpret_cast<FfnSmem*>(epi_buf + FF_EPI_WARPS * BUFS * FF_EPI_BUF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int cid = (int)cluster_id_x(), ncl = (int)num_clusters_x();

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], 2 * FF_EPI_WARPS);    // the epilogue warps of both CTAs
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
    pdl_wait();                                              // what the kernel before wrote or still reads
    // only now: the successor reads its weights before its own wait, which is safe once every CTA here
    // has seen the kernels before this one complete
    if (p.followed) pdl_launch_dependents();

    if (warp == 0) {
        // ------------------------------------------------ TMA copies of this CTA's halves
        int j = 0;
        for (int t = cid; t < p.total && !S.abort; t += ncl) {
            int m, n;
            const FfnProduct& q = ffn_tile(p, t, m, n);
            const int ra = m * FF_BM + (int)rank * 128;
            // the gate/up product: rank 0 holds the gate rows of W, rank 1 the up rows
            const int rb = EPI == FF_GATED ? n * (q.bn / 2) + (int)rank * q.N : n * q.bn + (int)rank * (q.bn / 2);
            const int KB = (q.K + FF_BK - 1) / FF_BK;
            const bool ok = q.amn ? ffn_copy_tile<1, 1, STAGES>(S, base, q, KB, ra, rb, rank, j)
                            : q.bmn ? ffn_copy_tile<0, 1, STAGES>(S, base, q, KB, ra, rb, rank, j)
                                    : ffn_copy_tile<0, 0, STAGES>(S, base, q, KB, ra, rb, rank, j);
            if (!ok) { S.abort = 1; break; }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issue
        if (rank == 0) {
            int j = 0, i = 0;
            for (int t = cid; t < p.total && !S.abort; t += ncl, ++i) {
                int m, n;
                const FfnProduct& q = ffn_tile(p, t, m, n);
                const int KB = (q.K + FF_BK - 1) / FF_BK;
                const int ab = i & 1;
                if (!__all_sync(0xffffffffu, mbar_spin(&S.acc_empty[ab], ((i >> 1) & 1) ^ 1))) { S.abort = 1; break; }
                tc_fence_after();
                const uint32_t d = tmem + ab * FF_BN;
                const bool ok = q.amn ? ffn_multiply_tile<1, 1, STAGES>(S, base, q.bn, KB, d, &S.acc_full[ab], j)
                                : q.bmn ? ffn_multiply_tile<0, 1, STAGES>(S, base, q.bn, KB, d, &S.acc_full[ab], j)
                                        : ffn_multiply_tile<0, 0, STAGES>(S, base, q.bn, KB, d, &S.acc_full[ab], j);
                if (!ok) { S.abort = 1; break; }
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ epilogue (lane quarter warp % 4)
        const int lq = warp & 3, first = 64 * ((warp - 2) >> 2);
        uint8_t* buf = epi_buf + (warp - 2) * BUFS * FF_EPI_BUF;
        // 32 columns of this lane's row: half a 64-column chunk in the staging buffer, or straight out
        // where a tile's width leaves fewer than 64 (the copies' boxes are 64 wide)
        auto put = [&](int b, int half, const uint32_t (&o)[16]) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<uint4*>(buf + b * FF_EPI_BUF + sw128_offset(lane, half * 4 + c)) =
                    make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        };
        auto put_out = [&](bf16* c, const FfnProduct& q, int row, int col, int end, const uint32_t (&o)[16]) {
            if (row >= q.M) return;
            bf16* r = c + row * q.ldc + col;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (col + 8 * k < end)
                    *reinterpret_cast<uint4*>(r + 8 * k) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        };
        int i = 0;
        for (int t = cid; t < p.total; t += ncl, ++i) {
            const int ab = i & 1;
            int m, n;
            const FfnProduct& q = ffn_tile(p, t, m, n);
            const int cols = EPI == FF_GATED ? q.bn / 2 : q.bn;
            const int cols4 = 2 * q.N / 4;                   // float4 columns of g and u
            const int row0 = m * FF_BM + (int)rank * 128 + lq * 32, row = row0 + lane;
            const int end = min(q.N, (n + 1) * cols);        // this tile's columns end here
            const bool kept = row0 < ((q.M + 127) & ~127);   // rows that the kept g and u hold
            float4 g4[8], u4[8];
            auto load_gu = [&](int col) {                    // FF_DGATE: g and u of 32 columns
                const float4* gu = reinterpret_cast<const float4*>(p.gu);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = kept && col + 4 * e < end;
                    g4[e] = in ? gu[ffn_gu_index(row, col / 4 + e, cols4)] : make_float4(0, 0, 0, 0);
                    u4[e] = in ? gu[ffn_gu_index(row, cols4 / 2 + col / 4 + e, cols4)] : make_float4(0, 0, 0, 0);
                }
            };
            if (EPI == FF_DGATE) {
                // while the products run: the tile's g and u into L2 (512 bytes per column group of
                // four and warp), the first 32 columns into registers
                if (kept)
                    for (int c0 = first; c0 < cols; c0 += 128) {
                        const int c = n * cols + c0 + 4 * (lane >> 1);        // 16 groups, two lanes each
                        if (c < end) {
                            const float4* g = reinterpret_cast<const float4*>(p.gu) + ffn_gu_index(row0, c / 4, cols4) + 16 * (lane & 1);
                            const float4* u = g + (size_t)(cols4 / 2) * 128;
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                asm volatile("prefetch.global.L2 [%0];" ::"l"(g + 8 * k));
                                asm volatile("prefetch.global.L2 [%0];" ::"l"(u + 8 * k));
                            }
                        }
                    }
                load_gu(n * cols + first);
            }
            const bool ok = !S.abort && mbar_wait_cluster(&S.acc_full[ab], (i >> 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) { S.abort = 1; break; }
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(lq * 32) << 16) + ab * FF_BN;
#pragma unroll 1
            for (int c0 = first; c0 < cols; c0 += 128) {
                const int col = n * cols + c0;
                if (col >= q.N) break;
                const bool whole = c0 + 64 <= cols;
                // the stores issued from this buffer before have read it
                if (lane == 0) bulk_wait_read<0>();
                __syncwarp();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int hc = c0 + half * 32, i4 = (col + half * 32) / 4;
                    if (hc >= cols) break;
                    uint32_t v[32], o[16];
                    tmem_ld32(acc + hc, v);
                    if (EPI == FF_PLAIN) {
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = pack_bf2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
                        if (whole) put(0, half, o); else put_out(q.c, q, row, col + half * 32, end, o);
                    } else if (EPI == FF_GATED) {
                        uint32_t w[32];
                        tmem_ld32(acc + cols + hc, w);
                        tmem_ld_wait();
                        if (p.gu && kept) {
                            float4* gu = reinterpret_cast<float4*>(p.gu);
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if ((i4 + e) * 4 < end) {
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
                        if (whole) put(0, half, o); else put_out(q.c, q, row, col + half * 32, end, o);
                    } else {
                        uint32_t o2[16];
                        tmem_ld_wait();
                        ffn_dgate32(v, g4, u4, o, o2);
                        // the next 32 columns of this warp are on their way while these are stored
                        const int next = half == 0 ? hc + 32 : c0 + 128;
                        if (next < cols) load_gu(n * cols + next);
                        if (whole) put(0, half, o); else put_out(q.c, q, row, col + half * 32, end, o);
                        if (whole) put(BUFS - 1, half, o2); else put_out(q.c2, q, row, col + half * 32, end, o2);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (row0 < q.M && whole) {
                        tma_store_2d(&q.tc, smem_u32(buf), col, row0);
                        if (EPI == FF_DGATE) tma_store_2d(&q.tc2, smem_u32(buf + FF_EPI_BUF), col, row0);
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
    if (!p.followed) pdl_launch_dependents();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

inline size_t ffn_gemm_smem(int epi) {
    return 1024 + (size_t)ff_stages(epi) * FF_STAGE + FF_EPI_WARPS * ff_epi_bufs(epi) * FF_EPI_BUF + sizeof(FfnSmem);
}

}  // namespace fnx
