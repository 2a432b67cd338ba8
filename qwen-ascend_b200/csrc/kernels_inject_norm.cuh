// The residual step between two blocks with the norms on both sides of it: the tail of one block
// (a norm of its output, its gate and residual scale, the residual sum) and the head of the next
// (its input norm) in one pass, and the gradients of both.  Per token t, branch b < HC, column c < H:
//   z[c]        = y[c] * rv * (1 + wp[c]),  rv = 1 / sqrt(mean(y^2) + eps)      (z = y without w_post)
//   state[b,c]  = hyper[b,c] + scale * gate[b] * z[c]
//   normed[b,c] = state[b,c] * rs[b] * (1 + wn[b,c]),  rs[b] = 1 / sqrt(mean(state[b]^2) + eps)
// (inject, fnx/engine.py:859-877, followed by the rms_norm that opens gated_residual,
// fnx/engine.py:156-190, 818-857, with a norm behind the block added).  Everything is fp32 inside
// and each output is rounded once: normed is the norm of the unrounded state.
//
// Backward, with e = d_normed * (1 + wn), D = d_state, from the stored state s and y alone:
//   d[b,c]      = D + rs * (e - s * rs^2 * mean(e * s))                          d_hyper
//   d_gate[b]   = scale * sum_c d * z
//   dz[c]       = scale * sum_b gate[b] * d[b,c]
//   d_y[c]      = rv * (dz (1 + wp) - y * rv^2 * mean(dz (1 + wp) * y))          (dz without w_post)
//   d_wn[b,c]   = sum_t d_normed * s * rs,   d_wp[c] = sum_t dz * y * rv
// The rms statistics are recomputed from s and y in the same reduction as the sums they scale, so
// nothing but the forward's inputs and outputs has to be kept.
#pragma once
#include "fnx_common.cuh"

namespace fnx {

// Sums of N values per thread over the block, in every thread (fixed order: deterministic).
// `red` holds N * 32 floats; the barrier at the end lets the caller reuse it at once.
template <int N>
FNX_DEV void block_sums(float (&v)[N], float* red) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int o = 16; o; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) red[i * 32 + warp] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = lane < nw ? red[i * 32 + lane] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        v[i] = s;
    }
    __syncthreads();
}

FNX_DEV void unpack8(const uint4& u, float (&f)[8]) {
    f[0] = bf_lo(u.x); f[1] = bf_hi(u.x); f[2] = bf_lo(u.y); f[3] = bf_hi(u.y);
    f[4] = bf_lo(u.z); f[5] = bf_hi(u.z); f[6] = bf_lo(u.w); f[7] = bf_hi(u.w);
}
FNX_DEV uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7]));
}
// Pairs of floats in one register pair: two fp32 operations per instruction, each rounded as the scalar
// one.  A bf16 pair widens to one in two instructions.
typedef unsigned long long f32x2;
FNX_DEV f32x2 f2_make(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
FNX_DEV float2 f2_get(f32x2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
FNX_DEV f32x2 f2_fma(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
FNX_DEV f32x2 f2_mul(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
FNX_DEV f32x2 f2_add(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
FNX_DEV float f2_sum(f32x2 a) {
    const float2 v = f2_get(a);
    return v.x + v.y;
}
FNX_DEV f32x2 f2_bf16(uint32_t u) { return f2_make(bf_lo(u), bf_hi(u)); }
FNX_DEV void widen8(const uint4& u, f32x2 (&f)[4]) {
    f[0] = f2_bf16(u.x); f[1] = f2_bf16(u.y); f[2] = f2_bf16(u.z); f[3] = f2_bf16(u.w);
}
FNX_DEV uint32_t f2_round(f32x2 a) {
    const float2 v = f2_get(a);
    return pack_bf2(v.x, v.y);
}
FNX_DEV uint4 round8(const f32x2 (&f)[4]) { return make_uint4(f2_round(f[0]), f2_round(f[1]), f2_round(f[2]), f2_round(f[3])); }

FNX_DEV float rms_scale(float sum_sq, int H, float eps) {
    return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum_sq, (float)H), eps)));
}

struct InjectNormParams {
    const bf16 *hyper, *gate, *values, *w_post, *w_next;
    bf16 *state, *normed;
    int H, HC;
    float scale, eps;
};

// One block per token and group of BR branches; thread i owns the 16-byte chunks i, i + blockDim, ...
// (NV of them).  All loads are issued before the first reduction; the branch data stay in registers.
// Bound: HBM, (3 HC + 1) * H * 2 bytes a token (8192 tokens of 4 x 2560 with both norms: 98.4 us, 5.5 TB/s).
// BR = 1 below one token per SM, where a branch per block spreads a token over four SMs.
template <int NV, int BR>
__global__ void __launch_bounds__(512) inject_norm_kernel(const InjectNormParams p) {
    __shared__ float red[32 * (BR > 1 ? BR : 1)];
    const int nc = p.H / 8;
    const long long t = blockIdx.x;
    const int b0 = blockIdx.y * BR;
    const uint4* yv = reinterpret_cast<const uint4*>(p.values) + t * nc;
    const uint4* hv = reinterpret_cast<const uint4*>(p.hyper) + (t * p.HC + b0) * nc;
    pdl_wait();

    uint4 y4[NV], h4[NV][BR];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        y4[j] = make_uint4(0, 0, 0, 0);
        if (c < nc) y4[j] = yv[c];
#pragma unroll
        for (int b = 0; b < BR; ++b) {
            h4[j][b] = make_uint4(0, 0, 0, 0);
            if (c < nc && b0 + b < p.HC) h4[j][b] = hv[(long long)b * nc + c];
        }
    }
    float g[BR];
#pragma unroll
    for (int b = 0; b < BR; ++b)
        g[b] = b0 + b < p.HC ? (p.gate ? bf2f(p.gate[t * p.HC + b0 + b]) : 1.0f) * p.scale : 0.f;

    float rv = 1.0f;
    if (p.w_post) {
        float ss[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float y[8];
            unpack8(y4[j], y);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss[0] = fmaf(y[e], y[e], ss[0]);
        }
        block_sums<1>(ss, red);
        rv = rms_scale(ss[0], p.H, p.eps);
    }
    float st[NV][BR][8], sq[BR];
#pragma unroll
    for (int b = 0; b < BR; ++b) sq[b] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        float z[8];
        unpack8(y4[j], z);
        if (p.w_post && c < nc) {
            float w[8];
            unpack8(reinterpret_cast<const uint4*>(p.w_post)[c], w);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = z[e] * rv * (1.0f + w[e]);
        }
#pragma unroll
        for (int b = 0; b < BR; ++b) {
            unpack8(h4[j][b], st[j][b]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                st[j][b][e] = fmaf(g[b], z[e], st[j][b][e]);
                sq[b] = fmaf(st[j][b][e], st[j][b][e], sq[b]);
            }
            if (c < nc && b0 + b < p.HC)
                reinterpret_cast<uint4*>(p.state)[(t * p.HC + b0 + b) * nc + c] = pack8(st[j][b]);
        }
    }
    if (!p.w_next) return;
    block_sums<BR>(sq, red);
#pragma unroll
    for (int b = 0; b < BR; ++b) {
        if (b0 + b >= p.HC) break;
        const float rs = rms_scale(sq[b], p.H, p.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = threadIdx.x + j * blockDim.x;
            if (c >= nc) continue;
            float w[8], o[8];
            unpack8(reinterpret_cast<const uint4*>(p.w_next)[(long long)(b0 + b) * nc + c], w);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = st[j][b][e] * rs * (1.0f + w[e]);
            reinterpret_cast<uint4*>(p.normed)[(t * p.HC + b0 + b) * nc + c] = pack8(o);
        }
    }
}

struct InjectNormBwdParams {
    const bf16 *d_state, *d_normed, *state, *gate, *values, *w_post, *w_next;
    bf16 *d_hyper, *d_gate, *d_values;
    float* part;                   // [gridDim.x, (HC + 1) * H]: each block's sums of d_wn, then d_wp
    int batch, H, HC;
    float scale, eps;
};

// Sums of 32 values per lane over a warp, value i in lane i: each step adds half of the values the
// lane pair holds and hands the other half over (31 shuffles for all 32).
FNX_DEV float warp_sums32(float (&v)[32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float mine = up ? v[i + o] : v[i], theirs = up ? v[i] : v[i + o];
            v[i] = mine + __shfl_xor_sync(0xffffffffu, theirs, o);
        }
    }
    return v[0];
}

// The backward for H <= 4096: persistent blocks, tokens blockIdx.x, + gridDim.x, ...; thread i owns
// chunk i of every branch, with its weights and its weight-gradient sums in registers.  The rows of a
// token (d_state, d_normed, state, values; (3 HC + 1) * H * 2 bytes) arrive by bulk copies in one of
// two stages while the token before is computed.  One reduction gives all sums over the rows, a second
// one the mean that the norm behind the block needs.
// Bound: HBM would be (4 HC + 2) * H * 2 bytes a token (46 us for 4095 tokens of 4 x 2048); it takes 68 us,
// with issue slots two thirds taken and the rest waiting at the token's two reductions (2 x 2048: 47 us with
// the column sums, 26 of them bytes).  Measured and not
// kept (times with the forward, 120 us as it is): half as wide chunks with twice the threads (146), the gates'
// sums moved to the second reduction (fewer instructions, a longer chain: 122).
template <int HC>
__global__ void __launch_bounds__(512, HC == 1 ? 2 : 1) inject_norm_bwd_kernel(const InjectNormBwdParams p) {
    extern __shared__ __align__(128) uint8_t stages[];
    __shared__ float red[16][32], red1[16];
    __shared__ uint64_t full[2];
    const int nc = p.H / 8, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nw = blockDim.x >> 5;
    const int rows = (p.d_state ? HC : 0) + (p.d_normed ? HC : 0) + HC + 1;
    const uint32_t row_bytes = p.H * 2, stage_bytes = rows * row_bytes;
    const bool mine = tid < nc;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        mbar_init(&full[0], 1);
        mbar_init(&full[1], 1);
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    // stage layout: state, values, d_state, d_normed
    const int off_D = HC + 1, off_n = off_D + (p.d_state ? HC : 0);
    auto fetch = [&](long long t, int s) {
        const uint32_t b = smem_u32(stages + (size_t)s * stage_bytes);
        mbar_arrive_expect_tx(&full[s], stage_bytes);
        const uint64_t once = l2_evict_first();
        bulk_load(b, p.state + t * HC * p.H, HC * row_bytes, &full[s], once);
        bulk_load(b + HC * row_bytes, p.values + t * p.H, row_bytes, &full[s], once);
        if (p.d_state) bulk_load(b + off_D * row_bytes, p.d_state + t * HC * p.H, HC * row_bytes, &full[s], once);
        if (p.d_normed) bulk_load(b + off_n * row_bytes, p.d_normed + t * HC * p.H, HC * row_bytes, &full[s], once);
    };
    if (tid == 0)
        for (int k = 0; k < 2; ++k)
            if (blockIdx.x + (long long)k * gridDim.x < p.batch) fetch(blockIdx.x + (long long)k * gridDim.x, k);

    const f32x2 one2 = f2_make(1.f, 1.f), zero2 = f2_make(0.f, 0.f);
    uint4 wn[HC], wp = zero;
    f32x2 an[HC][4], ap[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) ap[k] = zero2;
#pragma unroll
    for (int b = 0; b < HC; ++b) {
        wn[b] = mine && p.w_next ? reinterpret_cast<const uint4*>(p.w_next)[b * nc + tid] : zero;
#pragma unroll
        for (int k = 0; k < 4; ++k) an[b][k] = zero2;
    }
    if (mine && p.w_post) wp = reinterpret_cast<const uint4*>(p.w_post)[tid];

    int it = 0;
    for (long long t = blockIdx.x; t < p.batch; t += gridDim.x, ++it) {
        const int st = it & 1;
        const bool landed = mbar_wait(&full[st], (it >> 1) & 1);
        const uint4* S = reinterpret_cast<const uint4*>(stages + (size_t)st * stage_bytes);
        const uint4 y4 = mine ? S[HC * nc + tid] : zero;
        // per branch s^2, e s, D z0, e z0, s z0 (five each), and y^2 last; z0 = y (1 + wp)
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
        if (mine) {
            f32x2 z0[4], x[4], w[4], q0 = zero2;
            widen8(y4, x);
            widen8(wp, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                z0[k] = f2_mul(x[k], f2_add(one2, w[k]));
                q0 = f2_fma(x[k], x[k], q0);
            }
            v[5 * HC] = f2_sum(q0);
#pragma unroll
            for (int b = 0; b < HC; ++b) {
                f32x2 s[4], q1 = zero2;
                q0 = zero2;
                widen8(S[b * nc + tid], s);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    q0 = f2_fma(s[k], s[k], q0);
                    q1 = f2_fma(s[k], z0[k], q1);
                }
                v[5 * b] = f2_sum(q0);
                v[5 * b + 4] = f2_sum(q1);
                if (p.d_state) {
                    q0 = zero2;
                    widen8(S[(off_D + b) * nc + tid], x);
#pragma unroll
                    for (int k = 0; k < 4; ++k) q0 = f2_fma(x[k], z0[k], q0);
                    v[5 * b + 2] = f2_sum(q0);
                }
                if (p.d_normed) {
                    q0 = q1 = zero2;
                    widen8(S[(off_n + b) * nc + tid], x);
                    widen8(wn[b], w);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const f32x2 e = f2_mul(x[k], f2_add(one2, w[k]));
                        q0 = f2_fma(e, s[k], q0);
                        q1 = f2_fma(e, z0[k], q1);
                    }
                    v[5 * b + 1] = f2_sum(q0);
                    v[5 * b + 3] = f2_sum(q1);
                }
            }
        }
        red[warp][lane] = warp_sums32(v);
        // the block gives up as one (each thread's wait ends by its own clock)
        if (!__syncthreads_and(landed)) {
            for (int i = 0; i < 200; ++i) __nanosleep(1000); // time for the copies in flight to end
            break;
        }
        float tot = 0.f;                                     // value `lane`, over the block
        for (int i = 0; i < nw; ++i) tot += red[i][lane];
        // lane b: the scalars of branch b
        const int lb = lane < HC ? lane : 0;
        const float ss = __shfl_sync(0xffffffffu, tot, 5 * lb), es = __shfl_sync(0xffffffffu, tot, 5 * lb + 1);
        const float dz_D = __shfl_sync(0xffffffffu, tot, 5 * lb + 2), dz_e = __shfl_sync(0xffffffffu, tot, 5 * lb + 3);
        const float dz_s = __shfl_sync(0xffffffffu, tot, 5 * lb + 4), yy = __shfl_sync(0xffffffffu, tot, 5 * HC);
        const float rv = p.w_post ? rms_scale(yy, p.H, p.eps) : 1.0f;
        const float rs_l = rms_scale(ss, p.H, p.eps), m_l = es / (float)p.H * rs_l * rs_l;
        const float g_l = (p.gate ? bf2f(p.gate[t * HC + lb]) : 1.0f) * p.scale;
        if (tid < HC && p.d_gate) p.d_gate[t * HC + tid] = f2bf(p.scale * rv * (dz_D + rs_l * (dz_e - m_l * dz_s)));
        f32x2 dz[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) dz[k] = zero2;
#pragma unroll
        for (int b = 0; b < HC; ++b) {
            const float rs1 = __shfl_sync(0xffffffffu, rs_l, b), m1 = -__shfl_sync(0xffffffffu, m_l, b);
            const float g1 = __shfl_sync(0xffffffffu, g_l, b);
            if (mine) {
                const f32x2 rs = f2_make(rs1, rs1), m = f2_make(m1, m1), gb = f2_make(g1, g1);
                f32x2 s[4], D[4], n[4], w[4];
                widen8(S[b * nc + tid], s);
                widen8(p.d_state ? S[(off_D + b) * nc + tid] : zero, D);
                widen8(p.d_normed ? S[(off_n + b) * nc + tid] : zero, n);
                widen8(wn[b], w);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x2 e = f2_mul(n[k], f2_add(one2, w[k]));
                    D[k] = f2_fma(rs, f2_fma(s[k], m, e), D[k]);
                    dz[k] = f2_fma(gb, D[k], dz[k]);
                    an[b][k] = f2_fma(f2_mul(n[k], rs), s[k], an[b][k]);
                }
                reinterpret_cast<uint4*>(p.d_hyper)[(t * HC + b) * nc + tid] = round8(D);
            }
        }
        f32x2 y[4], w[4];
        float q = 0.f;
        widen8(y4, y);
        widen8(wp, w);
        if (p.w_post) {
            f32x2 q0 = zero2;                                // zero where !mine
#pragma unroll
            for (int k = 0; k < 4; ++k) q0 = f2_fma(f2_mul(dz[k], f2_add(one2, w[k])), y[k], q0);
            q = f2_sum(q0);
#pragma unroll
            for (int o = 16; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
            if (lane == 0) red1[warp] = q;
        }
        __syncthreads();                                     // the stage and `red` are read; red1 is written
        if (tid == 0 && t + 2LL * gridDim.x < p.batch) fetch(t + 2LL * gridDim.x, st);
        if (p.w_post) {
            q = 0.f;
            for (int i = 0; i < nw; ++i) q += red1[i];
            const float mq = -q / (float)p.H * rv * rv;
            const f32x2 mq2 = f2_make(mq, mq), rv2 = f2_make(rv, rv);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                ap[k] = f2_fma(f2_mul(dz[k], rv2), y[k], ap[k]);
                dz[k] = f2_mul(rv2, f2_fma(y[k], mq2, f2_mul(dz[k], f2_add(one2, w[k]))));
            }
        }
        if (mine) reinterpret_cast<uint4*>(p.d_values)[t * nc + tid] = round8(dz);
    }
    if (mine) {
        float4* out = reinterpret_cast<float4*>(p.part + (size_t)blockIdx.x * (HC + 1) * p.H) + 2 * tid;
        auto put = [&](size_t at, const f32x2 (&a)[4]) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 lo = f2_get(a[2 * k]), hi = f2_get(a[2 * k + 1]);
                out[at + k] = make_float4(lo.x, lo.y, hi.x, hi.y);
            }
        };
#pragma unroll
        for (int b = 0; b < HC; ++b) put((size_t)b * 2 * nc, an[b]);
        put((size_t)HC * 2 * nc, ap);
    }
}

// The backward for wider rows: every thread owns several chunks, whose weight-gradient sums it keeps in
// shared memory over all of its block's tokens, and reads the rows twice, with one block on an SM (its 512
// threads take the registers).  Bound: the latency of those reads and of a block reduction for every branch
// and token, with nothing in flight under them: 4096 tokens of 2 x 4104 take 463 us with the forward, where the
// bytes would be 72.
__global__ void __launch_bounds__(512) inject_norm_bwd_wide_kernel(const InjectNormBwdParams p) {
    extern __shared__ __align__(16) float acc[];           // [(HC + 1) * H], then dz [H]
    __shared__ float red[32 * 6];
    const int nc = p.H / 8;
    float* dzs = acc + (size_t)(p.HC + 1) * p.H;
    for (int i = threadIdx.x; i < (p.HC + 1) * p.H; i += blockDim.x) acc[i] = 0.f;
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (long long t = blockIdx.x; t < p.batch; t += gridDim.x) {
        const uint4* yv = reinterpret_cast<const uint4*>(p.values) + t * nc;
        for (int i = threadIdx.x; i < p.H; i += blockDim.x) dzs[i] = 0.f;
        __syncthreads();
        float rv = 1.0f;
        for (int b = 0; b < p.HC; ++b) {
            const long long row = (t * p.HC + b) * nc;
            const uint4* sv = reinterpret_cast<const uint4*>(p.state) + row;
            const uint4* Dv = p.d_state ? reinterpret_cast<const uint4*>(p.d_state) + row : nullptr;
            const uint4* Nv = p.d_normed ? reinterpret_cast<const uint4*>(p.d_normed) + row : nullptr;
            const uint4* wn = reinterpret_cast<const uint4*>(p.w_next) + (long long)b * nc;
            // s^2, e s, D z0, e z0, s z0, y^2  with z0 = y (1 + wp)
            float v[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (int c = threadIdx.x; c < nc; c += blockDim.x) {
                float s[8], D[8], n[8], y[8], w[8], wp[8];
                unpack8(sv[c], s);
                unpack8(Dv ? Dv[c] : zero, D);
                unpack8(Nv ? Nv[c] : zero, n);
                unpack8(Nv ? wn[c] : zero, w);
                unpack8(yv[c], y);
                unpack8(p.w_post ? reinterpret_cast<const uint4*>(p.w_post)[c] : zero, wp);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float e = n[k] * (1.0f + w[k]), z0 = y[k] * (1.0f + wp[k]);
                    v[0] = fmaf(s[k], s[k], v[0]);
                    v[1] = fmaf(e, s[k], v[1]);
                    v[2] = fmaf(D[k], z0, v[2]);
                    v[3] = fmaf(e, z0, v[3]);
                    v[4] = fmaf(s[k], z0, v[4]);
                    v[5] = fmaf(y[k], y[k], v[5]);
                }
            }
            block_sums<6>(v, red);
            if (p.w_post) rv = rms_scale(v[5], p.H, p.eps);
            const float rs = rms_scale(v[0], p.H, p.eps);
            const float m = v[1] / (float)p.H * rs * rs;
            const float gb = (p.gate ? bf2f(p.gate[t * p.HC + b]) : 1.0f) * p.scale;
            if (threadIdx.x == 0 && p.d_gate)
                p.d_gate[t * p.HC + b] = f2bf(p.scale * rv * (v[2] + rs * (v[3] - m * v[4])));
            for (int c = threadIdx.x; c < nc; c += blockDim.x) {
                float s[8], D[8], n[8], w[8];
                unpack8(sv[c], s);
                unpack8(Dv ? Dv[c] : zero, D);
                unpack8(Nv ? Nv[c] : zero, n);
                unpack8(Nv ? wn[c] : zero, w);
                float* a = acc + ((long long)b * nc + c) * 8;
                float* dz = dzs + c * 8;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    D[k] = fmaf(rs, n[k] * (1.0f + w[k]) - s[k] * m, D[k]);
                    dz[k] = fmaf(gb, D[k], dz[k]);
                    a[k] = fmaf(n[k] * rs, s[k], a[k]);
                }
                reinterpret_cast<uint4*>(p.d_hyper)[row + c] = pack8(D);
            }
        }
        float q[1] = {0.f};
        if (p.w_post) {
            for (int c = threadIdx.x; c < nc; c += blockDim.x) {
                float y[8], wp[8];
                unpack8(yv[c], y);
                unpack8(reinterpret_cast<const uint4*>(p.w_post)[c], wp);
#pragma unroll
                for (int k = 0; k < 8; ++k) q[0] = fmaf(dzs[c * 8 + k] * (1.0f + wp[k]), y[k], q[0]);
            }
            block_sums<1>(q, red);
        }
        const float mq = q[0] / (float)p.H * rv * rv;
        for (int c = threadIdx.x; c < nc; c += blockDim.x) {
            float y[8], wp[8], o[8];
            unpack8(yv[c], y);
            unpack8(p.w_post ? reinterpret_cast<const uint4*>(p.w_post)[c] : zero, wp);
            float* a = acc + ((long long)p.HC * nc + c) * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float dz = dzs[c * 8 + k];
                o[k] = p.w_post ? rv * (dz * (1.0f + wp[k]) - y[k] * mq) : dz;
                if (p.w_post) a[k] = fmaf(dz * rv, y[k], a[k]);
            }
            reinterpret_cast<uint4*>(p.d_values)[t * nc + c] = pack8(o);
        }
        __syncthreads();
    }
    float* out = p.part + (size_t)blockIdx.x * (p.HC + 1) * p.H;
    for (int i = threadIdx.x; i < (p.HC + 1) * p.H; i += blockDim.x) out[i] = acc[i];
}

// out[c] = bf16(sum over rows of part[row, c]) for c < n, rows in ascending order within each of the
// block's eight row groups, whose sums are added in order (deterministic).  Column c < n0 goes to
// out0, the rest to out1 (either may be NULL).  The kernel before it still writes `part` while these
// blocks start, so the pointers carry no __restrict__: its loads may not move above the wait.
__global__ void __launch_bounds__(256) column_sum_kernel(const float* part, bf16* out0, bf16* out1, int rows, int n0, int n) {
    __shared__ float red[8][33];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < n) {
#pragma unroll 8
        for (int r = grp; r < rows; r += 8) s += part[(size_t)r * n + c];
    }
    red[grp][lane] = s;
    __syncthreads();
    if (grp == 0 && c < n) {
        float v = red[0][lane];
#pragma unroll
        for (int i = 1; i < 8; ++i) v += red[i][lane];
        if (c < n0) {
            if (out0) out0[c] = f2bf(v);
        } else if (out1) {
            out1[c - n0] = f2bf(v);
        }
    }
}

}  // namespace fnx
