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
template <int NV, int BR>
__global__ void __launch_bounds__(512) inject_norm_kernel(const InjectNormParams p) {
    __shared__ float red[32 * (BR > 1 ? BR : 1)];
    const int nc = p.H / 8;
    const long long t = blockIdx.x;
    const int b0 = blockIdx.y * BR;
    const uint4* yv = reinterpret_cast<const uint4*>(p.values) + t * nc;
    const uint4* hv = reinterpret_cast<const uint4*>(p.hyper) + (t * p.HC + b0) * nc;

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

// Persistent blocks, tokens blockIdx.x, + gridDim.x, ...: every thread owns fixed columns, whose
// weight-gradient sums it keeps in shared memory over all of its block's tokens.
__global__ void __launch_bounds__(512) inject_norm_bwd_kernel(const InjectNormBwdParams p) {
    extern __shared__ __align__(16) float acc[];           // [(HC + 1) * H], then dz [H]
    __shared__ float red[32 * 6];
    const int nc = p.H / 8;
    float* dzs = acc + (size_t)(p.HC + 1) * p.H;
    for (int i = threadIdx.x; i < (p.HC + 1) * p.H; i += blockDim.x) acc[i] = 0.f;
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
// out0, the rest to out1 (either may be NULL).
__global__ void __launch_bounds__(256) column_sum_kernel(const float* __restrict__ part, bf16* __restrict__ out0,
                                                         bf16* __restrict__ out1, int rows, int n0, int n) {
    __shared__ float red[8][33];
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < n)
        for (int r = grp; r < rows; r += 8) s += part[(size_t)r * n + c];
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
