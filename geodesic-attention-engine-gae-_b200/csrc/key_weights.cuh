// key_weights.cuh -- the attention weight that a block of queries puts on each
// key: w[b, hk, j] = sum over the heads h of key head hk and the queries i that
// see key j of exp(scale <q_i, k_j> - lse_i), from the forward's log-sum-exp.
// No reference counterpart; it is what an eviction after a prompt goes by.
#pragma once
#include "attn_f32.cuh"
#include "sm100.cuh"

namespace gae {

struct KeyWeightsParams {
    const void *q, *k;
    const float *lse;
    float *out;
    int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, l_sb, l_sh, o_sb, o_sh;
    int B, H, Hkv, Nq, Nkv, D, causal, accumulate;
    int64_t off;  // query row r sees key c iff c <= r + off (causal)
    float scale_log2;
};

// One CTA per (64-key tile, key head, batch): 16 x 16 threads, each 4 keys x 4
// queries of a 64 x 64 tile of scores, queries streamed.
template <typename T>
__global__ void __launch_bounds__(256) key_weights_kernel(const KeyWeightsParams p) {
    extern __shared__ float smem_kw[];
    float *sk = smem_kw, *sq = smem_kw + 64 * (p.D + 1);
    __shared__ float slse[64], red[64][17];
    const int hk = blockIdx.y, b = blockIdx.z, k0 = blockIdx.x * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;  // tx: queries, ty: keys
    const int G = p.H / p.Hkv, ld = p.D + 1;
    const T *kp = static_cast<const T *>(p.k) + b * p.k_sb + hk * p.k_sh;
    for (int i = threadIdx.x; i < 64 * p.D; i += 256) {
        const int r = i / p.D, d = i % p.D;
        sk[r * ld + d] = k0 + r < p.Nkv ? to_f<T>(kp[(k0 + r) * p.k_ss + d]) : 0.f;
    }
    float w[4] = {};
    for (int g = 0; g < G; ++g) {
        const int h = hk * G + g;
        const T *qp = static_cast<const T *>(p.q) + b * p.q_sb + h * p.q_sh;
        for (int q0 = 0; q0 < p.Nq; q0 += 64) {
            if (p.causal && k0 > q0 + 63 + p.off) continue;
            __syncthreads();
            for (int i = threadIdx.x; i < 64 * p.D; i += 256) {
                const int r = i / p.D, d = i % p.D;
                sq[r * ld + d] = q0 + r < p.Nq ? to_f<T>(qp[(q0 + r) * p.q_ss + d]) : 0.f;
            }
            if (threadIdx.x < 64) {
                const int r = q0 + threadIdx.x;
                const float l = r < p.Nq ? p.lse[b * p.l_sb + h * p.l_sh + r] : -INFINITY;
                slse[threadIdx.x] = l == -INFINITY ? INFINITY : l * 1.4426950408889634f;  // such a row weighs nothing
            }
            __syncthreads();
            float s[4][4] = {};
            for (int d = 0; d < p.D; ++d) {
                float a[4], c[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = sk[(ty * 4 + e) * ld + d], c[e] = sq[(tx * 4 + e) * ld + d];
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int f = 0; f < 4; ++f) s[e][f] = fmaf(a[e], c[f], s[e][f]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                    const int key = k0 + ty * 4 + e, row = q0 + tx * 4 + f;
                    if (row < p.Nq && (!p.causal || key <= row + p.off))
                        w[e] += exp2f(fmaf(s[e][f], p.scale_log2, -slse[tx * 4 + f]));
                }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) red[ty * 4 + e][tx] = w[e];
    __syncthreads();
    if (threadIdx.x < 64 && k0 + threadIdx.x < p.Nkv) {
        float t = 0.f;
        for (int x = 0; x < 16; ++x) t += red[threadIdx.x][x];
        float *o = p.out + b * p.o_sb + hk * p.o_sh + k0 + threadIdx.x;
        *o = p.accumulate ? *o + t : t;
    }
}

}  // namespace gae
