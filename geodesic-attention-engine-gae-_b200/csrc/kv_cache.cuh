// kv_cache.cuh -- the paged key-value cache: writing tokens into it, attention
// of one new token per sequence over it, and its eviction to a budget by
// accumulated attention weight.  The reference has no cache; these kernels are
// the serving-side callers' form of its operator.
//
// Layout: position t of sequence b is row t % page_size of page
// table[b][t / page_size]; a table entry outside [0, num_pages) holds no keys.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_f32.cuh"
#include "sm100.cuh"

namespace gae {

// K and V pools [num_pages, kv_heads, page_size, head_dim], element strides.
struct KvPool {
    void *k, *v;
    int64_t k_sp, k_sh, k_ss, v_sp, v_sh, v_ss;
    int64_t num_pages;
    int Hkv, page, D;
};

struct PageTable {
    const int *entry;
    int64_t stride;  // elements between two sequences' rows
    int max_pages;
};

// Page of position `pos` of sequence b (the caller keeps pos in [0, max_pages
// * page_size)); -1 where the entry names no page.
__device__ __forceinline__ int page_of(const PageTable &t, int64_t num_pages, int b, int page_idx) {
    const int p = __ldg(t.entry + b * t.stride + page_idx);
    return (p >= 0 && p < num_pages) ? p : -1;
}

__device__ __forceinline__ int clamp_len(int len, int cap) { return max(0, min(len, cap)); }

// ------------------------------------------------------------------ append
struct AppendParams {
    KvPool pool;
    PageTable table;
    const void *k_new, *v_new;
    int64_t kn_sb, kn_sh, kn_st, vn_sb, vn_sh, vn_st;  // element strides: batch, head, token
    const int *start, *counts;                         // counts may be NULL: all tokens
    int tokens, chunks;                                // chunks: 16-byte pieces of a row
};

// One thread per 16-byte piece of a new row, K and V both.
template <int ESIZE>
__global__ void paged_append_kernel(const AppendParams p) {
    const int b = blockIdx.y;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int c = (int)(i % p.chunks);
    const int h = (int)(i / p.chunks % p.pool.Hkv);
    const int64_t t = i / p.chunks / p.pool.Hkv;
    const int n = p.counts ? min(p.counts[b], p.tokens) : p.tokens;
    if (t >= n) return;
    const int64_t pos = (int64_t)p.start[b] + t;
    if (pos < 0 || pos >= (int64_t)p.table.max_pages * p.pool.page) return;
    const int pg = page_of(p.table, p.pool.num_pages, b, (int)(pos / p.pool.page));
    if (pg < 0) return;
    const int64_t slot = pos % p.pool.page;
    const int4 *ks = reinterpret_cast<const int4 *>(static_cast<const char *>(p.k_new) +
                                                    (b * p.kn_sb + h * p.kn_sh + t * p.kn_st) * ESIZE);
    const int4 *vs = reinterpret_cast<const int4 *>(static_cast<const char *>(p.v_new) +
                                                    (b * p.vn_sb + h * p.vn_sh + t * p.vn_st) * ESIZE);
    int4 *kd = reinterpret_cast<int4 *>(static_cast<char *>(p.pool.k) +
                                        (pg * p.pool.k_sp + h * p.pool.k_sh + slot * p.pool.k_ss) * ESIZE);
    int4 *vd = reinterpret_cast<int4 *>(static_cast<char *>(p.pool.v) +
                                        (pg * p.pool.v_sp + h * p.pool.v_sh + slot * p.pool.v_ss) * ESIZE);
    kd[c] = __ldg(ks + c);
    vd[c] = __ldg(vs + c);
}

// ------------------------------------------------- single-token attention
struct PagedAttnParams {
    KvPool pool;
    PageTable table;
    const void *q;
    void *o;
    int64_t q_sb, q_sh, o_sb, o_sh;
    const int *lens;
    float *lse;           // [B, H], may be NULL
    float *scores;        // [B, H, cap], with weights only
    const float *w_in;    // [B, Hkv, >= len], with weights only
    float *w_out;
    int64_t wi_sb, wi_sh, wo_sb, wo_sh;
    int B, H, cap;        // cap = max_pages * page_size
    float scale_log2;
};

// One CTA per (head, sequence), one warp per key, lanes across head_dim.
template <typename T>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttnParams p) {
    constexpr int kPer = 8;  // head_dim <= 256
    const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = h / (p.H / p.pool.Hkv), D = p.pool.D;
    const int len = clamp_len(p.lens[b], p.cap);
    float q[kPer], acc[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int d = lane + 32 * j;
        q[j] = d < D ? to_f<T>(static_cast<const T *>(p.q)[b * p.q_sb + h * p.q_sh + d]) : 0.f;
        acc[j] = 0.f;
    }
    for (int pos = warp; pos < len; pos += 4) {
        const int pg = page_of(p.table, p.pool.num_pages, b, pos / p.pool.page);
        float *sc = p.scores ? p.scores + ((int64_t)b * p.H + h) * p.cap + pos : nullptr;
        if (pg < 0) {
            if (sc && lane == 0) *sc = -INFINITY;
            continue;
        }
        const int slot = pos % p.pool.page;
        const T *k = static_cast<const T *>(p.pool.k) + pg * p.pool.k_sp + hk * p.pool.k_sh + slot * p.pool.k_ss;
        const T *v = static_cast<const T *>(p.pool.v) + pg * p.pool.v_sp + hk * p.pool.v_sh + slot * p.pool.v_ss;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int d = lane + 32 * j;
            if (d < D) s = fmaf(q[j], to_f<T>(k[d]), s);
        }
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= p.scale_log2;
        if (sc && lane == 0) *sc = s;
        // A row of -inf scores only has no weight anywhere; a NaN score reaches l and the output.
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
        const float a = exp2f(m - base), w = exp2f(s - base);
        m = mn;
        l = l * a + w;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int d = lane + 32 * j;
            acc[j] = acc[j] * a + (d < D ? w * to_f<T>(v[d]) : 0.f);
        }
    }
    __shared__ float sm[4], sl[4], so[4][256];
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int j = 0; j < kPer; ++j) so[warp][lane + 32 * j] = acc[j];
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float f[4];
    l = 0.f;
    for (int w = 0; w < 4; ++w) {
        f[w] = exp2f(sm[w] - (m == -INFINITY ? 0.f : m));
        l += f[w] * sl[w];
    }
    for (int d = threadIdx.x; d < D; d += 128) {
        float o = 0.f;
        for (int w = 0; w < 4; ++w) o += f[w] * so[w][d];
        static_cast<T *>(p.o)[b * p.o_sb + h * p.o_sh + d] = from_f<T>(l == 0.f ? 0.f : o / l);
    }
    if (threadIdx.x == 0 && p.lse)
        p.lse[(int64_t)b * p.H + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// w_out = w_in + sum over the group's heads of exp(score - lse), in head order.
__global__ void paged_weights_kernel(const PagedAttnParams p) {
    const int hk = blockIdx.y, b = blockIdx.z, pos = blockIdx.x * blockDim.x + threadIdx.x;
    if (pos >= clamp_len(p.lens[b], p.cap)) return;
    if (page_of(p.table, p.pool.num_pages, b, pos / p.pool.page) < 0) return;
    const int G = p.H / p.pool.Hkv;
    float w = 0.f;
    for (int g = 0; g < G; ++g) {
        const int64_t row = (int64_t)b * p.H + hk * G + g;
        const float l = p.lse[row] * 1.4426950408889634f;
        if (l != -INFINITY) w += exp2f(p.scores[row * p.cap + pos] - l);
    }
    p.w_out[b * p.wo_sb + hk * p.wo_sh + pos] = p.w_in[b * p.wi_sb + hk * p.wi_sh + pos] + w;
}

// ---------------------------------------------------------------- eviction
struct EvictParams {
    KvPool pool;
    PageTable src, dst;
    const int *lens;
    const float *w;       // [B, Hkv, >= len]
    int64_t w_sb, w_sh;
    int keep, recent, cap;
    int *new_lens;        // [B]
    int *kept;            // [B, Hkv, keep]
    float *w_out;         // [B, Hkv, keep]
    int chunks;
};

// Whole-number order of the weights: NaN above +inf, -0 equal to 0.  Every
// float maps into [0x007fffff, 0xfffffffe]; 0 is "no key" and 0xffffffff "kept
// whatever its weight".
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint32_t evict_key(const EvictParams &p, int b, int hk, int pos, int len) {
    if (page_of(p.src, p.pool.num_pages, b, pos / p.pool.page) < 0) return 0u;
    if (pos >= len - p.recent) return 0xffffffffu;
    return weight_key(__ldg(p.w + b * p.w_sb + hk * p.w_sh + pos));
}

// One CTA per (kv head, sequence).  The keep-th largest key is found by four
// passes over its 8-bit digits; positions above it, and the first of those
// equal to it, are listed in ascending order.
__global__ void __launch_bounds__(1024) evict_select_kernel(const EvictParams p) {
    const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = clamp_len(p.lens[b], p.cap);
    __shared__ int hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left, s_total, s_gt[32], s_eq[32];
    // Keys that may be kept.
    int mine = 0;
    for (int i = tid; i < len; i += 1024) mine += evict_key(p, b, hk, i, len) != 0u;
    if (tid == 0) s_total = 0;
    __syncthreads();
    atomicAdd(&s_total, mine);
    __syncthreads();
    const int n_keep = min(p.keep, s_total);
    uint32_t prefix = 0;
    int left = n_keep;  // how many of the keys that share the prefix are kept
    for (int shift = 24; shift >= 0 && n_keep > 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < len; i += 1024) {
            const uint32_t k = evict_key(p, b, hk, i, len);
            if (k != 0u && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))))
                atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255, n = left;
            while (d > 0 && hist[d] < n) n -= hist[d--];
            s_prefix = prefix | ((uint32_t)d << shift);
            s_left = n;
        }
        __syncthreads();
        prefix = s_prefix;
        left = s_left;
    }
    int *kept = p.kept + ((int64_t)b * p.pool.Hkv + hk) * p.keep;
    float *wo = p.w_out + ((int64_t)b * p.pool.Hkv + hk) * p.keep;
    int done = 0, eq_done = 0;
    for (int i0 = 0; i0 < len && n_keep > 0; i0 += 1024) {
        const int i = i0 + tid;
        const uint32_t k = i < len ? evict_key(p, b, hk, i, len) : 0u;
        const bool gt = k > prefix, eq = k == prefix && k != 0u;
        const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
        __syncthreads();
        if (lane == 0) s_gt[warp] = __popc(bg), s_eq[warp] = __popc(be);
        __syncthreads();
        int g = 0, e = 0, gall = 0, eall = 0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) g += s_gt[w], e += s_eq[w];
            gall += s_gt[w], eall += s_eq[w];
        }
        g += __popc(bg & ((1u << lane) - 1u));
        e += __popc(be & ((1u << lane) - 1u));
        const int e_before = min(left, eq_done + e);
        if (gt || (eq && eq_done + e < left)) {
            const int at = done + g + (e_before - min(left, eq_done));
            kept[at] = i;
            wo[at] = p.w[b * p.w_sb + hk * p.w_sh + i];
        }
        done += gall + (min(left, eq_done + eall) - min(left, eq_done));
        eq_done += eall;
    }
    for (int i = n_keep + tid; i < p.keep; i += 1024) kept[i] = -1, wo[i] = 0.f;
    if (hk == 0 && tid == 0) p.new_lens[b] = n_keep;
}

// Kept row i of (b, hk) -> position i of the destination table's pages.
template <int ESIZE>
__global__ void evict_gather_kernel(const EvictParams p) {
    const int hk = blockIdx.y, b = blockIdx.z;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int c = (int)(i % p.chunks);
    const int64_t to = i / p.chunks;
    if (to >= p.keep) return;
    const int from = p.kept[((int64_t)b * p.pool.Hkv + hk) * p.keep + to];
    if (from < 0) return;
    const int sp = page_of(p.src, p.pool.num_pages, b, from / p.pool.page);
    const int dp = page_of(p.dst, p.pool.num_pages, b, (int)to / p.pool.page);
    if (sp < 0 || dp < 0) return;
    const int64_t ss = from % p.pool.page, ds = to % p.pool.page;
    char *k = static_cast<char *>(p.pool.k), *v = static_cast<char *>(p.pool.v);
    reinterpret_cast<int4 *>(k + (dp * p.pool.k_sp + hk * p.pool.k_sh + ds * p.pool.k_ss) * ESIZE)[c] =
        reinterpret_cast<const int4 *>(k + (sp * p.pool.k_sp + hk * p.pool.k_sh + ss * p.pool.k_ss) * ESIZE)[c];
    reinterpret_cast<int4 *>(v + (dp * p.pool.v_sp + hk * p.pool.v_sh + ds * p.pool.v_ss) * ESIZE)[c] =
        reinterpret_cast<const int4 *>(v + (sp * p.pool.v_sp + hk * p.pool.v_sh + ss * p.pool.v_ss) * ESIZE)[c];
}

}  // namespace gae
