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

// Division of positions (< 2^31) by a run-time constant: q = (umulhi(n, mul) +
// n) >> shift with shift = ceil(log2 d), mul = floor(2^32 (2^shift - d) / d) + 1
// (T. Granlund, P. Montgomery, "Division by Invariant Integers using
// Multiplication", 1994).  n < 2^31 keeps the sum within 32 bits.
struct FastDiv {
    uint32_t d, mul, shift;
    static FastDiv of(uint32_t d) {
        uint32_t s = 0;
        while ((1ull << s) < d) ++s;
        return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
#ifdef __CUDA_ARCH__
        return (__umulhi(n, mul) + n) >> shift;
#else
        return (uint32_t)((((uint64_t)n * mul) >> 32) + n) >> shift;
#endif
    }
};

// K and V pools [num_pages, kv_heads, page_size, head_dim], element strides.
struct KvPool {
    void *k, *v;
    int64_t k_sp, k_sh, k_ss, v_sp, v_sh, v_ss;
    int64_t num_pages;
    int Hkv, page, D;
    FastDiv by_page;
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
