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
    FastDiv by_chunks, by_heads;
};

// A thread copies 16 bytes of kAppendRows new rows, K and V both; all of its
// reads are on their way before it writes.  Bound by memory: 335 MB of a prompt
// read and written take 57 us (89% of the copy rate), 66 with one row to a thread.
constexpr int kAppendRows = 4;

template <int ESIZE>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
    const int b = blockIdx.y;
    const int n = p.counts ? min(p.counts[b], p.tokens) : p.tokens, start = p.start[b];
    const int64_t cap = (int64_t)p.table.max_pages * p.pool.page;
    int64_t k_to[kAppendRows], v_to[kAppendRows];
    int4 x[kAppendRows], y[kAppendRows];
    bool live[kAppendRows];
#pragma unroll
    for (int e = 0; e < kAppendRows; ++e) {
        const uint32_t i = ((uint32_t)blockIdx.x * kAppendRows + e) * 256u + threadIdx.x;
        const uint32_t row = p.by_chunks.div(i), t = p.by_heads.div(row);
        const int c = (int)(i - row * p.chunks), h = (int)(row - t * p.pool.Hkv);
        const int64_t pos = (int64_t)start + t;
        live[e] = (int64_t)t < n && pos >= 0 && pos < cap;
        int pg = -1;
        int64_t slot = 0;
        if (live[e]) {
            const uint32_t idx = p.pool.by_page.div((uint32_t)pos);
            pg = page_of(p.table, p.pool.num_pages, b, (int)idx);
            slot = pos - (int64_t)idx * p.pool.page;
            x[e] = __ldg(reinterpret_cast<const int4 *>(static_cast<const char *>(p.k_new) +
                                                       (b * p.kn_sb + h * p.kn_sh + t * p.kn_st) * ESIZE) + c);
            y[e] = __ldg(reinterpret_cast<const int4 *>(static_cast<const char *>(p.v_new) +
                                                       (b * p.vn_sb + h * p.vn_sh + t * p.vn_st) * ESIZE) + c);
        }
        live[e] = pg >= 0;
        k_to[e] = (pg * p.pool.k_sp + h * p.pool.k_sh + slot * p.pool.k_ss) * ESIZE + c * 16;
        v_to[e] = (pg * p.pool.v_sp + h * p.pool.v_sh + slot * p.pool.v_ss) * ESIZE + c * 16;
    }
#pragma unroll
    for (int e = 0; e < kAppendRows; ++e)
        if (live[e]) {
            *reinterpret_cast<int4 *>(static_cast<char *>(p.pool.k) + k_to[e]) = x[e];
            *reinterpret_cast<int4 *>(static_cast<char *>(p.pool.v) + v_to[e]) = y[e];
        }
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
    int chunks, esize;    // 16-byte pieces of a row, bytes of an element
};

// Whole-number order of the weights: NaN above +inf, -0 equal to 0.  Every
// float maps into [0x007fffff, 0xfffffffe]; 0 is "no key" and 0xffffffff "kept
// whatever its weight".
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Kept rows first, first + step, ... of (b, hk), their 16-byte piece c of K and
// V, to the same positions of the destination table: kRows copies on their
// way at once.
constexpr int kGatherRows = 4;

template <int kRows>
__device__ __forceinline__ void evict_gather(const EvictParams &p, int b, int hk, int first, int step, int c) {
    const int *kept = p.kept + ((int64_t)b * p.pool.Hkv + hk) * p.keep;
    char *k = static_cast<char *>(p.pool.k) + hk * p.pool.k_sh * p.esize + c * 16;
    char *v = static_cast<char *>(p.pool.v) + hk * p.pool.v_sh * p.esize + c * 16;
    int from[kRows], page[kRows], to_page[kRows];
    int4 x[kRows], y[kRows];
#pragma unroll
    for (int e = 0; e < kRows; ++e) from[e] = first + e * step < p.keep ? kept[first + e * step] : -1;
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
        page[e] = to_page[e] = -1;
        if (from[e] < 0) continue;
        const uint32_t idx = p.pool.by_page.div(from[e]);
        page[e] = page_of(p.src, p.pool.num_pages, b, (int)idx);
        from[e] -= (int)idx * p.pool.page;
        to_page[e] = page_of(p.dst, p.pool.num_pages, b, (int)p.pool.by_page.div((uint32_t)(first + e * step)));
    }
#pragma unroll
    for (int e = 0; e < kRows; ++e)
        if (page[e] >= 0) {
            x[e] = *reinterpret_cast<const int4 *>(k + (page[e] * p.pool.k_sp + from[e] * p.pool.k_ss) * p.esize);
            y[e] = *reinterpret_cast<const int4 *>(v + (page[e] * p.pool.v_sp + from[e] * p.pool.v_ss) * p.esize);
        }
#pragma unroll
    for (int e = 0; e < kRows; ++e)
        if (page[e] >= 0 && to_page[e] >= 0) {
            const uint32_t to = (uint32_t)(first + e * step);
            const int64_t slot = to - (int64_t)p.pool.by_page.div(to) * p.pool.page;
            *reinterpret_cast<int4 *>(k + (to_page[e] * p.pool.k_sp + slot * p.pool.k_ss) * p.esize) = x[e];
            *reinterpret_cast<int4 *>(v + (to_page[e] * p.pool.v_sp + slot * p.pool.v_ss) * p.esize) = y[e];
        }
}

// The weights of kept positions first, first + step, ...; 0 beyond the length.
template <int kRows>
__device__ __forceinline__ void evict_weights(const EvictParams &p, int b, int hk, int first, int step) {
    const int64_t row = ((int64_t)b * p.pool.Hkv + hk) * p.keep;
    const float *w = p.w + b * p.w_sb + hk * p.w_sh;
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
        const int i = first + e * step;
        if (i >= p.keep) break;
        const int pos = p.kept[row + i];
        p.w_out[row + i] = pos >= 0 ? __ldg(w + pos) : 0.f;
    }
}

// The keep-th largest key of a (key head, sequence) row is found by a radix
// search over its 11, 11 and 10 highest bits; positions above it, and the first
// of those equal to it, are then listed in ascending order.  A cluster of up to
// 8 CTAs shares a row where there are few rows, each with its run of positions:
// the keys are formed once and stay in shared memory (positions beyond
// kEvictMaxKeys are formed again), only histograms and counts cross the cluster.
// What bounds it is latency: one barrier of the cluster to a digit.
// Where a row's CTAs have little to copy they do it themselves (a launch less:
// 18 -> 16.4 us a call at 1024 positions of two sequences x 12 heads, though 13
// -> 15 us replayed from a graph); larger shares are left to a kernel that fills
// the GPU (50000 positions to 8192: 69 us, of which the copies take 43).
constexpr int kEvictThreads = 1024, kEvictWarps = kEvictThreads / 32, kEvictBins = 2048;
constexpr int kEvictMaxCluster = 8, kEvictMaxKeys = 40960;

// A cluster barrier after which the CTAs see what the others wrote before it:
// one thread's fence stands for the CTA (its threads have met before), where a
// releasing arrival would be a fence of every thread.
__device__ __forceinline__ void cluster_publish() {
    __syncthreads();
    if (threadIdx.x == 0) asm volatile("fence.acq_rel.cluster;" ::: "memory");
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint2 ld_cluster_u2(uint32_t addr, uint32_t rank) {
    uint2 v;
    asm volatile("ld.shared::cluster.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(mapa_shared(addr, rank)) : "memory");
    return v;
}

__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(const EvictParams p, int cluster, int max_keys, int copy) {
    extern __shared__ __align__(16) uint32_t smem_ev[];
    uint32_t *hist = smem_ev;                    // [2][bins], one digit's after the other's
    uint32_t *keys = smem_ev + 2 * kEvictBins;  // [max_keys], a multiple of 4
    __shared__ uint32_t s_warp[kEvictWarps], s_digit, s_left;
    __shared__ __align__(8) uint32_t s_counts[2];
    const int rank = (int)cluster_ctarank(), row = blockIdx.x / cluster, hk = row % p.pool.Hkv, b = row / p.pool.Hkv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int len = clamp_len(p.lens[b], p.cap);
    const int per = (len + cluster - 1) / cluster, lo = min(len, rank * per), n = min(len, lo + per) - lo;
    const float *w = p.w + b * p.w_sb + hk * p.w_sh + lo;
    const int *table = p.src.entry + b * p.src.stride;
    const int pages = (int)p.pool.num_pages, forced = len - p.recent - lo;
    auto key_of = [&](int i, int pg, float x) -> uint32_t {
        return (uint32_t)pg >= (uint32_t)pages ? 0u : i >= forced ? 0xffffffffu : weight_key(x);
    };
    auto form = [&](int i) -> uint32_t {  // the key of this CTA's position i
        return key_of(i, __ldg(table + p.pool.by_page.div(lo + i)), __ldg(w + i));
    };
    const bool all_held = n <= max_keys;
    auto get4 = [&](int i, uint32_t (&k)[4]) {  // keys i .. i + 3, 0 beyond the end; i a multiple of 4
        if (all_held) {
            const uint4 v = *reinterpret_cast<const uint4 *>(keys + i);
            k[0] = v.x, k[1] = v.y, k[2] = v.z, k[3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = i + e >= n ? 0u : i + e < max_keys ? keys[i + e] : form(i + e);
        }
    };
    for (int i = tid; i < 2 * kEvictBins; i += kEvictThreads) hist[i] = 0;
    const int held = min(n, max_keys);
    for (int i0 = tid; i0 < held; i0 += 8 * kEvictThreads) {  // eight pages and weights on their way at once
        int pg[8];
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = min(i0 + e * kEvictThreads, held - 1);
            pg[e] = __ldg(table + p.pool.by_page.div(lo + i));
            x[e] = __ldg(w + i);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = i0 + e * kEvictThreads;
            if (i < held) keys[i] = key_of(i, pg[e], x[e]);
        }
    }
    if (tid < (-held & 3)) keys[held + tid] = 0;
    uint32_t prefix = 0, left = 0;
    int n_keep = 0;
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
        const uint32_t mask = digit == 2 ? 1023u : 2047u;
        // the bits above this digit have to be the prefix's
        const uint32_t above = digit == 0 ? 0u : digit == 1 ? 0xffe00000u : 0xfffffc00u;
        uint32_t *h = hist + (digit & 1) * kEvictBins;
        __syncthreads();
        for (int i = tid * 4; i < n; i += kEvictThreads * 4) {
            uint32_t k[4];
            get4(i, k);
            // few keys share the upper digits: mostly none of four
            uint32_t off = 0xffffffffu;
#pragma unroll
            for (int e = 0; e < 4; ++e) off = min(off, (k[e] ^ prefix) & above);
            if (off == 0u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k[e] != 0u && ((k[e] ^ prefix) & above) == 0u) atomicAdd(h + ((k[e] >> shift) & mask), 1u);
        }
        cluster_publish();
        // Every CTA adds up the whole cluster's bins, kBins to a thread from the top.
        constexpr int kBins = kEvictBins / kEvictThreads;
        const uint32_t ha = smem_u32(h) + (kEvictBins - (tid + 1) * kBins) * 4;
        uint32_t c[kBins] = {}, mine = 0;
#pragma unroll
        for (int r = 0; r < kEvictMaxCluster; ++r)
            if (r < cluster)
#pragma unroll
                for (int e = 0; e < kBins; e += 2) {
                    const uint2 x = ld_cluster_u2(ha + (kBins - 2 - e) * 4, (uint32_t)r);
                    c[e] += x.y, c[e + 1] += x.x;
                }
#pragma unroll
        for (int e = 0; e < kBins; ++e) mine += c[e];
        uint32_t incl = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += up;
        }
        if (lane == 31) s_warp[warp] = incl;
        __syncthreads();
        const uint32_t sums = lane < kEvictWarps ? s_warp[lane] : 0u;
        uint32_t before = incl - mine + __reduce_add_sync(0xffffffffu, lane < warp ? sums : 0u);
        if (digit == 0) {
            n_keep = min(p.keep, (int)__reduce_add_sync(0xffffffffu, sums));
            left = (uint32_t)n_keep;
        }
        // the thread in whose bins the running count reaches `left`
        if (before < left && before + mine >= left)
#pragma unroll
            for (int e = 0; e < kBins; ++e) {
                if (before < left && before + c[e] >= left) {
                    s_digit = kEvictBins - 1 - tid * kBins - e;
                    s_left = left - before;
                }
                before += c[e];
            }
        __syncthreads();
        if (n_keep == 0) break;  // the same in every CTA of the cluster
        prefix |= s_digit << shift;
        left = s_left;
        // The third digit uses the first one's bins: every CTA has read them once
        // all have passed the second's barrier.
        if (digit == 1)
            for (int i = tid; i < kEvictBins; i += kEvictThreads) hist[i] = 0;
    }
    // Keys above the threshold and equal to it: every warp a run of positions,
    // counted, then listed from where the runs before it end.
    const int run = (((n + kEvictWarps - 1) / kEvictWarps) + 127) / 128 * 128, first = warp * run, last = min(n, first + run);
    uint32_t gt = 0, eq = 0;
    if (n_keep > 0)
        for (int i = first + lane * 4; i < last; i += 128) {
            uint32_t k[4];
            get4(i, k);
#pragma unroll
            for (int e = 0; e < 4; ++e) gt += k[e] > prefix, eq += k[e] == prefix && k[e] != 0u;
        }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    __shared__ uint32_t s_gt[kEvictWarps], s_eq[kEvictWarps];
    if (lane == 0) s_gt[warp] = gt, s_eq[warp] = eq;
    __syncthreads();
    const uint32_t gts = lane < kEvictWarps ? s_gt[lane] : 0u, eqs = lane < kEvictWarps ? s_eq[lane] : 0u;
    if (warp == 0) {
        const uint32_t g = __reduce_add_sync(0xffffffffu, gts), e = __reduce_add_sync(0xffffffffu, eqs);
        if (lane == 0) s_counts[0] = g, s_counts[1] = e;
    }
    cluster_publish();
    uint32_t g0 = __reduce_add_sync(0xffffffffu, lane < warp ? gts : 0u);
    uint32_t e0 = __reduce_add_sync(0xffffffffu, lane < warp ? eqs : 0u);
#pragma unroll
    for (int r = 0; r < kEvictMaxCluster - 1; ++r)
        if (r < rank) {
            const uint2 x = ld_cluster_u2(smem_u32(s_counts), (uint32_t)r);
            g0 += x.x, e0 += x.y;
        }
    int *kept = p.kept + ((int64_t)b * p.pool.Hkv + hk) * p.keep;
    if (n_keep > 0)
        for (int i0 = first; i0 < last; i0 += 128) {
            const int i = i0 + lane * 4;
            uint32_t k[4] = {};
            if (i < last) get4(i, k);
            uint32_t mine = 0;  // above in the low half, equal in the high half: 128 at most
#pragma unroll
            for (int e = 0; e < 4; ++e) mine += (k[e] > prefix ? 1u : 0u) + (k[e] == prefix && k[e] != 0u ? 0x10000u : 0u);
            uint32_t incl = mine;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, incl, s);
                if (lane >= s) incl += up;
            }
            if (mine) {
                uint32_t g = g0 + ((incl - mine) & 0xffffu), q = e0 + ((incl - mine) >> 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool above = k[e] > prefix, equal = k[e] == prefix && k[e] != 0u;
                    if (above || (equal && q < left)) kept[g + min(q, left)] = lo + i + e;
                    g += above, q += equal;
                }
            }
            const uint32_t all = __shfl_sync(0xffffffffu, incl, 31);
            g0 += all & 0xffffu;
            e0 += all >> 16;
        }
    for (int i = n_keep + rank * kEvictThreads + tid; i < p.keep; i += cluster * kEvictThreads) kept[i] = -1;
    if (hk == 0 && rank == 0 && tid == 0) p.new_lens[b] = n_keep;
    if (!copy) {
        // no CTA leaves while another reads its counts
        asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
        return;
    }
    cluster_publish();  // the row's list is complete
    for (int i = rank * kEvictThreads + tid; i < p.keep; i += cluster * kEvictThreads) evict_weights<1>(p, b, hk, i, 0);
    const int rows = kEvictThreads / p.chunks, r = tid / p.chunks;
    if (r < rows)
        for (int i = rank * rows * 2 + r; i < n_keep; i += cluster * rows * 2)
            evict_gather<2>(p, b, hk, i, rows, tid % p.chunks);
}

// The copies of a large share: blocks of their own, the first ones the weights,
// 1024 each.
__global__ void __launch_bounds__(256) evict_gather_kernel(const EvictParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int hk = blockIdx.y, b = blockIdx.z, weight_blocks = (p.keep + 1023) / 1024;
    if ((int)blockIdx.x < weight_blocks) {
        evict_weights<4>(p, b, hk, blockIdx.x * 1024 + threadIdx.x, 256);
        return;
    }
    const int rows = 256 / p.chunks, r = threadIdx.x / p.chunks;
    if (r < rows)
        evict_gather<kGatherRows>(p, b, hk, (int)(blockIdx.x - weight_blocks) * rows * kGatherRows + r, rows,
                                  threadIdx.x % p.chunks);
}

}  // namespace gae
