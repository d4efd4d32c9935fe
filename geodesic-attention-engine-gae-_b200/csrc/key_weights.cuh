// key_weights.cuh -- the attention weight that a block of queries puts on each
// key, from the forward's log-sum-exp:
//
//   w[b, hk, j] = sum over the heads h of key head hk, sum over the queries i
//                 that see key j of exp(scale <q_i, k_j> - lse_i)
//
// No reference counterpart; it is what an eviction after a prompt goes by.
//
// The scores are computed transposed, keys as the 128 rows of a tcgen05 tile
// and queries as its columns: a TMEM lane is then one key, so a thread adds up
// its key's weights in registers and no two threads ever share a sum (no
// atomics, the same bits every time).  One CTA per (two 128-key tiles, key head,
// batch), two CTAs to an SM: K stays in shared memory, the tiles of 128 queries
// of all the head's query heads stream through TMA, and each key tile has an S
// tile in TMEM and a warpgroup that exponentiates it while the other three
// tiles' products and exponentials run.  One key tile to a CTA read every query
// tile from L2 twice as often and was bound by that, at 6.2 TB/s.
//
// What bounds it: one exponential per score.  The MUFU gives 16 a cycle and
// SM, a 128 x 128 tile takes it 1024 cycles where the products at head_dim 128
// take 512.  All exponentials are the MUFU's, which keeps NaN, gives +inf from
// 2^128 on and 0 below 2^-126 whatever column a query stands in.  A polynomial
// on the FMA pipe for every third pair took as long within 2% and had none of
// that.  8192 x 8192 causal, 16 heads x 128: 182 us, MUFU 78% and tensor pipe 40%
// busy; 200 x 32768, 32 heads on 8, 128: 93 us, 66% and 37%.
#pragma once
#include <cfloat>

#include "attn_bwd_sm100.cuh"
#include "sm100.cuh"

namespace gae {

struct KeyWeightsParams {
    CUtensorMap tm_q, tm_k;  // dims {D, N, H, B}, box {64 elements, 128 rows}, 128B swizzle
    const float *lse;
    float *out;              // [B, Hkv, Nkv], or the splits' parts
    int64_t l_sb, l_sh, o_sb, o_sh;
    int64_t part;            // elements between two splits' parts; 0: one split, written to out
    int B, H, Hkv, Nq, Nkv, causal, accumulate, splits;
    int64_t off;             // query row r sees key c iff c <= r + off (causal)
    float scale_log2;
};

enum KeyWeightsWaitSite : unsigned {
    kSiteKwK = 0x501, kSiteKwQFull = 0x502, kSiteKwQEmpty = 0x503, kSiteKwS = 0x504, kSiteKwSEmpty = 0x505,
    kSiteKwDone = 0x506, kSiteKwSmem = 0x507,
};

template <int D>
struct KeyWeightsCfg {
    static constexpr int kBox = 128 * 128, kPanels = D * 2 / 128, kTile = kPanels * kBox;
    static constexpr int kStages = D == 128 ? 1 : 3;
    static constexpr int kOffK = 0, kOffQ = 2 * kTile, kOffLse = kOffQ + kStages * kTile;  // lse: 2 tiles of 128
    static constexpr int kOffBar = kOffLse + 2 * 128 * 4;
    static constexpr int kNumBars = 2 + 2 * kStages + 4;  // k, done, q_full/q_empty, s_full/s_empty [2]
    static constexpr int kPayload = kOffBar + kNumBars * 8 + 16;
    static constexpr int kSmem = kPayload + 1024;  // slack for the 1024-byte alignment of the swizzle atoms
    static constexpr int kTmaWarp = 8, kMmaWarp = 9, kLseWarp = 10, kThreads = 11 * 32;
    static constexpr uint32_t kTmemCols = 256;
    static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs to an SM");
};

template <int D, bool kBF16>
__global__ void __launch_bounds__(KeyWeightsCfg<D>::kThreads, 2)
    key_weights_kernel(const __grid_constant__ KeyWeightsParams p) {
    using Cfg = KeyWeightsCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw), base = (raw_addr + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (base - raw_addr);
    if (base - raw_addr + Cfg::kPayload > (uint32_t)Cfg::kSmem) {
        if (threadIdx.x == 0) record_error(kSiteKwSmem);
        return;
    }
    const uint32_t sK = base + Cfg::kOffK, sBar = base + Cfg::kOffBar;
    auto sQ = [&](int st) { return base + Cfg::kOffQ + st * Cfg::kTile; };
    float *s_lse = reinterpret_cast<float *>(smem + Cfg::kOffLse);
    const uint32_t bar_k = sBar, bar_done = sBar + 8;
    auto bar_q_full = [&](int st) { return sBar + 8u * (2 + st); };
    auto bar_q_empty = [&](int st) { return sBar + 8u * (2 + Cfg::kStages + st); };
    auto bar_s_full = [&](int kt) { return sBar + 8u * (2 + 2 * Cfg::kStages + kt); };
    auto bar_s_empty = [&](int kt) { return sBar + 8u * (4 + 2 * Cfg::kStages + kt); };
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Cfg::kOffBar + Cfg::kNumBars * 8);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int no_abort = 0;
    volatile int *s_none = reinterpret_cast<volatile int *>(tmem_slot + 2);  // [2] a query of the tile saw no key
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // Pairs of key tiles in ascending order: under a causal mask the first have the most queries.
    const int rows = p.B * p.Hkv;
    const int j = blockIdx.x / rows, b = blockIdx.x % rows / p.Hkv, hk = blockIdx.x % rows % p.Hkv, split = blockIdx.y;
    const int G = p.H / p.Hkv, nq = (p.Nq + 127) / 128;
    const int n_kt = (int64_t)j * 256 + 128 < p.Nkv ? 2 : 1;  // key tiles that exist
    int i0 = 0;  // first query tile that sees a key of this pair
    if (p.causal) i0 = (int)min64(nq, max64(0, (int64_t)j * 256 - p.off) / 128);
    const int per_head = nq - i0, all = per_head * G;
    const int t0 = (int)((int64_t)all * split / p.splits), t1 = (int)((int64_t)all * (split + 1) / p.splits);
    const int n_it = t1 - t0;
    // The query tile at hand: head h, tile i of those that see these keys.
    int h = hk * G, i = 0;
    if (n_it > 0) h += t0 / per_head, i = t0 % per_head;
    auto next_tile = [&] {
        if (++i == per_head) i = 0, ++h;
    };

    if (threadIdx.x == 0) {
        mbar_init(bar_k, 1);
        mbar_init(bar_done, 1);
        for (int st = 0; st < Cfg::kStages; ++st) {
            mbar_init(bar_q_full(st), 1);
            mbar_init(bar_q_empty(st), 1);
        }
        for (int kt = 0; kt < 2; ++kt) {
            mbar_init(bar_s_full(kt), 1 + 32);  // the products, and the lanes of the lse warp
            mbar_init(bar_s_empty(kt), 128);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == Cfg::kMmaWarp) {
        tmem_alloc(smem_u32(tmem_slot), Cfg::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == Cfg::kTmaWarp) {
        if (lane == 0 && n_it > 0) {
            tma_prefetch_desc(&p.tm_q);
            mbar_expect_tx(bar_k, n_kt * Cfg::kTile);
            for (int kt = 0; kt < n_kt; ++kt)
                for (int hf = 0; hf < Cfg::kPanels; ++hf)
                    tma_load_4d(sK + kt * Cfg::kTile + hf * Cfg::kBox, &p.tm_k, bar_k, hf * 64, j * 256 + kt * 128, hk, b);
            int it = 0;
            for (; it < n_it; ++it) {
                const int st = it % Cfg::kStages, use = it / Cfg::kStages;
                if (use > 0 && !mbar_wait(bar_q_empty(st), (use - 1) & 1, kSiteKwQEmpty, abort_flag)) break;
                mbar_expect_tx(bar_q_full(st), Cfg::kTile);
                for (int hf = 0; hf < Cfg::kPanels; ++hf)
                    tma_load_4d(sQ(st) + hf * Cfg::kBox, &p.tm_q, bar_q_full(st), hf * 64, (i0 + i) * 128, h, b);
                next_tile();
            }
            // the copies issued have landed before the CTA exits
            mbar_wait(bar_k, 0, kSiteKwK, &no_abort);
            for (int u = max(0, it - Cfg::kStages); u < it; ++u)
                mbar_wait(bar_q_full(u % Cfg::kStages), (u / Cfg::kStages) & 1, kSiteKwQFull, &no_abort);
        }
    } else if (warp == Cfg::kMmaWarp) {
        if (lane == 0 && n_it > 0) {
            constexpr uint32_t id = idesc_f16(128, 128, kBF16, false, false);
            bool ok = mbar_wait(bar_k, 0, kSiteKwK, abort_flag);
            for (int it = 0; it < n_it && ok; ++it) {
                const int st = it % Cfg::kStages;
                if (!(ok = mbar_wait(bar_q_full(st), (it / Cfg::kStages) & 1, kSiteKwQFull, abort_flag))) break;
                for (int kt = 0; kt < n_kt; ++kt) {
                    if (it > 0 && !(ok = mbar_wait(bar_s_empty(kt), (it - 1) & 1, kSiteKwSEmpty, abort_flag))) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t o = (kk >> 2) * Cfg::kBox + (kk & 3) * 32;
                        umma_f16_ss(tmem + kt * 128, smem_desc_sw128(sK + kt * Cfg::kTile + o, 16, 1024),
                                    smem_desc_sw128(sQ(st) + o, 16, 1024), id, kk > 0);
                    }
                    umma_commit(bar_s_full(kt));
                }
                umma_commit(bar_q_empty(st));
            }
            umma_commit(bar_done);
            mbar_wait(bar_done, 0, kSiteKwDone, &no_abort);
        }
    } else if (warp == Cfg::kLseWarp) {
        // -lse of the tile's queries in log2.  +inf marks a row that saw no key
        // (lse = -inf) or does not exist: its weights are 0 whatever its scores,
        // and s_none sends its tile to the epilogue's selecting path.  A finite
        // lse whose negative passes fp32's range stays finite: no mark.  Two
        // buffers: warpgroups that have let go of S tile it - 1 are done with
        // tile it - 2.
        auto fetch = [&](float (&v)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = (i0 + i) * 128 + e * 32 + lane;
                const float l = r < p.Nq ? __ldg(p.lse + b * p.l_sb + h * p.l_sh + r) : -INFINITY;
                v[e] = -l * 1.4426950408889634f;
                if (v[e] == INFINITY && l != -INFINITY) v[e] = FLT_MAX;
            }
            next_tile();
        };
        float v[4];
        if (n_it > 0) fetch(v);
        for (int it = 0; it < n_it; ++it) {
            bool ok = true;
            for (int kt = 0; kt < n_kt && it > 0; ++kt)
                ok = ok && mbar_wait(bar_s_empty(kt), (it - 1) & 1, kSiteKwSEmpty, abort_flag);
            if (!ok) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) s_lse[(it & 1) * 128 + e * 32 + lane] = v[e];
            const int none = __any_sync(0xffffffffu, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) == INFINITY);
            if (lane == 0) s_none[it & 1] = none;
            if (it + 1 < n_it) fetch(v);
            for (int kt = 0; kt < n_kt; ++kt) mbar_arrive(bar_s_full(kt));
        }
    } else {
        // ------------------------ epilogue: warpgroup g has key tile g, thread = key
        const int g = warp >> 2, key = (warp & 3) * 32 + lane;
        const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + g * 128;
        const uint64_t sl2 = f2_pack(p.scale_log2, p.scale_log2);
        float total = 0.f;
        // Query rows before this are before this thread's key (this warp's lowest,
        // its highest): all an epilogue has to know of the mask, within [0, Nq].
        auto first_row = [&](int k) {
            return p.causal ? (int)max64(0, min64(p.Nq, (int64_t)j * 256 + g * 128 + k - p.off)) : 0;
        };
        const int first = first_row(key), first_low = first_row(key - lane), first_high = first_row(key - lane + 31);
        for (int it = 0; it < n_it && g < n_kt; ++it) {
            const int q0 = (i0 + i) * 128;
            next_tile();
            if (!mbar_wait(bar_s_full(g), it & 1, kSiteKwS, abort_flag)) break;
            tc_fence_after();
            const uint32_t sl = base + Cfg::kOffLse + (it & 1) * 512;
            uint64_t acc[4] = {};
            // every key of the warp is seen by all 128 queries, each of which saw one
            if (first_high <= q0 && !s_none[it & 1]) {
#pragma unroll
                for (int c0 = 0; c0 < 128; c0 += 32) {
                    uint32_t r[32];
                    tmem_ld32(tS + c0, r);
                    tmem_wait_ld();
                    if (c0 == 96) {
                        tc_fence_before();
                        mbar_arrive(bar_s_empty(g));
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        uint64_t n[2];
                        asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];" : "=l"(n[0]), "=l"(n[1]) : "r"(sl + c0 * 4 + e * 8));
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int c = 2 * (e + u);
                            float x0, x1;
                            f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), sl2, n[u]), x0, x1);
                            const uint64_t w = f2_pack(ex2_approx(x0), ex2_approx(x1));
                            acc[(e + u) & 3] = f2_add(acc[(e + u) & 3], w);
                        }
                    }
                }
            } else {
                // Columns [lo, hi) count (from hi on there are no queries), but for
                // those marked as having seen no key: a select, since their scores
                // may be NaN or infinite.  32 columns that no key of the warp counts
                // are passed over.
                const int lo = first - q0, hi = min(128, p.Nq - q0);
#pragma unroll 1
                for (int c0 = max(0, first_low - q0) & ~31; c0 < hi; c0 += 32) {
                    uint32_t r[32];
                    tmem_ld32(tS + c0, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        uint64_t n0;
                        asm volatile("ld.shared.b64 %0, [%1];" : "=l"(n0) : "r"(sl + c0 * 4 + e * 8));
                        const int c = c0 + 2 * e;
                        float x0, x1, l0, l1;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), sl2, n0), x0, x1);
                        f2_unpack(n0, l0, l1);
                        const float w0 = c >= lo && l0 != INFINITY ? ex2_approx(x0) : 0.f;
                        const float w1 = c + 1 >= lo && l1 != INFINITY ? ex2_approx(x1) : 0.f;
                        acc[e & 3] = f2_add(acc[e & 3], f2_pack(w0, w1));
                    }
                }
                tc_fence_before();
                mbar_arrive(bar_s_empty(g));
            }
            // a tile's sum first, then the total: the longest chains stay short
            float a, c;
            f2_unpack(f2_add(f2_add(acc[0], acc[1]), f2_add(acc[2], acc[3])), a, c);
            total += a + c;
        }
        const int64_t c = (int64_t)j * 256 + g * 128 + key;
        if (c < p.Nkv) {
            if (p.part) {
                p.out[split * p.part + ((int64_t)b * p.Hkv + hk) * p.Nkv + c] = total;
            } else {
                float *o = p.out + b * p.o_sb + hk * p.o_sh + c;
                *o = p.accumulate ? *o + total : total;
            }
        }
    }
    __syncthreads();
    if (warp == Cfg::kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
}

// Adds the splits' parts in their order.
__global__ void key_weights_sum_kernel(const float *parts, float *out, int64_t o_sb, int64_t o_sh, int Hkv, int Nkv,
                                       int64_t part, int splits, int accumulate) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= part) return;
    float w = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) w += parts[s * part + i];
    const int64_t row = i / Nkv;
    float *o = out + row / Hkv * o_sb + row % Hkv * o_sh + i % Nkv;
    *o = accumulate ? *o + w : w;
}

// A block without queries: nothing to add, or zeros.
__global__ void key_weights_zero_kernel(float *out, int64_t o_sb, int64_t o_sh, int Hkv, int Nkv, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) out[i / Nkv / Hkv * o_sb + i / Nkv % Hkv * o_sh + i % Nkv] = 0.f;
}

}  // namespace gae
