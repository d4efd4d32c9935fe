// paged_attn.cuh -- attention of one new token per sequence over the paged
// cache, split over the cache's length and joined.
//
//   o = sum_t softmax_t(scale <q, k_t>) v_t,  t < len,  per (sequence, head)
//
// Every cached row is read once for up to 16 query heads that share it (8 in
// fp32; once for each such group where more do), so the work is bound by the
// cache's bytes; the kernels are built to keep enough of them in flight.  A row (sequence, key head, group of up to 16 query heads) is cut
// into tiles of kKeys positions to a warp and the tiles of all rows, in order, are
// dealt in equal runs to a grid that fills the GPU once, whatever the lengths
// are: they are read on the device, so a captured graph stays balanced when
// they change.  A block that ends inside a row leaves (max, sum, O) of its part
// in the workspace; paged_attn_join_kernel adds those parts in a fixed order.
//
// Inside a block the warps take 16 rows (8 for fp32) of each tile each,
// with their own ring of cp.async stages, maximum, sum and accumulator: nothing
// is shared until the row ends, so no barrier stands between tiles.
//
// Measured (one B200, 6.55 TB/s as a copy): 32 sequences x 32 heads x 128, up to
// 4096 positions, bf16, 1.11 GB: 168 us in the kernel (6.6 TB/s), 174 us with the
// join; 131072 positions, 32 heads on 8, f16, 537 MB: 83 and 91 us; 16 sequences
// up to 8191 positions with weights, 290 MB: 50 and 61 us (the weights' second
// pass over 8.4 MB of scores is latency: 10 us).  What made it so: three blocks
// of two stages to an SM over two of three (172 against 180 us at the first
// size), the next tile's loads before this tile's products, the next row's q
// before the merge, and one page look-up to a tile (all four: 262 to 172 us).  At
// head_dim 256 six warps to a block: 16 x 16 heads, up to 4096 positions, bf16,
// 95 us, 103 with four.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_bwd_sm100.cuh"  // unpack2
#include "kv_cache.cuh"

namespace gae {

struct PagedAttnParams {
    KvPool pool;
    PageTable table;
    const void *q;
    void *o;
    int64_t q_sb, q_sh, o_sb, o_sh;
    const int *lens;
    float *lse;           // [B, H], may be NULL
    float *scores;        // [B, Hkv, cap, H / Hkv] scaled by log2(e), with weights only
    const float *w_in;    // [B, Hkv, >= cap]
    float *w_out;
    int64_t wi_sb, wi_sh, wo_sb, wo_sh;
    int B, H, G, cap;     // G = H / Hkv, cap = max_pages * page_size
    int groups;           // rows of a key head: ceil(G / heads of a tile)
    int whole_rows;       // a block to a row, no join
    float scale_log2;
    // workspace
    int2 *parts;          // [rows] first and last block of the row
    float *lse2;          // [B, H] log2-sum-exp2 of rows that one block finished
    float *part_ml;       // [blocks][2][heads of a tile][2] maximum and sum
    float *part_o;        // [blocks][2][heads of a tile][D]
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool pred) {
    // src-size 0 writes zeros and reads nothing
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(pred ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <bool kBF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kBF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// How far a score may pass the maximum so far (log2) before the accumulator is
// rescaled.
constexpr float kPaSlack = 8.f;

// 16 cached rows against up to NT * 8 query heads on the tensor cores, keys as
// the rows of the product (S^T = K Q^T, O^T = V^T P): the 8 columns of an
// m16n8k16 are then query heads, of which a key head rarely has more, where
// heads as rows would pad them to 16 and double the products and the
// accumulator.  mma.sync, not tcgen05: at one query per head the products are
// 1/20 of what even these reach while the cache's bytes take the whole time,
// and operands come from shared memory in the layout that cp.async can gather
// from pages of any size.
template <typename T, int DM, int NT>
struct PaMmaTile {
    static constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kHeads = NT * 8, kKeys = 16, kChunks = DM * 2 / 16;
    // f16 probabilities are held times 2^13, so that they end where f16 does: the
    // largest lies in [2^13, 2^15], and the steps of 2^-24 at f16's lower end are
    // 2^-37 of it (from 2^-24 of it on they would round to nothing: of 131072 keys,
    // 2^-24 as heavy as the heaviest each, that is 2^-7 of the output).
    static constexpr float kSlack = kBF16 ? kPaSlack : 2.f, kUp = kBF16 ? 0.f : 13.f;
    static constexpr int kWarpScratch = 0;
    using Elem = T;
    __device__ explicit PaMmaTile(const float *) {}
    uint32_t qf[NT][DM / 16][2];
    float o[NT][DM / 16][4], l[NT][2];
    float m[NT][2];  // the exponents' base: kUp below the maximum that it was last set by

    // Shared-memory byte offset of 16-byte chunk c of row r (ldmatrix reads 8
    // rows of one chunk: the swizzle puts them in different banks).
    static __device__ __forceinline__ uint32_t at(int r, int c) { return r * (DM * 2) + ((c ^ (r & 7)) << 4); }

    __device__ __forceinline__ void load_q(const T *q, int64_t q_sh, int heads, int D, int lane) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int h = n * 8 + (lane >> 2);
#pragma unroll
            for (int kk = 0; kk < DM / 16; ++kk)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = kk * 16 + e * 8 + (lane & 3) * 2;
                    qf[n][kk][e] =
                        (h < heads && d < D) ? __ldg(reinterpret_cast<const unsigned *>(q + h * q_sh + d)) : 0u;
                }
        }
    }

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.f;
#pragma unroll
            for (int dd = 0; dd < DM / 16; ++dd)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][dd][e] = 0.f;
        }
    }

    // `valid`: bit r set where row r holds a key.  scores: this tile's first
    // row, G apart from row to row, or NULL.
    __device__ __forceinline__ void step(uint32_t sk, uint32_t sv, uint32_t valid, float scale_log2, int lane,
                                         float *scores, int G, int heads, float *) {
        float s[2][NT][4] = {};  // even and odd products apart: two chains
#pragma unroll
        for (int kk = 0; kk < DM / 16; ++kk) {
            uint32_t a[4];
            ldmatrix_x4(sk + at(lane & 15, kk * 2 + (lane >> 4)), a);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<kBF16>(s[kk & 1][n], a, qf[n][kk][0], qf[n][kk][1]);
        }
        const int r = lane >> 2;
        const bool ok[2] = {((valid >> r) & 1u) != 0, ((valid >> (r + 8)) & 1u) != 0};
        bool grow = false;
        float x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = (s[0][n][e] + s[1][n][e]) * scale_log2;
                if (scores && ok[e >> 1]) {
                    const int h = n * 8 + (lane & 3) * 2 + (e & 1);
                    if (h < heads) scores[(int64_t)(r + 8 * (e >> 1)) * G + h] = v;
                }
                x[n][e] = ok[e >> 1] ? v : -INFINITY;
                grow |= x[n][e] > m[n][e & 1] + (kUp + kSlack);
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mx = fmaxf(x[n][e], x[n][e + 2]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)) - kUp, m[n][e]);
                    const float alpha = m[n][e] == -INFINITY ? 0.f : ex2_approx(m[n][e] - mx);
                    m[n][e] = mx;
                    l[n][e] *= alpha;
#pragma unroll
                    for (int dd = 0; dd < DM / 16; ++dd) o[n][dd][e] *= alpha, o[n][dd][e + 2] *= alpha;
                }
        }
        uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // base 0 where no key had a finite score: -inf still maps to 0, NaN to NaN
                p[e] = ex2_approx(x[n][e] - (m[n][e & 1] == -INFINITY ? 0.f : m[n][e & 1]));
                l[n][e & 1] += p[e];
            }
            // P as the sum of two 16-bit numbers (17 bits): one would round every
            // probability by 2^-9 and cost as much precision as the output's own rounding.
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t w = kBF16 ? pack_bf16x2(p[2 * e], p[2 * e + 1]) : pack_f16x2(p[2 * e], p[2 * e + 1]);
                float f0, f1;
                unpack2<kBF16>(w, f0, f1);
                const uint32_t v = kBF16 ? pack_bf16x2(p[2 * e] - f0, p[2 * e + 1] - f1)
                                         : pack_f16x2(p[2 * e] - f0, p[2 * e + 1] - f1);
                hi[n][e] = movmatrix_trans(w);
                lo[n][e] = movmatrix_trans(v);
            }
        }
#pragma unroll
        for (int dd = 0; dd < DM / 16; ++dd) {
            uint32_t a[4];
            ldmatrix_x4_trans(sv + at((lane & 7) + ((lane >> 4) & 1) * 8, dd * 2 + ((lane >> 3) & 1)), a);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma_16816<kBF16>(o[n][dd], a, hi[n][0], hi[n][1]);
                mma_16816<kBF16>(o[n][dd], a, lo[n][0], lo[n][1]);
            }
        }
    }

    // O of this warp as fp32 [head][DM] (columns swizzled, see pa_swizzle), its
    // maximum and sum as ml[head][2].
    __device__ __forceinline__ void finish(float *so, float *ml, int lane) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float t = l[n][e];
                t += __shfl_xor_sync(0xffffffffu, t, 4);
                t += __shfl_xor_sync(0xffffffffu, t, 8);
                t += __shfl_xor_sync(0xffffffffu, t, 16);
                const int h = n * 8 + (lane & 3) * 2 + e;
                if (lane < 4) ml[2 * h] = m[n][e], ml[2 * h + 1] = t;
#pragma unroll
                for (int dd = 0; dd < DM / 16; ++dd)
#pragma unroll
                    for (int f = 0; f < 2; ++f)
                        so[h * DM + ((dd * 16 + f * 8 + (lane >> 2)) ^ (((h >> 1) & 3) << 3))] = o[n][dd][e + 2 * f];
            }
    }
};

// 8 cached fp32 rows against up to HG query heads on the CUDA cores, in fp32
// throughout: four lanes to a key for the scores, all lanes across head_dim for
// the products with V.
template <int DM, int HG>
struct PaFmaTile {
    static constexpr int kHeads = HG, kKeys = 8, kChunks = DM * 4 / 16;
    static constexpr int kWarpScratch = kKeys * HG;  // probabilities, floats
    static constexpr int kVec = DM / 32;             // columns of a lane
    using Elem = float;
    uint32_t q;  // [HG][DM] in shared memory
    uint64_t o[HG][kVec / 2];  // pairs of columns
    float m[HG], l[HG];
    __device__ explicit PaFmaTile(const float *q_smem) : q(smem_u32(q_smem)) {}

    // Eight lanes (two rows, four chunks) read 128 bytes at a time.
    static __device__ __forceinline__ uint32_t at(int r, int c) { return r * (DM * 4) + ((c ^ ((r & 1) << 2)) << 4); }

    __device__ __forceinline__ void load_q(const float *, int64_t, int, int, int) {}

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.f;
#pragma unroll
            for (int j = 0; j < kVec / 2; ++j) o[g][j] = 0;
        }
    }

    // 16 bytes as two pairs for the packed arithmetic
    static __device__ __forceinline__ void lds_pairs(uint32_t a, uint64_t &lo, uint64_t &hi) {
        asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];" : "=l"(lo), "=l"(hi) : "r"(a) : "memory");
    }
    static __device__ __forceinline__ float sum2(uint64_t v) {
        float a, b;
        f2_unpack(v, a, b);
        return a + b;
    }

    __device__ __forceinline__ void step(uint32_t sk, uint32_t sv, uint32_t valid, float scale_log2, int lane,
                                         float *scores, int G, int heads, float *sp) {
        const int r = lane >> 2, quarter = lane & 3;
        float s[HG];
        {
            uint64_t acc[HG] = {};
#pragma unroll
            for (int i = 0; i < DM / 16; ++i) {
                uint64_t k0, k1;
                lds_pairs(sk + at(r, i * 4 + quarter), k0, k1);
#pragma unroll
                for (int g = 0; g < HG; ++g) {
                    uint64_t q0, q1;
                    lds_pairs(q + (g * DM + (i * 4 + quarter) * 4) * 4, q0, q1);
                    acc[g] = f2_fma(k0, q0, acc[g]);
                    acc[g] = f2_fma(k1, q1, acc[g]);
                }
            }
#pragma unroll
            for (int g = 0; g < HG; ++g) s[g] = sum2(acc[g]);
        }
        const bool ok = ((valid >> r) & 1u) != 0;
        bool grow = false;
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            s[g] += __shfl_xor_sync(0xffffffffu, s[g], 1);
            s[g] += __shfl_xor_sync(0xffffffffu, s[g], 2);
            s[g] *= scale_log2;
            if (scores && ok && quarter == 0 && g < heads) scores[(int64_t)r * G + g] = s[g];
            if (!ok) s[g] = -INFINITY;
            grow |= s[g] > m[g] + kPaSlack;
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                float mx = fmaxf(s[g], __shfl_xor_sync(0xffffffffu, s[g], 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)), m[g]);
                const float alpha = m[g] == -INFINITY ? 0.f : ex2_approx(m[g] - mx);
                m[g] = mx;
                l[g] *= alpha;
#pragma unroll
                for (int j = 0; j < kVec / 2; ++j) o[g][j] = f2_mul(o[g][j], f2_pack(alpha, alpha));
            }
        }
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            const float p = ex2_approx(s[g] - (m[g] == -INFINITY ? 0.f : m[g]));
            l[g] += p;  // four lanes hold the same key: finish() takes one of them
            if (quarter == 0) sp[r * HG + g] = p;
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
            uint64_t v[kVec / 2];
            if constexpr (kVec == 2) {
                asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v[0]) : "r"(sv + at(k, lane >> 1) + (lane & 1) * 8) : "memory");
            } else {
#pragma unroll
                for (int j = 0; j < kVec / 4; ++j) lds_pairs(sv + at(k, j * 32 + lane), v[2 * j], v[2 * j + 1]);
            }
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                const float pg = sp[k * HG + g];
                const uint64_t p2 = f2_pack(pg, pg);
#pragma unroll
                for (int j = 0; j < kVec / 2; ++j) o[g][j] = f2_fma(p2, v[j], o[g][j]);
            }
        }
        __syncwarp();  // sp is rewritten by the next step
    }

    __device__ __forceinline__ void finish(float *so, float *ml, int lane) {
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            float t = l[g];
            t += __shfl_xor_sync(0xffffffffu, t, 4);
            t += __shfl_xor_sync(0xffffffffu, t, 8);
            t += __shfl_xor_sync(0xffffffffu, t, 16);
            if (lane == 0) ml[2 * g] = m[g], ml[2 * g + 1] = t;
#pragma unroll
            for (int j = 0; j < kVec / 2; ++j) {
                const int d = kVec == 2 ? lane * 2 : (j >> 1) * 128 + lane * 4 + (j & 1) * 2;
                *reinterpret_cast<uint64_t *>(so + g * DM + (d ^ (((g >> 1) & 3) << 3))) = o[g][j];
            }
        }
    }
};

template <class Tile, int DM>
struct PaCfg {
    static constexpr int kSlot = Tile::kKeys * DM * (int)sizeof(typename Tile::Elem) * 2;  // K and V rows of a warp
    // Two stages and as many warps as the shared memory feeds: three blocks of
    // four, or at head_dim 256 one of six.
    static constexpr int kWarps = DM == 256 ? 6 : 4, kThreads = kWarps * 32, kTileKeys = kWarps * Tile::kKeys;
    static constexpr int kStages = DM == 64 ? 4 : 2;
    static constexpr int kRing = kWarps * kStages * kSlot;
    static constexpr int kOffMl = kRing;                                   // [warps][heads][2]
    static constexpr int kOffQ = kOffMl + kWarps * Tile::kHeads * 8;     // fp32 tiles: q [heads][DM]
    static constexpr bool kQ = sizeof(typename Tile::Elem) == 4;
    static constexpr int kOffP = kOffQ + (kQ ? Tile::kHeads * DM * 4 : 0);  // fp32 tiles: probabilities
    static constexpr int kOffValid = kOffP + kWarps * Tile::kWarpScratch * 4;
    static constexpr int kOffScan = kOffValid + kWarps * kStages * 4;
    static constexpr int kSmem = (kOffScan + kWarps * 8 + 16 + 15) / 16 * 16;
    static constexpr int kPerSm = 3 * (kSmem + 1024) <= 228 * 1024 ? 3 : 2 * (kSmem + 1024) <= 228 * 1024 ? 2 : 1;
    // the merge reuses a stage: fp32 [heads][DM]
    static_assert(Tile::kHeads * DM * 4 <= kSlot, "a warp's O has to fit its stage");
    static_assert(kSmem <= 227 * 1024, "shared memory budget");
};

// Walks the tiles of all rows in order.
struct PaCursor {
    int b, r, tile, tiles, len;
};

template <class Tile, int DM>
__global__ void __launch_bounds__(PaCfg<Tile, DM>::kThreads, PaCfg<Tile, DM>::kPerSm)
    paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
    using Cfg = PaCfg<Tile, DM>;
    using T = typename Tile::Elem;
    constexpr int kKeys = Tile::kKeys, kWarps = Cfg::kWarps, kTileKeys = Cfg::kTileKeys, kThreads = Cfg::kThreads;
    extern __shared__ __align__(128) uint8_t smem_pa[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int R = p.pool.Hkv * p.groups;  // rows of a sequence
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    auto tiles_of = [&](int len) { return max(1, (len + kTileKeys - 1) / kTileKeys); };  // an empty row is a tile too

    // --- this block's run of tiles: [begin, end) of the total
    PaCursor ld, cp;
    int64_t total, blocks, begin, end;
    if (p.whole_rows) {  // few short rows: a block each, nothing to join
        ld.b = blockIdx.x / R;
        ld.r = blockIdx.x % R;
        ld.tile = 0;
        ld.len = clamp_len(__ldg(p.lens + ld.b), p.cap);
        ld.tiles = tiles_of(ld.len);
        total = end = ld.tiles;
        blocks = 1;
        begin = 0;
    } else {
        int64_t *scan = reinterpret_cast<int64_t *>(smem_pa + Cfg::kOffScan);  // [kWarps] warp sums
        int *found = reinterpret_cast<int *>(scan + kWarps);                   // b, r, tile
        const int per = (p.B + kThreads - 1) / kThreads;
        const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
        int64_t mine = 0;
        for (int b = b0; b < b1; ++b) mine += tiles_of(clamp_len(__ldg(p.lens + b), p.cap));
        mine *= R;
        int64_t incl = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += up;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        int64_t excl = incl - mine;
        total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) excl += scan[w];
            total += scan[w];
        }
        blocks = min64(gridDim.x, total);  // none of them without a tile
        if (blockIdx.x >= blocks) return;
        begin = total * blockIdx.x / blocks;
        end = total * (blockIdx.x + 1) / blocks;
        if (begin >= excl && begin < excl + mine) {
            int64_t at = excl;
            for (int b = b0; b < b1; ++b) {
                const int t = tiles_of(clamp_len(__ldg(p.lens + b), p.cap));
                if (begin < at + (int64_t)t * R) {
                    found[0] = b;
                    found[1] = (int)((begin - at) / t);
                    found[2] = (int)((begin - at) % t);
                    break;
                }
                at += (int64_t)t * R;
            }
        }
        __syncthreads();
        ld.b = found[0];
        ld.r = found[1];
        ld.tile = found[2];
        ld.len = clamp_len(__ldg(p.lens + ld.b), p.cap);
        ld.tiles = tiles_of(ld.len);
    }
    cp = ld;
    int64_t row_begin = begin - cp.tile;  // first tile of the current row, in the total

    // --- loader: pages are looked up one tile ahead of their copies
    const uint32_t ring = smem_u32(smem_pa) + warp * (Cfg::kStages * Cfg::kSlot);
    uint32_t *valid = reinterpret_cast<uint32_t *>(smem_pa + Cfg::kOffValid) + warp * Cfg::kStages;
    constexpr int kRowChunks = Tile::kChunks, kPasses = kKeys * kRowChunks / 32, kElems = 16 / (int)sizeof(T);
    constexpr int kRowsPerPass = 32 / kRowChunks > 0 ? 32 / kRowChunks : 1;
    const int live_chunks = p.pool.D / kElems;
    // Where a page holds whole warp tiles (its size a multiple of kKeys), the
    // rows of a tile share one page and lie at one stride; full rows of such a
    // tile need no predicate.
    const bool one_page = p.pool.page % kKeys == 0;
    const bool full_rows = live_chunks == kRowChunks;
    const int *ld_table = p.table.entry + ld.b * p.table.stride;
    const T *ld_k, *ld_v;
    auto ld_head = [&] {
        const int hk = ld.r / p.groups;
        ld_k = static_cast<const T *>(p.pool.k) + hk * p.pool.k_sh;
        ld_v = static_cast<const T *>(p.pool.v) + hk * p.pool.v_sh;
    };
    ld_head();
    int next_page = -1, next_slot = 0, next_rows = 0;
    auto look_up = [&] {  // the tile at ld
        const int pos0 = ld.tile * kTileKeys + warp * kKeys;
        const int pos = one_page ? pos0 : pos0 + (lane & (kKeys - 1));
        next_page = -1;
        next_rows = min(kKeys, ld.len - pos0);
        if (pos < ld.len) {
            const uint32_t idx = p.pool.by_page.div(pos);
            next_slot = pos - (int)idx * p.pool.page;
            next_page = __ldg(ld_table + idx);
            if ((int64_t)next_page >= p.pool.num_pages) next_page = -1;
        }
    };
    auto ld_advance = [&] {
        if (++ld.tile >= ld.tiles) {
            ld.tile = 0;
            if (++ld.r >= R) {
                ld.r = 0;
                ++ld.b;  // another tile is issued only where there is another sequence
                ld.len = 0;
                if (ld.b < p.B) {
                    ld.len = clamp_len(__ldg(p.lens + ld.b), p.cap);
                    ld.tiles = tiles_of(ld.len);
                    ld_table = p.table.entry + ld.b * p.table.stride;
                }
            }
            ld_head();
        }
        look_up();
    };
    auto load = [&](int stage) {  // the rows that look_up found
        const uint32_t sk = ring + stage * Cfg::kSlot, sv = sk + Cfg::kSlot / 2;
        if (one_page) {
            const int rows = next_page >= 0 ? max(next_rows, 0) : 0;
            if (lane == 0) valid[stage] = (1u << rows) - 1u;
            if (rows == 0) return;
            // Pass i: row row0 + i * kRowsPerPass, or half a row where it has 64 pieces.
            constexpr int kHalves = kRowChunks > 32 ? kRowChunks / 32 : 1;
            const int row0 = lane / kRowChunks, c0 = lane % kRowChunks;
            const T *ks = ld_k + next_page * p.pool.k_sp + (next_slot + row0) * p.pool.k_ss + c0 * kElems;
            const T *vs = ld_v + next_page * p.pool.v_sp + (next_slot + row0) * p.pool.v_ss + c0 * kElems;
            const int64_t kst = kRowsPerPass * p.pool.k_ss, vst = kRowsPerPass * p.pool.v_ss;
            if (rows == kKeys && full_rows) {
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    const int r = row0 + i / kHalves * kRowsPerPass, half = i % kHalves * 32;
                    cp_async16(sk + Tile::at(r, c0 + half), ks + half * kElems);
                    cp_async16(sv + Tile::at(r, c0 + half), vs + half * kElems);
                    if (i % kHalves == kHalves - 1) ks += kst, vs += vst;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    const int r = row0 + i / kHalves * kRowsPerPass, half = i % kHalves * 32;
                    const bool live = r < rows && c0 + half < live_chunks;
                    cp_async16(sk + Tile::at(r, c0 + half), live ? ks + half * kElems : ld_k, live);
                    cp_async16(sv + Tile::at(r, c0 + half), live ? vs + half * kElems : ld_v, live);
                    if (i % kHalves == kHalves - 1) ks += kst, vs += vst;
                }
            }
            return;
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, next_page >= 0 && lane < kKeys);
        if (lane == 0) valid[stage] = mask;
        if (mask == 0) return;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int row = (i * 32 + lane) / kRowChunks, c = (i * 32 + lane) % kRowChunks;
            const int pg = __shfl_sync(0xffffffffu, next_page, row), sl = __shfl_sync(0xffffffffu, next_slot, row);
            const bool live = pg >= 0 && c < live_chunks;
            const T *ks = ld_k, *vs = ld_v;
            if (live) {
                ks += pg * p.pool.k_sp + sl * p.pool.k_ss + c * kElems;
                vs += pg * p.pool.v_sp + sl * p.pool.v_ss + c * kElems;
            }
            cp_async16(sk + Tile::at(row, c), ks, live);
            cp_async16(sv + Tile::at(row, c), vs, live);
        }
    };

    const int n_tiles = (int)(end - begin);
    int issued = 0;
    look_up();
#pragma unroll
    for (int s = 0; s < Cfg::kStages - 1; ++s) {
        if (issued < n_tiles) {
            load(s);
            ++issued;
            ld_advance();
        }
        cp_async_commit();
    }

    float *q_smem = reinterpret_cast<float *>(smem_pa + Cfg::kOffQ);
    Tile tile(q_smem);
    float *sp = reinterpret_cast<float *>(smem_pa + Cfg::kOffP) + warp * Tile::kWarpScratch;
    int64_t row_start_tile = begin;  // where this block's part of the row starts
    // The row at cp: its key head, first query head, their number, q and scores.
    struct Row {
        int b, r, hk, h0, heads;
        const T *q;
        float *scores;
    } row;
    auto set_row = [&] {
        row.b = cp.b;
        row.r = cp.r;
        row.hk = cp.r / p.groups;
        row.h0 = (cp.r % p.groups) * Tile::kHeads;
        row.heads = min(Tile::kHeads, p.G - row.h0);
        row.q = static_cast<const T *>(p.q) + cp.b * p.q_sb + (int64_t)(row.hk * p.G + row.h0) * p.q_sh;
        row.scores =
            p.scores ? p.scores + ((int64_t)cp.b * p.pool.Hkv + row.hk) * p.cap * p.G + row.h0 : nullptr;
        tile.load_q(row.q, p.q_sh, row.heads, p.pool.D, lane);
    };
    auto stage_q = [&] {  // the fp32 tiles' q
        for (int i = tid; i < (Cfg::kQ ? Tile::kHeads * DM : 0); i += kThreads) {
            const int h = i / DM, d = i % DM;
            q_smem[i] = (h < row.heads && d < p.pool.D) ? to_f<T>(row.q[h * p.q_sh + d]) : 0.f;
        }
    };
    set_row();
    stage_q();
    tile.reset();
    if constexpr (Cfg::kQ) __syncthreads();
    int stage = 0;
    for (int it = 0; it < n_tiles; ++it) {
        cp_async_wait<Cfg::kStages - 2>();
        __syncwarp();
        // The stage before this one was read in the last turn: it is filled
        // first, so that all stages but this are on their way meanwhile.
        if (issued < n_tiles) {
            load(stage == 0 ? Cfg::kStages - 1 : stage - 1);
            ++issued;
            ld_advance();
        }
        cp_async_commit();
        const uint32_t sk = ring + stage * Cfg::kSlot;
        const uint32_t mask = valid[stage];
        if (mask != 0) {
            float *sc = row.scores ? row.scores + (int64_t)(cp.tile * kTileKeys + warp * kKeys) * p.G : nullptr;
            tile.step(sk, sk + Cfg::kSlot / 2, mask, p.scale_log2, lane, sc, p.G, row.heads, sp);
        }
        __syncwarp();
        const bool last = cp.tile + 1 == cp.tiles;
        if (last || it + 1 == n_tiles) {
            // --- the row's end here: the warps' parts become one.  The next
            // row's q is on its way meanwhile.
            const Row done = row;
            const int row_tiles = cp.tiles;
            cp.tile = -1;
            if (it + 1 < n_tiles) {
                if (++cp.r == R) {
                    cp.r = 0;
                    ++cp.b;
                    cp.len = clamp_len(__ldg(p.lens + cp.b), p.cap);
                    cp.tiles = tiles_of(cp.len);
                }
                set_row();
            }
            float *so = reinterpret_cast<float *>(smem_pa + warp * (Cfg::kStages * Cfg::kSlot) + stage * Cfg::kSlot);
            float *sml = reinterpret_cast<float *>(smem_pa + Cfg::kOffMl);
            tile.finish(so, sml + warp * Tile::kHeads * 2, lane);
            __syncthreads();
            if (it + 1 < n_tiles) stage_q();
            const bool first = row_start_tile == row_begin, whole = first && last;
            const int part = blockIdx.x * 2 + (first ? 1 : 0);
            if (first && tid == 0 && !p.whole_rows) {
                // the block that holds tile t of the total is floor(((t + 1) * blocks - 1) / total)
                const int64_t t = row_begin + row_tiles - 1;
                p.parts[done.b * R + done.r] = make_int2((int)blockIdx.x, (int)(((t + 1) * blocks - 1) / total));
            }
            for (int i = tid; i < done.heads * (DM / 4); i += kThreads) {
                const int h = i / (DM / 4), d = i % (DM / 4) * 4;
                float mw[kWarps], mx = -INFINITY, l = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    mw[w] = sml[(w * Tile::kHeads + h) * 2];
                    mx = fmaxf(mx, mw[w]);
                }
                const float base = mx == -INFINITY ? 0.f : mx;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float f = ex2_approx(mw[w] - base);
                    l += f * sml[(w * Tile::kHeads + h) * 2 + 1];
                    const float4 x = *reinterpret_cast<const float4 *>(
                        smem_pa + w * (Cfg::kStages * Cfg::kSlot) + stage * Cfg::kSlot +
                        (h * DM + (d ^ (((h >> 1) & 3) << 3))) * 4);
                    acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
                }
                if (d >= p.pool.D) continue;
                if (whole) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    T *o = static_cast<T *>(p.o) + done.b * p.o_sb + (int64_t)(done.hk * p.G + done.h0 + h) * p.o_sh + d;
                    if constexpr (sizeof(T) == 4) {
                        *reinterpret_cast<float4 *>(o) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                    } else {
                        alignas(8) T v[4] = {from_f<T>(acc.x * inv), from_f<T>(acc.y * inv), from_f<T>(acc.z * inv),
                                             from_f<T>(acc.w * inv)};
                        *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<const uint2 *>(v);
                    }
                    if (d == 0) {
                        const float l2 = l == 0.f ? -INFINITY : base + log2f(l);
                        const int64_t hh = (int64_t)done.b * p.H + done.hk * p.G + done.h0 + h;
                        p.lse2[hh] = l2;
                        if (p.lse) p.lse[hh] = l2 * kLn2;
                    }
                } else {
                    const int64_t at = (int64_t)part * Tile::kHeads + h;
                    *reinterpret_cast<float4 *>(p.part_o + at * p.pool.D + d) = acc;
                    if (d == 0) p.part_ml[at * 2] = mx, p.part_ml[at * 2 + 1] = l;
                }
            }
            __syncthreads();  // the stage may be loaded again
            tile.reset();
            row_begin += row_tiles;
            row_start_tile = row_begin;
        }
        ++cp.tile;
        stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;
    }
    cp_async_wait<0>();
}

// Joins the parts of rows that more than one block worked on: block (row, y), y
// < join_heads, joins head y; further blocks of the row's key head add up the
// keys' weights, kJoinKeys positions at a time (512 to 2048 measure alike).  The
// kernel is all latency: every thread reads its parts' statistics and sums side by
// side and scales as it goes, so that one trip to memory follows the row's entry
// in `parts`.
constexpr int kJoinThreads = 256, kJoinKeys = 1024;

// (m, l) and (m2, l2), sums relative to 2^m, become one; f and f2 scale what
// was summed beside them.
__device__ __forceinline__ void join_sums(float &m, float &l, float m2, float l2, float &f, float &f2) {
    const float mx = fmaxf(m, m2), base = mx == -INFINITY ? 0.f : mx;
    f = ex2_approx(m - base);
    f2 = ex2_approx(m2 - base);
    l = f * l + f2 * l2;
    m = mx;
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads)
    paged_attn_join_kernel(const __grid_constant__ PagedAttnParams p, int tile_heads, int join_heads) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int R = p.pool.Hkv * p.groups, row = blockIdx.x, b = row / R, r = row % R, D = p.pool.D;
    const int hk = r / p.groups, tid = threadIdx.x;
    auto part_at = [&](int2 ps, int i, int h) {  // the first block's part starts the row
        return ((int64_t)(ps.x + i) * 2 + (i == 0 ? 1 : 0)) * tile_heads + h;
    };
    const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml);
    if ((int)blockIdx.y < join_heads) {
        const int h = blockIdx.y, h0 = (r % p.groups) * tile_heads;
        if (h0 + h >= p.G) return;
        const int2 ps = p.parts[row];
        if (ps.x == ps.y) return;
        // float4 columns across threads, parts across what is left of them
        __shared__ float4 sum[kJoinThreads];
        __shared__ float2 stat[kJoinThreads];
        const int cols = D / 4, lanes = kJoinThreads / cols, c = tid % cols, lane0 = tid / cols;
        const int n = ps.y - ps.x + 1;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float m = -INFINITY, l = 0.f, f, f2;
        if (lane0 < lanes)
#pragma unroll 4
            for (int i = lane0; i < n; i += lanes) {
                const int64_t at = part_at(ps, i, h);
                const float2 s = ml[at];
                const float4 x = *reinterpret_cast<const float4 *>(p.part_o + at * D + c * 4);
                join_sums(m, l, s.x, s.y, f, f2);
                acc.x = f * acc.x + f2 * x.x, acc.y = f * acc.y + f2 * x.y;
                acc.z = f * acc.z + f2 * x.z, acc.w = f * acc.w + f2 * x.w;
            }
        sum[tid] = acc;
        if (c == 0 && lane0 < lanes) stat[lane0] = make_float2(m, l);
        __syncthreads();
        if (tid < cols) {
            for (int i = 1; i < min(lanes, n); ++i) {
                const float4 x = sum[i * cols + tid];
                join_sums(m, l, stat[i].x, stat[i].y, f, f2);
                acc.x = f * acc.x + f2 * x.x, acc.y = f * acc.y + f2 * x.y;
                acc.z = f * acc.z + f2 * x.z, acc.w = f * acc.w + f2 * x.w;
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            T *o = static_cast<T *>(p.o) + b * p.o_sb + (int64_t)(hk * p.G + h0 + h) * p.o_sh + tid * 4;
            o[0] = from_f<T>(acc.x * inv), o[1] = from_f<T>(acc.y * inv);
            o[2] = from_f<T>(acc.z * inv), o[3] = from_f<T>(acc.w * inv);
            if (tid == 0 && p.lse)
                p.lse[(int64_t)b * p.H + hk * p.G + h0 + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
        return;
    }
    // weights: once per key head, by its first row's blocks
    if (r % p.groups) return;
    const int len = clamp_len(__ldg(p.lens + b), p.cap);
    int first = ((int)blockIdx.y - join_heads) * kJoinKeys;
    if (first >= len) return;
    constexpr int kPer = kJoinKeys / kJoinThreads, kWarps = kJoinThreads / 32;
    __shared__ __align__(16) float lse2[kWarps * 2];
    const int warp = tid >> 5, lane = tid & 31;
    const float *scores = p.scores + ((int64_t)b * p.pool.Hkv + hk) * p.cap * p.G;
    for (; first < len; first += ((int)gridDim.y - join_heads) * kJoinKeys) {
        float was[kPer], w[kPer] = {};
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int pos = first + i * kJoinThreads + tid;
            was[i] = pos < len ? p.w_in[b * p.wi_sb + hk * p.wi_sh + pos] : 0.f;
        }
        for (int g0 = 0; g0 < p.G; g0 += kWarps * 2) {  // 16 heads' statistics at a time, two to a warp
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int g = g0 + warp + e * kWarps;
                if (g >= p.G) break;
                const int2 ps = p.parts[row + g / tile_heads];
                float l2;
                if (ps.x == ps.y) {
                    l2 = p.lse2[(int64_t)b * p.H + hk * p.G + g];
                } else {
                    float m = -INFINITY, l = 0.f, f, f2;
                    for (int i = lane; i <= ps.y - ps.x; i += 32) {
                        const float2 s = ml[part_at(ps, i, g % tile_heads)];
                        join_sums(m, l, s.x, s.y, f, f2);
                    }
                    float top = m;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    l *= ex2_approx(m - (top == -INFINITY ? 0.f : top));
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                    m = top;
                    l2 = l == 0.f ? -INFINITY : m + log2f(l);
                }
                // a row without a finite score has no weight to hand out
                if (lane == 0) lse2[warp + e * kWarps] = l2 == -INFINITY ? INFINITY : l2;
            }
            __syncthreads();
            const int many = min(p.G - g0, kWarps * 2);
            const float *s = scores + (int64_t)(first + tid) * p.G + g0;
            if (p.G % 4 == 0) {  // four heads of a position at a time
                for (int g = 0; g < many; g += 4) {
                    const float4 l4 = *reinterpret_cast<const float4 *>(lse2 + g);
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        if (first + i * kJoinThreads + tid < len) {
                            const float4 x = *reinterpret_cast<const float4 *>(s + (int64_t)i * kJoinThreads * p.G + g);
                            w[i] += (ex2_approx(x.x - l4.x) + ex2_approx(x.y - l4.y)) +
                                    (ex2_approx(x.z - l4.z) + ex2_approx(x.w - l4.w));
                        }
                }
            } else {
                for (int g = 0; g < many; ++g)
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        if (first + i * kJoinThreads + tid < len)
                            w[i] += ex2_approx(s[(int64_t)i * kJoinThreads * p.G + g] - lse2[g]);
            }
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int pos = first + i * kJoinThreads + tid;
            if (pos >= len || page_of(p.table, p.pool.num_pages, b, (int)p.pool.by_page.div(pos)) < 0) continue;
            p.w_out[b * p.wo_sb + hk * p.wo_sh + pos] = was[i] + w[i];
        }
    }
}

}  // namespace gae
