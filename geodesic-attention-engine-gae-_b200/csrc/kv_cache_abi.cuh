// kv_cache_abi.cuh -- the C ABI of the paged key-value cache and of the key
// weights: argument checks and launches.  Included by gae_abi.cu after its
// helpers (fail, set_smem, num_sms): one translation unit.
#pragma once
#include <initializer_list>

namespace {

int dtype_size(gae_dtype t) { return t == GAE_DTYPE_F32 ? 4 : t == GAE_DTYPE_BF16 || t == GAE_DTYPE_F16 ? 2 : 0; }

// Strides that keep every row on a 16-byte boundary; what stands for a
// dimension of one element is never used.
bool row_strides(const int64_t *s, std::initializer_list<int64_t> sizes, int esize) {
    for (int64_t n : sizes) {
        if (n > 1 && (*s < 0 || (*s * esize) % 16)) return false;
        ++s;
    }
    return true;
}

// Fits an int with room for one page more (positions are 32-bit, rows 64-bit).
constexpr int64_t kMaxPositions = 1ll << 30;

gae_status check_pool(const gae_kv_pool *pl, gae::KvPool *out) {
    if (!pl) return fail(GAE_ERR_INVALID_ARG, "pool is NULL");
    const int es = dtype_size(pl->dtype);
    if (!es) return fail(GAE_ERR_INVALID_ARG, "unknown dtype %d", (int)pl->dtype);
    if (pl->num_pages < 0 || pl->kv_heads < 1 || pl->page_size < 1 || pl->head_dim < 1)
        return fail(GAE_ERR_INVALID_ARG, "invalid pool shape [%lld, %lld, %lld, %lld]", (long long)pl->num_pages,
                    (long long)pl->kv_heads, (long long)pl->page_size, (long long)pl->head_dim);
    if (pl->num_pages > INT32_MAX || pl->kv_heads > 65535 || pl->page_size > kMaxPositions)
        return fail(GAE_ERR_UNSUPPORTED, "pool beyond 2^31 - 1 pages, 65535 heads or 2^30 rows to a page");
    if (pl->head_dim > 256 || (pl->head_dim * es) % 16)
        return fail(GAE_ERR_UNSUPPORTED, "the cache needs head_dim <= 256 in rows of a multiple of 16 bytes, got %lld",
                    (long long)pl->head_dim);
    if (pl->num_pages > 0 && (!pl->k || !pl->v)) return fail(GAE_ERR_INVALID_ARG, "pool pointers are NULL");
    if (!aligned16(pl->k) || !aligned16(pl->v)) return fail(GAE_ERR_INVALID_ARG, "pools must be 16-byte aligned");
    if (!row_strides(pl->k_stride, {pl->num_pages, pl->kv_heads, pl->page_size}, es) ||
        !row_strides(pl->v_stride, {pl->num_pages, pl->kv_heads, pl->page_size}, es))
        return fail(GAE_ERR_INVALID_ARG, "pool strides must be non-negative multiples of 16 bytes");
    out->k = pl->k; out->v = pl->v;
    out->k_sp = pl->k_stride[0]; out->k_sh = pl->k_stride[1]; out->k_ss = pl->k_stride[2];
    out->v_sp = pl->v_stride[0]; out->v_sh = pl->v_stride[1]; out->v_ss = pl->v_stride[2];
    out->num_pages = pl->num_pages;
    out->Hkv = (int)pl->kv_heads; out->page = (int)pl->page_size; out->D = (int)pl->head_dim;
    out->by_page = gae::FastDiv::of((uint32_t)pl->page_size);
    return GAE_OK;
}

gae_status check_table(const int32_t *entry, int64_t stride, int64_t max_pages, int64_t batch, int64_t page,
                       gae::PageTable *out) {
    if (max_pages < 0 || stride < 0) return fail(GAE_ERR_INVALID_ARG, "negative page table size or stride");
    if (max_pages > 0 && batch > 0 && !entry) return fail(GAE_ERR_INVALID_ARG, "page table is NULL");
    if (max_pages > kMaxPositions / page)
        return fail(GAE_ERR_UNSUPPORTED, "a page table of more than 2^30 positions");
    out->entry = entry; out->stride = stride; out->max_pages = (int)max_pages;
    return GAE_OK;
}

// Workspace of one paged attention call (bytes, each region 256-byte aligned).
struct PagedWs {
    size_t parts, lse2, ml, o, scores, total;
};
PagedWs paged_ws(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t cap, bool weights) {
    const size_t blocks = (size_t)num_sms() * 3, heads = H / Hkv <= 8 ? 8 : 16;  // most of either, any type
    PagedWs w;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t was = at;
        at += (n + 255) & ~(size_t)255;
        return was;
    };
    w.parts = take((size_t)B * H * sizeof(int2));
    w.lse2 = take((size_t)B * H * 4);
    w.ml = take(blocks * 2 * heads * 2 * 4);
    w.o = take(blocks * 2 * heads * D * 4);
    w.scores = take(weights ? (size_t)B * H * cap * 4 : 0);
    w.total = at;
    return w;
}

// How many CTAs share a pair of key tiles' queries: enough to fill the GPU (two
// CTAs to an SM) as long as each is left with 4 query tiles (1000 x 1000, 24
// heads x 64: 13.1 us replayed from a graph with 4, 13.2 with 2, 16.8 with 8 and
// thus one launch).  (Four times as many, so that a causal mask's long units end
// together, gained nothing: 178 against 180 us at 8192 x 8192, 16 heads.)
int key_weights_splits(int64_t B, int64_t H, int64_t Hkv, int64_t Nq, int64_t Nkv) {
    const int64_t units = B * Hkv * ((Nkv + 255) / 256), tiles = H / Hkv * ((Nq + 127) / 128);
    return (int)gae::max64(1, gae::min64((2 * num_sms() + units - 1) / units, tiles / 4));
}

template <int D, bool kBF16>
gae_status launch_key_weights(const gae::KeyWeightsParams &p, dim3 grid, cudaStream_t st) {
    using Cfg = gae::KeyWeightsCfg<D>;
    gae_status s = set_smem(gae::key_weights_kernel<D, kBF16>, Cfg::kSmem);
    if (s != GAE_OK) return s;
    gae::key_weights_kernel<D, kBF16><<<grid, Cfg::kThreads, Cfg::kSmem, st>>>(p);
    GAE_CUDA_TRY(cudaGetLastError());
    return GAE_OK;
}

// A launch that may begin while the one before it ends (it waits for it by griddepcontrol.wait).
template <typename... Params, typename... Args>
gae_status launch_after(void (*kern)(Params...), dim3 grid, int threads, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t c;
    memset(&c, 0, sizeof(c));
    c.gridDim = grid;
    c.blockDim = dim3((unsigned)threads);
    c.stream = st;
    cudaLaunchAttribute at;
    memset(&at, 0, sizeof(at));
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    GAE_CUDA_TRY(cudaLaunchKernelEx(&c, kern, args...));
    return GAE_OK;
}

template <class Tile, int DM>
gae_status launch_paged_attn(gae::PagedAttnParams p, cudaStream_t st) {
    using Cfg = gae::PaCfg<Tile, DM>;
    using T = typename Tile::Elem;
    gae_status s;
    if ((s = set_smem(gae::paged_attn_kernel<Tile, DM>, Cfg::kSmem)) != GAE_OK) return s;
    p.groups = (p.G + Tile::kHeads - 1) / Tile::kHeads;
    const int64_t rows = (int64_t)p.B * p.pool.Hkv * p.groups;
    constexpr int tile_keys = Cfg::kTileKeys;
    const int64_t most = rows * gae::max64(1, (p.cap + tile_keys - 1) / tile_keys);
    const int64_t slots = (int64_t)num_sms() * Cfg::kPerSm;
    // Rows of up to 6 tiles are left whole where each has a block at once: one
    // launch, no join.  5 tiles, 12 heads x 64: 5.8 against 6.1 us replayed from
    // a graph, 16.5 against 18.7 a call from Python; 8 tiles: 7.6 against 6.3.
    p.whole_rows = !p.scores && p.cap <= 6 * tile_keys && rows <= slots;
    const unsigned blocks = (unsigned)(p.whole_rows ? rows : gae::min64(most, slots));
    gae::paged_attn_kernel<Tile, DM><<<blocks, Cfg::kThreads, Cfg::kSmem, st>>>(p);
    GAE_CUDA_TRY(cudaGetLastError());
    if (p.whole_rows || (p.cap <= tile_keys && !p.scores)) return GAE_OK;  // nothing was split
    const int64_t chunks = p.scores ? gae::min64((p.cap + gae::kJoinKeys - 1) / gae::kJoinKeys, 32768) : 0;
    const int heads = p.G < Tile::kHeads ? p.G : Tile::kHeads;
    return launch_after(gae::paged_attn_join_kernel<T>, dim3((unsigned)rows, (unsigned)(heads + chunks)),
                        gae::kJoinThreads, st, p, (int)Tile::kHeads, heads);
}

template <int DM>
gae_status launch_paged_attn_d(const gae::PagedAttnParams &p, gae_dtype t, cudaStream_t st) {
    const bool few = p.G <= 8;
    if (t == GAE_DTYPE_F32)
        return p.G <= 2 ? launch_paged_attn<gae::PaFmaTile<DM, 2>, DM>(p, st) : launch_paged_attn<gae::PaFmaTile<DM, 8>, DM>(p, st);
    if (t == GAE_DTYPE_BF16)
        return few ? launch_paged_attn<gae::PaMmaTile<__nv_bfloat16, DM, 1>, DM>(p, st)
                   : launch_paged_attn<gae::PaMmaTile<__nv_bfloat16, DM, 2>, DM>(p, st);
    return few ? launch_paged_attn<gae::PaMmaTile<__half, DM, 1>, DM>(p, st)
               : launch_paged_attn<gae::PaMmaTile<__half, DM, 2>, DM>(p, st);
}

}  // namespace

extern "C" {

gae_status gae_paged_append(const gae_kv_pool *pool, const gae_paged_append_args *a, void *stream) {
    gae::AppendParams p;
    memset(&p, 0, sizeof(p));
    gae_status s;
    if ((s = check_pool(pool, &p.pool)) != GAE_OK) return s;
    if (!a) return fail(GAE_ERR_INVALID_ARG, "args is NULL");
    if (a->batch < 0 || a->tokens < 0) return fail(GAE_ERR_INVALID_ARG, "negative batch or tokens");
    if ((s = check_table(a->page_table, a->table_stride, a->max_pages, a->batch, pool->page_size, &p.table)) != GAE_OK)
        return s;
    if (a->batch == 0 || a->tokens == 0) return GAE_OK;
    const int es = dtype_size(pool->dtype);
    if (!a->k_new || !a->v_new || !a->start) return fail(GAE_ERR_INVALID_ARG, "NULL pointer in append arguments");
    if (!aligned16(a->k_new) || !aligned16(a->v_new) ||
        !row_strides(a->k_new_stride, {a->batch, pool->kv_heads, a->tokens}, es) ||
        !row_strides(a->v_new_stride, {a->batch, pool->kv_heads, a->tokens}, es))
        return fail(GAE_ERR_INVALID_ARG, "new rows must be 16-byte aligned, with non-negative strides of 16 bytes");
    if (a->batch > 65535) return fail(GAE_ERR_UNSUPPORTED, "batch > 65535");
    p.k_new = a->k_new; p.v_new = a->v_new;
    p.kn_sb = a->k_new_stride[0]; p.kn_sh = a->k_new_stride[1]; p.kn_st = a->k_new_stride[2];
    p.vn_sb = a->v_new_stride[0]; p.vn_sh = a->v_new_stride[1]; p.vn_st = a->v_new_stride[2];
    p.start = a->start; p.counts = a->counts;
    p.chunks = (int)(pool->head_dim * es / 16);
    if (a->tokens > kMaxPositions) return fail(GAE_ERR_UNSUPPORTED, "more than 2^30 new tokens");
    p.tokens = (int)a->tokens;
    p.by_chunks = gae::FastDiv::of((uint32_t)p.chunks);
    p.by_heads = gae::FastDiv::of((uint32_t)p.pool.Hkv);
    const int64_t pieces = a->tokens * p.chunks * pool->kv_heads, per_block = 256 * gae::kAppendRows;
    if (pieces > INT32_MAX - per_block) return fail(GAE_ERR_UNSUPPORTED, "more than 2^31 pieces of new rows to a sequence");
    const int64_t blocks = (pieces + per_block - 1) / per_block;
    const dim3 grid((unsigned)blocks, (unsigned)a->batch);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (es == 4) gae::paged_append_kernel<4><<<grid, 256, 0, st>>>(p);
    else gae::paged_append_kernel<2><<<grid, 256, 0, st>>>(p);
    GAE_CUDA_TRY(cudaGetLastError());
    return GAE_OK;
}

size_t gae_paged_attn_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                      int64_t capacity, int with_weights) {
    if (batch < 1 || heads < 1 || kv_heads < 1 || head_dim < 1 || capacity < 0 || batch > 65535 || heads > 65535 ||
        capacity > kMaxPositions || heads % kv_heads || head_dim > 256 || batch * heads > INT32_MAX)
        return 0;
    return paged_ws(batch, heads, kv_heads, head_dim, capacity, with_weights != 0).total;
}

gae_status gae_paged_attn_fwd(const gae_kv_pool *pool, const gae_paged_attn_args *a, void *stream) {
    gae::PagedAttnParams p;
    memset(&p, 0, sizeof(p));
    gae_status s;
    if ((s = check_pool(pool, &p.pool)) != GAE_OK) return s;
    if (!a) return fail(GAE_ERR_INVALID_ARG, "args is NULL");
    if (a->batch < 0 || a->heads < 1) return fail(GAE_ERR_INVALID_ARG, "invalid batch or heads");
    if (a->heads % pool->kv_heads) return fail(GAE_ERR_INVALID_ARG, "heads must be a multiple of kv_heads");
    if ((s = check_table(a->page_table, a->table_stride, a->max_pages, a->batch, pool->page_size, &p.table)) != GAE_OK)
        return s;
    if (a->batch == 0) return GAE_OK;
    if (a->batch > 65535 || a->heads > 65535 || a->batch * a->heads > INT32_MAX)
        return fail(GAE_ERR_UNSUPPORTED, "batch or heads > 65535, or more than 2^31 - 1 rows");
    const int es = dtype_size(pool->dtype);
    if (!a->q || !a->o || !a->seq_lens) return fail(GAE_ERR_INVALID_ARG, "NULL pointer in paged attention arguments");
    if (!aligned16(a->q) || !aligned16(a->o) || !row_strides(a->q_stride, {a->batch, a->heads}, es) ||
        !row_strides(a->o_stride, {a->batch, a->heads}, es))
        return fail(GAE_ERR_INVALID_ARG, "q and o must be 16-byte aligned, with non-negative strides of 16 bytes");
    if (!(a->scale >= 0.f)) return fail(GAE_ERR_UNSUPPORTED, "negative or NaN scale");
    if ((a->weights != nullptr) != (a->weights_out != nullptr))
        return fail(GAE_ERR_INVALID_ARG, "weights and weights_out go together");
    // Rows that lie on one another cannot be written.
    if ((a->batch > 1 && a->o_stride[0] == 0) || (a->heads > 1 && a->o_stride[1] == 0) ||
        (a->weights_out && ((a->batch > 1 && a->w_out_stride[0] == 0) || (pool->kv_heads > 1 && a->w_out_stride[1] == 0))))
        return fail(GAE_ERR_INVALID_ARG, "output stride of 0");
    if (a->weights_out && (a->w_stride[0] < 0 || a->w_stride[1] < 0 || a->w_out_stride[0] < 0 || a->w_out_stride[1] < 0))
        return fail(GAE_ERR_INVALID_ARG, "negative weights stride");
    const int64_t cap = a->max_pages * pool->page_size;
    if (a->weights_out && a->weights_len < cap)
        return fail(GAE_ERR_INVALID_ARG, "weights rows of %lld entries for %lld positions", (long long)a->weights_len,
                    (long long)cap);
    const size_t need =
        gae_paged_attn_workspace_bytes(a->batch, a->heads, pool->kv_heads, pool->head_dim, cap, a->weights_out != nullptr);
    if (!a->workspace || !aligned16(a->workspace))
        return fail(GAE_ERR_INVALID_ARG, "workspace is NULL or not 16-byte aligned");
    if (a->workspace_bytes < need)
        return fail(GAE_ERR_INVALID_ARG, "workspace too small: %zu < %zu", a->workspace_bytes, need);
    p.q = a->q; p.o = a->o; p.lse = a->lse; p.lens = a->seq_lens;
    p.q_sb = a->q_stride[0]; p.q_sh = a->q_stride[1]; p.o_sb = a->o_stride[0]; p.o_sh = a->o_stride[1];
    p.B = (int)a->batch; p.H = (int)a->heads; p.cap = (int)cap;
    p.G = p.H / p.pool.Hkv;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    const PagedWs w = paged_ws(a->batch, a->heads, pool->kv_heads, pool->head_dim, cap, a->weights_out != nullptr);
    char *ws = static_cast<char *>(a->workspace);
    p.parts = reinterpret_cast<int2 *>(ws + w.parts);
    p.lse2 = reinterpret_cast<float *>(ws + w.lse2);
    p.part_ml = reinterpret_cast<float *>(ws + w.ml);
    p.part_o = reinterpret_cast<float *>(ws + w.o);
    if (a->weights_out) {
        p.scores = reinterpret_cast<float *>(ws + w.scores);
        p.w_in = a->weights; p.w_out = a->weights_out;
        p.wi_sb = a->w_stride[0]; p.wi_sh = a->w_stride[1];
        p.wo_sb = a->w_out_stride[0]; p.wo_sh = a->w_out_stride[1];
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Narrower heads than the tile's are padded with zeros in shared memory only.
    if (pool->head_dim <= 64) return launch_paged_attn_d<64>(p, pool->dtype, st);
    if (pool->head_dim <= 128) return launch_paged_attn_d<128>(p, pool->dtype, st);
    return launch_paged_attn_d<256>(p, pool->dtype, st);
}

size_t gae_key_weights_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq_q, int64_t seq_kv) {
    if (batch < 1 || heads < 1 || kv_heads < 1 || seq_q < 1 || seq_kv < 1 || heads % kv_heads ||
        batch * heads > 65535 || seq_q > kMaxPositions || seq_kv > kMaxPositions)
        return 0;
    const int splits = key_weights_splits(batch, heads, kv_heads, seq_q, seq_kv);
    return splits == 1 ? 0 : (size_t)splits * batch * kv_heads * seq_kv * 4;
}

gae_status gae_key_weights(const gae_key_weights_args *a, void *stream) {
    if (!a) return fail(GAE_ERR_INVALID_ARG, "args is NULL");
    if (a->batch < 1 || a->heads < 1 || a->kv_heads < 1 || a->seq_q < 0 || a->seq_kv < 0 || a->head_dim < 1)
        return fail(GAE_ERR_INVALID_ARG, "invalid key weights shape");
    if (a->heads % a->kv_heads) return fail(GAE_ERR_INVALID_ARG, "heads must be a multiple of kv_heads");
    if (a->head_dim != 64 && a->head_dim != 128)
        return fail(GAE_ERR_UNSUPPORTED, "key weights support head_dim 64 or 128, got %lld", (long long)a->head_dim);
    if (a->dtype != GAE_DTYPE_BF16 && a->dtype != GAE_DTYPE_F16)
        return fail(GAE_ERR_UNSUPPORTED, "key weights support bf16 and f16");
    if (a->batch * a->heads > 65535) return fail(GAE_ERR_UNSUPPORTED, "batch*heads > 65535");
    if (a->seq_q > kMaxPositions || a->seq_kv > kMaxPositions)
        return fail(GAE_ERR_UNSUPPORTED, "sequence longer than 2^30");
    if (a->heads / a->kv_heads * ((a->seq_q + 127) / 128) > INT32_MAX)  // a CTA counts its query tiles in an int
        return fail(GAE_ERR_UNSUPPORTED, "more than 2^31 - 1 query tiles to a key head");
    if (!(a->scale >= 0.f)) return fail(GAE_ERR_UNSUPPORTED, "negative or NaN scale");
    if (a->seq_kv == 0) return GAE_OK;
    if (!a->out || (a->seq_q > 0 && (!a->q || !a->k || !a->lse)))
        return fail(GAE_ERR_INVALID_ARG, "NULL pointer in key weights arguments");
    if (!aligned16(a->q) || !aligned16(a->k) || !row_strides(a->q_stride, {a->batch, a->heads, a->seq_q}, 2) ||
        !row_strides(a->k_stride, {a->batch, a->kv_heads, a->seq_kv}, 2))
        return fail(GAE_ERR_INVALID_ARG, "q and k must be 16-byte aligned, with non-negative strides of 16 bytes");
    for (int i = 0; i < 2; ++i)
        if (a->lse_stride[i] < 0 || a->out_stride[i] < 0)
            return fail(GAE_ERR_INVALID_ARG, "negative lse or out stride");
    if ((a->batch > 1 && a->out_stride[0] == 0) || (a->kv_heads > 1 && a->out_stride[1] == 0))
        return fail(GAE_ERR_INVALID_ARG, "output stride of 0");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->seq_q == 0) {
        const int64_t n = a->batch * a->kv_heads * a->seq_kv, blocks = (n + 255) / 256;
        if (a->accumulate) return GAE_OK;
        if (blocks > INT32_MAX) return fail(GAE_ERR_UNSUPPORTED, "too many keys");
        gae::key_weights_zero_kernel<<<(unsigned)blocks, 256, 0, st>>>(a->out, a->out_stride[0], a->out_stride[1],
                                                                       (int)a->kv_heads, (int)a->seq_kv, n);
        GAE_CUDA_TRY(cudaGetLastError());
        return GAE_OK;
    }
    const size_t need = gae_key_weights_workspace_bytes(a->batch, a->heads, a->kv_heads, a->seq_q, a->seq_kv);
    if (a->workspace_bytes < need || (need && (!a->workspace || !aligned16(a->workspace))))
        return fail(GAE_ERR_INVALID_ARG, "workspace too small or not 16-byte aligned: %zu < %zu", a->workspace_bytes, need);
    gae::KeyWeightsParams p;
    memset(&p, 0, sizeof(p));
    gae_status s;
    const bool bf16 = a->dtype == GAE_DTYPE_BF16;
    const int64_t D = a->head_dim;
    const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    auto stride = [&](int64_t st, int64_t n) { return n > 1 ? st : D; };  // a map checks the unused ones too
    if ((s = make_map_4d(&p.tm_q, a->q, dt, 2, a->batch, a->heads, a->seq_q, D, stride(a->q_stride[0], a->batch),
                         stride(a->q_stride[1], a->heads), stride(a->q_stride[2], a->seq_q), 128)) != GAE_OK ||
        (s = make_map_4d(&p.tm_k, a->k, dt, 2, a->batch, a->kv_heads, a->seq_kv, D, stride(a->k_stride[0], a->batch),
                         stride(a->k_stride[1], a->kv_heads), stride(a->k_stride[2], a->seq_kv), 128)) != GAE_OK)
        return s;
    p.lse = a->lse;
    p.l_sb = a->lse_stride[0]; p.l_sh = a->lse_stride[1];
    p.o_sb = a->out_stride[0]; p.o_sh = a->out_stride[1];
    p.B = (int)a->batch; p.H = (int)a->heads; p.Hkv = (int)a->kv_heads;
    p.Nq = (int)a->seq_q; p.Nkv = (int)a->seq_kv;
    p.causal = a->causal ? 1 : 0;
    p.accumulate = a->accumulate ? 1 : 0;
    // Beyond the longest sequence all offsets mean the same.
    const __int128 off = (__int128)a->q_offset - a->kv_offset, most = 2 * (__int128)kMaxPositions;
    p.off = (int64_t)(off > most ? most : off < -most ? -most : off);
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.splits = key_weights_splits(a->batch, a->heads, a->kv_heads, a->seq_q, a->seq_kv);
    p.part = p.splits > 1 ? a->batch * a->kv_heads * a->seq_kv : 0;
    p.out = p.splits > 1 ? static_cast<float *>(a->workspace) : a->out;
    const int64_t units = a->batch * a->kv_heads * ((a->seq_kv + 255) / 256);
    if (units > INT32_MAX) return fail(GAE_ERR_UNSUPPORTED, "too many key tiles");
    const dim3 grid((unsigned)units, (unsigned)p.splits);
    if (D == 128) s = bf16 ? launch_key_weights<128, true>(p, grid, st) : launch_key_weights<128, false>(p, grid, st);
    else s = bf16 ? launch_key_weights<64, true>(p, grid, st) : launch_key_weights<64, false>(p, grid, st);
    if (s != GAE_OK || p.splits == 1) return s;
    const int64_t blocks = (p.part + 255) / 256;
    return launch_after(gae::key_weights_sum_kernel, dim3((unsigned)blocks), 256, st, (const float *)p.out, a->out, p.o_sb,
                        p.o_sh, p.Hkv, p.Nkv, p.part, p.splits, p.accumulate);
}

gae_status gae_paged_evict(const gae_kv_pool *pool, const gae_paged_evict_args *a, void *stream) {
    gae::EvictParams p;
    memset(&p, 0, sizeof(p));
    gae_status s;
    if ((s = check_pool(pool, &p.pool)) != GAE_OK) return s;
    if (!a) return fail(GAE_ERR_INVALID_ARG, "args is NULL");
    if (a->batch < 0) return fail(GAE_ERR_INVALID_ARG, "negative batch");
    if ((s = check_table(a->page_table, a->table_stride, a->max_pages, a->batch, pool->page_size, &p.src)) != GAE_OK ||
        (s = check_table(a->dst_table, a->dst_stride, a->dst_max_pages, a->batch, pool->page_size, &p.dst)) != GAE_OK)
        return s;
    if (a->keep < 1 || a->recent < 0 || a->recent > a->keep)
        return fail(GAE_ERR_INVALID_ARG, "eviction needs 1 <= keep and 0 <= recent <= keep, got %lld and %lld",
                    (long long)a->keep, (long long)a->recent);
    if (a->keep > a->dst_max_pages * pool->page_size)
        return fail(GAE_ERR_INVALID_ARG, "dst_table has room for %lld positions, keep is %lld",
                    (long long)(a->dst_max_pages * pool->page_size), (long long)a->keep);
    if (a->batch == 0) return GAE_OK;
    if (a->batch > 65535) return fail(GAE_ERR_UNSUPPORTED, "batch > 65535");
    if (!a->seq_lens || !a->new_lens || !a->kept || !a->kept_weights || (a->max_pages > 0 && a->weights_len > 0 && !a->weights))
        return fail(GAE_ERR_INVALID_ARG, "NULL pointer in eviction arguments");
    if (a->page_table == a->dst_table) return fail(GAE_ERR_INVALID_ARG, "dst_table must name other pages than page_table");
    if (a->new_lens == a->seq_lens || a->kept_weights == a->weights)
        return fail(GAE_ERR_INVALID_ARG, "eviction cannot write its lengths or weights over those it reads");
    if (a->w_stride[0] < 0 || a->w_stride[1] < 0 || a->weights_len < 0)
        return fail(GAE_ERR_INVALID_ARG, "negative weights stride or length");
    p.lens = a->seq_lens; p.w = a->weights;
    p.w_sb = a->w_stride[0]; p.w_sh = a->w_stride[1];
    p.keep = (int)a->keep; p.recent = (int)a->recent; p.cap = (int)gae::min64(a->max_pages * pool->page_size, a->weights_len);
    p.new_lens = a->new_lens; p.kept = a->kept; p.w_out = a->kept_weights;
    const int es = dtype_size(pool->dtype);
    p.chunks = (int)(pool->head_dim * es / 16);
    p.esize = es;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // As many CTAs to a row as the GPU has room for beside the other rows', each
    // with 4096 positions at least; more where a CTA could not hold its keys.
    const int64_t rows = a->batch * pool->kv_heads;
    int cluster = 1;
    while (cluster < gae::kEvictMaxCluster &&
           ((int64_t)cluster * gae::kEvictMaxKeys < p.cap ||
            ((int64_t)cluster * 4096 < p.cap && rows * cluster * 2 <= num_sms())))
        cluster *= 2;
    const int max_keys = (int)gae::min64(((p.cap + cluster - 1) / cluster + 3) / 4 * 4, gae::kEvictMaxKeys);
    if (rows * cluster > INT32_MAX) return fail(GAE_ERR_UNSUPPORTED, "too many rows");
    const int smem = (2 * gae::kEvictBins + max_keys) * 4;
    // The limit belongs to the kernel, not to this call: always the largest, so
    // that no other thread's call lowers it between here and the launch.
    if ((s = set_smem(gae::evict_select_kernel, (2 * gae::kEvictBins + gae::kEvictMaxKeys) * 4)) != GAE_OK) return s;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    cfg.blockDim = dim3(gae::kEvictThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    memset(&at, 0, sizeof(at));
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    // A row's own CTAs copy what it keeps where that is little to each; else
    // blocks of their own do.
    const int copy = a->keep * pool->head_dim * es * 2 / cluster <= (256 << 10);
    GAE_CUDA_TRY(cudaLaunchKernelEx(&cfg, gae::evict_select_kernel, (const gae::EvictParams)p, cluster, max_keys, copy));
    if (copy) return GAE_OK;
    const int64_t block_rows = 256 / p.chunks * gae::kGatherRows;
    const dim3 grid((unsigned)((a->keep + block_rows - 1) / block_rows + (a->keep + 1023) / 1024), (unsigned)pool->kv_heads,
                    (unsigned)a->batch);
    return launch_after(gae::evict_gather_kernel, grid, 256, st, p);
}

}  // extern "C"
