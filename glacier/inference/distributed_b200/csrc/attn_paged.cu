// attn_paged.cu -- causal attention with grouped heads over packed prompts and
// over a paged fp16 KV cache (a batch of sequences, each with its own number of
// new tokens), for the attention half of a stage that takes more than one token
// at a time (IClusterStageModel.ForwardBatchStage, IClusterStageModel.cs:24; the
// reference runs a batch's tokens one position after another).
//
// Query i of a sequence's n new tokens sees keys j <= kv_len - n + i:
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,  zero where no key is seen.
// Query head h reads KV head h / G (G = n_heads / n_kv_heads).
//
// Two kernels, by the rows a sequence brings to a KV head (its new tokens times
// their G heads): up to 16 take attn_rows_kernel, which lives by the bytes of K
// and V; more take attn_tiles_kernel on 128-row tensor-memory tiles.
//
// fp32 queries are carried as two fp16 halves after a power-of-two scale per
// row, and so are the exponentials (two products each, ~22 bits of q and p
// against the fp16 cache values); fp16 queries take one product.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>

#include "attn.cuh"

namespace glc {

namespace {

// Differs from call to call, and from what a workspace may hold by chance (2^-56).
unsigned long long next_nonce() {
    static std::atomic<unsigned long long> n{(unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count()};
    unsigned long long z = n.fetch_add(0x9E3779B97F4A7C15ull, std::memory_order_relaxed);
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;   // SplitMix64
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return ((z ^ (z >> 31)) & ~0xffull) | 0x100ull;
}

// Tokens of a row tile of the tile kernel, 128 rows.
constexpr int kRowTileTokens(int G) { return kTileRows / 2 / G; }

// Descriptor of fp16 queries as [2 halves][tokens][heads][64]: a box is a row tile's
// tokens times the heads of a KV head of one 64-element half, 128-byte swizzled.
int query_map(CUtensorMap* map, const AttnBatch& p) {
    const cuuint64_t dims[4] = {64, (cuuint64_t)p.n_heads, (cuuint64_t)p.T, 2};
    const cuuint64_t strides[3] = {kHd * 2, (cuuint64_t)p.q_stride * 2, 128};
    const cuuint32_t box[4] = {64, (cuuint32_t)p.G, (cuuint32_t)p.row_tile_tokens, 1};
    return paged_encode(map, p.q, 4, dims, strides, box);
}

// How a call runs, from what the host knows of it.
struct AttnPlan {
    bool rows, tiles;     // kernels that are launched
    bool split;           // units of the tile kernel may be cut
    int row_tiles;        // of a unit of the tile kernel
    long long items;      // most items of it
    int slots;            // and of their partials
    size_t work;          // workspace bytes
    size_t tile_work;     // where the partials of the tile kernel begin
};
AttnPlan plan_attention(int n_heads, int n_kv, int B, int T, int max_new, bool workspace) {
    const int G = n_heads / n_kv;
    AttnPlan a{};
    // A sequence of up to 16 rows a KV head is the row kernel's.  With longer ones
    // in the batch the row kernel comes first where there may be several short
    // ones; a batch of up to four is left to the tiles, where the short ones fill SMs
    // that would idle.  300 tokens at 2,000 keys (48 heads over 8, fp16) next to k
    // single ones at 4,000, both kernels against tiles alone: k = 1 64 against 72 us,
    // 3 74 against 64, 4 78 against 87, 16 107 against 140.
    a.tiles = (long long)max_new * G > kRows;
    a.rows = !a.tiles || (workspace && B > 4);
    const auto units_of = [&](int row_tiles) {   // at most
        return ((long long)T / (row_tiles * kRowTileTokens(G)) + std::min(B, T)) * n_kv;
    };
    // Two row tiles share a CTA's keys and hide each other's chain; packed prompts that
    // would leave half of the SMs without any take one a unit (40 heads over 8, fp32:
    // 33 tokens 14.8 against 17.0 us, 300 21.6 against 25.3; at 450, 208 units, 24.7
    // against 28.7, but at 600, 264 units, 36 against 32).  Over pages keys are cut
    // instead (300 tokens at 8,000 keys: 102 us as pairs in parts, 165 singly).
    a.row_tiles = !workspace && units_of(1) <= 148 ? 1 : 2;
    const long long units = units_of(a.row_tiles);
    // The kernel cuts up to kCutUnits units; the host, which does not know the lengths,
    // leaves the joining launch out where there may be many more.
    a.split = a.tiles && workspace && units <= 8 * kCutUnits;
    a.items = units + (a.split ? kTileExtra : 0);
    // (room for parts also where none are cut: a workspace serves every smaller call)
    a.slots = a.tiles && workspace ? (int)std::min<long long>(units * kTileParts, 2 * kTileExtra) : 0;
    a.tile_work = kRowsWorkBytes + ((size_t)(a.slots + 1) * kTileUnitBytes + 255) / 256 * 256;
    a.work = a.tile_work + (size_t)a.slots * kTilePartFloats * sizeof(float);
    return a;
}

int attn_launch(const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& ttk, const CUtensorMap& ttv, AttnBatch p,
                const AttnPlan& a, bool f32, cudaStream_t st) {
    p.nonce = next_nonce();
    p.rows_take = a.rows ? kRows : 0;
    p.split = a.split;
    p.slots = a.slots;
    p.tile_work = p.work ? p.work + a.tile_work / sizeof(float) : nullptr;
    if (a.rows) {
        p.tokens_per_tile = kRows / p.G;
        if (int rc = attn_rows_launch(f32, tk, tv, p, st)) return rc;
    }
    if (!a.tiles) return GLC_OK;
    p.row_tile_tokens = kRowTileTokens(p.G);
    p.tokens_per_tile = a.row_tiles * p.row_tile_tokens;
    // ceil(2^(31 + l) / d) with 2^(l - 1) < d <= 2^l: exact below 2^31 (d is 8 at least)
    int l = 1;
    while ((1 << l) < p.tokens_per_tile) ++l;
    p.unit_mul = (unsigned)(((1ull << (31 + l)) + p.tokens_per_tile - 1) / p.tokens_per_tile);
    p.unit_shift = l - 1;
    CUtensorMap tq = ttk;   // fp32 queries are not read through a descriptor
    if (!f32)
        if (int rc = query_map(&tq, p)) return rc;
    return attn_tiles_launch(f32, tq, ttk, ttv, p, a.items, st);
}

// What both attentions ask of their queries, outputs and heads.
int check_rows(const void* q, int q_type, int64_t q_stride, const void* out, int64_t out_stride, int n_heads, int n_kv,
               int head_dim, float scale, int B, int T) {
    if (head_dim != kHd) return paged_fail(GLC_ERR_UNSUPPORTED, "head_dim %d (only 128)", head_dim);
    if (q_type != GLC_GGUF_F32 && q_type != GLC_GGUF_F16)
        return paged_fail(GLC_ERR_UNSUPPORTED, "query type %d (GLC_GGUF_F32 or GLC_GGUF_F16)", q_type);
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || n_heads / n_kv > kRows || n_kv > 65535)
        return paged_fail(GLC_ERR_UNSUPPORTED, "%d heads over %d KV heads (a multiple, at most %d per KV head)", n_heads,
                          n_kv, kRows);
    if (B < 0 || T < 0) return paged_fail(GLC_ERR_INVALID_ARG, "%d sequences, %d rows", B, T);
    const int align = q_type == GLC_GGUF_F32 ? 4 : 8;
    if ((((uintptr_t)q | (uintptr_t)out) & 15u) || q_stride % align || out_stride % align)
        return paged_fail(GLC_ERR_INVALID_ARG, "query and output rows must be 16-byte aligned");
    if (q_stride < (int64_t)n_heads * kHd || out_stride < (int64_t)n_heads * kHd)
        return paged_fail(GLC_ERR_INVALID_ARG, "row strides shorter than a row");
    if (!(scale >= 0.f) || std::isinf(scale))
        return paged_fail(GLC_ERR_INVALID_ARG, "softmax scale must be finite and not negative");
    return GLC_OK;
}

AttnBatch make_batch(const void* q, int64_t q_stride, void* out, int64_t out_stride, const int32_t* cu, int B, int T,
                     int n_heads, int n_kv, float scale) {
    AttnBatch p{};
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.cu = cu;
    p.B = B;
    p.T = T;
    p.n_heads = n_heads;
    p.n_kv = n_kv;
    p.G = n_heads / n_kv;
    p.scale_log2 = (float)((scale > 0.f ? (double)scale : 1.0 / std::sqrt((double)kHd)) * 1.4426950408889634);
    return p;
}

}  // namespace

}  // namespace glc

using glc::paged_fail;

extern "C" int glc_attn_prompt_dev(const void* q, int32_t q_type, int64_t q_stride, const void* k, const void* v,
                                   int64_t kv_stride, const int32_t* cu_seqlens, int32_t B, int32_t T, int32_t n_heads,
                                   int32_t n_kv_heads, int32_t head_dim, float scale, void* out, int64_t out_stride,
                                   void* stream) {
    if (!q || !k || !v || !cu_seqlens || !out) return paged_fail(GLC_ERR_INVALID_ARG, "null pointer");
    if (int rc = glc::check_rows(q, q_type, q_stride, out, out_stride, n_heads, n_kv_heads, head_dim, scale, B, T))
        return rc;
    if ((((uintptr_t)k | (uintptr_t)v) & 15u) || (kv_stride & 7) || kv_stride < (int64_t)n_kv_heads * 128 ||
        kv_stride >= ((int64_t)1 << 38))
        return paged_fail(GLC_ERR_INVALID_ARG, "key and value rows must be 16-byte aligned and a row apart");
    if (B == 0 || T == 0) return GLC_OK;
    if (int rc = glc::paged_check_devices({{q, "q"}, {k, "k"}, {v, "v"}, {cu_seqlens, "cu_seqlens"}, {out, "out"}})) return rc;
    glc::AttnBatch p = glc::make_batch(q, q_stride, out, out_stride, cu_seqlens, B, T, n_heads, n_kv_heads, scale);
    if (int rc = glc::paged_error_word(&p.err)) return rc;
    p.box_rows = glc::kTile;  // the packed rows are one page of T rows
    CUtensorMap tk, tv;
    if (int rc = glc::paged_tensor_map(&tk, k, T, kv_stride, n_kv_heads, 128, 1, kv_stride, p.box_rows, 2)) return rc;
    if (int rc = glc::paged_tensor_map(&tv, v, T, kv_stride, n_kv_heads, 128, 1, kv_stride, p.box_rows, 2)) return rc;
    return glc::attn_launch(tk, tv, tk, tv, p, glc::plan_attention(n_heads, n_kv_heads, B, T, T, false),
                            q_type == GLC_GGUF_F32, (cudaStream_t)stream);
}

extern "C" int glc_attn_paged_workspace_bytes(int32_t n_heads, int32_t n_kv_heads, int32_t B, int32_t T,
                                              int32_t max_new, uint64_t* bytes) {
    if (!bytes) return paged_fail(GLC_ERR_INVALID_ARG, "null pointer");
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > glc::kRows || B < 0 || T < 0 ||
        max_new < 0)
        return paged_fail(GLC_ERR_INVALID_ARG, "bad attention shape (%d heads, %d KV heads, %d sequences, %d rows)",
                          n_heads, n_kv_heads, B, T);
    *bytes = glc::plan_attention(n_heads, n_kv_heads, B, T, max_new, true).work;
    return GLC_OK;
}

extern "C" int glc_attn_paged_dev(const void* q, int32_t q_type, int64_t q_stride, const glc_kv_pages* cache,
                                  const int32_t* block_table, int32_t max_pages, const int32_t* cu_new,
                                  const int32_t* kv_lens, int32_t B, int32_t T, int32_t max_new, int32_t n_heads,
                                  float scale, void* out, int64_t out_stride, void* workspace, uint64_t workspace_bytes,
                                  void* stream) {
    if (!q || !cache || !block_table || !cu_new || !kv_lens || !out || !workspace)
        return paged_fail(GLC_ERR_INVALID_ARG, "null pointer");
    if (int rc = glc::paged_check_pages(cache)) return rc;
    if (int rc = glc::check_rows(q, q_type, q_stride, out, out_stride, n_heads, cache->n_kv_heads, cache->head_dim,
                                 scale, B, T))
        return rc;
    // (the kernels round key counts up to whole tiles in 32 bits)
    if (max_pages <= 0 || max_new < 0 || (int64_t)max_pages * cache->page_size > 0x80000000ll - glc::kTile)
        return paged_fail(GLC_ERR_INVALID_ARG, "tables of %d pages, up to %d new tokens", max_pages, max_new);
    uint64_t need = 0;
    if (int rc = glc_attn_paged_workspace_bytes(n_heads, cache->n_kv_heads, B, T, max_new, &need)) return rc;
    if (((uintptr_t)workspace & 15u) || workspace_bytes < need)
        return paged_fail(GLC_ERR_INVALID_ARG, "workspace of %llu bytes is too small or not 16-byte aligned",
                          (unsigned long long)workspace_bytes);
    if (B == 0 || T == 0) return GLC_OK;
    if (int rc = glc::paged_check_devices({{q, "q"}, {cache->k, "the cache's k"}, {cache->v, "the cache's v"},
                                           {block_table, "block_table"}, {cu_new, "cu_new"}, {kv_lens, "kv_lens"},
                                           {out, "out"}, {workspace, "workspace"}}))
        return rc;
    glc::AttnBatch p = glc::make_batch(q, q_stride, out, out_stride, cu_new, B, T, n_heads, cache->n_kv_heads, scale);
    if (int rc = glc::paged_error_word(&p.err)) return rc;
    p.work = static_cast<float*>(workspace);
    p.kv_lens = kv_lens;
    p.table = block_table;
    p.max_pages = max_pages;
    p.max_new = max_new;
    p.n_pages = cache->n_pages;
    while ((1 << p.ps_log2) < cache->page_size) ++p.ps_log2;
    p.box_rows = std::min(cache->page_size, glc::kTile);
    const glc::AttnPlan a = glc::plan_attention(n_heads, cache->n_kv_heads, B, T, max_new, true);
    CUtensorMap tk{}, tv{}, ttk{}, ttv{};   // of the row kernel, of the tile kernel
    const auto map = [&](CUtensorMap* m, const void* base, int halves) {
        return glc::paged_tensor_map(m, base, cache->page_size, cache->row_stride, cache->n_kv_heads, cache->head_stride,
                                     cache->n_pages, cache->page_stride, p.box_rows, halves);
    };
    if (a.rows) {
        if (int rc = map(&tk, cache->k, 2)) return rc;
        if (int rc = map(&tv, cache->v, 2)) return rc;
    }
    // the tile kernel's K and V lie as two blocks of 64 dims: a box that covers part
    // of a tile's keys is one block's, one that covers them all takes both
    const int halves = p.box_rows < glc::kTile ? 1 : 2;
    if (a.tiles) {
        if (int rc = map(&ttk, cache->k, halves)) return rc;
        if (int rc = map(&ttv, cache->v, halves)) return rc;
    }
    return glc::attn_launch(tk, tv, ttk, ttv, p, a, q_type == GLC_GGUF_F32, (cudaStream_t)stream);
}
