// attn.cuh -- what the two kernels of the batched attention share: the batch, the
// page loads, the fp16 halves and the partials in the workspace.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.cuh"

namespace glc {

constexpr int kHd = 128;
constexpr int kTile = 128;                     // keys per tile
constexpr int kTileBytes = kTile * kHd * 2;    // K or V of a tile
constexpr int kRows = 16;                      // most query rows of a KV head in the row kernel
constexpr float kPShift = 10.f;                // exponentials are stored as 2^10 2^(s - m): see below

constexpr float kMinFactor = 1.2e-38f;         // a factor of zero would turn a masked -inf into NaN

// p = 2^(s - m) lies in [0, 1]; stored as 2^10 p its fp16 form (or the high one of two
// halves) stays normal down to 2^-24 of the row's largest weight.  The factor cancels in
// o / l.  Both kernels do so but for fp16 queries on tiles: there m may lag behind the
// row's maximum by 11 powers of two, so 2^4 p is stored, normal down to 2^-18 of the
// largest (see kShift16).  One fp16 weight is off by half a step, 2^-11: with the outputs'
// own rounding rows of fp16 queries come out 2.5e-4 to 2.8e-4 off (2-norm), 2.1e-4 of it
// from the outputs.

struct AttnBatch {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;   // elements between tokens
    const int32_t* cu;              // [B + 1] first row of each sequence
    const int32_t* kv_lens;         // [B]; null: packed keys, rows cu[b] .. cu[b + 1]
    const int32_t* table;           // [B][max_pages]
    int max_pages, ps_log2, n_pages, box_rows;
    int B, T, max_new, n_heads, n_kv, G, tokens_per_tile;
    int row_tile_tokens;            // tokens of a row tile of the tile kernel: one or two make a unit
    unsigned unit_mul;              // x / tokens_per_tile = (x * unit_mul >> 32) >> unit_shift, 0 <= x < 2^31
    int unit_shift;
    float scale_log2;               // softmax scale times log2(e)
    float* work;                    // partials of the row kernel, then of the tiles
    int rows_take;                  // most query rows of a KV head that the row kernel takes (0: not launched)
    int split;                      // whether the tile kernel may cut a unit's keys into parts
    int slots;                      // places of its partials
    float* tile_work;
    unsigned long long nonce;       // this call's mark in the workspace's counters (low 8 bits zero)
    int* err;
};

__device__ __forceinline__ void tma_load_kv(void* dst, const CUtensorMap* tm, int half, int row, int head, int page,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(tm), "r"(0), "r"(row), "r"(half), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// One instruction; the division's subroutine call costs the callers' registers.
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The fp16 high halves of a and b, and what is left of them
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack2(a - f.x, b - f.y);
}

// Power of two that takes a query row's largest value to [2^12, 2^13), where the
// low halves stay normal far below it, and the score factor that undoes it.
__device__ __forceinline__ void row_scale(float mx, float scale_log2, float& up, float& f) {
    const int x = (int)(__float_as_uint(mx) >> 23);    // biased exponent; zeros, infinities and NaN stay as they are
    const int e = x == 0 || x == 255 ? 0 : min(139 - x, 126);
    up = __uint_as_float((uint32_t)(127 + e) << 23);
    f = fmaxf(scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23), kMinFactor);
}

// Rows of sequence b, held inside [0, T] whatever cu holds.
__device__ __forceinline__ void seq_rows(const AttnBatch& p, int b, int& first, int& n) {
    first = min(max(p.cu[b], 0), p.T);
    n = min(max(p.cu[b + 1], first), p.T) - first;
}

// ---- partials in the workspace
// Units whose keys several CTAs share are joined by the last CTA to bring its
// partial (maximum, sum, unnormalised outputs), told by a counter: no CTA waits
// for another, and the order of arrival changes no result.  A counter starts from
// whatever the workspace holds: before it counts, a CTA sets a counter that does
// not carry this call's nonce to the nonce (compare and swap); the last one
// clears it, so a replayed graph starts over.
__device__ __forceinline__ void part_open(unsigned long long* n, unsigned long long nonce) {
    unsigned long long old = *reinterpret_cast<volatile unsigned long long*>(n);
    while ((old & ~0xffull) != nonce) {
        const unsigned long long seen = atomicCAS(n, old, nonce);
        if (seen == old) break;
        old = seen;
    }
}

constexpr int kRowCtas = 148;                  // CTAs of the row kernel
constexpr int kPartFloats = kRows * (kHd + 2); // a partial: outputs, then (maximum, sum) of each row
constexpr size_t kRowsWorkBytes =
    (size_t)kRowCtas * (2 * kPartFloats * sizeof(float) + sizeof(unsigned long long));

// Two outputs of a row, times inv (zeros where the row sees no key)
template <bool F32>
__device__ __forceinline__ void store_pair(void* out, int64_t off, float2 a, float inv, bool none) {
    if constexpr (F32)
        *reinterpret_cast<float2*>(static_cast<float*>(out) + off) =
            none ? make_float2(0.f, 0.f) : make_float2(a.x * inv, a.y * inv);
    else
        *reinterpret_cast<uint32_t*>(static_cast<__half*>(out) + off) = none ? 0u : pack2(a.x * inv, a.y * inv);
}

// ---- the kernels, and what a call needs of them
constexpr int kTileRows = 256;                  // query rows of an item of the tile kernel
constexpr int kTileParts = 8;                   // most parts of a unit's keys
// From two units an SM on, whole units of about the same length fill the SMs better than
// parts with their join: 192 units of 130 key tiles take 456 us cut and 565 whole, 312
// units of 65 take 490 cut and 430 whole (48 heads over 8, fp16 queries).  The rule counts
// units whatever their length, so one long chunk among many short sequences is not cut: 64
// fp32 tokens against 32,000 keys take 140 us alone, 202 next to 100 single tokens against
// 500 keys, 915 next to 300 of them and 817 next to 40 sequences of four tokens.
constexpr int kCutUnits = 2 * 148;
constexpr int kTileExtra = 3 * 148;             // most items that cutting units into parts adds
constexpr int kTilePartFloats = kTileRows * (kHd + 2);
constexpr int kTileUnitBytes = 32;              // a place's entry for the join
int attn_rows_launch(bool f32, const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p, cudaStream_t st);
// tq: the fp16 queries (unused with fp32 ones)
int attn_tiles_launch(bool f32, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p,
                      long long items, cudaStream_t st);

}  // namespace glc
