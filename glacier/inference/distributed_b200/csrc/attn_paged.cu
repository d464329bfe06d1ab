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
// attn_rows_kernel: up to 16 query rows of one KV head, so every K and V row is
// read once for all the heads that share it.  Eight warps take 16 of a tile's
// 128 keys each and keep their own running maximum, sum and output in registers
// (one pass, no exchange between warps until a unit's end, where the eight
// partials are joined in warp order); two more stream the pages with TMA
// into a ring of six 32 KB slots, one the keys, one the values.  Products run as mma.sync m16n8k16 with
// fp32 accumulators: 16 rows cannot fill a 128-row tensor-memory tile.
// fp32 queries are carried as two fp16 halves after a power-of-two scale per
// row, and so are the exponentials (two products each, ~22 bits of q and p
// against the fp16 cache values); fp16 queries take one product.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>

#include "common.cuh"
#include "paged.cuh"

namespace glc {

namespace {

constexpr int kHd = 128;
constexpr int kTile = 128;                     // keys per tile
constexpr int kTileBytes = kTile * kHd * 2;    // K or V of a tile
constexpr int kRowWarps = 8;
constexpr int kRowThreads = (kRowWarps + 2) * 32;
constexpr int kRows = 16;                      // query rows of a tile
constexpr float kPShift = 10.f;                // exponentials are stored as 2^10 e^(s - m): see below

constexpr float kMinFactor = 1.2e-38f;         // a factor of zero would turn a masked -inf into NaN

// p = 2^(s - m) lies in [0, 1]; stored as 2^10 p its fp16 form stays normal down
// to 2^-24 of the row's largest weight.  The factor cancels in o / l.

struct AttnBatch {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;   // elements between tokens
    const int32_t* cu;              // [B + 1] first row of each sequence
    const int32_t* kv_lens;         // [B]; null: packed keys, rows cu[b] .. cu[b + 1]
    const int32_t* table;           // [B][max_pages]
    int max_pages, ps_log2, n_pages, box_rows;
    int B, T, max_new, n_heads, n_kv, G, tokens_per_tile;
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

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// ------------------------------------------------------------ few rows (decode)
// A unit is one KV head of one sequence; its keys come in tiles of 128.  The
// tiles of all units, one unit after another, are cut into kRowCtas equal runs,
// one CTA each: every SM streams the same number of bytes whatever the lengths.
// A run holds whole units, which are finished in place, and at most two that it
// shares with its neighbours.  Their partials (maximum, sum, unnormalised output)
// go to the workspace, two places a CTA; the last CTA to bring its own, told by a
// counter per shared unit, joins them in key order.  No CTA waits for another,
// and the order of arrival changes no result.
// A counter starts from whatever the workspace holds: at its start every CTA that
// has a part of the unit sets a counter that does not carry this call's nonce to
// the nonce (compare and swap), and counts up only after that; the last one
// clears it, so a replayed graph starts over.
constexpr int kRowCtas = 148;
constexpr int kRowSlots = 6;                   // 32 KB each: K and V tiles in turn
constexpr int kUnitCache = 256;                // sequences whose lengths are kept in shared memory
constexpr int kPartFloats = kRows * (kHd + 2); // a partial: outputs, then (maximum, sum) of each row
constexpr size_t kRowsWorkBytes =
    (size_t)kRowCtas * (2 * kPartFloats * sizeof(float) + sizeof(unsigned long long));

struct RowsUnit {
    int first, n, kv_len, tiles;
};

struct RowsSmem {
    uint8_t ring[kRowSlots][kTileBytes];
    uint4 q[2][8][32];                         // A fragments of the unit's rows: high and low halves, 8 steps of 16 dims
    float o[kRowWarps][8][72];                 // joins the warps' outputs, 8 rows x 64 dims at a time (rows 8 banks apart)
    float m[kRowWarps][kRows], l[kRowWarps][kRows], qmax[kRowWarps][kRows];
    int first[kUnitCache], n[kUnitCache], kv[kUnitCache];
    uint64_t full[kRowSlots], empty[kRowSlots], opened;
    long long sums[kRowWarps], rest[kRowWarps];
    long long W, x0;                           // tiles in all, first tile of the CTA's run
    int b, g, tile, left;                      // where that is
    int last;
};

__device__ __forceinline__ RowsUnit load_unit(const AttnBatch& p, int b, bool record = false) {
    RowsUnit u;
    int len = 0;
    if (p.kv_lens) len = p.kv_lens[b];
    seq_rows(p, b, u.first, u.n);
    u.kv_len = u.n;
    if (p.kv_lens) {
        const long long room = (long long)p.max_pages << p.ps_log2;
        u.kv_len = (int)min((long long)max(len, 0), room);
        if (record && (len != u.kv_len || u.n > p.max_new)) atomicExch(p.err, kDevBadArg);
    }
    if (u.n * p.G > p.rows_take) u.n = 0;   // the tile kernel's
    u.tiles = u.n > 0 ? (u.kv_len + kTile - 1) / kTile : 0;
    return u;
}
__device__ __forceinline__ RowsUnit get_unit(const AttnBatch& p, const RowsSmem& S, int b) {
    if (p.B > kUnitCache) return load_unit(p, b);
    RowsUnit u;
    u.first = S.first[b];
    u.n = S.n[b];
    u.kv_len = S.kv[b];
    u.tiles = u.n > 0 ? (u.kv_len + kTile - 1) / kTile : 0;
    return u;
}

// A position in the flattened tiles, and how many are left of the CTA's run.
struct RowsWalk {
    int b, g, tile, left;
    __device__ __forceinline__ int end(const RowsUnit& u) const { return min(u.tiles, tile + left); }
    __device__ __forceinline__ void next(const AttnBatch& p, const RowsSmem& S, const RowsUnit& u) {
        left -= end(u) - tile;
        tile = 0;
        if (left > 0 && ++g == p.n_kv) {
            g = 0;
            do ++b;
            while (b + 1 < p.B && get_unit(p, S, b).tiles == 0);
        }
    }
};

// CTA that holds tile x of W: the last c with c * W / kRowCtas <= x.
__device__ __forceinline__ int rows_cta(long long x, long long W) {
    const long long n = (x + 1) * kRowCtas - 1;
    return W <= 0xffffffff / kRowCtas ? (int)((uint32_t)n / (uint32_t)W) : (int)(n / W);
}
__device__ __forceinline__ bool rows_cta_empty(int c, long long W) {
    return W * c / kRowCtas == W * (c + 1) / kRowCtas;
}
// Partials: place 2c for a unit that began before CTA c's run, 2c + 1 for one
// that goes on behind it.
__device__ __forceinline__ float* part_at(const AttnBatch& p, int place) { return p.work + (size_t)place * kPartFloats; }
// Counter of the unit whose first tile CTA c holds and whose last one it does not.
__device__ __forceinline__ unsigned long long* part_count(const AttnBatch& p, int c) {
    return reinterpret_cast<unsigned long long*>(p.work + (size_t)2 * kRowCtas * kPartFloats) + c;
}
__device__ __forceinline__ void part_open(unsigned long long* n, unsigned long long nonce) {
    unsigned long long old = *reinterpret_cast<volatile unsigned long long*>(n);
    while ((old & ~0xffull) != nonce) {
        const unsigned long long seen = atomicCAS(n, old, nonce);
        if (seen == old) break;
        old = seen;
    }
}

// Two outputs of a row, times inv (zeros where the row sees no key)
template <bool F32>
__device__ __forceinline__ void store_pair(void* out, int64_t off, float2 a, float inv, bool none) {
    if constexpr (F32)
        *reinterpret_cast<float2*>(static_cast<float*>(out) + off) =
            none ? make_float2(0.f, 0.f) : make_float2(a.x * inv, a.y * inv);
    else
        *reinterpret_cast<uint32_t*>(static_cast<__half*>(out) + off) = none ? 0u : pack2(a.x * inv, a.y * inv);
}

template <bool F32>
__global__ void __launch_bounds__(kRowThreads, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const __grid_constant__ AttnBatch p) {
    extern __shared__ uint8_t smem_raw[];
    RowsSmem& S = *reinterpret_cast<RowsSmem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kConsumers = kRowWarps * 32;

    if (threadIdx.x == kConsumers) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tv) : "memory");
        for (int i = 0; i < kRowSlots; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], kRowWarps);
        }
        mbar_init(&S.opened, 1);
        fence_mbar_init();
    }
    // where the CTA's run of tiles begins: sums over the sequences, 256 at a time
    if (warp < kRowWarps) {
        const int tid = threadIdx.x;
        RowsUnit u = tid < p.B ? load_unit(p, tid, blockIdx.x == 0) : RowsUnit{0, 0, 0, 0};
        if (p.B <= kUnitCache && tid < p.B) {
            S.first[tid] = u.first;
            S.n[tid] = u.n;
            S.kv[tid] = u.kv_len;
        }
        if (tid == 0) S.left = 0;
        long long rest = 0;   // tiles of the sequences behind the first 256
        for (int b = tid + kConsumers; b < p.B; b += kConsumers) rest += load_unit(p, b, blockIdx.x == 0).tiles;
        long long before = 0, W = 0, x0 = 0, x1 = 1;
        for (int b0 = 0; b0 < p.B && x1 > x0 && before * p.n_kv <= x0; b0 += kConsumers) {
            if (b0) u = b0 + tid < p.B ? load_unit(p, b0 + tid) : RowsUnit{0, 0, 0, 0};
            long long end = u.tiles;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const long long o = __shfl_up_sync(0xffffffffu, end, off);
                if (lane >= off) end += o;
            }
            if (b0) named_bar_sync(1, kConsumers);
            if (b0 == 0 && p.B > kConsumers) {
#pragma unroll
                for (int off = 16; off >= 1; off >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, off);
                if (lane == 0) S.rest[warp] = rest;
            }
            if (lane == 31) S.sums[warp] = end;
            named_bar_sync(1, kConsumers);
            long long all = 0;
            for (int x = 0; x < kRowWarps; ++x) {
                if (x == warp) end += all + before;
                all += S.sums[x];
            }
            if (b0 == 0) {
                W = all;
                if (p.B > kConsumers)
                    for (int x = 0; x < kRowWarps; ++x) W += S.rest[x];
                W *= p.n_kv;
                x0 = W * blockIdx.x / kRowCtas;
                x1 = W * (blockIdx.x + 1) / kRowCtas;
            }
            const long long in = x0 - (end - u.tiles) * p.n_kv;   // tiles into this thread's sequence
            if (x1 > x0 && in >= 0 && in < (long long)u.tiles * p.n_kv) {
                S.b = b0 + tid;
                S.g = (int)(in / u.tiles);
                S.tile = (int)(in - (long long)S.g * u.tiles);
                S.left = (int)min(x1 - x0, (long long)0x7fffffff);
                S.x0 = x0;
                S.W = W;
            }
            before += all;
        }
    }
    __syncthreads();
    RowsWalk w{S.b, S.g, S.tile, S.left};

    if (warp >= kRowWarps) {
        // ---------------------------------- page stream: keys, and values
        const int m = warp - kRowWarps;
        const CUtensorMap* tm = m ? &tv : &tk;
        const int nbox = kTile / p.box_rows, ps = 1 << p.ps_log2;
        bool ok = true;
        int it = m;
        while (w.left > 0 && ok) {
            const RowsUnit u = get_unit(p, S, w.b);
            const int end = w.end(u);
            for (int j = w.tile; j < end; ++j, it += 2) {
                const int r0 = j * kTile + lane * p.box_rows, st = it % kRowSlots;
                const bool mine = lane < nbox && r0 < u.kv_len;
                const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
                int page = 0, row = u.first + r0;
                if (mine && p.table) {
                    page = p.table[(long long)w.b * p.max_pages + (r0 >> p.ps_log2)];
                    row = r0 & (ps - 1);
                    if ((unsigned)page >= (unsigned)p.n_pages) {  // reads as zeros
                        atomicExch(p.err, kDevBadArg);
                        page = p.n_pages;
                    }
                }
                ok = mbar_wait(&S.empty[st], ((uint32_t)(it / kRowSlots) & 1u) ^ 1u, p.err, kDevTimeoutEmpty);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&S.full[st], (uint32_t)(boxes * p.box_rows * kHd * 2));
                __syncwarp();
                if (mine)
                    tma_load_kv(S.ring[st] + lane * p.box_rows * kHd * 2, tm, 0, row, w.g, page, &S.full[st]);
                __syncwarp();
                // the counters of the units this CTA shares (at most its first and its
                // last), once the first keys are on their way
                if (it == 0 && lane == 0) {
                    if (w.tile > 0 || w.left < u.tiles) part_open(part_count(p, rows_cta(S.x0 - w.tile, S.W)), p.nonce);
                    if (w.left > u.tiles - w.tile) part_open(part_count(p, blockIdx.x), p.nonce);   // (unused if whole)
                    mbar_arrive(&S.opened);
                }
                __syncwarp();
            }
            w.next(p, S, u);
        }
        // the tiles in flight land before the CTA can exit
        if (lane == 0)
            for (int i = it - kRowSlots < m ? m : it - kRowSlots; i < it; i += 2)
                mbar_wait(&S.full[i % kRowSlots], (uint32_t)(i / kRowSlots) & 1u, nullptr, 0);
        return;
    }

    // zero rows of sequences without keys: CTA b % kRowCtas sees to b
    for (int b = blockIdx.x; b < p.B; b += kRowCtas) {
        const RowsUnit u = get_unit(p, S, b);
        if (u.n > 0 && u.tiles == 0)
            for (int i = threadIdx.x; i < min(u.n, p.tokens_per_tile) * p.n_heads * (kHd / 2); i += kConsumers) {
                const int tok = i / (p.n_heads * (kHd / 2)), d = i - tok * p.n_heads * (kHd / 2);
                store_pair<F32>(p.out, (int64_t)(u.first + tok) * p.out_stride + 2 * d, make_float2(0.f, 0.f), 0.f, true);
            }
    }

    const int gr = lane >> 2, gc = lane & 3;
    // the warp's 16 keys of a tile: box and row inside the box are fixed
    const int k0 = 16 * warp, box_b = p.box_rows * kHd;  // bytes of a 64-element half of a box
    const uint32_t warp_off = (uint32_t)((k0 / p.box_rows) * box_b * 2 + (k0 % p.box_rows) * 128);
    // ldmatrix lane addresses (rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7))
    const int lr = (lane & 7) + ((lane >> 4) << 3), lc = (lane >> 3) & 1;          // K: matrices (keys 0-7, c), (keys 0-7, c + 1), (keys 8-15, ..)
    const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;          // V (transposed): (keys 0-7, c), (keys 8-15, c), (.., c + 1)
    long long x = S.x0;                            // flattened position
    bool ok = true;
    int it = 0;
    while (w.left > 0) {
        const RowsUnit u = get_unit(p, S, w.b);
        const int g = w.g, tile0 = w.tile, tile1 = w.end(u);
        const int ntok = min(u.n, p.tokens_per_tile), rows = ntok * p.G;
        const int see0 = u.kv_len - u.n + 1;           // keys the first token sees (may be <= 0)

        // ------------------------------------------------------------ queries
        // warp ks brings step ks of the A fragments: thread (gr, gc) holds rows
        // gr, gr + 8, columns 16 ks + 2 gc + {0, 1} and + 8
        float f[2];                                    // score factor: scale * log2(e) * the row's power of two
        int lim[2];                                    // keys seen by the thread's two rows
        {
            uint32_t hi[4], lo[4];
            float2 a[2][2];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int r = gr + 8 * hh, tok = r / p.G, h = r - tok * p.G;
                const bool live = r < rows;
                lim[hh] = live ? max(0, min(u.kv_len, see0 + tok)) : 0;
                f[hh] = p.scale_log2;
                const int64_t off =
                    (int64_t)(u.first + tok) * p.q_stride + (int64_t)(g * p.G + h) * kHd + 16 * warp + 2 * gc;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if constexpr (F32)
                        a[hh][c] = live ? __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + off + 8 * c))
                                        : make_float2(0.f, 0.f);
                    else
                        hi[2 * c + hh] = live ? __ldg(reinterpret_cast<const uint32_t*>(static_cast<const __half*>(p.q) +
                                                                                        off + 8 * c))
                                              : 0u;
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    float mx = fmaxf(fmaxf(fabsf(a[hh][0].x), fabsf(a[hh][0].y)), fmaxf(fabsf(a[hh][1].x), fabsf(a[hh][1].y)));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    if (gc == 0) S.qmax[warp][gr + 8 * hh] = mx;
                }
                named_bar_sync(1, kConsumers);
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    float mx = 0.f;
#pragma unroll
                    for (int i = 0; i < kRowWarps; ++i) mx = fmaxf(mx, S.qmax[i][gr + 8 * hh]);
                    float up;
                    row_scale(mx, p.scale_log2, up, f[hh]);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        split2(a[hh][c].x * up, a[hh][c].y * up, hi[2 * c + hh], lo[2 * c + hh]);
                }
                S.q[1][warp][lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            S.q[0][warp][lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            named_bar_sync(1, kConsumers);
        }

        const bool whole = tile0 == 0 && tile1 == u.tiles;
        int c0 = 0, c1 = 0, parts = 0;                 // CTAs that share the unit
        if (!whole) {
            c0 = rows_cta(x - tile0, S.W);
            c1 = rows_cta(x - tile0 + u.tiles - 1, S.W);
            for (int c = c0 + lane; c <= c1; c += 32) parts += !rows_cta_empty(c, S.W);
            parts = __reduce_add_sync(0xffffffffu, parts);
        }

        float o[16][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][e] = 0.f;

        for (int j = tile0; j < tile1 && ok; ++j, it += 2) {
            const int j0 = j * kTile + k0;             // first key of the warp's 16
            const bool any = j0 < u.kv_len;
            uint32_t ph[4], pl[4];
            // ------------------------------------------------ scores, weights
            int st = it % kRowSlots;
            ok = mbar_wait(&S.full[st], (uint32_t)(it / kRowSlots) & 1u, p.err, kDevTimeoutFull);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (any) {
                const uint32_t kb = smem_u32(S.ring[st]) + warp_off;
                float s[2][4], sl[2][4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][e] = sl[t][e] = 0.f;
#pragma unroll
                for (int kh = 0; kh < 2; ++kh) {       // the loads of four steps ahead of their products
                    uint32_t b[4][4];
                    uint4 q[4], r[4];
#pragma unroll
                    for (int k4 = 0; k4 < 4; ++k4) {
                        ldsm4(kb + kh * box_b + lr * 128 + (((2 * k4 + lc) ^ (lr & 7)) << 4), b[k4]);
                        q[k4] = S.q[0][4 * kh + k4][lane];
                        if constexpr (F32) r[k4] = S.q[1][4 * kh + k4][lane];
                    }
#pragma unroll
                    for (int k4 = 0; k4 < 4; ++k4) {
                        const uint32_t qa[4] = {q[k4].x, q[k4].y, q[k4].z, q[k4].w};
                        mma_f16(s[0], qa, b[k4][0], b[k4][1]);
                        mma_f16(s[1], qa, b[k4][2], b[k4][3]);
                        if constexpr (F32) {
                            const uint32_t ra[4] = {r[k4].x, r[k4].y, r[k4].z, r[k4].w};
                            mma_f16(sl[0], ra, b[k4][0], b[k4][1]);
                            mma_f16(sl[1], ra, b[k4][2], b[k4][3]);
                        }
                    }
                }
                if constexpr (F32) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[t][e] += sl[t][e];
                }
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int k = j0 + 8 * (e >> 1) + 2 * gc + (e & 1);
                        v[e] = k < lim[hh] ? s[e >> 1][2 * hh + (e & 1)] * f[hh] : -INFINITY;
                    }
                    float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float mn = fmaxf(m[hh], mx), mu = (mn == -INFINITY) ? 0.f : mn - kPShift;
                    if (mn > m[hh]) {
                        const float corr = ex2(m[hh] - mn);
                        l[hh] *= corr;
#pragma unroll
                        for (int t = 0; t < 16; ++t) {
                            o[t][2 * hh] *= corr;
                            o[t][2 * hh + 1] *= corr;
                        }
                        m[hh] = mn;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = ex2(v[e] - mu);
                    l[hh] += (v[0] + v[1]) + (v[2] + v[3]);
                    // P as an A fragment: register hh holds keys 2 gc, 2 gc + 1; register hh + 2 the same + 8
                    if constexpr (F32) {
                        split2(v[0], v[1], ph[hh], pl[hh]);
                        split2(v[2], v[3], ph[hh + 2], pl[hh + 2]);
                    } else {
                        ph[hh] = pack2(v[0], v[1]);
                        ph[hh + 2] = pack2(v[2], v[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.empty[st]);
            // -------------------------------------------------------- outputs
            st = (it + 1) % kRowSlots;
            ok = mbar_wait(&S.full[st], (uint32_t)((it + 1) / kRowSlots) & 1u, p.err, kDevTimeoutFull);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (any) {
                const uint32_t vb = smem_u32(S.ring[st]) + warp_off;
                // values past the last key may be anything, NaN included: they count as zeros
                const bool tail = j0 + 16 > u.kv_len;
                const int left = u.kv_len - j0 - 2 * gc;   // keys left from this thread's first
                const uint32_t k0m = (left > 0 ? 0xffffu : 0u) | (left > 1 ? 0xffff0000u : 0u);
                const uint32_t k1m = (left > 8 ? 0xffffu : 0u) | (left > 9 ? 0xffff0000u : 0u);
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    uint32_t b[4];
                    const int c = 2 * (t & 3) + vc;
                    ldsm4_t(vb + (t >> 2) * box_b + vr * 128 + ((c ^ (vr & 7)) << 4), b);
                    if (tail) {
                        b[0] &= k0m;
                        b[1] &= k1m;
                        b[2] &= k0m;
                        b[3] &= k1m;
                    }
                    if constexpr (F32) {
                        // the tensor core cuts its sums: the 16 keys' products are
                        // added to the running output by fp32 additions
                        float a0[4] = {0.f, 0.f, 0.f, 0.f}, a1[4] = {0.f, 0.f, 0.f, 0.f};
                        mma_f16(a0, pl, b[0], b[1]);
                        mma_f16(a1, pl, b[2], b[3]);
                        mma_f16(a0, ph, b[0], b[1]);
                        mma_f16(a1, ph, b[2], b[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[2 * t][e] += a0[e];
                            o[2 * t + 1][e] += a1[e];
                        }
                    } else {
                        mma_f16(o[2 * t], ph, b[0], b[1]);
                        mma_f16(o[2 * t + 1], ph, b[2], b[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.empty[st]);
        }

        // ------------------------------------- the warps' partials, in warp order
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 1);
            l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 2);
            if (gc == 0) {
                S.m[warp][gr + 8 * hh] = m[hh];
                S.l[warp][gr + 8 * hh] = l[hh];
            }
        }
        named_bar_sync(1, kConsumers);
        const int place = 2 * blockIdx.x + (tile0 > 0 ? 0 : 1);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            if (8 * hh >= rows) break;
            float M = -INFINITY;
#pragma unroll
            for (int i = 0; i < kRowWarps; ++i) M = fmaxf(M, S.m[i][gr + 8 * hh]);
            const float corr = m[hh] == -INFINITY ? 0.f : ex2(m[hh] - M);
            const int row = warp + 8 * hh;             // the thread's row when it joins
            float MR = -INFINITY, L = 0.f;
#pragma unroll
            for (int i = 0; i < kRowWarps; ++i) MR = fmaxf(MR, S.m[i][row]);
#pragma unroll
            for (int i = 0; i < kRowWarps; ++i) L += S.m[i][row] == -INFINITY ? 0.f : S.l[i][row] * ex2(S.m[i][row] - MR);
            const int tok = row / p.G;
            const bool none = max(0, min(u.kv_len, see0 + tok)) == 0;
            const float inv = none ? 0.f : rcp(L);
            const int64_t off = (int64_t)(u.first + tok) * p.out_stride + (int64_t)(g * p.G + row - tok * p.G) * kHd;
            if (!whole && row < rows && lane == 0)
                *reinterpret_cast<float2*>(part_at(p, place) + kRows * kHd + 2 * row) = make_float2(MR, L);
#pragma unroll
            for (int dh = 0; dh < 2; ++dh) {
#pragma unroll
                for (int t = 0; t < 8; ++t)
                    *reinterpret_cast<float2*>(&S.o[warp][gr][8 * t + 2 * gc]) =
                        make_float2(o[8 * dh + t][2 * hh] * corr, o[8 * dh + t][2 * hh + 1] * corr);
                named_bar_sync(1, kConsumers);
                float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < kRowWarps; ++i) {
                    const float2 y = *reinterpret_cast<const float2*>(&S.o[i][warp][2 * lane]);
                    acc.x += y.x;
                    acc.y += y.y;
                }
                if (row < rows) {
                    const int d = 64 * dh + 2 * lane;
                    if (whole) store_pair<F32>(p.out, off + d, acc, inv, none);
                    else *reinterpret_cast<float2*>(part_at(p, place) + row * kHd + d) = acc;
                }
                named_bar_sync(1, kConsumers);
            }
        }
        // --------------------------------------- a shared unit: the last one joins
        if (!whole) {
            // (the barrier above orders the CTA's stores before thread 0's release)
            if (threadIdx.x == 0) {
                ok = ok && mbar_wait(&S.opened, 0, p.err, kDevTimeoutFull);
                const bool last = ok && atom_add_acq_rel_gpu_u64(part_count(p, c0), 1ull) + 1 == p.nonce + parts;
                if (last) *part_count(p, c0) = 0;
                S.last = last;
            }
            named_bar_sync(1, kConsumers);
            if (S.last) {
#pragma unroll 1
                for (int row = warp; row < rows; row += kRowWarps) {
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    float M = -INFINITY, L = 0.f, k = 0.f;
#pragma unroll 1
                    for (int cb = c0; cb <= c1; cb += 32) {   // lane i: part cb + i
                        const int c = cb + lane;
                        const bool part = c <= c1 && !rows_cta_empty(c, S.W);
                        const unsigned have = __ballot_sync(0xffffffffu, part);
                        float2 ml = make_float2(-INFINITY, 0.f);
                        if (part)
                            ml = __ldcg(reinterpret_cast<const float2*>(part_at(p, 2 * c + (c == c0)) + kRows * kHd + 2 * row));
#pragma unroll 1
                        for (int i0 = 0; i0 < 32 && cb + i0 <= c1; i0 += 16) {   // sixteen parts' outputs at once
                            float4 y[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                                const int q = cb + i0 + i;
                                if (have >> (i0 + i) & 1u)
                                    y[i] = __ldcg(reinterpret_cast<const float4*>(part_at(p, 2 * q + (q == c0)) + row * kHd) +
                                                  lane);
                            }
                            if (i0 == 0) {   // the maximum so far and the parts' weights
                                float mn = fmaxf(M, ml.x);
#pragma unroll
                                for (int d = 16; d >= 1; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
                                const float old = M == -INFINITY ? 0.f : ex2(M - mn);
                                k = ml.x == -INFINITY ? 0.f : ex2(ml.x - mn);
                                L = fmaf(L, old, warp_sum(ml.y * k));
                                acc = make_float4(acc.x * old, acc.y * old, acc.z * old, acc.w * old);
                                M = mn;
                            }
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float ki = __shfl_sync(0xffffffffu, k, i0 + i);
                                acc.x = fmaf(y[i].x, ki, acc.x);
                                acc.y = fmaf(y[i].y, ki, acc.y);
                                acc.z = fmaf(y[i].z, ki, acc.z);
                                acc.w = fmaf(y[i].w, ki, acc.w);
                            }
                        }
                    }
                    const int tok = row / p.G;
                    const bool none = max(0, min(u.kv_len, see0 + tok)) == 0;
                    const float inv = none ? 0.f : rcp(L);
                    const int64_t off =
                        (int64_t)(u.first + tok) * p.out_stride + (int64_t)(g * p.G + row - tok * p.G) * kHd + 4 * lane;
                    store_pair<F32>(p.out, off, make_float2(acc.x, acc.y), inv, none);
                    store_pair<F32>(p.out, off + 2, make_float2(acc.z, acc.w), inv, none);
                }
            }
        }
        x += tile1 - tile0;
        w.next(p, S, u);
    }
}

// ------------------------------------------------- tensor-memory tiles (prompts)
// attn_tiles_kernel: 256 query rows of one KV head per CTA, as two row tiles A
// and B of 128 (floor(128 / G) tokens times their G heads) that share every K
// and V tile of 128 keys.  Per key tile and row tile:
//   S = Q K^T   tcgen05.mma, Q and K from shared memory, S in tensor memory;
//   P = 2^(S f - m)  one warpgroup per row tile, one row per thread: no
//               exchange between threads; P overwrites S in tensor memory;
//   PV          tcgen05.mma, P from tensor memory, V from shared memory, into a
//               tile of its own that the row's thread adds to its fp32 output
//               in registers: o = o 2^(m_old - m) + PV.
// While one row tile's warpgroup works on its softmax the tensor core runs the
// other's products.  Keeping o out of the tensor-memory accumulator costs a
// 128-column read per tile, and keeps the rounding of the sum over the keys
// that of fp32 additions: the tensor core's own accumulation cuts the sum at
// every 16 keys, which over 32,000 keys costs fp32 queries a decimal digit.
// fp32 queries: S and PV take two products each (halves of q and of p, low
// halves first).  Warps 0-7: softmax; warp 8: TMA; warps 9 and 10: MMA issue.
constexpr int kTcThreads = 12 * 32;
constexpr int kTcRows = 128;
constexpr uint32_t kTcCols = 512;        // S_A, S_B, PV_A, PV_B
constexpr int kMaxStages = 5;

// A CTA's work: 256 rows (tile) of a KV head of a sequence, and a part of its keys.
struct TileItem {
    int seq, tile, g, part, parts;   // parts: the most a unit of this sequence has
    int part_tiles;                  // key tiles of a part
    int slot;                        // workspace place of the unit's first part
};

struct TilesSmem {
    float f[2][kTcRows];                  // score factor of each row
    uint64_t kv_full[kMaxStages], kv_empty[kMaxStages], s_full[2], p_full[2][2], o_full[2], turn[2], q_full, v_clean,
        drain[2];
    uint32_t tmem;
    TileItem item;
    int found;
};

// Few units with many keys: a unit's key tiles are cut into up to kMaxParts parts
// of kMinPart tiles or more, one CTA each, whose partials (unnormalised outputs,
// maximum, sum) are joined through the workspace as in the row kernel.  At most
// kMaxExtra CTAs more than there are units, so twice as many places.
constexpr int kMaxParts = 8, kMinPart = 8, kMaxExtra = 3 * 148;
constexpr int kTilePartFloats = 2 * kTcRows * (kHd + 2);
__device__ __forceinline__ unsigned long long* tile_count(const AttnBatch& p, int slot) {
    return reinterpret_cast<unsigned long long*>(p.work + kRowsWorkBytes / sizeof(float)) + slot;
}

template <bool F32>
struct TilesLayout {
    static constexpr int kQBytes = 2 * (F32 ? 2 : 1) * kTileBytes;   // [row tile][half of q][2 x 64 dims][128 rows]
    static constexpr int kStages = F32 ? 3 : 5;
    static constexpr int kBytes = kQBytes + kStages * kTileBytes + (int)sizeof(TilesSmem) + 1024;
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_arrive(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// SWIZZLE_128B matrix descriptors, the low word only: start address and the
// leading offset; kDescHi holds 1024 bytes between groups of 8 rows (or keys),
// the version and the swizzle.  K-major (Q, K: 64 dims a row of 128 bytes) has
// no leading offset; MN-major (V: the dims run along a row, the keys down the
// rows) has 16 KB between its blocks of 64 dims.  The 64-bit descriptors are put
// together inside the instruction's block: kept as values, the issuing thread's
// 64 loop-invariant descriptors spilled to local memory (10x the kernel's time
// with 227 KB of shared memory, which leaves no first-level cache).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) {
    return ((addr >> 4) & 0x3FFFu) | (((uint32_t)(kTileBytes / 2) >> 4) << 16);
}
// D[tmem] (+)= A[smem] B[smem]^T and D[tmem] (+)= A[tmem] B[smem], fp16 operands, fp32 accumulators
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc),
        "r"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc),
        "r"(kDescHi)
        : "memory");
}
constexpr uint32_t kIdescS = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);   // f32 += f16 x f16, M = N = 128
constexpr uint32_t kIdescO = kIdescS | (1u << 16);                                     // B MN-major

#define TMEM_LD32(taddr, r)                                                                                        \
    asm volatile(                                                                                                  \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"         \
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"                                     \
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),           \
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),     \
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),   \
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])    \
        : "r"(taddr)                                                                                               \
        : "memory")
#define TMEM_LD16(taddr, r)                                                                                        \
    asm volatile(                                                                                                  \
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"     \
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),           \
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])      \
        : "r"(taddr)                                                                                               \
        : "memory")
#define TMEM_ST16(taddr, r)                                                                                        \
    asm volatile(                                                                                                  \
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"    \
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),       \
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])              \
        : "memory")
#define TMEM_ST8(taddr, r)                                                                                         \
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),  \
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])                        \
                 : "memory")
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Units and key tiles of sequence b.
__device__ __forceinline__ void seq_tiles(const AttnBatch& p, int b, int& units, int& tiles) {
    units = tiles = 0;
    if (b >= p.B || b < 0) return;
    int first, n;
    seq_rows(p, b, first, n);
    if (n * p.G <= p.rows_take) return;   // none, or the row kernel's
    units = (n + p.tokens_per_tile - 1) / p.tokens_per_tile * p.n_kv;
    const long long room = (long long)p.max_pages << p.ps_log2;
    const int len = p.kv_lens ? (int)min((long long)max(p.kv_lens[b], 0), room) : n;
    tiles = (len + kTile - 1) / kTile;
}

// The x-th item of the batch (called by one warp).  Sequences are taken from the
// batch's end and tiles from a sequence's end: the last ones see the most keys,
// so they start first and the short ones fill the gaps.
//
// With a workspace, keys are cut into parts of L tiles: of the longest sequence's
// tiles in 1 to 8 parts, the L with the least rounds of 148 CTAs times L, 3 % more
// for each further part's own prologue and join.
__device__ __forceinline__ bool find_item(const AttnBatch& p, int x, TileItem& item) {
    const int lane = threadIdx.x & 31;
    int L = 0x7fffffff;
    if (p.split) {
        int most = 0;
        for (int b0 = 0; b0 < p.B; b0 += 32) {
            int units, tiles;
            seq_tiles(p, b0 + lane, units, tiles);
            most = max(most, tiles);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        int len[kMaxParts], count[kMaxParts];
#pragma unroll
        for (int i = 0; i < kMaxParts; ++i) {
            len[i] = max(kMinPart, (most + i) / (i + 1));
            count[i] = 0;
        }
        if (most > kMinPart) {
            for (int b0 = 0; b0 < p.B; b0 += 32) {
                int units, tiles;
                seq_tiles(p, b0 + lane, units, tiles);
#pragma unroll
                for (int i = 0; i < kMaxParts; ++i) count[i] += units * max(1, (tiles + len[i] - 1) / len[i]);
            }
            float best = 3.4e38f;
            int units = 0;
#pragma unroll
            for (int i = 0; i < kMaxParts; ++i) {
                count[i] = __reduce_add_sync(0xffffffffu, count[i]);
                if (i == 0) units = count[0];
                const float cost = (float)((count[i] + 147) / 148) * (float)len[i] * (1.f + 0.03f * i);
                if (cost < best && count[i] - units <= kMaxExtra) {
                    best = cost;
                    L = len[i];
                }
            }
        }
    }
    int before = 0, slots = 0;
    for (int b0 = p.B - 1; b0 >= 0; b0 -= 32) {
        int units, tiles;
        seq_tiles(p, b0 - lane, units, tiles);
        const int parts = max(1, (tiles - 1) / L + 1), count = units * parts, split = parts > 1 ? count : 0;
        int end = count, send = split;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, end, off), q = __shfl_up_sync(0xffffffffu, send, off);
            if (lane >= off) {
                end += o;
                send += q;
            }
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + end > x);
        if (hit) {
            const int l = __ffs(hit) - 1;
            const int np = __shfl_sync(0xffffffffu, parts, l), nu = __shfl_sync(0xffffffffu, units, l);
            const int in = x - before - __shfl_sync(0xffffffffu, end - count, l);
            const int u = in / np;                            // unit of the sequence, from its end
            item.seq = b0 - l;
            item.part = in - u * np;
            item.parts = np;
            item.part_tiles = L;
            item.tile = nu / p.n_kv - 1 - u / p.n_kv;
            item.g = u % p.n_kv;
            item.slot = slots + __shfl_sync(0xffffffffu, send - split, l) + u * np;
            // first rows that do not ascend may name more units than the workspace has room for
            const bool room = np == 1 || item.slot + np <= p.slots;
            if (!room && lane == 0) atomicExch(p.err, kDevBadArg);
            return room;
        }
        before += __shfl_sync(0xffffffffu, end, 31);
        slots += __shfl_sync(0xffffffffu, send, 31);
    }
    return false;
}

// Pairs of fp32 values in one 64-bit register: half the issue slots of scalar
// arithmetic.  Volatile on purpose: the compiler otherwise sinks a chunk's
// arithmetic below the next chunk's tensor-memory load, keeps several chunks
// alive next to the row's 128 outputs, and spills.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 unpair(uint64_t a) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
    return d;
}
// o = o * c + (a, b)
__device__ __forceinline__ void fma_pair(uint64_t& o, uint64_t c, uint32_t a, uint32_t b) {
    asm volatile("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tfma.rn.f32x2 %0, %0, %3, t;\n\t}"
                 : "+l"(o)
                 : "r"(a), "r"(b), "l"(c));
}
__device__ __forceinline__ void mul_pair(uint32_t& a, uint32_t& b, uint64_t c) {
    asm volatile("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tmul.rn.f32x2 t, t, %2;\n\tmov.b64 {%0, %1}, t;\n\t}"
                 : "+r"(a), "+r"(b)
                 : "l"(c));
}
// 16 bytes of output: the pairs times c
__device__ __forceinline__ void store_f32(uint4* d, uint64_t a, uint64_t b, uint64_t c) {
    asm volatile(
        "{\n\t.reg .b64 t, u;\n\tmul.rn.f32x2 t, %1, %3;\n\tmul.rn.f32x2 u, %2, %3;\n\tst.global.v2.b64 [%0], {t, u};\n\t}" ::
            "l"(d),
        "l"(a), "l"(b), "l"(c)
        : "memory");
}
// 2^((a, b) * f - mu)
__device__ __forceinline__ void exp_pair(uint32_t a, uint32_t b, uint64_t f, uint64_t mu, float& x, float& y) {
    asm volatile(
        "{\n\t.reg .b64 t;\n\tmov.b64 t, {%2, %3};\n\tfma.rn.f32x2 t, t, %4, %5;\n\tmov.b64 {%0, %1}, t;\n\t"
        "ex2.approx.ftz.f32 %0, %0;\n\tex2.approx.ftz.f32 %1, %1;\n\t}"
        : "=f"(x), "=f"(y)
        : "r"(a), "r"(b), "l"(f), "l"(mu));
}
__device__ __forceinline__ void add_pair(uint64_t& s, float a, float b) {
    asm volatile("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;\n\t}" : "+l"(s) : "f"(a), "f"(b));
}
__device__ __forceinline__ void max3(float& m, uint32_t a, uint32_t b) {
    asm volatile("max.f32 %0, %0, %1, %2;" : "+f"(m) : "r"(a), "r"(b));
}

// 16 scores of a row: MASK takes keys at or past lim out
template <bool MASK>
__device__ __forceinline__ void mask16(uint32_t (&r)[16], int lim) {
    if (MASK) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e >= lim) r[e] = 0xff800000u;
    }
}
__device__ __forceinline__ void max16(const uint32_t (&r)[16], float& m0, float& m1) {
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        max3(m0, r[e], r[e + 1]);
        max3(m1, r[e + 2], r[e + 3]);
    }
}
// The weights of 16 scores over the scores' columns: 8 columns of high halves,
// then 8 of low halves
__device__ __forceinline__ void exp16(const uint32_t (&r)[16], uint32_t col, uint64_t f, uint64_t mu, uint64_t& s0,
                                      uint64_t& s1) {
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
        float a, b;
        exp_pair(r[e], r[e + 1], f, mu, a, b);
        add_pair((e & 2) ? s1 : s0, a, b);
        split2(a, b, hi[e >> 1], lo[e >> 1]);
    }
    TMEM_ST8(col, hi);
    TMEM_ST8(col + 8, lo);
}

// The two warpgroups take turns at the exponentials: one row tile's run while the
// other's products do.  Left alone the two fall into step, and the tensor core
// and the exponential unit wait for each other (4.2k cycles a key tile against
// 2.9k in turns, fp16 queries).  Warpgroup 0 starts; a turn is passed on before
// the last quarter of the exponentials.
struct Turn {
    uint64_t *mine, *other;   // null: this tile has no partner
    uint32_t phase;
    bool wait;
    int* err;
    __device__ __forceinline__ bool take() const {
        return !wait || mbar_wait(mine, phase, err, kDevTimeoutFull);
    }
    __device__ __forceinline__ void pass() const {
        if (other && (threadIdx.x & 31) == 0) mbar_arrive(other);
    }
};

// One arrival per warp: its rows' weights of 64 keys are in tensor memory.
__device__ __forceinline__ void weights_ready(uint64_t* bar) {
    tmem_wait_st();
    tc_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// fp32 queries: softmax of one row against one key tile.  Two passes over the
// scores in tensor memory (a row's 128 scores next to its 128 outputs would not
// fit the registers): the maximum, then the exponentials.  Both loop over 32
// scores as two loads of 16, the next in flight while one is worked on, and stay
// rolled: unrolled, all the loads move to the top and their values spill.  MASK:
// keys at or past lim count as -inf.  Returns the rescale of what came before.
template <bool MASK>
__device__ __forceinline__ float softmax_row(uint32_t trow, int lim, float f, float& m, float& l, uint64_t* p_full,
                                             const Turn& turn, bool& ok) {
    uint32_t a[16], b[16];
    float mx0 = -INFINITY, mx1 = -INFINITY;
    TMEM_LD16(trow, a);
    tmem_wait_ld();
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        TMEM_LD16(trow + 32 * c + 16, b);
        mask16<MASK>(a, lim - 32 * c);
        max16(a, mx0, mx1);
        tmem_wait_ld();
        TMEM_LD16(trow + ((32 * c + 32) & 127), a);   // after the last chunk: the first again, for the second pass
        mask16<MASK>(b, lim - 32 * c - 16);
        max16(b, mx0, mx1);
        tmem_wait_ld();
    }
    const float mn = fmaxf(m, fmaxf(mx0, mx1) * f);
    const float mu = mn == -INFINITY ? 0.f : mn - kPShift;
    const float corr = ex2(m - (mn == -INFINITY ? 0.f : mn));
    m = mn;
    const uint64_t f2 = pair(f, f), mu2 = pair(-mu, -mu);
    uint64_t s0 = 0, s1 = 0;
    ok = turn.take();
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        if (c == 3) turn.pass();
        TMEM_LD16(trow + 32 * c + 16, b);
        mask16<MASK>(a, lim - 32 * c);
        exp16(a, trow + 32 * c, f2, mu2, s0, s1);
        tmem_wait_ld();
        if (c < 3) TMEM_LD16(trow + 32 * c + 32, a);
        mask16<MASK>(b, lim - 32 * c - 16);
        exp16(b, trow + 32 * c + 16, f2, mu2, s0, s1);
        tmem_wait_ld();
        if (c & 1) weights_ready(p_full + (c >> 1));
    }
    const float2 u = unpair(s0), v = unpair(s1);
    l = fmaf(l, corr, (u.x + u.y) + (v.x + v.y));
    return corr;
}

// fp16 queries: the row's 128 scores in registers, its outputs in tensor memory.
// The maximum in use may lag the row's by kLazy before the outputs are rescaled
// (the weights then reach 2^(kPShift + kLazy), inside fp16): after the first
// tiles that hardly happens.
constexpr float kLazy = 5.f;
template <bool MASK>
__device__ __forceinline__ void softmax_row_f16(uint32_t trow, int lim, float f, bool first, float& m, float& l,
                                                uint64_t* p_full, const Turn& turn, bool& ok) {
    uint32_t s[kTile];
    TMEM_LD32(trow, s);
    TMEM_LD32(trow + 32, (s + 32));
    TMEM_LD32(trow + 64, (s + 64));
    TMEM_LD32(trow + 96, (s + 96));
    tmem_wait_ld();
    if (MASK) {
#pragma unroll
        for (int e = 0; e < kTile; ++e)
            if (e >= lim) s[e] = 0xff800000u;
    }
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < kTile; e += 2) max3(mx[(e >> 1) & 3], s[e], s[e + 1]);
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * f;
    if (__any_sync(0xffffffffu, top > m + kLazy)) {
        const float mn = fmaxf(m, top);
        const float corr = mn == -INFINITY ? 1.f : ex2(m - mn);
        m = mn;
        l *= corr;
        if (!first) {   // S of this tile is there, so the product before it is done
            const uint64_t corr2 = pair(corr, corr);
#pragma unroll 1
            for (int c = 0; c < kHd; c += 16) {
                uint32_t r[16];
                TMEM_LD16(trow + 256u + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e += 2) mul_pair(r[e], r[e + 1], corr2);
                TMEM_ST16(trow + 256u + c, r);
            }
        }
    }
    const float mu = m == -INFINITY ? 0.f : m - kPShift;
    const uint64_t f2 = pair(f, f), mu2 = pair(-mu, -mu);
    uint64_t s0 = 0, s1 = 0;
    ok = turn.take();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (c == 3) turn.pass();
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            float a, b;
            exp_pair(s[32 * c + e], s[32 * c + e + 1], f2, mu2, a, b);
            add_pair((e & 2) ? s1 : s0, a, b);
            w[e >> 1] = pack2(a, b);
        }
        TMEM_ST16(trow + 16 * c, w);
        if (c & 1) weights_ready(p_full + (c >> 1));
    }
    const float2 u = unpair(s0), v = unpair(s1);
    l += (u.x + u.y) + (v.x + v.y);
}

template <bool F32>
__global__ void __launch_bounds__(kTcThreads, 1)
    attn_tiles_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                      const __grid_constant__ AttnBatch p) {
    using L = TilesLayout<F32>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* qs = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint8_t* ring = qs + L::kQBytes;
    TilesSmem& S = *reinterpret_cast<TilesSmem*>(ring + L::kStages * kTileBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(&S.kv_full[i], 1);
            mbar_init(&S.kv_empty[i], 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&S.s_full[t], 1);
            mbar_init(&S.p_full[t][0], 4);
            mbar_init(&S.p_full[t][1], 4);
            mbar_init(&S.o_full[t], 1);
            mbar_init(&S.turn[t], 4);
        }
        mbar_init(&S.q_full, 8);
        mbar_init(&S.v_clean, 1);
        mbar_init(&S.drain[0], 1);
        mbar_init(&S.drain[1], 1);
        fence_mbar_init();
    }
    if (warp == 0) {
        TileItem item;
        const bool ok = find_item(p, blockIdx.x, item);
        if (lane == 0) {
            S.item = item;
            S.found = ok;
        }
    }
    __syncthreads();
    if (!S.found) return;
    const TileItem item = S.item;
    const int seq = item.seq, g = item.g, part = item.part;
    const int tpt = p.tokens_per_tile >> 1;   // tokens per row tile
    int first, n;
    seq_rows(p, seq, first, n);
    const int tok0 = item.tile * p.tokens_per_tile;
    int kv_len = n;
    if (p.kv_lens) {
        const long long room = (long long)p.max_pages << p.ps_log2;
        kv_len = p.kv_lens[seq];
        if ((kv_len < 0 || kv_len > room || n > p.max_new) && threadIdx.x == 0) atomicExch(p.err, kDevBadArg);
        kv_len = kv_len < 0 ? 0 : (kv_len > room ? (int)room : kv_len);
    }
    // row tile t: tokens [tok0 + t tpt, +ntok[t]), keys [0, end)
    int ntok[2], nt[2], kv_end = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        ntok[t] = max(0, min(tpt, n - tok0 - t * tpt));
        const int end = ntok[t] ? max(0, min(kv_len, kv_len - n + tok0 + t * tpt + ntok[t])) : 0;
        nt[t] = (end + kTile - 1) / kTile;
        kv_end = max(kv_end, end);
    }
    // this CTA's part of the key tiles, [j0, j1); a tile early in its sequence has fewer parts
    const int all_tiles = max(nt[0], nt[1]), parts = min(item.parts, max(1, (all_tiles - 1) / item.part_tiles + 1));
    if (part >= parts) return;
    const int j0 = (int)((long long)all_tiles * part / parts), j1 = (int)((long long)all_tiles * (part + 1) / parts);
    const int ntiles = j1 - j0;
#pragma unroll
    for (int t = 0; t < 2; ++t) nt[t] = max(0, min(nt[t], j1) - j0);   // of them, row tile t's

    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem)),
                     "r"(kTcCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = S.tmem;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == 11 && lane == 0 && parts > 1) {
            part_open(tile_count(p, item.slot), p.nonce);
        } else if (warp == 8) {
            // --------------------------------------------------- K and V tiles
            const int ps = 1 << p.ps_log2, nbox = kTile / p.box_rows, halves = nbox == 1 ? 1 : 2;
            const int box = lane / halves, half = lane - box * halves;
            bool ok = true;
            int it = 0;
            for (int j = 0; j < ntiles && ok; ++j) {
                const int r0 = (j0 + j) * kTile + box * p.box_rows;
                const bool mine = box < nbox && r0 < kv_end;
                const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
                const uint32_t bytes = (uint32_t)(boxes * p.box_rows * (nbox == 1 ? 256 : 128));
                int page = 0, row = first + r0;
                if (mine && p.table) {
                    page = p.table[(long long)seq * p.max_pages + (r0 >> p.ps_log2)];
                    row = r0 & (ps - 1);
                    if ((unsigned)page >= (unsigned)p.n_pages) {  // reads as zeros
                        atomicExch(p.err, kDevBadArg);
                        page = p.n_pages;
                    }
                }
#pragma unroll
                for (int m = 0; m < 2; ++m, ++it) {
                    const int st = it % L::kStages;
                    ok = mbar_wait_backoff(&S.kv_empty[st], ((uint32_t)(it / L::kStages) & 1u) ^ 1u, p.err,
                                           kDevTimeoutEmpty, 32);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&S.kv_full[st], bytes);
                    __syncwarp();
                    uint8_t* dst = ring + st * kTileBytes;
                    if (mine)
                        tma_load_kv(dst + half * (kTileBytes / 2) + box * p.box_rows * 128, m ? &tv : &tk, half, row, g,
                                    page, &S.kv_full[st]);
                    __syncwarp();
                    // values past the last key may be anything, NaN included: zeros
                    // before the tensor core reads them
                    if (m == 1 && j == ntiles - 1 && kv_end < (j0 + j + 1) * kTile) {
                        ok = mbar_wait(&S.kv_full[st], (uint32_t)(it / L::kStages) & 1u, p.err, kDevTimeoutFull);
                        for (int r = kv_end - (j0 + j) * kTile + (lane >> 3); r < kTile; r += 4)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                *reinterpret_cast<uint4*>(dst + h * (kTileBytes / 2) + r * 128 + (lane & 7) * 16) =
                                    make_uint4(0u, 0u, 0u, 0u);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&S.v_clean);
                    }
                }
            }
            if (lane == 0) drain_issued_stages(S.kv_full, L::kStages, it, kWaitLimitNs);
        } else if (warp <= 10 && lane == 0 && ntiles > 0) {
            // ------------------------------------------------------------- MMA
            // One issuer per row tile: an issuing thread's waits queue behind its
            // own products (~200 cycles each, measured), and the other issuer's
            // products run meanwhile.
            const int t = warp - 9;
            const uint32_t qb = desc_k(smem_u32(qs + t * (F32 ? 2 : 1) * kTileBytes));
            const uint32_t s_col = tmem + 128u * t, o_col = tmem + 256u + 128u * t;
            auto wait_kv = [&](int it) {
                return mbar_wait(&S.kv_full[it % L::kStages], (uint32_t)(it / L::kStages) & 1u, p.err, kDevTimeoutFull);
            };
            auto qk = [&](int it) {   // S = Q K^T
                const uint32_t kb = desc_k(smem_u32(ring + (it % L::kStages) * kTileBytes));
#pragma unroll
                for (int part = F32 ? 1 : 0; part >= 0; --part)
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t off = ((uint32_t)(ks >> 2) * (kTileBytes / 2) + (uint32_t)(ks & 3) * 32u) >> 4;
                        mma_ss(s_col, qb + (uint32_t)(part * (kTileBytes >> 4)) + off, kb + off, kIdescS,
                               (ks == 0 && part == (F32 ? 1 : 0)) ? 0u : 1u);
                    }
                tc_arrive(&S.s_full[t]);
            };
            auto pv = [&](int it, int half, bool fresh) {   // PV (+)= P V over 64 of the tile's keys
                const uint32_t vb = desc_mn(smem_u32(ring + (it % L::kStages) * kTileBytes)) + (uint32_t)half * (8192u >> 4);
#pragma unroll
                for (int part = F32 ? 1 : 0; part >= 0; --part)
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const uint32_t col = (uint32_t)(4 * half + ks) * (F32 ? 16u : 8u) + 8u * part;
                        mma_ts(o_col, s_col + col, vb + (uint32_t)ks * (2048u >> 4), kIdescO,
                               (fresh && ks == 0 && part == (F32 ? 1 : 0)) ? 0u : 1u);
                    }
            };
            const int mine = nt[t];
            bool ok = mbar_wait(&S.q_full, 0, p.err, kDevTimeoutFull) && wait_kv(0);
            tc_after();
            if (ok) {
                if (mine > 0) qk(0);
                tc_arrive(&S.kv_empty[0]);
            }
            for (int j = 0; j < ntiles && ok; ++j) {
                const int iv = 2 * j + 1, ik = 2 * j + 2;
                ok = wait_kv(iv);
                if (ok && j == ntiles - 1 && kv_end < j1 * kTile) ok = mbar_wait(&S.v_clean, 0, p.err, kDevTimeoutFull);
                // the next keys too, while the weights are on their way (fp16 queries; the
                // three slots of fp32 ones do not hold them yet)
                if (!F32 && ok && j + 1 < ntiles) ok = wait_kv(ik);
                if (j < mine) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        ok = ok && mbar_wait(&S.p_full[t][half], (uint32_t)j & 1u, p.err, kDevTimeoutFull);
                        if (!ok) break;
                        tc_after();
                        pv(iv, half, half == 0 && (F32 || j == 0));
                    }
                    if (ok && (F32 || j + 1 == mine)) tc_arrive(&S.o_full[t]);
                }
                if (!ok) break;
                if (F32) {
                    tc_arrive(&S.kv_empty[iv % L::kStages]);
                    if (j + 1 < ntiles && !wait_kv(ik)) break;
                }
                if (j + 1 < mine) qk(ik);
                if (!F32) tc_arrive(&S.kv_empty[iv % L::kStages]);
                if (j + 1 < ntiles) tc_arrive(&S.kv_empty[ik % L::kStages]);
            }
            // every product is done before the CTA frees its tensor memory
            tc_arrive(&S.drain[t]);
            mbar_wait(&S.drain[t], 0, nullptr, 0, kWaitLimitNs);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int t = warp >> 2, wrow = 32 * (warp & 3);
        const int rows = ntok[t] * p.G;
        // ------------------------------------------------------------- queries
        // a warp's 32 rows to shared memory, 64 dims a 128-byte swizzled row
        uint8_t* qt = qs + t * (F32 ? 2 : 1) * kTileBytes;
        const int64_t tok_first = first + tok0 + t * tpt;
        if constexpr (F32) {
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += 16) {
                float4 a[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = wrow + r0 + i, tok = r / p.G, h = r - tok * p.G;
                    a[i] = r < rows ? __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.q) +
                                                                            (tok_first + tok) * p.q_stride +
                                                                            (int64_t)(g * p.G + h) * kHd) +
                                            lane)
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = wrow + r0 + i;
                    float mx = fmaxf(fmaxf(fabsf(a[i].x), fabsf(a[i].y)), fmaxf(fabsf(a[i].z), fabsf(a[i].w)));
#pragma unroll
                    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                    float up, fr;
                    row_scale(mx, p.scale_log2, up, fr);
                    if (lane == 0) S.f[t][r] = fr;
                    uint2 hi, lo;
                    split2(a[i].x * up, a[i].y * up, hi.x, lo.x);
                    split2(a[i].z * up, a[i].w * up, hi.y, lo.y);
                    const int c = lane >> 1;
                    uint8_t* d = qt + (c >> 3) * (kTileBytes / 2) + r * 128 + (((c & 7) ^ (r & 7)) << 4) + (lane & 1) * 8;
                    *reinterpret_cast<uint2*>(d) = hi;
                    *reinterpret_cast<uint2*>(d + kTileBytes) = lo;
                }
            }
        } else {
            const int c = lane & 15;
            uint4 a[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = wrow + 2 * i + (lane >> 4), tok = r / p.G, h = r - tok * p.G;
                a[i] = make_uint4(0u, 0u, 0u, 0u);
                if (r < rows)
                    a[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(p.q) +
                                                                (tok_first + tok) * p.q_stride +
                                                                (int64_t)(g * p.G + h) * kHd) +
                                 c);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = wrow + 2 * i + (lane >> 4);
                *reinterpret_cast<uint4*>(qt + (c >> 3) * (kTileBytes / 2) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = a[i];
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.q_full);

        // ------------------------------------------------------------- softmax
        const int row = wrow + lane, tok = row / p.G;
        const bool live = row < rows;
        const int lim = live ? max(0, min(kv_len, kv_len - n + tok0 + t * tpt + tok + 1)) : 0;
        const int lim0 = max(0, kv_len - n + tok0 + t * tpt + 1);   // keys the tile's first row sees
        const float f = F32 ? S.f[t][row] : p.scale_log2;
        const uint32_t trow = tmem + 128u * t + ((uint32_t)wrow << 16);
        const int64_t out_off = (tok_first + tok) * p.out_stride + (int64_t)(g * p.G + row - tok * p.G) * kHd;
        float* part_out = p.tile_work + (size_t)(item.slot + part) * kTilePartFloats;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        const int both = min(nt[0], nt[1]);
        auto turn_of = [&](int j) {   // warpgroup 0 waits for 1's turn at the tile before, 1 for 0's at this one
            return Turn{&S.turn[t], j < both ? &S.turn[t ^ 1] : nullptr, (uint32_t)(j - 1 + t) & 1u,
                        j < both && j + t > 0, p.err};
        };
        if constexpr (F32) {
            uint64_t o[kHd / 2];   // the row's outputs in pairs
#pragma unroll
            for (int d = 0; d < kHd / 2; ++d) o[d] = 0;
            for (int j = 0; j < nt[t]; ++j) {
                const uint32_t ph = (uint32_t)j & 1u;
                ok = mbar_wait(&S.s_full[t], ph, p.err, kDevTimeoutFull);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_after();
                const Turn turn = turn_of(j);
                const float corr = (j0 + j + 1) * kTile > lim0
                                       ? softmax_row<true>(trow, lim - (j0 + j) * kTile, f, m, l, S.p_full[t], turn, ok)
                                       : softmax_row<false>(trow, 0, f, m, l, S.p_full[t], turn, ok);
                ok = ok && mbar_wait(&S.o_full[t], ph, p.err, kDevTimeoutFull);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_after();
                const uint64_t corr2 = pair(corr, corr);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    // the barrier once more: a branch that keeps the later loads from
                    // moving to the top, where their values would spill
                    if (c == 2 && !mbar_wait(&S.o_full[t], ph, p.err, kDevTimeoutFull)) ok = false;
                    uint32_t r[32];
                    TMEM_LD32(trow + 256u + 32 * c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) fma_pair(o[16 * c + e], corr2, r[2 * e], r[2 * e + 1]);
                }
                tc_before();
            }
            if (parts > 1) {
                if (live && ok) {   // unnormalised, to the workspace
                    *reinterpret_cast<float2*>(part_out + 2 * kTcRows * kHd + 2 * (kTcRows * t + row)) = make_float2(m, l);
                    uint4* d = reinterpret_cast<uint4*>(part_out + (size_t)(kTcRows * t + row) * kHd);
#pragma unroll
                    for (int e = 0; e < kHd / 2; e += 2) store_f32(d + e / 2, o[e], o[e + 1], pair(1.f, 1.f));
                }
            } else if (live && ok) {
                uint4* d = reinterpret_cast<uint4*>(static_cast<float*>(p.out) + out_off);
                if (lim > 0) {
                    const float rl = rcp(l);
                    const uint64_t inv = pair(rl, rl);
#pragma unroll
                    for (int e = 0; e < kHd / 2; e += 2) store_f32(d + e / 2, o[e], o[e + 1], inv);
                } else {   // no key seen
#pragma unroll
                    for (int e = 0; e < kHd / 4; ++e) d[e] = make_uint4(0u, 0u, 0u, 0u);
                }
            }
        } else {
            for (int j = 0; j < nt[t]; ++j) {
                ok = mbar_wait(&S.s_full[t], (uint32_t)j & 1u, p.err, kDevTimeoutFull);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_after();
                const Turn turn = turn_of(j);
                if ((j0 + j + 1) * kTile > lim0)
                    softmax_row_f16<true>(trow, lim - (j0 + j) * kTile, f, j == 0, m, l, S.p_full[t], turn, ok);
                else softmax_row_f16<false>(trow, 0, f, j == 0, m, l, S.p_full[t], turn, ok);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
            }
            if (parts > 1 && live)
                *reinterpret_cast<float2*>(part_out + 2 * kTcRows * kHd + 2 * (kTcRows * t + row)) = make_float2(m, l);
            if (ok && nt[t] > 0) {
                ok = mbar_wait(&S.o_full[t], 0, p.err, kDevTimeoutFull);
                ok = __all_sync(0xffffffffu, ok);
                tc_after();
            }
            if (ok) {
                const float rl = rcp(l);
                uint4* d = reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + out_off);
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[32];
                    if (nt[t] > 0) TMEM_LD32(trow + 256u + 32 * c, r);
                    tmem_wait_ld();
                    if (parts > 1) {   // unnormalised, to the workspace
                        uint4* x = reinterpret_cast<uint4*>(part_out + (size_t)(kTcRows * t + row) * kHd + 32 * c);
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            if (live)
                                x[e >> 2] = nt[t] > 0 ? make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3])
                                                      : make_uint4(0u, 0u, 0u, 0u);
                        __syncwarp();
                        continue;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint4 u = make_uint4(0u, 0u, 0u, 0u);
                        if (lim > 0) {
                            u.x = pack2(__uint_as_float(r[e]) * rl, __uint_as_float(r[e + 1]) * rl);
                            u.y = pack2(__uint_as_float(r[e + 2]) * rl, __uint_as_float(r[e + 3]) * rl);
                            u.z = pack2(__uint_as_float(r[e + 4]) * rl, __uint_as_float(r[e + 5]) * rl);
                            u.w = pack2(__uint_as_float(r[e + 6]) * rl, __uint_as_float(r[e + 7]) * rl);
                        }
                        if (live) d[4 * c + (e >> 3)] = u;
                    }
                    __syncwarp();
                }
            }
        }
    }
    tc_before();
    __syncthreads();
    if (warp == 9) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTcCols) : "memory");
    }
    if (parts == 1) return;

    // ------------------------- parts of a unit: the last CTA to end joins them
    if (threadIdx.x == 0) {
        const unsigned long long n = atom_add_acq_rel_gpu_u64(tile_count(p, item.slot), 1ull) + 1;
        S.found = n == p.nonce + parts;
        if (S.found) *tile_count(p, item.slot) = 0;
    }
    __syncthreads();
    if (!S.found || warp >= 8) return;
    const float* part0 = p.tile_work + (size_t)item.slot * kTilePartFloats;
    const int t = warp >> 2, rows = ntok[t] * p.G;
#pragma unroll 1
    for (int row = 32 * (warp & 3); row < min(rows, 32 * (warp & 3) + 32); ++row) {
        const int r = kTcRows * t + row, tok = row / p.G;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < parts)
            ml = __ldcg(reinterpret_cast<const float2*>(part0 + (size_t)lane * kTilePartFloats + 2 * kTcRows * kHd + 2 * r));
        float4 y[kMaxParts];
#pragma unroll
        for (int i = 0; i < kMaxParts; ++i)
            if (i < parts)
                y[i] = __ldcg(reinterpret_cast<const float4*>(part0 + (size_t)i * kTilePartFloats + (size_t)r * kHd) + lane);
        float M = ml.x;
#pragma unroll
        for (int d = 4; d >= 1; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
        M = __shfl_sync(0xffffffffu, M, 0);
        const float k = ml.x == -INFINITY ? 0.f : ex2(ml.x - M), kl = warp_sum(k * ml.y);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kMaxParts; ++i) {
            const float ki = __shfl_sync(0xffffffffu, k, i);
            if (i < parts)
                acc = make_float4(fmaf(y[i].x, ki, acc.x), fmaf(y[i].y, ki, acc.y), fmaf(y[i].z, ki, acc.z),
                                  fmaf(y[i].w, ki, acc.w));
        }
        const bool none = kv_len - n + tok0 + t * tpt + tok + 1 <= 0 || kv_len == 0;
        const float inv = none ? 0.f : rcp(kl);
        const int64_t off = (int64_t)(first + tok0 + t * tpt + tok) * p.out_stride +
                            (int64_t)(g * p.G + row - tok * p.G) * kHd + 4 * lane;
        store_pair<F32>(p.out, off, make_float2(acc.x, acc.y), inv, none);
        store_pair<F32>(p.out, off + 2, make_float2(acc.z, acc.w), inv, none);
    }
}

// Differs from call to call, and from what a workspace may hold by chance (2^-56).
unsigned long long next_nonce() {
    static std::atomic<unsigned long long> n{(unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count()};
    unsigned long long z = n.fetch_add(0x9E3779B97F4A7C15ull, std::memory_order_relaxed);
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;   // SplitMix64
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return ((z ^ (z >> 31)) & ~0xffull) | 0x100ull;
}

template <bool F32>
int attn_rows_launch(const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p, cudaStream_t st) {
    constexpr int smem = (int)sizeof(RowsSmem) + 1024;
    static_assert(smem <= 232448, "shared memory of a CTA");
    cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) {
        attn_rows_kernel<F32><<<kRowCtas, kRowThreads, smem, st>>>(tk, tv, p);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "attention: %s", cudaGetErrorString(e));
    return GLC_OK;
}

template <bool F32>
int attn_tiles_launch(const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p, long long items, cudaStream_t st) {
    constexpr int smem = TilesLayout<F32>::kBytes;
    static_assert(smem <= 232448, "shared memory of a CTA");
    cudaError_t e = cudaFuncSetAttribute(attn_tiles_kernel<F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "attention: %s", cudaGetErrorString(e));
    if (items > 0x7fffffffLL) return paged_fail(GLC_ERR_UNSUPPORTED, "%d rows are too many for one call", p.T);
    attn_tiles_kernel<F32><<<(unsigned)items, kTcThreads, smem, st>>>(tk, tv, p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "attention: %s", cudaGetErrorString(e));
    return GLC_OK;
}

// How a call runs, from what the host knows of it.
struct AttnPlan {
    bool rows, tiles;     // kernels that are launched
    bool split;           // units of the tile kernel may be cut
    long long items;      // most CTAs of it that have work
    int slots;            // and of their partials
    size_t work;          // workspace bytes
    size_t tile_work;     // where the partials of the tile kernel begin
};
AttnPlan plan_attention(int n_heads, int n_kv, int B, int T, int max_new, bool workspace) {
    const int G = n_heads / n_kv;
    AttnPlan a{};
    // A sequence of up to 16 rows a KV head is the row kernel's.  With longer ones
    // in the batch the row kernel comes first where there may be several short
    // ones; a batch of up to four is left to the tiles, the empty launch costs 3 us.
    a.tiles = (long long)max_new * G > kRows;
    a.rows = !a.tiles || (workspace && B > 4);
    const long long units = ((long long)T / (2 * (kTcRows / G)) + std::min(B, T)) * n_kv;
    // Many units fill the SMs by themselves, and each CTA looks through all sequences
    a.split = a.tiles && workspace && units <= 16 * 148;
    a.items = units + (a.split ? kMaxExtra : 0);
    a.slots = a.split ? (int)std::min<long long>(units * kMaxParts, 2 * kMaxExtra) : 0;
    a.tile_work = kRowsWorkBytes + ((size_t)a.slots * sizeof(unsigned long long) + 255) / 256 * 256;
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
        if (int rc = f32 ? attn_rows_launch<true>(tk, tv, p, st) : attn_rows_launch<false>(tk, tv, p, st)) return rc;
    }
    if (!a.tiles) return GLC_OK;
    p.tokens_per_tile = 2 * (kTcRows / p.G);
    return f32 ? attn_tiles_launch<true>(ttk, ttv, p, a.items, st) : attn_tiles_launch<false>(ttk, ttv, p, a.items, st);
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
    if (int rc = glc::paged_check_device(k, "k")) return rc;
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
    if (max_pages <= 0 || max_new < 0 || (int64_t)max_pages * cache->page_size > 0x7fffffff)
        return paged_fail(GLC_ERR_INVALID_ARG, "tables of %d pages, up to %d new tokens", max_pages, max_new);
    uint64_t need = 0;
    if (int rc = glc_attn_paged_workspace_bytes(n_heads, cache->n_kv_heads, B, T, max_new, &need)) return rc;
    if (((uintptr_t)workspace & 15u) || workspace_bytes < need)
        return paged_fail(GLC_ERR_INVALID_ARG, "workspace of %llu bytes is too small or not 16-byte aligned",
                          (unsigned long long)workspace_bytes);
    if (B == 0 || T == 0) return GLC_OK;
    if (int rc = glc::paged_check_device(cache->k, "the cache")) return rc;
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
    CUtensorMap tk, tv, ttk, ttv;
    const auto map = [&](CUtensorMap* m, const void* base, int halves) {
        return glc::paged_tensor_map(m, base, cache->page_size, cache->row_stride, cache->n_kv_heads, cache->head_stride,
                                     cache->n_pages, cache->page_stride, p.box_rows, halves);
    };
    if (int rc = map(&tk, cache->k, 2)) return rc;
    if (int rc = map(&tv, cache->v, 2)) return rc;
    // the tile kernel's K and V lie as two blocks of 64 dims: a box that covers part
    // of a tile's keys is one block's, one that covers them all takes both
    const int halves = p.box_rows < glc::kTile ? 1 : 2;
    if (int rc = map(&ttk, cache->k, halves)) return rc;
    if (int rc = map(&ttv, cache->v, halves)) return rc;
    return glc::attn_launch(tk, tv, ttk, ttv, p, a, q_type == GLC_GGUF_F32, (cudaStream_t)stream);
}
