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
// Row kernel (attn_rows_kernel): a tile is up to 16 query rows of one KV head --
// floor(16 / G) tokens times their G heads -- so every K and V row is read once
// for all the heads that share it.  Eight warps take 16 of a stage's 128 keys
// each and keep their own running maximum, sum and output in registers (one
// pass, no exchange between warps until the tile's end, where the eight
// partials are merged in warp order); a ninth warp streams the pages with TMA
// into a ring of three 64 KB stages.  Products run as mma.sync m16n8k16 with
// fp32 accumulators: 16 rows cannot fill a 128-row tensor-memory tile, and at
// these row counts the bytes of K and V bound the time.
// fp32 queries are carried as two fp16 halves after a power-of-two scale per
// row, and so are the exponentials (two products each, ~22 bits of q and p
// against the fp16 cache values); fp16 queries take one product.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "paged.cuh"

namespace glc {

namespace {

constexpr int kHd = 128;
constexpr int kTile = 128;                     // keys per stage
constexpr int kStages = 3;
constexpr int kTileBytes = kTile * kHd * 2;    // one matrix of a stage
constexpr int kRowWarps = 8;
constexpr int kRowThreads = (kRowWarps + 1) * 32;
constexpr int kRows = 16;                      // query rows of a tile
constexpr float kPShift = 10.f;                // exponentials are stored as 2^10 e^(s - m): see below

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

// Rows of sequence b, held inside [0, T] whatever cu holds.
__device__ __forceinline__ void seq_rows(const AttnBatch& p, int b, int& first, int& n) {
    first = min(max(p.cu[b], 0), p.T);
    n = min(max(p.cu[b + 1], first), p.T) - first;
}

// Sequence and tile of the x-th tile of the batch (called by one warp): the
// tiles of a sequence are its tokens in runs of tokens_per_tile.
__device__ __forceinline__ bool find_tile(const AttnBatch& p, int x, int& seq, int& tile) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int b = b0 + lane;
        int nt = 0;
        if (b < p.B) {
            int first, n;
            seq_rows(p, b, first, n);
            nt = (n + p.tokens_per_tile - 1) / p.tokens_per_tile;
        }
        int end = nt;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, end, off);
            if (lane >= off) end += o;
        }
        const unsigned m = __ballot_sync(0xffffffffu, before + end > x);
        if (m) {
            const int l = __ffs(m) - 1;
            seq = b0 + l;
            tile = x - before - __shfl_sync(0xffffffffu, end - nt, l);
            return true;
        }
        before += __shfl_sync(0xffffffffu, end, 31);
    }
    return false;
}

struct RowsSmem {
    uint8_t ring[kStages][2][kTileBytes];
    float m[kRowWarps][kRows];
    float l[kRowWarps][kRows];
    uint64_t full[kStages], empty[kStages];
    int seq, tile, found;
};
// the merge of a tile's partials: four warps' outputs at a time
struct RowsSmemAll {
    RowsSmem s;
    float o[4][kRows][kHd];
};

template <bool F32>
__global__ void __launch_bounds__(kRowThreads, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const __grid_constant__ AttnBatch p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    RowsSmemAll& A = *reinterpret_cast<RowsSmemAll*>(base);
    RowsSmem& S = A.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = blockIdx.y;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], kRowWarps);
        }
        fence_mbar_init();
    }
    if (warp == 0) {
        int seq = 0, tile = 0;
        const bool ok = find_tile(p, blockIdx.x, seq, tile);
        if (lane == 0) {
            S.seq = seq;
            S.tile = tile;
            S.found = ok;
        }
    }
    __syncthreads();
    if (!S.found) return;
    const int seq = S.seq, tok0 = S.tile * p.tokens_per_tile;
    int first, n;
    seq_rows(p, seq, first, n);
    const int ntok = min(p.tokens_per_tile, n - tok0), rows = ntok * p.G;
    int kv_len = n;
    if (p.kv_lens) {
        if (n > p.max_new && threadIdx.x == 0) atomicExch(p.err, kDevBadArg);
        const long long room = (long long)p.max_pages << p.ps_log2;
        kv_len = p.kv_lens[seq];
        if (kv_len < 0 || kv_len > room) {
            if (threadIdx.x == 0) atomicExch(p.err, kDevBadArg);
            kv_len = kv_len < 0 ? 0 : (int)room;
        }
    }
    const int see0 = kv_len - n + tok0 + 1;            // keys the tile's first token sees (may be <= 0)
    const int kv_end = max(0, min(kv_len, see0 + ntok - 1));
    const int ntiles = (kv_end + kTile - 1) / kTile;

    if (warp == kRowWarps) {
        // ------------------------------------------------------- page stream
        const int nbox = kTile / p.box_rows, ps = 1 << p.ps_log2;
        bool ok = true;
        int it = 0;
        for (; it < ntiles && ok; ++it) {
            const int st = it % kStages;
            ok = mbar_wait_backoff(&S.empty[st], ((uint32_t)(it / kStages) & 1u) ^ 1u, p.err, kDevTimeoutEmpty, 32);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int r0 = it * kTile + lane * p.box_rows;
            const bool mine = lane < nbox && r0 < kv_end;
            const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
            if (lane == 0) mbar_arrive_expect_tx(&S.full[st], (uint32_t)(boxes * p.box_rows * kHd * 2 * 2));
            int page = 0, row = first + r0;
            if (mine && p.table) {
                page = p.table[(long long)seq * p.max_pages + (r0 >> p.ps_log2)];
                row = r0 & (ps - 1);
                if ((unsigned)page >= (unsigned)p.n_pages) {  // reads as zeros
                    atomicExch(p.err, kDevBadArg);
                    page = p.n_pages;
                }
            }
            __syncwarp();
            if (mine) {
                tma_load_kv(S.ring[st][0] + lane * p.box_rows * kHd * 2, &tk, 0, row, g, page, &S.full[st]);
                tma_load_kv(S.ring[st][1] + lane * p.box_rows * kHd * 2, &tv, 0, row, g, page, &S.full[st]);
            }
            __syncwarp();
        }
        if (lane == 0) drain_issued_stages(S.full, kStages, it, kWaitLimitNs);
        __syncthreads();  // matches the consumers' first barrier of the merge
        for (int i = 0; i < 4; ++i) __syncthreads();
        return;
    }

    // ---------------------------------------------------------------- queries
    // A fragments of the tile's 16 rows: thread (gr, gc) holds rows gr, gr + 8,
    // columns 16 ks + 2 gc + {0, 1} and + 8
    const int gr = lane >> 2, gc = lane & 3;
    uint32_t qh[8][4], ql[F32 ? 8 : 1][4];
    float f[2];                                        // S row factor: scale * log2(e) * the row's power of two
    int lim[2];                                        // keys seen by the thread's two rows
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        const int r = gr + 8 * hh, tok = r / p.G, h = r - tok * p.G;
        const bool live = r < rows;
        lim[hh] = live ? max(0, min(kv_len, see0 + tok)) : 0;
        f[hh] = p.scale_log2;
        const int64_t off = (int64_t)(first + tok0 + tok) * p.q_stride + (int64_t)(g * p.G + h) * kHd + 2 * gc;
        if constexpr (F32) {
            float2 a[8][2];
            float mx = 0.f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    a[ks][c] = live ? __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + off +
                                                                            16 * ks + 8 * c))
                                    : make_float2(0.f, 0.f);
                    mx = fmaxf(mx, fmaxf(fabsf(a[ks][c].x), fabsf(a[ks][c].y)));
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // largest value to [2^12, 2^13): the low halves stay normal far below it
            const int e = (mx > 0.f && mx < INFINITY) ? 12 - ilogbf(mx) : 0;
            const float up = exp2f((float)max(-126, min(126, e)));
            f[hh] = p.scale_log2 / up;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    split2(a[ks][c].x * up, a[ks][c].y * up, qh[ks][2 * c + hh], ql[ks][2 * c + hh]);
        } else {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    qh[ks][2 * c + hh] = live ? __ldg(reinterpret_cast<const uint32_t*>(
                                                    static_cast<const __half*>(p.q) + off + 16 * ks + 8 * c))
                                              : 0u;
        }
    }

    float o[16][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 16; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] = 0.f;

    // the warp's 16 keys of a stage: box and row inside the box are fixed
    const int k0 = 16 * warp, box_b = p.box_rows * kHd;  // bytes of a 64-element half of a box
    const uint32_t warp_off = (uint32_t)((k0 / p.box_rows) * box_b * 2 + (k0 % p.box_rows) * 128);
    // ldmatrix lane addresses (rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7))
    const int lr = (lane & 7) + ((lane >> 4) << 3), lc = (lane >> 3) & 1;          // K: matrices (keys 0-7, c), (keys 0-7, c + 1), (keys 8-15, ..)
    const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;          // V (transposed): (keys 0-7, c), (keys 8-15, c), (.., c + 1)

    bool ok = true;
    for (int it = 0; it < ntiles && ok; ++it) {
        const int st = it % kStages;
        ok = mbar_wait(&S.full[st], (uint32_t)(it / kStages) & 1u, p.err, kDevTimeoutFull);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t kb = smem_u32(S.ring[st][0]) + warp_off, vb = smem_u32(S.ring[st][1]) + warp_off;
        const int j0 = it * kTile + k0;                // first key of the warp's 16
        if (j0 < kv_end) {
            float s[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                uint32_t b[4];
                const int c = 2 * (ks & 3) + lc;
                ldsm4(kb + (ks >> 2) * box_b + lr * 128 + ((c ^ (lr & 7)) << 4), b);
                mma_f16(s[0], qh[ks], b[0], b[1]);
                mma_f16(s[1], qh[ks], b[2], b[3]);
                if constexpr (F32) {
                    mma_f16(s[0], ql[ks], b[0], b[1]);
                    mma_f16(s[1], ql[ks], b[2], b[3]);
                }
            }
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j0 + 8 * (e >> 1) + 2 * gc + (e & 1);
                    v[e] = j < lim[hh] ? s[e >> 1][2 * hh + (e & 1)] * f[hh] : -INFINITY;
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
            // values past the last key may be anything, NaN included: they count as zeros
            const bool tail = j0 + 16 > kv_end;
            const int left = kv_end - j0 - 2 * gc;     // keys left from this thread's first
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
                mma_f16(o[2 * t], ph, b[0], b[1]);
                mma_f16(o[2 * t + 1], ph, b[2], b[3]);
                if constexpr (F32) {
                    mma_f16(o[2 * t], pl, b[0], b[1]);
                    mma_f16(o[2 * t + 1], pl, b[2], b[3]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.empty[st]);
    }

    // ------------------------------------------------------------------ merge
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 1);
        l[hh] += __shfl_xor_sync(0xffffffffu, l[hh], 2);
        if (gc == 0) {
            S.m[warp][gr + 8 * hh] = m[hh];
            S.l[warp][gr + 8 * hh] = l[hh];
        }
    }
    __syncthreads();
    float corr[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, S.m[w][gr + 8 * hh]);
        corr[hh] = m[hh] == -INFINITY ? 0.f : ex2(m[hh] - M);
    }
    constexpr int kPer = kRows * kHd / (kRowWarps * 32);  // outputs per thread: row tid / 16, dims 8 (tid % 16) ..
    const int orow = threadIdx.x >> 4, od = (threadIdx.x & 15) * kPer;
    float acc[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if ((warp >> 2) == half) {
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                const int d = 8 * t + 2 * gc;
                *reinterpret_cast<float2*>(&A.o[warp & 3][gr][d]) = make_float2(o[t][0] * corr[0], o[t][1] * corr[0]);
                *reinterpret_cast<float2*>(&A.o[warp & 3][gr + 8][d]) = make_float2(o[t][2] * corr[1], o[t][3] * corr[1]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int e = 0; e < kPer; ++e) acc[e] += A.o[w][orow][od + e];
        __syncthreads();
    }
    if (orow < rows) {
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, S.m[w][orow]);
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w)
            L += S.m[w][orow] == -INFINITY ? 0.f : S.l[w][orow] * ex2(S.m[w][orow] - M);
        const int tok = orow / p.G, h = orow - tok * p.G;
        // no key seen: zeros.  A NaN score leaves m at -inf or l at NaN: the row's sum says which
        const bool none = max(0, min(kv_len, see0 + tok)) == 0;
        const float inv = none ? 0.f : 1.f / L;
        const int64_t off = (int64_t)(first + tok0 + tok) * p.out_stride + (int64_t)(g * p.G + h) * kHd + od;
        if constexpr (F32) {
            float* d = static_cast<float*>(p.out) + off;
#pragma unroll
            for (int e = 0; e < kPer; ++e) d[e] = none ? 0.f : acc[e] * inv;
        } else {
            __half* d = static_cast<__half*>(p.out) + off;
#pragma unroll
            for (int e = 0; e < kPer; ++e) d[e] = __float2half_rn(none ? 0.f : acc[e] * inv);
        }
    }
}

int attn_rows_launch(const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p, bool f32, cudaStream_t st) {
    const int smem = (int)sizeof(RowsSmemAll) + 1024;
    const void* fn = f32 ? (const void*)attn_rows_kernel<true> : (const void*)attn_rows_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "attention: %s", cudaGetErrorString(e));
    const long long tiles = (long long)p.T / p.tokens_per_tile + std::min(p.B, p.T);
    if (tiles > 0x7fffffffLL) return paged_fail(GLC_ERR_UNSUPPORTED, "%d rows are too many for one call", p.T);
    const dim3 grid((unsigned)tiles, (unsigned)p.n_kv);
    if (f32)
        attn_rows_kernel<true><<<grid, kRowThreads, smem, st>>>(tk, tv, p);
    else
        attn_rows_kernel<false><<<grid, kRowThreads, smem, st>>>(tk, tv, p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "attention: %s", cudaGetErrorString(e));
    return GLC_OK;
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
    p.tokens_per_tile = kRows / p.G;
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
    return glc::attn_rows_launch(tk, tv, p, q_type == GLC_GGUF_F32, (cudaStream_t)stream);
}

extern "C" int glc_attn_paged_workspace_bytes(int32_t n_heads, int32_t n_kv_heads, int32_t B, int32_t T,
                                              int32_t max_new, uint64_t* bytes) {
    if (!bytes) return paged_fail(GLC_ERR_INVALID_ARG, "null pointer");
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > glc::kRows || B < 0 || T < 0 ||
        max_new < 0)
        return paged_fail(GLC_ERR_INVALID_ARG, "bad attention shape (%d heads, %d KV heads, %d sequences, %d rows)",
                          n_heads, n_kv_heads, B, T);
    *bytes = 256;
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
    p.kv_lens = kv_lens;
    p.table = block_table;
    p.max_pages = max_pages;
    p.max_new = max_new;
    p.n_pages = cache->n_pages;
    while ((1 << p.ps_log2) < cache->page_size) ++p.ps_log2;
    p.box_rows = std::min(cache->page_size, glc::kTile);
    CUtensorMap tk, tv;
    if (int rc = glc::paged_tensor_map(&tk, cache->k, cache->page_size, cache->row_stride, cache->n_kv_heads,
                                       cache->head_stride, cache->n_pages, cache->page_stride, p.box_rows, 2))
        return rc;
    if (int rc = glc::paged_tensor_map(&tv, cache->v, cache->page_size, cache->row_stride, cache->n_kv_heads,
                                       cache->head_stride, cache->n_pages, cache->page_stride, p.box_rows, 2))
        return rc;
    return glc::attn_rows_launch(tk, tv, p, q_type == GLC_GGUF_F32, (cudaStream_t)stream);
}
