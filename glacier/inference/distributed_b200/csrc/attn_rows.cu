// attn_rows.cu -- attention of few query rows (decode tokens) over pages or packed
// keys: see attn_paged.cu for the operator.
//
// attn_rows_kernel: up to 16 query rows of one KV head, so every K and V row is
// read once for all the heads that share it.  Eight warps take 16 of a tile's
// 128 keys each and keep their own running maximum, sum and output in registers
// (one pass, no exchange between warps until a unit's end, where the eight
// partials are joined in warp order); two more stream the pages with TMA
// into a ring of six 32 KB slots, one the keys, one the values.  Products run as
// mma.sync m16n8k16 with fp32 accumulators: 16 rows cannot fill a 128-row
// tensor-memory tile.
// The tensor core cuts its running sums by up to 2^-23 a product.  fp32 queries add each
// tile's products up outside it; fp16 ones leave the sum there, which costs n / 2 x 2^-23
// of it over a CTA's n tiles: 2^-13 at 2,048 tiles (262,144 keys), a quarter of the
// fp16 output's own half step.
// Bound by the bytes of K and V: 64 sequences of 100 to 16,000 rows (48 heads over
// 8) take 140 to 145 us, 90 to 94 % of the copy rate, with fp16 queries and with fp32
// ones.  One sequence of 2,048 rows (40 heads over 8, fp32 queries) takes 11 us a call,
// 9.5 in a replayed graph: the chain of lengths, page table, keys, merge of the warps and
// join of the CTAs, not the 8.4 MB.
#include <type_traits>

#include "attn.cuh"

namespace glc {

namespace {

constexpr int kRowWarps = 8;
constexpr int kRowThreads = (kRowWarps + 2) * 32;

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
// ------------------------------------------------------------ few rows (decode)
// A unit is one KV head of one sequence; its keys come in tiles of 128.  The
// tiles of all units, one unit after another, are cut into kRowCtas equal runs,
// one CTA each: every SM streams the same number of bytes whatever the lengths.
// A unit counts kUnitOver tiles more than it has, one before and one behind, for its
// queries and its merge (3.5k cycles against 2k a tile).  A run holds whole units,
// which are finished in place, and at most two that it shares with its neighbours;
// their partials go to the workspace, two places a CTA, and the last CTA to bring
// its own joins them in key order.
constexpr int kUnitOver = 2;
constexpr int kRowSlots = 6;                   // 32 KB each: K and V tiles in turn
constexpr int kUnitCache = 256;                // sequences whose lengths are kept in shared memory
struct RowsUnit {
    int first, n, kv_len, tiles;
    __device__ __forceinline__ int weight() const { return tiles ? tiles + kUnitOver : 0; }
};

struct RowsSmem {
    uint8_t ring[kRowSlots][kTileBytes];
    uint4 q[2][8][32];                         // A fragments of the unit's rows: high and low halves, 8 steps of 16 dims
    float o[kRowWarps][8][72];                 // joins the warps' outputs, 8 rows x 64 dims at a time (rows 8 banks apart)
    float m[kRowWarps][kRows], l[kRowWarps][kRows], qmax[kRowWarps][kRows];
    int first[kUnitCache], n[kUnitCache], kv[kUnitCache];
    uint64_t full[kRowSlots], empty[kRowSlots];
    uint64_t opened[2];                        // the CTA's shared units: at most its first and its last
    long long sums[kRowWarps], rest[kRowWarps];
    long long W, x0, x1, u0;                   // weight in all, the CTA's run of it, start of the run's first unit
    int b, g;                                  // which that is
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
        if (record && u.n > 0 && (len != u.kv_len || u.n > p.max_new)) record_bad_arg(p.err);
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

// A unit of the CTA's run [x0, x1): it begins at u0, and its tile j lies at u0 + 1 + j.
struct RowsWalk {
    int b, g;
    long long u0, x0, x1;
    __device__ __forceinline__ bool more() const { return u0 < x1; }
    __device__ __forceinline__ int first(const RowsUnit& u) const { return (int)max(0ll, min((long long)u.tiles, x0 - u0 - 1)); }
    __device__ __forceinline__ int end(const RowsUnit& u) const { return (int)max(0ll, min((long long)u.tiles, x1 - u0 - 1)); }
    __device__ __forceinline__ void next(const AttnBatch& p, const RowsSmem& S, const RowsUnit& u) {
        u0 += u.weight();
        if (u0 < x1 && ++g == p.n_kv) {
            g = 0;
            do ++b;
            while (b + 1 < p.B && get_unit(p, S, b).tiles == 0);
        }
    }
};

// CTA that holds position x of W: the last c with c * W / kRowCtas <= x.
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
template <bool F32>
__global__ void __launch_bounds__(kRowThreads, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const __grid_constant__ AttnBatch p) {
    extern __shared__ uint8_t smem_raw[];
    RowsSmem& S = *reinterpret_cast<RowsSmem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kConsumers = kRowWarps * 32;

    // the tile kernel of the same call, where there is one, reads nothing that this one writes
    if ((long long)p.max_new * p.G > kRows) grid_dep_launch_dependents();
    if (threadIdx.x == kConsumers) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tv) : "memory");
        for (int i = 0; i < kRowSlots; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], kRowWarps);
        }
        mbar_init(&S.opened[0], 1);
        mbar_init(&S.opened[1], 1);
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
        if (tid == 0) S.u0 = S.x1 = 0;
        long long rest = 0;   // weight of the sequences behind the first 256
        for (int b = tid + kConsumers; b < p.B; b += kConsumers) rest += load_unit(p, b, blockIdx.x == 0).weight();
        long long before = 0, W = 0, x0 = 0, x1 = 1;
        for (int b0 = 0; b0 < p.B && x1 > x0 && before * p.n_kv <= x0; b0 += kConsumers) {
            if (b0) u = b0 + tid < p.B ? load_unit(p, b0 + tid) : RowsUnit{0, 0, 0, 0};
            long long end = u.weight();
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
            const long long in = x0 - (end - u.weight()) * p.n_kv;   // into this thread's sequence
            if (x1 > x0 && in >= 0 && in < (long long)u.weight() * p.n_kv) {
                S.b = b0 + tid;
                S.g = (int)(in / u.weight());
                S.u0 = x0 - (in - (long long)S.g * u.weight());
                S.x0 = x0;
                S.x1 = x1;
                S.W = W;
            }
            before += all;
        }
    }
    __syncthreads();
    RowsWalk w{S.b, S.g, S.u0, S.x0, S.x1};

    if (warp >= kRowWarps) {
        // ---------------------------------- page stream: keys, and values
        const int m = warp - kRowWarps;
        const CUtensorMap* tm = m ? &tv : &tk;
        const int nbox = kTile / p.box_rows, ps = 1 << p.ps_log2;
        bool ok = true;
        int it = m, shared = 0;
        while (w.more() && ok) {
            const RowsUnit u = get_unit(p, S, w.b);
            const int tile0 = w.first(u), end = w.end(u);
            for (int j = tile0; j < end; ++j, it += 2) {
                const int r0 = j * kTile + lane * p.box_rows, st = it % kRowSlots;
                const bool mine = lane < nbox && r0 < u.kv_len;
                const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
                int page = 0, row = u.first + r0;
                if (mine && p.table) {
                    page = p.table[(long long)w.b * p.max_pages + (r0 >> p.ps_log2)];
                    row = r0 & (ps - 1);
                    if ((unsigned)page >= (unsigned)p.n_pages) {  // reads as zeros
                        record_bad_arg(p.err);
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
                // the counter of a unit this CTA shares, once its first keys are on their way
                if (m == 0 && j == tile0 && lane == 0 && (tile0 > 0 || end < u.tiles)) {
                    part_open(part_count(p, rows_cta(w.u0 + 1, S.W)), p.nonce);
                    mbar_arrive(&S.opened[shared++]);
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
    // a unit's queries on their way: warp ks brings step ks of the A fragments, thread
    // (gr, gc) rows gr, gr + 8, columns 16 ks + 2 gc + {0, 1} and + 8.  The next unit's
    // are loaded while this one's keys are worked on.
    using QRaw = std::conditional_t<F32, float2, uint32_t>;
    QRaw qraw[2][2];
    auto load_q = [&](const RowsUnit& u, int g) {
        const int rows = min(u.n, p.tokens_per_tile) * p.G;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const int r = gr + 8 * hh, tok = r / p.G, h = r - tok * p.G;
            const int64_t off = (int64_t)(u.first + tok) * p.q_stride + (int64_t)(g * p.G + h) * kHd + 16 * warp + 2 * gc;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                qraw[hh][c] = QRaw{};
                if (r < rows)
                    qraw[hh][c] = __ldg(reinterpret_cast<const QRaw*>(
                        reinterpret_cast<const char*>(p.q) + (off + 8 * c) * (F32 ? sizeof(float) : sizeof(__half))));
            }
        }
    };
    auto skip = [&](RowsWalk& v) {   // to the next unit that has tiles in the run
        while (v.more()) {
            const RowsUnit u = get_unit(p, S, v.b);
            if (v.first(u) < v.end(u)) return;
            v.next(p, S, u);
        }
    };
    skip(w);
    if (w.more()) load_q(get_unit(p, S, w.b), w.g);
    bool ok = true;
    int it = 0, shared = 0;
    while (w.more()) {
        const RowsUnit u = get_unit(p, S, w.b);
        const int g = w.g, tile0 = w.first(u), tile1 = w.end(u);
        const int ntok = min(u.n, p.tokens_per_tile), rows = ntok * p.G;
        const int see0 = u.kv_len - u.n + 1;           // keys the first token sees (may be <= 0)

        // ------------------------------------------------------------ queries
        float f[2];                                    // score factor: scale * log2(e) * the row's power of two
        int lim[2];                                    // keys seen by the thread's two rows
        {
            uint32_t hi[4], lo[4];
            float2 a[2][2];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int r = gr + 8 * hh, tok = r / p.G;
                lim[hh] = r < rows ? max(0, min(u.kv_len, see0 + tok)) : 0;
                f[hh] = p.scale_log2;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if constexpr (F32) a[hh][c] = qraw[hh][c];
                    else hi[2 * c + hh] = qraw[hh][c];
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
        RowsWalk nw = w;
        nw.next(p, S, u);
        skip(nw);
        if (nw.more()) load_q(get_unit(p, S, nw.b), nw.g);

        const bool whole = tile0 == 0 && tile1 == u.tiles;
        int c0 = 0, c1 = 0, parts = 0;                 // CTAs that share the unit
        if (!whole) {
            c0 = rows_cta(w.u0 + 1, S.W);
            c1 = rows_cta(w.u0 + u.tiles, S.W);
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
                ok = ok && mbar_wait(&S.opened[shared], 0, p.err, kDevTimeoutFull);
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
        shared += !whole;
        w = nw;
    }
}

template <bool F32>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p, cudaStream_t st) {
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

}  // namespace

int attn_rows_launch(bool f32, const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p, cudaStream_t st) {
    return f32 ? launch<true>(tk, tv, p, st) : launch<false>(tk, tv, p, st);
}

}  // namespace glc
