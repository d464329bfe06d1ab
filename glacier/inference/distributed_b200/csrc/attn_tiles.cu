// attn_tiles.cu -- attention of many query rows (prompts, chunks of prompts) over
// packed keys or pages: see attn_paged.cu for the operator.
//
// An item is 256 query rows of one KV head, as two row tiles A and B of 128
// (floor(128 / G) tokens times their G heads) that share every K and V tile of
// 128 keys.  One CTA per SM works through items.  Per key tile and row tile:
//   S = Q K^T   tcgen05.mma, S in tensor memory;
//   P = 2^(S f - m)  one warpgroup per row tile, one row per thread: no
//               exchange between threads; P overwrites S in tensor memory;
//   PV          tcgen05.mma, P from tensor memory, V from shared memory.
// While one row tile's warpgroup works on its softmax the tensor core runs the
// other's products.
// fp16 queries: PV adds up in tensor memory; a row is rescaled there when its
// maximum has grown by more than 2^kLazy, which after the first tiles hardly happens.
// fp32 queries: S and PV take two products each (halves of q and of p, low
// halves first), and PV is a tile of its own that the row's thread adds to its
// fp32 output in registers: the tensor core cuts its running sum at every 16
// keys, which over 32,000 keys costs a decimal digit.  The low halves of q are
// read from tensor memory and the two row tiles share one PV tile, so both types
// leave room for five K or V tiles in flight.
// Warps 0-7: softmax; 8: TMA; 9 and 10: MMA issue; 11: the next items.
// Bound by the chain of a row tile (its products wait for its exponentials and the
// next scores for its PV, as P lies over S and tensor memory has no room for another
// S): a key tile of a pair takes 3,600 cycles with fp16 queries, of which the tensor
// core works 2,500 (a product of 128 x 128 x 16 takes 87 cycles with both operands in
// shared memory, 67 with A in tensor memory) and the exponentials 2,050, and 6,200
// with fp32 ones (4,600 and 2,050).  Calls one after another, where the power limit holds
// the clock down: 16,384 tokens (48 heads over 8, fp16) take 3.44 ms, 958 TFLOP/s; 512
// tokens against 32,513 keys (40 over 8, fp32) 672 us, two products each.  At the full
// clock 3.1 ms and 575 us.
// An item costs 4,000 cycles more for its outputs, and fp32 queries 7,000 to load.
#include <algorithm>
#include <type_traits>

#include "attn.cuh"

namespace glc {

namespace {

constexpr int kTcThreads = 12 * 32;
constexpr int kTcRows = 128;
constexpr uint32_t kTcCols = 512;
// tensor memory: S_A, S_B, then O_A, O_B (fp16 queries) or PV, low halves of Q_A, Q_B (fp32)
constexpr uint32_t kColO = 256, kColQlo = 384;
constexpr int kSlots = 5;                 // K and V tiles in flight
constexpr int kItemBufs = 2;

// Few units with many keys: a unit's key tiles are cut into up to kMaxParts parts
// of kMinPart tiles or more, one item each, whose partials (unnormalised outputs,
// maximum, sum) go to the workspace and are joined by a second launch.  (The last
// CTA of a unit joining them itself took 30 to 45 thousand cycles for 256 rows of
// five parts: with nearly all of the first-level cache given to shared memory an SM
// loads 25 bytes a cycle.)  At most kMaxExtra items more than there are units, so
// twice as many places.
constexpr int kMaxParts = kTileParts, kMinPart = 8, kMaxExtra = kTileExtra;

// One item, as the roles need it.
struct TileItem {
    int seq;          // -1: no more
    int g;
    int row0;         // first token of row tile A in q and out
    int see0;         // keys its first token sees
    int kv_len, kv_end, kv_row0;
    int ntok[2];      // tokens of the row tiles
    int nt[2];        // key tiles of this part that row tile t sees
    int j0, ntiles;   // this part's key tiles
    int part, parts, slot;
};

struct TilesSmem {
    float f[2][kTcRows];                  // score factor of each row
    uint64_t kv_full[kSlots], kv_empty[kSlots], s_full[2], p_full[2][2], o_full[2], turn[2], q_full[2], q_free[2], landed,
        item_full[kItemBufs], item_empty[kItemBufs], drain[2];
    uint32_t tmem;
    int reads[2];                         // fp32: PV tiles read by each row tile's four warps, counted per warp
    TileItem item[kItemBufs];
};
template <bool F32>
constexpr int tiles_smem_bytes() {
    return 2 * kTileBytes + kSlots * kTileBytes + (int)sizeof(TilesSmem) + 1024;
}

// Places of the workspace in use, and what each holds, for the launch that joins the
// parts: a unit whose keys are cut at the place of its first part, nothing at the
// others.  Every place in use is written by every call.
struct TileUnit {
    int parts, g, row0, see0, kv_len, ntok[2];   // parts 0: nothing
};
static_assert(sizeof(TileUnit) <= kTileUnitBytes, "places of the units");
__device__ __forceinline__ int* tile_places(const AttnBatch& p) { return reinterpret_cast<int*>(p.work + kRowsWorkBytes / sizeof(float)); }
__device__ __forceinline__ TileUnit* tile_unit(const AttnBatch& p, int slot) {
    return reinterpret_cast<TileUnit*>(tile_places(p) + (slot + 1) * (kTileUnitBytes / (int)sizeof(int)));
}

__device__ __forceinline__ void tma_load_q(void* dst, const CUtensorMap* tm, int head, int token, int half, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
        "l"(tm), "r"(0), "r"(head), "r"(token), "r"(half), "r"(smem_u32(bar))
        : "memory");
}

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

// Units of sequence b whose key tiles number up to x: the tiles a unit sees grow along
// the sequence.
struct SeqUnits {
    int n, kv_len, first;         // new tokens, keys, first row
    __device__ __forceinline__ int upto(const AttnBatch& p, int x) const {
        if (x < 0) return 0;
        if ((unsigned)kv_len <= (unsigned)x * kTile) return all(p);
        const int t = (int)((unsigned)x * kTile) - kv_len + n;   // tokens whose keys fit x tiles
        return t <= 0 ? 0 : min(all(p) - 1, div_unit(p, t));
    }
    __device__ __forceinline__ int all(const AttnBatch& p) const { return div_unit(p, n + p.tokens_per_tile - 1); }
    __device__ __forceinline__ int tiles() const { return (int)(((unsigned)kv_len + kTile - 1) / kTile); }
    // x / tokens_per_tile, 0 <= x < 2^31 (with divisions the first item of the last CTA,
    // five classes down, was there after 14,600 cycles instead of 9,800)
    static __device__ __forceinline__ int div_unit(const AttnBatch& p, int x) {
        return (int)(__umulhi((unsigned)x, p.unit_mul) >> p.unit_shift);
    }
};
__device__ __forceinline__ SeqUnits seq_units(const AttnBatch& p, int b, bool record = false) {
    SeqUnits u{0, 0, 0};
    if (b < 0) return u;
    seq_rows(p, b, u.first, u.n);
    if (u.n * p.G <= p.rows_take) u.n = 0;   // none, or the row kernel's
    u.kv_len = u.n;
    if (p.kv_lens) {
        const long long room = (long long)p.max_pages << p.ps_log2;
        const int len = p.kv_lens[b];
        u.kv_len = (int)min((long long)max(len, 0), room);
        if (record && u.n > 0 && (len != u.kv_len || u.n > p.max_new)) record_bad_arg(p.err);
    }
    return u;
}

// Walks a CTA's items (one warp), long ones first: the units in kBuckets classes of
// their key tiles, from the class with the most down, the sequences of a class
// from the batch's end.  CTA c takes items c, 2 * CTAs - 1 - c, and so on back and
// forth, which evens the sums out.
//
// With a workspace, keys are cut into parts of up to L tiles: of the longest
// sequence's tiles in 1 to 8 parts, the L with the least rounds of all CTAs times
// an item's cost, in key tiles: its own, two for its prologue and epilogue, and a
// third of one for each part that the join reads.
constexpr int kBuckets = 16;
static_assert(kMaxParts == 8, "a lane for each number of parts");
constexpr int kSeqCache = 4;       // chunks of 32 sequences, from the last down, kept in registers
struct ItemWalk {
    int seq_first[kSeqCache], seq_n[kSeqCache], seq_kv[kSeqCache];   // of the lane's sequences
    int first, n, kv_len;         // of the lane's sequence in the chunk at hand
    int L, most, total, cut;      // tiles of a part, of the longest unit; items in all, and those of cut units
    int bucket, b0, before, slots;   // class; chunk of 32 sequences (the one of lane 0); items and places before it
    int low, units, parts, count, split, end, send, chunk, schunk;   // of the lane's sequence; sums of the chunk

    __device__ __forceinline__ int parts_of(int tiles) const { return tiles <= L ? 1 : (int)((unsigned)(tiles - 1) / (unsigned)L) + 1; }

    __device__ __forceinline__ SeqUnits seq(const AttnBatch& p, int chunk) const {
        if (p.B > 32 * kSeqCache) return seq_units(p, p.B - 1 - 32 * chunk - (int)(threadIdx.x & 31));
        SeqUnits u{0, 0, 0};
#pragma unroll
        for (int k = 0; k < kSeqCache; ++k)
            if (k == chunk) {
                u.n = seq_n[k];
                u.kv_len = seq_kv[k];
                u.first = seq_first[k];
            }
        return u;
    }
    __device__ __forceinline__ void load(const AttnBatch& p) {
        const int lane = threadIdx.x & 31;
        const SeqUnits u = seq(p, (p.B - 1 - b0) >> 5);
        first = u.first;
        n = u.n;
        kv_len = u.kv_len;
        // classes (lo, hi] of key tiles; the last one takes units without keys too
        const int hi = most * (bucket + 1) / kBuckets, lo = bucket ? most * bucket / kBuckets : -1;   // (most < 2^24)
        low = u.upto(p, lo);
        units = u.n > 0 ? u.upto(p, hi) - low : 0;
        parts = parts_of(u.tiles());
        count = units * p.n_kv * parts;
        split = parts > 1 ? count : 0;
        end = count;
        send = split;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, end, off), q = __shfl_up_sync(0xffffffffu, send, off);
            if (lane >= off) {
                end += o;
                send += q;
            }
        }
        chunk = __shfl_sync(0xffffffffu, end, 31);
        schunk = __shfl_sync(0xffffffffu, send, 31);
    }

    __device__ __forceinline__ void init(const AttnBatch& p) {
        const int lane = threadIdx.x & 31;
        L = 0x7fffffff;
        most = total = cut = 0;
        long long rows = 0;
        const int chunks = (p.B + 31) >> 5;
#pragma unroll
        for (int k = 0; k < kSeqCache; ++k) {
            const SeqUnits u = seq_units(p, p.B - 1 - 32 * k - lane, blockIdx.x == 0);
            seq_first[k] = u.first;
            seq_n[k] = u.n;
            seq_kv[k] = u.kv_len;
        }
        for (int c = 0; c < chunks; ++c) {
            const SeqUnits u = seq(p, c);
            if (c >= kSeqCache && blockIdx.x == 0) seq_units(p, p.B - 1 - 32 * c - lane, true);
            if (u.n > 0) {
                rows += u.n;
                most = max(most, u.tiles());
                total += u.all(p) * p.n_kv;
            }
        }
        total = __reduce_add_sync(0xffffffffu, total);
        most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) rows += __shfl_xor_sync(0xffffffffu, rows, off);
        // first rows that do not ascend may name more units than there is room for: no items
        if (rows > p.T) {
            if (lane == 0) record_bad_arg(p.err);
            total = 0;
            return;
        }
        if (p.split && most > kMinPart && total <= kCutUnits) {
            // lane: choice lane & 7, of the sequences 4 k + lane / 8
            const int i = lane % kMaxParts, len = max(kMinPart, (most + i) / (i + 1));
            int items = 0, of_cut = 0;
            L = len;
#pragma unroll 1
            for (int c = 0; c < chunks; ++c) {
                const SeqUnits u = seq(p, c);
                const int units = u.all(p) * p.n_kv, tiles = u.tiles();
                const unsigned some = __ballot_sync(0xffffffffu, units > 0);
#pragma unroll 1
                for (int k = 0; k < 32; k += 4) {
                    if ((some >> k & 15u) == 0) continue;
                    const int parts = parts_of(__shfl_sync(0xffffffffu, tiles, k + lane / kMaxParts));
                    const int count = __shfl_sync(0xffffffffu, units, k + lane / kMaxParts) * parts;
                    items += count;
                    if (parts > 1) of_cut += count;
                }
            }
#pragma unroll
            for (int off = 16; off >= kMaxParts; off >>= 1) {
                items += __shfl_xor_sync(0xffffffffu, items, off);
                of_cut += __shfl_xor_sync(0xffffffffu, of_cut, off);
            }
            const int ctas = gridDim.x;
            float cost = (float)((items + ctas - 1) / ctas) * ((float)len + 2.f) + 0.33f * i;
            if (items - total > kMaxExtra) cost = INFINITY;   // (never the first: no parts)
            float best = cost;
#pragma unroll
            for (int off = kMaxParts / 2; off >= 1; off >>= 1) best = fminf(best, __shfl_xor_sync(0xffffffffu, best, off));
            const int pick = __ffs(__ballot_sync(0xffffffffu, cost == best)) - 1;
            L = __shfl_sync(0xffffffffu, len, pick);
            total = __shfl_sync(0xffffffffu, items, pick);
            cut = __shfl_sync(0xffffffffu, of_cut, pick);
        }
        bucket = kBuckets - 1;
        b0 = p.B - 1;
        before = slots = 0;
        load(p);
    }

    // item x (ascending from call to call); false when this one has no work
    __device__ __forceinline__ bool get(const AttnBatch& p, int x, TileItem& it) {
        while (before + chunk <= x) {
            before += chunk;
            slots += schunk;
            b0 -= 32;
            if (b0 < 0) {
                if (--bucket < 0) return false;   // (x < total: a chunk holds it)
                b0 = p.B - 1;
            }
            load(p);
        }
        const int l = __ffs(__ballot_sync(0xffffffffu, before + end > x)) - 1;
        const int np = __shfl_sync(0xffffffffu, parts, l), nu = __shfl_sync(0xffffffffu, units, l);
        const int in = x - before - __shfl_sync(0xffffffffu, end - count, l);
        const int u = np == 1 ? in : (int)((unsigned)in / (unsigned)np), part = in - u * np;   // unit of the class's, from its end
        const int ul = (int)((unsigned)u / (unsigned)p.n_kv);
        const int slot = slots + __shfl_sync(0xffffffffu, send - split, l) + u * np;
        const int tpt = p.row_tile_tokens;
        it.seq = b0 - l;
        it.g = u - ul * p.n_kv;
        const int tok0 = (__shfl_sync(0xffffffffu, low, l) + nu - 1 - ul) * p.tokens_per_tile;
        const int first = __shfl_sync(0xffffffffu, this->first, l), n = __shfl_sync(0xffffffffu, this->n, l);
        it.kv_len = __shfl_sync(0xffffffffu, kv_len, l);
        it.kv_row0 = p.kv_lens ? 0 : first;
        it.row0 = first + tok0;
        it.see0 = it.kv_len - n + tok0 + 1;
        it.kv_end = 0;
        int nt[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            it.ntok[t] = max(0, min(tpt, min(n - tok0, p.tokens_per_tile) - t * tpt));
            const int see = it.ntok[t] ? max(0, min(it.kv_len, it.see0 - 1 + t * tpt + it.ntok[t])) : 0;
            nt[t] = (see + kTile - 1) / kTile;
            it.kv_end = max(it.kv_end, see);
        }
        // a tile early in its sequence has fewer parts
        const int all = max(nt[0], nt[1]);
        it.part = part;
        it.parts = min(np, parts_of(all));
        it.slot = slot;
        if (np > 1 && (threadIdx.x & 31) == 0)
            *tile_unit(p, slot + part) = TileUnit{part == 0 && it.parts > 1 ? it.parts : 0, it.g, it.row0, it.see0, it.kv_len,
                                                  {it.ntok[0], it.ntok[1]}};
        if (part >= it.parts) return false;
        it.j0 = 0;
        it.ntiles = all;
        if (it.parts > 1) {   // (fewer than 2^24 tiles, eight parts)
            it.j0 = (int)((unsigned)(all * part) / (unsigned)it.parts);
            it.ntiles = (int)((unsigned)(all * (part + 1)) / (unsigned)it.parts) - it.j0;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) it.nt[t] = max(0, min(nt[t], it.j0 + it.ntiles) - it.j0);
        return true;
    }
};

// The scheduler warp: hands the CTA's items out, an end marker behind them.  After a
// wait that gave up it hands out no more but walks on, as every place of the workspace
// that the joining launch reads is written on this walk.
__device__ __forceinline__ void hand_out_items(const AttnBatch& p, TilesSmem& S) {
    const int lane = threadIdx.x & 31;
    ItemWalk w;
    w.init(p);
    if (p.split && blockIdx.x == 0 && lane == 0) *tile_places(p) = min(w.cut, p.slots);
    const int ctas = gridDim.x, c = blockIdx.x;
    bool ok = true;
    int i = 0;
    for (int r = 0;; ++r) {
        const int x = r * ctas + ((r & 1) ? ctas - 1 - c : c);
        TileItem it;
        if (r * ctas >= w.total) it.seq = -1;
        else if (x >= w.total || !w.get(p, x, it)) continue;
        if (ok) {
            const int buf = i % kItemBufs;
            ok = mbar_wait_backoff(&S.item_empty[buf], ((uint32_t)(i / kItemBufs) & 1u) ^ 1u, p.err, kDevTimeoutEmpty, 64);
            ok = __all_sync(0xffffffffu, ok);
            if (ok && lane == 0) {
                S.item[buf] = it;
                mbar_arrive(&S.item_full[buf]);
            }
            __syncwarp();
            ++i;
        }
        if (it.seq < 0) break;
    }
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
__device__ __forceinline__ uint4 mul_pairs(uint64_t a, uint64_t b, uint64_t c) {
    uint4 u;
    asm("{\n\t.reg .b64 t;\n\tmul.rn.f32x2 t, %4, %6;\n\tmov.b64 {%0, %1}, t;\n\tmul.rn.f32x2 t, %5, %6;\n\t"
        "mov.b64 {%2, %3}, t;\n\t}"
        : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
        : "l"(a), "l"(b), "l"(c));
    return u;
}
// Four lanes' 16-byte pieces of their rows, turned: u[i] becomes piece `lane & 3` of
// row i of the four, so that a store of the four covers 64 bytes of a row (an item's
// epilogue 4,000 cycles; 4,000 to 5,600 with stores of one row a lane, 32 lines each).
__device__ __forceinline__ uint4 shfl_xor4(const uint4& a, int x) {
    return make_uint4(__shfl_xor_sync(0xffffffffu, a.x, x), __shfl_xor_sync(0xffffffffu, a.y, x),
                      __shfl_xor_sync(0xffffffffu, a.z, x), __shfl_xor_sync(0xffffffffu, a.w, x));
}
__device__ __forceinline__ uint4 pick4(bool c, const uint4& a, const uint4& b) {
    return make_uint4(c ? a.x : b.x, c ? a.y : b.y, c ? a.z : b.z, c ? a.w : b.w);
}
__device__ __forceinline__ void turn_pieces(uint4 (&u)[4]) {
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        const bool up = threadIdx.x & x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (!(i & x)) {
                const uint4 r = shfl_xor4(pick4(up, u[i], u[i + x]), x);
                u[i] = pick4(up, r, u[i]);
                u[i + x] = pick4(up, u[i + x], r);
            }
    }
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
    float a[16];
#pragma unroll
    for (int e = 0; e < 16; e += 2) exp_pair(r[e], r[e + 1], f, mu, a[e], a[e + 1]);
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
        add_pair((e & 2) ? s1 : s0, a[e], a[e + 1]);
        split2(a[e], a[e + 1], hi[e >> 1], lo[e >> 1]);
    }
    TMEM_ST8(col, hi);
    TMEM_ST8(col + 8, lo);
}

// fp16 queries: the two warpgroups take turns at the exponentials, one row tile's
// run while the other's products do.  Warpgroup 0 starts; a turn is passed on before
// the last quarter.  Without turns (48 query heads over 8): 3.6 against 3.4 ms over
// 16,384 tokens, 188 against 163 us over 11 prompts of 1 to 2,048.  fp32 queries are
// 5 % faster without (40 heads over 8, three documents of 1,777 to 4,099 tokens:
// 491 against 516 us; 512 tokens against 32,513 keys: 595 against 630 us).
struct Turn {
    uint64_t *mine, *other;   // other null: this tile has no partner
    uint32_t phase;
    bool wait;
    int* err;
    __device__ __forceinline__ bool take() const {
        return !wait || mbar_wait_spin(mine, phase, err, kDevTimeoutFull);
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
// rolled: unrolled, all the loads move to the top and their values spill (the kernel as
// it is still stores 40 bytes a thread and loads 64, by ptxas' count).  MASK:
// keys at or past lim count as -inf.  Returns the rescale of what came before.
template <bool MASK>
__device__ __forceinline__ float softmax_row(uint32_t trow, int lim, float f, float& m, float& l, uint64_t* p_full) {
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
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
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
// (the weights, kept as 2^kShift16 p, then reach 2^15, inside fp16): after the
// first tiles that hardly happens (a lag of 2^5 was overtaken by one of a warp's
// 32 rows in most tiles).
constexpr float kShift16 = 4.f, kLazy = 11.f;
template <bool MASK>
__device__ __forceinline__ void softmax_row_f16(uint32_t trow, uint32_t orow, int lim, float f, bool first, float& m, float& l,
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
    const bool grow = top > m + kLazy;
    if (__any_sync(0xffffffffu, grow)) {   // each row by itself: its result does not depend on its neighbours
        const float corr = grow ? ex2(m - top) : 1.f;
        m = grow ? top : m;
        l *= corr;
        if (!first) {   // S of this tile is there, so the product before it is done
            const uint64_t corr2 = pair(corr, corr);
#pragma unroll 1
            for (int c = 0; c < kHd; c += 16) {
                uint32_t r[16];
                TMEM_LD16(orow + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e += 2) mul_pair(r[e], r[e + 1], corr2);
                TMEM_ST16(orow + c, r);
            }
        }
    }
    const float mu = m == -INFINITY ? 0.f : m - kShift16;
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

// Bounded wait for a counter that only grows (a row tile may run ahead of the other
// by any number of key tiles, which a barrier's one phase bit cannot tell).
__device__ __forceinline__ bool wait_reads(const int* count, int target, int* err) {
    const uint32_t a = smem_u32(count);
    uint64_t t0 = 0;
    for (int i = 0;; ++i) {
        int v;
        asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
        if (v >= target) return true;
        if (i == 0) t0 = global_timer_ns();
        else if ((i & 31) == 0 && global_timer_ns() - t0 > kWaitLimitNs) break;
    }
    if (err) atomicExch(err, kDevTimeoutFull);
    return false;
}

// fp32 queries of a row tile (a warp's 32 rows): scaled, their high halves to shared
// memory (64 dims a 128-byte swizzled row) and their low halves, by way of the same
// place, to tensor memory.
__device__ __forceinline__ void load_queries(const AttnBatch& p, TilesSmem& S, uint8_t* qt, uint32_t qlo, int t, int wrow,
                                             int rows, int64_t tok_first, int g) {
    const int lane = threadIdx.x & 31, c = lane >> 1;
    float4 a[32];
    {
        const int tok = wrow / p.G;
        int h = wrow - tok * p.G;
        const float* src = static_cast<const float*>(p.q) + (tok_first + tok) * p.q_stride + (int64_t)(g * p.G + h) * kHd;
        const int64_t next_token = p.q_stride - (int64_t)(p.G - 1) * kHd;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            a[i] = wrow + i < rows ? __ldg(reinterpret_cast<const float4*>(src) + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
            const bool wrap = ++h == p.G;
            src += wrap ? next_token : kHd;
            h = wrap ? 0 : h;
        }
    }
    // largest value of each row: 32 values a lane to one, lane i row i, by halving
    // (31 shuffles; a butterfly a row takes 160)
    float v[16];
    {
        auto top = [&](int i) {
            return fmaxf(fmaxf(fabsf(a[i].x), fabsf(a[i].y)), fmaxf(fabsf(a[i].z), fabsf(a[i].w)));
        };
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = top(i), y = top(16 + i);
            v[i] = fmaxf(lane & 16 ? y : x, __shfl_xor_sync(0xffffffffu, lane & 16 ? x : y, 16));
        }
#pragma unroll
        for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
            for (int i = 0; i < w; ++i)
                v[i] = fmaxf(lane & w ? v[w + i] : v[i], __shfl_xor_sync(0xffffffffu, lane & w ? v[i] : v[w + i], w));
    }
    float up, fr;
    row_scale(v[0], p.scale_log2, up, fr);
    S.f[t][wrow + lane] = fr;
    uint8_t* d0 = qt + (c >> 3) * (kTileBytes / 2) + wrow * 128 + (lane & 1) * 8;
    uint2 hi[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const float u = __shfl_sync(0xffffffffu, up, i);
        uint2 lo;
        split2(a[i].x * u, a[i].y * u, hi[i].x, lo.x);
        split2(a[i].z * u, a[i].w * u, hi[i].y, lo.y);
        *reinterpret_cast<uint2*>(d0 + i * 128 + (((c & 7) ^ (i & 7)) << 4)) = lo;
    }
    __syncwarp();
    // the thread's own row of low halves: 64 columns of fp16 pairs
    const uint8_t* mine = qt + (wrow + lane) * 128;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 v = lds128(mine + h * (kTileBytes / 2) + (((4 * q + k) ^ (lane & 7)) << 4));
                w[4 * k] = v.x;
                w[4 * k + 1] = v.y;
                w[4 * k + 2] = v.z;
                w[4 * k + 3] = v.w;
            }
            TMEM_ST16(qlo + 32 * h + 16 * q, w);
        }
    tmem_wait_st();
    tc_before();
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; ++i) *reinterpret_cast<uint2*>(d0 + i * 128 + (((c & 7) ^ (i & 7)) << 4)) = hi[i];
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&S.q_full[t]);
}

// A partial: [row tile][32 groups of 4 dims][128 rows][4], then (maximum, sum) of each
// row: a warp's rows are neighbours, for the thread that holds one and for the join.
template <typename T>
__device__ __forceinline__ auto part_at(T* part, int t, int d4, int row) {
    using V = std::conditional_t<std::is_const_v<T>, const float4, float4>;
    return reinterpret_cast<V*>(part) + (t * (kHd / 4) + d4) * kTcRows + row;
}

// Joins the parts of the units that were cut: 32 rows of a unit at a time, a row a
// lane, a warp four groups of four dims.
constexpr int kJoinCtas = 4 * 148;
template <bool F32>
__global__ void __launch_bounds__(256, 4) attn_tiles_join_kernel(const __grid_constant__ AttnBatch p) {
    grid_dep_wait();
    const int places = *tile_places(p), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tpt = p.row_tile_tokens;
    for (int w = blockIdx.x; w < 8 * places; w += kJoinCtas) {
        const TileUnit u = *tile_unit(p, w >> 3);
        const int t = (w >> 2) & 1, row = 32 * (w & 3) + lane;
        if (u.parts == 0 || row >= u.ntok[t] * p.G) continue;
        const float* part0 = p.tile_work + (size_t)(w >> 3) * kTilePartFloats;
        const int tok = row / p.G;
        const int64_t off = (int64_t)(u.row0 + t * tpt + tok) * p.out_stride + (int64_t)(u.g * p.G + row - tok * p.G) * kHd;
        float k[kMaxParts], M = -INFINITY, L = 0.f;
        float2 ml[kMaxParts];
#pragma unroll
        for (int i = 0; i < kMaxParts; ++i)
            ml[i] = i < u.parts ? *(reinterpret_cast<const float2*>(part0 + (size_t)i * kTilePartFloats + 2 * kTcRows * kHd) +
                                    kTcRows * t + row)
                                : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int i = 0; i < kMaxParts; ++i) M = fmaxf(M, ml[i].x);
#pragma unroll
        for (int i = 0; i < kMaxParts; ++i) {
            k[i] = ml[i].x == -INFINITY ? 0.f : ex2(ml[i].x - M);
            L = fmaf(k[i], ml[i].y, L);
        }
        const bool none = min(u.kv_len, u.see0 + t * tpt + tok) <= 0;   // a row that sees no key: zeros
        const float inv = none ? 0.f : rcp(L);
#pragma unroll 2
        for (int d = 4 * warp; d < 4 * warp + 4; ++d) {
            float4 y[kMaxParts], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < kMaxParts; ++c)
                y[c] = c < u.parts ? *part_at(part0 + (size_t)c * kTilePartFloats, t, d, row) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < kMaxParts; ++c)
                acc = make_float4(fmaf(y[c].x, k[c], acc.x), fmaf(y[c].y, k[c], acc.y), fmaf(y[c].z, k[c], acc.z),
                                  fmaf(y[c].w, k[c], acc.w));
            store_pair<F32>(p.out, off + 4 * d, make_float2(acc.x, acc.y), inv, none);
            store_pair<F32>(p.out, off + 4 * d + 2, make_float2(acc.z, acc.w), inv, none);
        }
    }
}

template <bool F32>
__global__ void __launch_bounds__(kTcThreads, 1)
    attn_tiles_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv, const __grid_constant__ AttnBatch p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* qs = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);   // fp16 queries or high halves, [row tile][2 x 64 dims][128 rows]
    uint8_t* ring = qs + 2 * kTileBytes;
    TilesSmem& S = *reinterpret_cast<TilesSmem*>(ring + kSlots * kTileBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&S.kv_full[i], 1);
            mbar_init(&S.kv_empty[i], 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&S.s_full[t], 1);
            mbar_init(&S.p_full[t][0], 4);
            mbar_init(&S.p_full[t][1], 4);
            mbar_init(&S.o_full[t], 1);
            S.reads[t] = 0;
            mbar_init(&S.turn[t], 4);
            mbar_init(&S.q_full[t], F32 ? 4 : 1);
            mbar_init(&S.q_free[t], 1);
            mbar_init(&S.drain[t], 1);
        }
        mbar_init(&S.landed, 1);
        for (int i = 0; i < kItemBufs; ++i) {
            mbar_init(&S.item_full[i], 1);
            mbar_init(&S.item_empty[i], 11);   // TMA, two issuers, eight softmax warps
        }
        fence_mbar_init();
    }
    if (warp == 8 && lane == 0) {
        if (!F32) asm volatile("prefetch.tensormap [%0];" ::"l"(&tq) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tv) : "memory");
    }
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
    grid_dep_launch_dependents();
    const int tpt = p.row_tile_tokens;   // tokens per row tile

    // the i-th item of the CTA, for a role (a whole warp): false at the end
    auto take = [&](int i, bool& ok) {
        const int buf = i % kItemBufs;
        ok = mbar_wait(&S.item_full[buf], (uint32_t)(i / kItemBufs) & 1u, p.err, kDevTimeoutFull);
        ok = __all_sync(0xffffffffu, ok);
        return ok && S.item[buf].seq >= 0;
    };
    auto give = [&](int i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.item_empty[i % kItemBufs]);
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 11) {
            // ------------------------------------------------------- next items
            hand_out_items(p, S);
        } else if (warp == 8) {
            // --------------------------------------------- Q (fp16), K and V tiles
            const int ps = 1 << p.ps_log2, nbox = kTile / p.box_rows, halves = nbox == 1 ? 1 : 2;
            const int box = lane / halves, half = lane - box * halves;
            bool ok = true;
            int slot = 0, landings = 0;         // K and V tiles so far, last ones of items among them
            int nq[2] = {0, 0};
            for (int i = 0; ok && take(i, ok); ++i) {
                const TileItem& it = S.item[i % kItemBufs];
                for (int j = 0; j < it.ntiles && ok; ++j) {
                    const int r0 = (it.j0 + j) * kTile + box * p.box_rows;
                    const bool mine = box < nbox && r0 < it.kv_end;
                    const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
                    const uint32_t bytes = (uint32_t)(boxes * p.box_rows * (nbox == 1 ? 256 : 128));
                    int page = 0, row = it.kv_row0 + r0;
                    if (mine && p.table) {
                        page = p.table[(long long)it.seq * p.max_pages + (r0 >> p.ps_log2)];
                        row = r0 & (ps - 1);
                        if ((unsigned)page >= (unsigned)p.n_pages) {  // reads as zeros
                            record_bad_arg(p.err);
                            page = p.n_pages;
                        }
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m, ++slot) {
                        const int st = slot % kSlots;
                        ok = mbar_wait_backoff(&S.kv_empty[st], ((uint32_t)(slot / kSlots) & 1u) ^ 1u, p.err,
                                               kDevTimeoutEmpty, 32);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        // values past the last key may be anything, NaN included: zeros
                        // before the tensor core reads them, so that tile lands on a
                        // barrier of its own
                        const bool tail = m == 1 && j == it.ntiles - 1 && it.kv_end < (it.j0 + j + 1) * kTile;
                        uint64_t* bar = tail ? &S.landed : &S.kv_full[st];
                        if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
                        __syncwarp();
                        uint8_t* dst = ring + st * kTileBytes;
                        if (mine)
                            tma_load_kv(dst + half * (kTileBytes / 2) + box * p.box_rows * 128, m ? &tv : &tk, half, row, it.g,
                                        page, bar);
                        __syncwarp();
                        if (!F32 && m == 0 && j == 0) {   // the queries, once the products on the last ones are done
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                if (it.nt[t] > 0) {
                                    if (nq[t]) ok = ok && mbar_wait(&S.q_free[t], (uint32_t)(nq[t] - 1) & 1u, p.err, kDevTimeoutEmpty);
                                    ++nq[t];
                                    if (ok && lane == 0) {
                                        mbar_arrive_expect_tx(&S.q_full[t], (uint32_t)(2 * tpt * p.G * 128));
                                        for (int h = 0; h < 2; ++h)
                                            tma_load_q(qs + t * kTileBytes + h * (kTileBytes / 2), &tq, it.g * p.G,
                                                       it.row0 + t * tpt, h, &S.q_full[t]);
                                    }
                                }
                            ok = __all_sync(0xffffffffu, ok);
                        }
                        if (tail) {
                            ok = ok && mbar_wait(&S.landed, (uint32_t)landings & 1u, p.err, kDevTimeoutFull);
                            ++landings;
                            for (int r = it.kv_end - (it.j0 + j) * kTile + (lane >> 3); r < kTile; r += 4)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    *reinterpret_cast<uint4*>(dst + h * (kTileBytes / 2) + r * 128 + (lane & 7) * 16) =
                                        make_uint4(0u, 0u, 0u, 0u);
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&S.kv_full[st]);
                            ok = __all_sync(0xffffffffu, ok);
                        }
                    }
                }
                give(i);
            }
            // the copies in flight land before the CTA can exit
            if (lane == 0) {
                drain_issued_stages(S.kv_full, kSlots, slot, kWaitLimitNs);
                if (!F32)
                    for (int t = 0; t < 2; ++t)
                        if (nq[t]) mbar_wait(&S.q_full[t], (uint32_t)(nq[t] - 1) & 1u, nullptr, 0);
            }
        } else {
            // ------------------------------------------------------------- MMA
            // One issuer per row tile: an issuing thread's waits queue behind its
            // own products (~200 cycles each, measured), and the other issuer's
            // products run meanwhile.
            const int t = warp - 9;
            const uint32_t qb = desc_k(smem_u32(qs + t * kTileBytes));
            const uint32_t s_col = tmem + 128u * t, o_col = tmem + kColO + (F32 ? 0u : 128u * t), q_col = tmem + kColQlo + 64u * t;
            auto wait_kv = [&](int i) {
                return mbar_wait_spin(&S.kv_full[i % kSlots], (uint32_t)(i / kSlots) & 1u, p.err, kDevTimeoutFull);
            };
            auto qk = [&](int i) {   // S = Q K^T
                const uint32_t kb = desc_k(smem_u32(ring + (i % kSlots) * kTileBytes));
#pragma unroll
                for (int part = F32 ? 1 : 0; part >= 0; --part)
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t off = ((uint32_t)(ks >> 2) * (kTileBytes / 2) + (uint32_t)(ks & 3) * 32u) >> 4;
                        const uint32_t acc = (ks == 0 && part == (F32 ? 1 : 0)) ? 0u : 1u;
                        if (part) mma_ts(s_col, q_col + 8u * ks, kb + off, kIdescS, acc);
                        else mma_ss(s_col, qb + off, kb + off, kIdescS, acc);
                    }
                tc_arrive(&S.s_full[t]);
            };
            auto pv = [&](int i, int half, bool fresh) {   // PV (+)= P V over 64 of the tile's keys
                const uint32_t vb = desc_mn(smem_u32(ring + (i % kSlots) * kTileBytes)) + (uint32_t)half * (8192u >> 4);
#pragma unroll
                for (int part = F32 ? 1 : 0; part >= 0; --part)
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const uint32_t col = (uint32_t)(4 * half + ks) * (F32 ? 16u : 8u) + 8u * part;
                        mma_ts(o_col, s_col + col, vb + (uint32_t)ks * (2048u >> 4), kIdescO,
                               (fresh && ks == 0 && part == (F32 ? 1 : 0)) ? 0u : 1u);
                    }
            };
            bool ok = true;
            int slot = 0, tiles = 0, nq = 0, others = 0;   // ring places, this row tile's key tiles, queries, the other's tiles
            for (int i = 0; ok && take(i, ok); ++i) {
                const TileItem& it = S.item[i % kItemBufs];
                const int mine = it.nt[t], theirs = it.nt[t ^ 1];
                if (lane == 0 && it.ntiles > 0) {
                    if (mine > 0) ok = mbar_wait_spin(&S.q_full[t], (uint32_t)nq & 1u, p.err, kDevTimeoutFull);
                    ok = ok && wait_kv(slot);
                    tc_after();
                    if (ok) {
                        if (mine > 0) qk(slot);
                        if (mine == 1) tc_arrive(&S.q_free[t]);
                        tc_arrive(&S.kv_empty[slot % kSlots]);
                    }
                    for (int j = 0; j < it.ntiles && ok; ++j) {
                        const int iv = slot + 2 * j + 1, ik = iv + 1;
                        const bool more = j + 1 < it.ntiles;
                        ok = wait_kv(iv);
                        // the next keys too, while the weights are on their way
                        if (ok && more) ok = wait_kv(ik);
                        if (j < mine) {
                            if (F32) {   // the other row tile's last PV has been read
                                const int reads = others + min(j + t, theirs);
                                if (reads) ok = ok && wait_reads(&S.reads[t ^ 1], 4 * reads, p.err);
                            }
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                ok = ok && mbar_wait_spin(&S.p_full[t][half], (uint32_t)(tiles + j) & 1u, p.err, kDevTimeoutFull);
                                if (!ok) break;
                                tc_after();
                                pv(iv, half, half == 0 && (F32 || j == 0));
                            }
                            if (!ok) break;
                            if (F32 || j + 1 == mine) tc_arrive(&S.o_full[t]);
                            if (j + 1 < mine) qk(ik);
                            if (j + 2 == mine) tc_arrive(&S.q_free[t]);
                        }
                        if (!ok) break;
                        tc_arrive(&S.kv_empty[iv % kSlots]);
                        if (more) tc_arrive(&S.kv_empty[ik % kSlots]);
                    }
                    nq += mine > 0;
                    tiles += mine;
                    others += theirs;
                    slot += 2 * it.ntiles;
                }
                give(i);
                ok = __all_sync(0xffffffffu, ok);
            }
            // every product is done before the CTA frees its tensor memory
            if (lane == 0) {
                tc_arrive(&S.drain[t]);
                mbar_wait(&S.drain[t], 0, nullptr, 0, kWaitLimitNs);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2, wrow = 32 * (warp & 3), row = wrow + lane, tok = row / p.G;
        const uint32_t trow = tmem + 128u * t + ((uint32_t)wrow << 16);
        const uint32_t orow = tmem + kColO + (F32 ? 0u : 128u * t) + ((uint32_t)wrow << 16);
        int tiles = 0, outs = 0, turns = 0;
        bool ok = true;
        for (int i = 0; ok && take(i, ok); ++i) {
            const TileItem& it = S.item[i % kItemBufs];
            const int rows = it.ntok[t] * p.G, nt = it.nt[t];
            if (F32 && nt > 0)
                load_queries(p, S, qs + t * kTileBytes, tmem + kColQlo + 64u * t + ((uint32_t)wrow << 16), t, wrow, rows,
                             it.row0 + t * tpt, it.g);

            // --------------------------------------------------------- softmax
            const bool live = row < rows;
            const int see = it.see0 + t * tpt;                       // keys the row tile's first token sees
            const int lim = live ? max(0, min(it.kv_len, see + tok)) : 0, lim0 = max(0, see);
            const float f = F32 ? S.f[t][row] : p.scale_log2;
            // (addresses are formed after the loops, which need the registers)
            auto out_off = [&] {
                return ((int64_t)it.row0 + t * tpt + tok) * p.out_stride + (int64_t)(it.g * p.G + row - tok * p.G) * kHd;
            };
            // rows of the thread's group of four lanes
            auto four_rows = [&](int64_t (&off)[4], bool (&on)[4]) {
                const int64_t mine = out_off();
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    off[e] = __shfl_sync(0xffffffffu, mine, (lane & ~3) + e);
                    on[e] = wrow + (lane & ~3) + e < rows;
                }
            };
            auto part_out = [&] { return p.tile_work + (size_t)(it.slot + it.part) * kTilePartFloats; };
            float m = -INFINITY, l = 0.f;
            const int both = min(it.nt[0], it.nt[1]);
            auto turn_of = [&](int j) {   // warpgroup 0 waits for 1's last turn, 1 for 0's of the same tile
                const int n = turns + j;
                return Turn{&S.turn[t], j < both ? &S.turn[t ^ 1] : nullptr, (uint32_t)(n - 1 + t) & 1u,
                            j < both && n + t > 0, p.err};
            };
            if constexpr (F32) {
                uint64_t o[kHd / 2];   // the row's outputs in pairs
#pragma unroll
                for (int d = 0; d < kHd / 2; ++d) o[d] = 0;
                for (int j = 0; j < nt; ++j) {
                    const uint32_t ph = (uint32_t)(tiles + j) & 1u;
                    ok = mbar_wait_spin(&S.s_full[t], ph, p.err, kDevTimeoutFull);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_after();
                    const int k0 = (it.j0 + j) * kTile;
                    const float corr = k0 + kTile > lim0 ? softmax_row<true>(trow, lim - k0, f, m, l, S.p_full[t])
                                                         : softmax_row<false>(trow, 0, f, m, l, S.p_full[t]);
                    ok = mbar_wait_spin(&S.o_full[t], ph, p.err, kDevTimeoutFull);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_after();
                    const uint64_t corr2 = pair(corr, corr);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        // the barrier once more: a branch that keeps the later loads from
                        // moving to the top, where their values would spill
                        if (c == 2 && !mbar_wait_spin(&S.o_full[t], ph, p.err, kDevTimeoutFull)) ok = false;
                        uint32_t r[32];
                        TMEM_LD32(orow + 32 * c, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) fma_pair(o[16 * c + e], corr2, r[2 * e], r[2 * e + 1]);
                    }
                    tc_before();
                    __syncwarp();
                    if (lane == 0)
                        asm volatile("red.release.cta.shared::cta.add.s32 [%0], 1;" ::"r"(smem_u32(&S.reads[t])) : "memory");
                }
                if (ok && it.parts > 1) {   // unnormalised, to the workspace
                    if (live) {
                        float* x = part_out();
                        *reinterpret_cast<float2*>(x + 2 * kTcRows * kHd + 2 * (kTcRows * t + row)) = make_float2(m, l);
                        const uint64_t one = pair(1.f, 1.f);
#pragma unroll
                        for (int e = 0; e < kHd / 2; e += 2)
                            store_f32(reinterpret_cast<uint4*>(part_at(x, t, e / 2, row)), o[e], o[e + 1], one);
                    }
                } else if (ok && rows > wrow) {
                    int64_t off[4];
                    bool on[4];
                    four_rows(off, on);
                    const bool some = lim > 0;   // no key seen: zeros
                    const float rl = rcp(l);
                    const uint64_t inv = pair(rl, rl);
#pragma unroll
                    for (int e = 0; e < kHd / 2; e += 8) {
                        uint4 u[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            u[k] = pick4(some, mul_pairs(o[e + 2 * k], o[e + 2 * k + 1], inv), make_uint4(0u, 0u, 0u, 0u));
                        turn_pieces(u);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (on[k])
                                *reinterpret_cast<uint4*>(static_cast<float*>(p.out) + off[k] + 2 * e + 4 * (lane & 3)) = u[k];
                    }
                }
            } else {
                for (int j = 0; j < nt; ++j) {
                    ok = mbar_wait_spin(&S.s_full[t], (uint32_t)(tiles + j) & 1u, p.err, kDevTimeoutFull);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_after();
                    const Turn turn = turn_of(j);
                    const int k0 = (it.j0 + j) * kTile;
                    if (k0 + kTile > lim0)
                        softmax_row_f16<true>(trow, orow, lim - k0, f, j == 0, m, l, S.p_full[t], turn, ok);
                    else
                        softmax_row_f16<false>(trow, orow, 0, f, j == 0, m, l, S.p_full[t], turn, ok);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                if (ok && nt > 0) {
                    ok = mbar_wait_spin(&S.o_full[t], (uint32_t)outs & 1u, p.err, kDevTimeoutFull);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_after();
                    ++outs;
                }
                if (ok) {
                    if (it.parts > 1 && live)
                        *reinterpret_cast<float2*>(part_out() + 2 * kTcRows * kHd + 2 * (kTcRows * t + row)) = make_float2(m, l);
                    const float rl = rcp(l);
                    int64_t off[4];
                    bool on[4];
                    four_rows(off, on);
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t r[32];
                        if (nt > 0) TMEM_LD32(orow + 32 * c, r);
                        tmem_wait_ld();
                        if (it.parts > 1) {   // unnormalised, to the workspace
                            uint4* x = reinterpret_cast<uint4*>(part_at(part_out(), t, 8 * c, row));
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                if (live)
                                    x[(e >> 2) * kTcRows] = nt > 0 ? make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3])
                                                                   : make_uint4(0u, 0u, 0u, 0u);
                            __syncwarp();
                            continue;
                        }
                        uint4 u[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            u[k] = make_uint4(0u, 0u, 0u, 0u);
                            if (lim > 0) {
                                const uint32_t* v = r + 8 * k;
                                u[k].x = pack2(__uint_as_float(v[0]) * rl, __uint_as_float(v[1]) * rl);
                                u[k].y = pack2(__uint_as_float(v[2]) * rl, __uint_as_float(v[3]) * rl);
                                u[k].z = pack2(__uint_as_float(v[4]) * rl, __uint_as_float(v[5]) * rl);
                                u[k].w = pack2(__uint_as_float(v[6]) * rl, __uint_as_float(v[7]) * rl);
                            }
                        }
                        turn_pieces(u);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (on[k])
                                *reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + off[k] + 32 * c + 8 * (lane & 3)) = u[k];
                    }
                    tc_before();   // the next item's products may overwrite the outputs
                }
            }
            tiles += nt;
            turns += both;
            give(i);
        }
    }
    tc_before();
    if (p.rows_take > 0 && threadIdx.x == 0) grid_dep_wait();   // what follows this launch waits for the row kernel too
    __syncthreads();
    if (warp == 9) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTcCols) : "memory");
    }
}

template <bool F32>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p, long long items,
           cudaStream_t st) {
    constexpr int smem = tiles_smem_bytes<F32>();
    static_assert(smem <= 232448, "shared memory of a CTA");
    cudaError_t e = cudaFuncSetAttribute(attn_tiles_kernel<F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.stream = st;
    cfg.attrs = attr;
    if (e == cudaSuccess) {
        // behind the row kernel of the same call: CTAs start as its CTAs leave their SMs
        cfg.gridDim = dim3((unsigned)std::min<long long>(items, 148));
        cfg.blockDim = dim3(kTcThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.numAttrs = p.rows_take > 0 ? 1 : 0;
        e = cudaLaunchKernelEx(&cfg, attn_tiles_kernel<F32>, tq, tk, tv, p);
    }
    if (e == cudaSuccess && p.split) {
        cfg.gridDim = dim3(kJoinCtas);
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, attn_tiles_join_kernel<F32>, p);
    }
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "attention: %s", cudaGetErrorString(e));
    return GLC_OK;
}

}  // namespace

int attn_tiles_launch(bool f32, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnBatch& p,
                      long long items, cudaStream_t st) {
    return f32 ? launch<true>(tq, tk, tv, p, items, st) : launch<false>(tq, tk, tv, p, items, st);
}

}  // namespace glc
