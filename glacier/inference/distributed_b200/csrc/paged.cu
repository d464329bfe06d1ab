// paged.cu -- what fills a paged fp16 KV cache: the page plan of a step (block
// tables and slot maps from request lengths) and the rotary embedding with the
// store of the new keys and values into their slots.
//
// The reference keeps one contiguous cache per stage model
// (IClusterStageModel.ResetKvCache, IClusterStageModel.cs:35) and runs one
// sequence, one token at a time (DistributedPipelineCoordinator.cs:72-137); a
// batch of sequences of different lengths has no counterpart there.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <utility>

#include "common.cuh"
#include "paged.cuh"

namespace glc {

static __device__ int g_paged_err;
static __device__ int g_paged_seen;   // what a poll took from it

// Read and cleared in one step: what another stream records meanwhile is in this
// poll or in the next.
static __global__ void take_error_kernel() { g_paged_seen = atomicExch(&g_paged_err, kDevOk); }

int paged_fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return set_last_error(code, buf);
}

int paged_error_word(int** err) {
    static int* addr[kMaxDevices] = {nullptr};
    static std::mutex mu;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "no CUDA device");
    if (dev < 0 || dev >= kMaxDevices) return paged_fail(GLC_ERR_INVALID_ARG, "device %d out of range", dev);
    std::lock_guard<std::mutex> lk(mu);
    if (!addr[dev]) {
        void* p = nullptr;
        const cudaError_t e = cudaGetSymbolAddress(&p, g_paged_err);
        if (e != cudaSuccess || !p)
            return paged_fail(GLC_ERR_CUDA, "address of the device error word: %s", cudaGetErrorString(e));
        addr[dev] = static_cast<int*>(p);
    }
    *err = addr[dev];
    return GLC_OK;
}

// Driver function by name, looked up once.
template <typename F>
static F driver_fn(const char* name) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint(name, &ptr, cudaEnableDefault, &qr) != cudaSuccess || qr != cudaDriverEntryPointSuccess)
        ptr = nullptr;
    return (F)ptr;
}

int paged_check_devices(std::initializer_list<DevicePtr> ptrs) {
    // (30 ns a pointer; 60 for the runtime's question, asked where this one does not settle it)
    static const auto attribute = driver_fn<CUresult (*)(void*, CUpointer_attribute, CUdeviceptr)>("cuPointerGetAttribute");
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "no CUDA device");
    for (const DevicePtr& d : ptrs) {
        int on = -1;
        if (!d.p || (attribute && attribute(&on, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, (CUdeviceptr)d.p) == CUDA_SUCCESS && on == dev))
            continue;
        cudaPointerAttributes at{};
        if (cudaPointerGetAttributes(&at, d.p) != cudaSuccess) {
            cudaGetLastError();
            return paged_fail(GLC_ERR_INVALID_ARG, "%s is not memory known to CUDA", d.what);
        }
        if (at.type == cudaMemoryTypeUnregistered)
            return paged_fail(GLC_ERR_INVALID_ARG, "%s is not device memory", d.what);
        if (at.type == cudaMemoryTypeDevice && at.device != dev)
            return paged_fail(GLC_ERR_INVALID_ARG, "%s is on device %d, the current device is %d", d.what, at.device, dev);
    }
    return GLC_OK;
}

int paged_check_pages(const glc_kv_pages* c) {
    if (!c || !c->k || !c->v) return paged_fail(GLC_ERR_INVALID_ARG, "null pointer");
    if (c->head_dim != 128) return paged_fail(GLC_ERR_UNSUPPORTED, "head_dim %d (only 128)", c->head_dim);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
        return paged_fail(GLC_ERR_UNSUPPORTED, "page_size %d (16, 32, 64, 128 or 256)", c->page_size);
    if (c->n_pages <= 0 || c->n_kv_heads <= 0)
        return paged_fail(GLC_ERR_INVALID_ARG, "%d pages, %d KV heads", c->n_pages, c->n_kv_heads);
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15u)
        return paged_fail(GLC_ERR_INVALID_ARG, "caches must be 16-byte aligned");
    const int64_t lim = (int64_t)1 << 38;  // halves; a descriptor's strides end at 2^40 bytes
    if (c->page_stride <= 0 || c->head_stride <= 0 || c->row_stride < 128 || c->page_stride >= lim ||
        c->head_stride >= lim || c->row_stride >= lim || ((c->page_stride | c->head_stride | c->row_stride) & 7))
        return paged_fail(GLC_ERR_INVALID_ARG, "cache strides must be positive multiples of 8 elements, rows 128 or more apart");
    return GLC_OK;
}

typedef CUresult (*PFN_encodeTiledKv)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                      const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                      CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int paged_encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                 const cuuint32_t* box) {
    static const auto fn = driver_fn<PFN_encodeTiledKv>("cuTensorMapEncodeTiled");
    if (!fn) return paged_fail(GLC_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box,
                          estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return paged_fail(GLC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return GLC_OK;
}

int paged_tensor_map(CUtensorMap* map, const void* base, int64_t rows, int64_t row_stride, int64_t heads,
                     int64_t head_stride, int64_t pages, int64_t page_stride, int box_rows, int box_halves) {
    const cuuint64_t dims[5] = {64, (cuuint64_t)rows, 2, (cuuint64_t)heads, (cuuint64_t)pages};
    const cuuint64_t strides[4] = {(cuuint64_t)row_stride * 2, 128, (cuuint64_t)head_stride * 2,
                                   (cuuint64_t)page_stride * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_halves, 1, 1};
    return paged_encode(map, base, 5, dims, strides, box);
}

namespace {

// ------------------------------------------------------------------ page plan
// held_i = ceil(ctx_i / ps), want_i = ceil((ctx_i + new_i) / ps).  Three prefix
// sums over the requests: rows (cu), pages given back by finished requests,
// pages needed by the others.  Request i is served when its rows fit T, its
// want fits the table's width and the pages needed up to and including it are
// there; page r of the step is entry top - r of the free list after the
// give-back.
//
// Bound by latency, not by bytes: a few hundred KB at most, behind three
// dependent sums.  Up to kPlanFlat requests (kv_plan_flat_kernel) every CTA forms
// all the sums itself, keeps them in shared memory and writes its share of the
// rows and entries; a page that is given back and taken in the same step is
// looked up in the row it comes from, so no CTA reads what another writes and
// nothing waits.  More requests (kv_plan_kernel) go 1024 at a time through one
// cluster of 8 CTAs, with a cluster barrier between the pages given back and the
// pages taken.
constexpr int kPlanCluster = 8;
constexpr int kPlanFlat = 4096;

struct PlanParams {
    const int32_t* ctx;
    const int32_t* nw;
    int32_t* table;
    int32_t* pool;
    const int32_t* free_in;
    int32_t* free_out;
    int32_t* cu;
    int32_t* kv;
    int32_t* pos;
    int64_t* slots;
    int32_t* status;
    int B, ps_log2, width, capacity, T;
};

// Inclusive prefix sum of v over the CTA's threads; total gets the CTA's sum.
// `part` holds one value per warp; the CTA synchronises twice.
__device__ __forceinline__ long long block_scan(long long v, long long* part, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += o;
    }
    __syncthreads();  // the previous scan's reads of part are done
    if (lane == 31) part[warp] = v;
    __syncthreads();
    long long w = lane < nw ? part[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, w, off);
        if (lane >= off) w += o;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const long long before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    return v + (warp > 0 ? before : 0);
}

// First index in [0, n) whose inclusive end is above x (ends ascending).
template <typename T>
__device__ __forceinline__ int upper(const T* end, int n, T x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int m = (lo + hi) >> 1;
        if (end[m] > x) hi = m;
        else lo = m + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(1024, 1) kv_plan_kernel(const __grid_constant__ PlanParams p) {
    __shared__ long long part[32];
    __shared__ long long row_end[1024];   // inclusive ends of the chunk's rows (or of the pages it gives back)
    __shared__ long long page_end[1024];  // inclusive ends of the pages the chunk's requests take
    __shared__ int s_ctx[1024], s_held[1024], s_ok[1024];
    const int tid = threadIdx.x, nt = blockDim.x;
    uint32_t rank, size;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int ps = 1 << p.ps_log2;
    const long long free0 = min(max(*p.free_in, 0), p.capacity);

    // finished requests push their pages on the free list, in request order
    long long back = 0;
    for (int base = 0; base < p.B; base += nt) {
        const int i = base + tid, nb = min(nt, p.B - base);
        long long give = 0;
        if (i < p.B && p.nw[i] < 0) {
            const long long c = max(p.ctx[i], 0);
            give = min((c + ps - 1) >> p.ps_log2, (long long)p.width);
        }
        long long sum;
        const long long end = block_scan(give, part, sum);
        if (sum) {
            row_end[tid] = end;
            __syncthreads();
            for (long long x = (long long)rank * nt + tid; x < sum; x += (long long)size * nt) {
                const int q = upper(row_end, nb, x);
                const long long at = free0 + back + x;
                const long long col = x - (q ? row_end[q - 1] : 0);
                if (at < p.capacity) p.pool[at] = p.table[(long long)(base + q) * p.width + col];
            }
        }
        back += sum;
    }
    const long long avail = min(free0 + back, (long long)p.capacity);
    // every push is visible to the cluster before any page is taken
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");

    long long rows = 0, need_sum = 0, used = 0;
    int bad = 0;
    for (int base = 0; base < p.B; base += nt) {
        const int i = base + tid, nb = min(nt, p.B - base);
        int ctx = 0, add = 0;
        bool live = false;
        if (i < p.B) {
            ctx = p.ctx[i];
            add = p.nw[i];
            live = add >= 0;
            add = max(add, 0);
        }
        long long sum_rows, sum_need;
        const long long rend = rows + block_scan(add, part, sum_rows);
        const long long held = ((long long)max(ctx, 0) + ps - 1) >> p.ps_log2;
        const long long want = ((long long)max(ctx, 0) + add + ps - 1) >> p.ps_log2;
        const bool fits = live && ctx >= 0 && rend <= p.T && want <= p.width;
        const long long need = fits ? want - held : 0;
        const long long nend = need_sum + block_scan(need, part, sum_need);
        const bool ok = fits && (need == 0 || nend <= avail);
        if (ok && need > 0) used = max(used, nend);
        bad += (i < p.B && live && !ok) ? 1 : 0;
        row_end[tid] = rend;
        page_end[tid] = nend;
        s_ctx[tid] = ctx;
        s_held[tid] = (int)min(held, (long long)p.width);
        s_ok[tid] = ok;
        if (i < p.B && (uint32_t)((base / nt) % size) == rank) {
            if (i == 0) p.cu[0] = 0;
            p.cu[i + 1] = (int)min(rend, (long long)p.T);
            p.kv[i] = ok ? ctx + add : 0;
        }
        __syncthreads();
        // table entries of the pages taken
        for (long long x = (long long)rank * nt + tid; x < sum_need; x += (long long)size * nt) {
            const long long r = need_sum + x;
            const int q = upper(page_end, nb, r);
            const long long first = q ? page_end[q - 1] : need_sum;
            if (s_ok[q]) p.table[(long long)(base + q) * p.width + s_held[q] + (r - first)] = p.pool[avail - 1 - r];
        }
        // positions and slots of the chunk's rows
        const long long lo = min(rows, (long long)p.T), hi = min(rows + sum_rows, (long long)p.T);
        for (long long t = lo + (long long)rank * nt + tid; t < hi; t += (long long)size * nt) {
            const int q = upper(row_end, nb, t);
            int pos = 0;
            long long slot = -1;
            if (s_ok[q]) {
                pos = s_ctx[q] + (int)(t - (q ? row_end[q - 1] : rows));
                const int col = pos >> p.ps_log2;
                int page;
                if (col < s_held[q]) {
                    page = p.table[(long long)(base + q) * p.width + col];
                } else {
                    const long long first = q ? page_end[q - 1] : need_sum;
                    page = p.pool[avail - 1 - (first + col - s_held[q])];
                }
                slot = ((long long)page << p.ps_log2) + (pos & (ps - 1));
            }
            p.pos[t] = pos;
            p.slots[t] = slot;
        }
        rows += sum_rows;
        need_sum += sum_need;
        __syncthreads();  // the next chunk overwrites the shared arrays
    }
    // rows behind the last request have no slot
    for (long long t = min(rows, (long long)p.T) + (long long)rank * nt + tid; t < p.T; t += (long long)size * nt) {
        p.pos[t] = 0;
        p.slots[t] = -1;
    }
    if (rank == 0) {  // pages taken (the largest served end) and requests not served
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
            used = max(used, __shfl_xor_sync(0xffffffffu, used, off));
            bad += __shfl_xor_sync(0xffffffffu, bad, off);
        }
        if ((tid & 31) == 0) {
            part[tid >> 5] = used;
            s_ok[tid >> 5] = bad;
        }
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < (nt >> 5); ++w) {
                used = max(used, part[w]);
                bad += s_ok[w];
            }
            *p.free_out = (int)(avail - used);
            *p.status = bad;
        }
    }
}

// All of the shared memory of kv_plan_flat_kernel
constexpr int plan_flat_smem(int B) { return 32 * (int)sizeof(long long) + 5 * (int)sizeof(int) * B; }

// Sums past what they are compared with (T rows, the pages there are) are held
// one above it, so 32 bits carry them.
__global__ void __launch_bounds__(1024, 1) kv_plan_flat_kernel(const __grid_constant__ PlanParams p) {
    extern __shared__ long long plan_smem[];
    long long* part = plan_smem;                            // [32]
    int* row_end = reinterpret_cast<int*>(plan_smem + 32);  // [B] inclusive ends: rows, pages given back, pages taken
    int* back_end = row_end + p.B;
    int* page_end = back_end + p.B;
    int* s_ctx = page_end + p.B;
    int* s_held = s_ctx + p.B;        // pages held, -1 - held for a request that is not served
    const int tid = threadIdx.x, nt = blockDim.x, items = (p.B + nt - 1) / nt, i0 = tid * items;
    const int ps = 1 << p.ps_log2;
    const int n = max(0, min(items, p.B - i0));
    const long long free0 = min(max(*p.free_in, 0), p.capacity);

    long long rows = 0, back = 0;
    for (int i = i0; i < i0 + n; ++i) {
        const int ctx = p.ctx[i], nw = p.nw[i];
        s_ctx[i] = ctx;
        s_held[i] = nw;
        rows += max(nw, 0);
        if (nw < 0) back += min(((long long)max(ctx, 0) + ps - 1) >> p.ps_log2, (long long)p.width);
    }
    long long all_rows, all_back, all_need;
    long long r = block_scan(rows, part, all_rows) - rows, g = block_scan(back, part, all_back) - back;
    const long long avail = min(free0 + all_back, (long long)p.capacity);
    long long need_sum = 0;
    for (int i = i0; i < i0 + n; ++i) {
        const int ctx = s_ctx[i], nw = s_held[i];
        const long long held = ((long long)max(ctx, 0) + ps - 1) >> p.ps_log2;
        const long long want = ((long long)max(ctx, 0) + max(nw, 0) + ps - 1) >> p.ps_log2;
        r += max(nw, 0);
        if (nw < 0) g += min(held, (long long)p.width);
        row_end[i] = (int)min(r, (long long)p.T + (p.T < 0x7fffffff));
        back_end[i] = (int)min(g, (long long)0x7fffffff);
        const bool fits = nw >= 0 && ctx >= 0 && r <= p.T && want <= p.width;
        page_end[i] = fits ? (int)(want - held) : -1;   // pages needed, for now
        if (fits) need_sum += want - held;
    }
    long long e = block_scan(need_sum, part, all_need) - need_sum;
    long long used = 0;
    int bad = 0;
    for (int i = i0; i < i0 + n; ++i) {
        const int ctx = s_ctx[i], nw = s_held[i], need = page_end[i];
        if (need > 0) e += need;
        const bool ok = need == 0 || (need > 0 && e <= avail);
        if (need > 0 && ok) used = e;
        bad += nw >= 0 && !ok;
        const int held = (int)min(((long long)max(ctx, 0) + ps - 1) >> p.ps_log2, (long long)p.width);
        page_end[i] = (int)min(e, avail + 1);
        s_held[i] = ok ? held : -1 - held;
        if (blockIdx.x == 0) {
            p.cu[i + 1] = min(row_end[i], p.T);
            p.kv[i] = ok ? ctx + nw : 0;
        }
    }
    if (blockIdx.x == 0) {
        if (tid == 0) p.cu[0] = 0;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
            used = max(used, __shfl_xor_sync(0xffffffffu, used, off));
            bad += __shfl_xor_sync(0xffffffffu, bad, off);
        }
        __syncthreads();
        if ((tid & 31) == 0) part[tid >> 5] = used << 32 | (unsigned)bad;
        __syncthreads();
        if (tid == 0) {
            used = 0;
            bad = 0;
            for (int w = 0; w < (nt >> 5); ++w) {
                used = max(used, part[w] >> 32);
                bad += (int)(part[w] & 0xffffffffll);
            }
            *p.free_out = (int)(avail - used);
            *p.status = bad;
        }
    }
    __syncthreads();

    const int first = blockIdx.x * nt + tid, step = gridDim.x * nt;
    auto page_of = [&](long long rank) -> int {         // the page of this rank among those taken
        const long long at = avail - 1 - rank;
        if (at < free0) return p.pool[at];
        const int x = (int)(at - free0), q = upper(back_end, p.B, x);
        return p.table[(long long)q * p.width + x - (q ? back_end[q - 1] : 0)];
    };
    for (long long x = first; x < min(all_back, (long long)p.capacity - free0); x += step) {
        const int q = upper(back_end, p.B, (int)x);
        p.pool[free0 + x] = p.table[(long long)q * p.width + x - (q ? back_end[q - 1] : 0)];
    }
    for (long long x = first; x < min(all_need, avail); x += step) {
        const int q = upper(page_end, p.B, (int)x);
        if (q < p.B && s_held[q] >= 0) {
            const long long at = x - (q ? page_end[q - 1] : 0);
            p.table[(long long)q * p.width + s_held[q] + at] = page_of(x);
        }
    }
    for (long long t = first; t < p.T; t += step) {
        int pos = 0;
        long long slot = -1;
        const int q = t < all_rows ? upper(row_end, p.B, (int)t) : p.B;
        if (q < p.B && s_held[q] >= 0) {
            pos = s_ctx[q] + (int)(t - (q ? row_end[q - 1] : 0));
            const int col = pos >> p.ps_log2;
            const int page = col < s_held[q] ? p.table[(long long)q * p.width + col]
                                             : page_of((q ? page_end[q - 1] : 0) + (long long)(col - s_held[q]));
            slot = ((long long)page << p.ps_log2) + (pos & (ps - 1));
        }
        p.pos[t] = pos;
        p.slots[t] = slot;
    }
}

// ------------------------------------------------- rotary embedding and store
// Pair (i, i + 64) of a head of a token at position s turns by s theta^(-2i/128);
// rotated queries go to q_out, rotated keys and the values as fp16 to row
// slot % ps of page slot / ps (and to k_out / v_out).
//
// HBM-bound: each fp32 row is read once and written once at its output width.
// One warp takes a run of a token's heads, two heads at a time: 16 lanes hold
// a head, lane l the pairs 4l .. 4l + 3, so every access is 16 bytes (8 for
// the fp16 halves) and the four angles of a lane, reduced in double, serve all
// the heads of its run.
struct RopeParams {
    const float* q;
    const float* k;
    const float* v;
    int64_t q_stride, kv_stride;
    void* q_out;
    __half* k_out;
    __half* v_out;
    const int32_t* pos;
    const int64_t* slots;
    __half* kc;
    __half* vc;
    int64_t page_stride, head_stride, row_stride, n_slots;
    int* err;
    int T, n_heads, n_kv, ps_log2, run;
    double inv_freq[64];
};

__device__ __forceinline__ void store4(__half* d, float4 a) {
    const __half2 x = __floats2half2_rn(a.x, a.y), y = __floats2half2_rn(a.z, a.w);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&x);
    u.y = *reinterpret_cast<const uint32_t*>(&y);
    *reinterpret_cast<uint2*>(d) = u;
}
__device__ __forceinline__ void store4(float* d, float4 a) { *reinterpret_cast<float4*>(d) = a; }

constexpr int kRopeBatch = 4;   // heads a thread has in flight

template <typename QO>
__global__ void __launch_bounds__(256) rope_append_kernel(const __grid_constant__ RopeParams p) {
    const int lane = threadIdx.x & 31, sub = lane & 15;
    const int heads = p.n_heads + 2 * p.n_kv, pairs = (heads + 1) >> 1;
    const int runs = (pairs + p.run - 1) / p.run;
    const long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const long long t = w / runs;
    if (t >= p.T) return;
    const int h0 = (int)(w - t * runs) * p.run * 2;
    const int pos = p.pos[t];
    const long long slot = p.slots ? p.slots[t] : -1;
    const bool store = p.kc != nullptr && slot >= 0 && slot < p.n_slots;
    if (p.kc != nullptr && slot >= p.n_slots && lane == 0) record_bad_arg(p.err);
    const long long page = slot >> p.ps_log2;
    const long long row_off = store ? page * p.page_stride + (slot - (page << p.ps_log2)) * p.row_stride : 0;
    const int hend = min(heads, h0 + 2 * p.run);
    // The loads of kRopeBatch heads, then their stores: coherent loads (in place the launch
    // writes these rows too) that no store holds up, the first ones under way while the
    // angles are formed.  A thread stores to an address only what it formed from the value
    // there.
    float4 a[kRopeBatch], b[kRopeBatch];
    auto load = [&](int hb) {
#pragma unroll
        for (int i = 0; i < kRopeBatch; ++i) {
            const int h = hb + 2 * i;
            if (h >= hend) break;
            const float* src = h < p.n_heads ? p.q + t * p.q_stride + (int64_t)h * 128
                               : h < p.n_heads + p.n_kv ? p.k + t * p.kv_stride + (int64_t)(h - p.n_heads) * 128
                                                        : p.v + t * p.kv_stride + (int64_t)(h - p.n_heads - p.n_kv) * 128;
            a[i] = *(reinterpret_cast<const float4*>(src) + sub);
            b[i] = *(reinterpret_cast<const float4*>(src + 64) + sub);
        }
    };
    load(h0 + (lane >> 4));
    float c[4], s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) rope_cs(pos, p.inv_freq[4 * sub + e], c[e], s[e]);
    for (int hb = h0 + (lane >> 4); hb < hend; hb += 2 * kRopeBatch) {
#pragma unroll
        for (int i = 0; i < kRopeBatch; ++i) {
            const int h = hb + 2 * i;
            if (h >= hend) break;
            const bool is_q = h < p.n_heads, is_k = !is_q && h < p.n_heads + p.n_kv;
            const int kh = h - p.n_heads - (is_k ? 0 : p.n_kv);
            float4 x = a[i], y = b[i];
            if (is_q || is_k) {
                x = make_float4(a[i].x * c[0] - b[i].x * s[0], a[i].y * c[1] - b[i].y * s[1], a[i].z * c[2] - b[i].z * s[2],
                                a[i].w * c[3] - b[i].w * s[3]);
                y = make_float4(b[i].x * c[0] + a[i].x * s[0], b[i].y * c[1] + a[i].y * s[1], b[i].z * c[2] + a[i].z * s[2],
                                b[i].w * c[3] + a[i].w * s[3]);
            }
            if (is_q) {
                QO* d = static_cast<QO*>(p.q_out) + ((int64_t)t * p.n_heads + h) * 128 + 4 * sub;
                store4(d, x);
                store4(d + 64, y);
            } else {
                if (store) {
                    __half* d = (is_k ? p.kc : p.vc) + row_off + (int64_t)kh * p.head_stride + 4 * sub;
                    store4(d, x);
                    store4(d + 64, y);
                }
                __half* o = is_k ? p.k_out : p.v_out;
                if (o) {
                    o += ((int64_t)t * p.n_kv + kh) * 128 + 4 * sub;
                    store4(o, x);
                    store4(o + 64, y);
                }
            }
        }
        load(hb + 2 * kRopeBatch);
    }
}

// Whether any of T fp32 rows (`stride` elements apart, `row` long, row <= stride) meets
// the bytes [at, end).
bool rows_overlap(const float* base, int64_t stride, int64_t row, int T, uintptr_t at, uintptr_t end) {
    if (row == 0 || at >= end) return false;
    const uintptr_t b = (uintptr_t)base, len = (uintptr_t)row * 4, step = (uintptr_t)stride * 4;
    const uintptr_t i = b + len > at ? 0 : (at - b - len) / step + 1;   // first row that ends behind `at`
    return i < (uintptr_t)T && b + i * step < end;
}

}  // namespace

}  // namespace glc

using glc::paged_fail;

extern "C" int glc_kv_plan_dev(const int32_t* ctx_lens, const int32_t* new_lens, int32_t B, int32_t page_size,
                               int32_t* block_table, int32_t max_pages, int32_t* free_list, int32_t capacity,
                               const int32_t* free_count, int32_t* free_count_out, int32_t T, int32_t* cu_new,
                               int32_t* kv_lens, int32_t* positions, int64_t* slots, int32_t* status, void* stream) {
    if (!ctx_lens || !new_lens || !block_table || !free_list || !free_count || !free_count_out || !cu_new || !kv_lens ||
        !status || (T > 0 && (!positions || !slots)))
        return paged_fail(GLC_ERR_INVALID_ARG, "null pointer");
    if (B < 0 || T < 0 || max_pages <= 0 || capacity < 0 || (int64_t)max_pages * std::max(page_size, 1) > 0x7fffffff ||
        capacity == 0x7fffffff)
        return paged_fail(GLC_ERR_INVALID_ARG, "page plan of %d requests, %d rows, %d pages a table row, %d pages", B, T,
                          max_pages, capacity);
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
        return paged_fail(GLC_ERR_UNSUPPORTED, "page_size %d (16, 32, 64, 128 or 256)", page_size);
    // the CTAs of a launch read the inputs while others write the outputs
    struct Range {
        const void* p;
        int64_t bytes;
    };
    for (const Range& i : {Range{ctx_lens, 4LL * B}, Range{new_lens, 4LL * B}, Range{free_count, 4}})
        for (const Range& o : {Range{block_table, 4LL * B * max_pages}, Range{free_list, 4LL * capacity}, Range{free_count_out, 4},
                               Range{cu_new, 4LL * B + 4}, Range{kv_lens, 4LL * B}, Range{positions, 4LL * T},
                               Range{slots, 8LL * T}, Range{status, 4}})
            if ((uintptr_t)i.p < (uintptr_t)o.p + o.bytes && (uintptr_t)o.p < (uintptr_t)i.p + i.bytes)
                return paged_fail(GLC_ERR_INVALID_ARG, "outputs must not alias ctx_lens, new_lens or free_count");
    const auto used = [](const void* ptr, int n) { return n ? ptr : nullptr; };   // arrays without elements may be anything
    if (int rc = glc::paged_check_devices({{used(ctx_lens, B), "ctx_lens"}, {used(new_lens, B), "new_lens"},
                                           {used(block_table, B), "block_table"}, {used(free_list, capacity), "free_list"},
                                           {free_count, "free_count"}, {free_count_out, "free_count_out"}, {cu_new, "cu_new"},
                                           {used(kv_lens, B), "kv_lens"}, {used(positions, T), "positions"},
                                           {used(slots, T), "slots"}, {status, "status"}}))
        return rc;
    glc::PlanParams p{};
    p.ctx = ctx_lens;
    p.nw = new_lens;
    p.table = block_table;
    p.pool = free_list;
    p.free_in = free_count;
    p.free_out = free_count_out;
    p.cu = cu_new;
    p.kv = kv_lens;
    p.pos = positions;
    p.slots = slots;
    p.status = status;
    p.B = B;
    while ((1 << p.ps_log2) < page_size) ++p.ps_log2;
    p.width = max_pages;
    p.capacity = capacity;
    p.T = T;
    cudaError_t e = cudaSuccess;
    if (B <= glc::kPlanFlat) {
        // every CTA repeats the sums: as many as one row or page a thread takes, up to all SMs
        const int threads = B <= 256 ? 256 : 1024;
        const long long work = std::max<long long>(T, B);
        const int grid = (int)std::min<long long>(148, (work + threads - 1) / threads);
        const int smem = glc::plan_flat_smem(B);
        // the limit belongs to the kernel, not to the call: always that of the largest plan, so
        // that no other host thread lowers it before this launch
        if (smem > 48 * 1024)
            e = cudaFuncSetAttribute(glc::kv_plan_flat_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     glc::plan_flat_smem(glc::kPlanFlat));
        if (e == cudaSuccess) {
            glc::kv_plan_flat_kernel<<<std::max(grid, 1), threads, smem, (cudaStream_t)stream>>>(p);
            e = cudaGetLastError();
        }
    } else {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(glc::kPlanCluster);
        cfg.blockDim = dim3(1024);
        cfg.stream = (cudaStream_t)stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = glc::kPlanCluster;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, glc::kv_plan_kernel, p);
    }
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "page plan: %s", cudaGetErrorString(e));
    return GLC_OK;
}

extern "C" int glc_rope_append_dev(const float* q, int64_t q_stride, const float* k, const float* v, int64_t kv_stride,
                                   int32_t T, int32_t n_heads, int32_t n_kv_heads, const int32_t* positions,
                                   const int64_t* slots, float rope_theta, const glc_kv_pages* cache, void* q_out,
                                   int32_t q_out_type, void* k_out, void* v_out, void* stream) {
    if (T < 0 || n_heads < 0 || n_kv_heads <= 0)
        return paged_fail(GLC_ERR_INVALID_ARG, "%d rows of %d query and %d KV heads", T, n_heads, n_kv_heads);
    if (!k || !v || !positions || (n_heads > 0 && (!q || !q_out)) || (cache && !slots) || (!k_out != !v_out))
        return paged_fail(GLC_ERR_INVALID_ARG, "null pointer");
    if (q_out_type != GLC_GGUF_F32 && q_out_type != GLC_GGUF_F16)
        return paged_fail(GLC_ERR_UNSUPPORTED, "query type %d (GLC_GGUF_F32 or GLC_GGUF_F16)", q_out_type);
    if (!(rope_theta > 0.f) || std::isinf(rope_theta))
        return paged_fail(GLC_ERR_INVALID_ARG, "rope_theta must be positive");
    if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out) & 15u) ||
        ((q_stride | kv_stride) & 3))
        return paged_fail(GLC_ERR_INVALID_ARG, "rows must be 16-byte aligned");
    if (q_stride < (int64_t)n_heads * 128 || kv_stride < (int64_t)n_kv_heads * 128)
        return paged_fail(GLC_ERR_INVALID_ARG, "row strides shorter than a row");
    if (q_out == q && n_heads > 0 && (q_out_type != GLC_GGUF_F32 || q_stride != (int64_t)n_heads * 128))
        return paged_fail(GLC_ERR_INVALID_ARG, "in place only as fp32 rows of n_heads x 128");
    const int64_t q_row = (int64_t)n_heads * 128, kv_row = (int64_t)n_kv_heads * 128;
    for (const auto& o : {std::make_pair(q_out, q_row * (q_out_type == GLC_GGUF_F32 ? 4 : 2)), std::make_pair(k_out, kv_row * 2),
                          std::make_pair(v_out, kv_row * 2)}) {
        const uintptr_t at = (uintptr_t)o.first, end = at + (uintptr_t)(T * o.second);
        if (o.first && ((o.first != q && glc::rows_overlap(q, q_stride, q_row, T, at, end)) ||
                        glc::rows_overlap(k, kv_stride, kv_row, T, at, end) || glc::rows_overlap(v, kv_stride, kv_row, T, at, end)))
            return paged_fail(GLC_ERR_INVALID_ARG, "outputs overlap the rows of q, k or v");
    }
    if (cache) {
        if (int rc = glc::paged_check_pages(cache)) return rc;
        if (cache->n_kv_heads != n_kv_heads)
            return paged_fail(GLC_ERR_INVALID_ARG, "%d KV heads for a cache of %d", n_kv_heads, cache->n_kv_heads);
    }
    if (T == 0) return GLC_OK;
    if (int rc = glc::paged_check_devices({{n_heads ? q : nullptr, "q"}, {k, "k"}, {v, "v"}, {positions, "positions"},
                                           {slots, "slots"}, {cache ? cache->k : nullptr, "the cache's k"},
                                           {cache ? cache->v : nullptr, "the cache's v"},
                                           {n_heads ? q_out : nullptr, "q_out"}, {k_out, "k_out"}, {v_out, "v_out"}}))
        return rc;
    glc::RopeParams p{};
    if (int rc = glc::paged_error_word(&p.err)) return rc;
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride = q_stride;
    p.kv_stride = kv_stride;
    p.q_out = q_out;
    p.k_out = static_cast<__half*>(k_out);
    p.v_out = static_cast<__half*>(v_out);
    p.pos = positions;
    p.slots = slots;
    if (cache) {
        p.kc = static_cast<__half*>(cache->k);
        p.vc = static_cast<__half*>(cache->v);
        p.page_stride = cache->page_stride;
        p.head_stride = cache->head_stride;
        p.row_stride = cache->row_stride;
        p.n_slots = (int64_t)cache->n_pages * cache->page_size;
        while ((1 << p.ps_log2) < cache->page_size) ++p.ps_log2;
    }
    p.T = T;
    p.n_heads = n_heads;
    p.n_kv = n_kv_heads;
    // theta^(-i/64) as products of six powers: 64 exponentials take 1 us, as long as the
    // launch; five roundings in double do not show in an fp32 angle
    const double step = -std::log((double)rope_theta) / 64.0;
    p.inv_freq[0] = 1.0;
    for (int n = 1; n < 64; n *= 2) {
        const double f = std::exp(n * step);
        for (int i = 0; i < n; ++i) p.inv_freq[n + i] = p.inv_freq[i] * f;
    }
    const long long pairs = (n_heads + 2LL * n_kv_heads + 1) / 2;
    // A warp's four angles (double reduction, sincosf: ~200 instructions) serve its
    // run of head pairs: the shortest run whose warps are resident at once (three CTAs an
    // SM), up to eight pairs, and one pair a warp where the call is short (8192 rows of
    // 48 / 8 heads, fp16 out: 234 us with runs of one pair, 68 us with eight: 5.9 TB/s;
    // 300 rows of 28 / 4: 8.3 us with one, 6.3 with two).
    p.run = (int)std::min<long long>(8, ((long long)T * pairs + 148 * 24 - 1) / (148 * 24));
    const long long warps = (long long)T * ((pairs + p.run - 1) / p.run);
    const long long blocks = (warps + 7) / 8;
    if (blocks > 0x7fffffffLL) return paged_fail(GLC_ERR_UNSUPPORTED, "%d rows are too many for one call", T);
    if (q_out_type == GLC_GGUF_F32)
        glc::rope_append_kernel<float><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
    else
        glc::rope_append_kernel<__half><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "rotary store: %s", cudaGetErrorString(e));
    return GLC_OK;
}

extern "C" int glc_paged_poll_error(void) {
    static std::mutex mu;   // one poll at a time has the word it was read to
    std::lock_guard<std::mutex> lk(mu);
    int code = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) {
        glc::take_error_kernel<<<1, 1, 0, cudaStreamLegacy>>>();
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&code, glc::g_paged_seen, sizeof(int));
    if (e != cudaSuccess) return paged_fail(GLC_ERR_CUDA, "device error word: %s", cudaGetErrorString(e));
    if (code == glc::kDevOk) return GLC_OK;
    if (code == glc::kDevBadArg)
        return paged_fail(GLC_ERR_INVALID_ARG, "a page id, slot or length on the device was out of range");
    return paged_fail(GLC_ERR_TIMEOUT, "a device-side wait of the paged attention gave up (code %d)", code);
}
