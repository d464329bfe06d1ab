// The scheduler warp of the tile kernel by itself, with nobody to take its items:
// its wait runs out, is recorded, and every place that the joining launch reads
// is written all the same, with rows and parts inside their bounds.  (The kernel of
// a call would go on to its joining launch, which trusts the places; it is not run
// here.)
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "attn_tiles.cu"

#define MUST(x)                                              \
    do {                                                     \
        if (!(x)) {                                          \
            std::printf("line %d: %s\n", __LINE__, #x);      \
            std::exit(1);                                    \
        }                                                    \
    } while (0)

__global__ void scheduler_alone(const __grid_constant__ glc::AttnBatch p) {
    __shared__ glc::TilesSmem S;
    if (threadIdx.x == 0) {
        for (int i = 0; i < glc::kItemBufs; ++i) {
            glc::mbar_init(&S.item_full[i], 1);
            glc::mbar_init(&S.item_empty[i], 11);
        }
        glc::fence_mbar_init();
    }
    __syncwarp();
    glc::hand_out_items(p, S);
}

int main() {
    // one sequence of 300 new tokens of 3,000, four KV heads of four query heads: 20
    // units on 8 CTAs, cut into parts
    const int T = 300, n_kv = 4, G = 4, tpt = 128 / G, slots = 160, ctas = 8;
    const std::vector<int32_t> cu = {0, T}, kv = {3000};
    int32_t *d_cu = nullptr, *d_kv = nullptr, *err = nullptr;
    uint8_t* work = nullptr;
    const size_t bytes = glc::kRowsWorkBytes + (size_t)(slots + 1) * glc::kTileUnitBytes;
    MUST(cudaMalloc(&d_cu, 8) == cudaSuccess && cudaMalloc(&d_kv, 4) == cudaSuccess);
    MUST(cudaMalloc(&err, 4) == cudaSuccess && cudaMalloc(&work, bytes) == cudaSuccess);
    MUST(cudaMemcpy(d_cu, cu.data(), 8, cudaMemcpyHostToDevice) == cudaSuccess);
    MUST(cudaMemcpy(d_kv, kv.data(), 4, cudaMemcpyHostToDevice) == cudaSuccess);
    MUST(cudaMemset(err, 0, 4) == cudaSuccess && cudaMemset(work, 0xff, bytes) == cudaSuccess);
    glc::AttnBatch p{};
    p.cu = d_cu;
    p.kv_lens = d_kv;
    p.max_pages = 200;
    p.ps_log2 = 4;
    p.B = 1;
    p.T = p.max_new = T;
    p.n_kv = n_kv;
    p.n_heads = n_kv * G;
    p.G = G;
    p.row_tile_tokens = tpt;
    p.tokens_per_tile = 2 * tpt;      // 64: a shift
    p.unit_mul = 1u << 31;
    p.unit_shift = 5;
    p.split = 1;
    p.slots = slots;
    p.work = reinterpret_cast<float*>(work);
    p.err = err;
    scheduler_alone<<<ctas, 32>>>(p);
    MUST(cudaDeviceSynchronize() == cudaSuccess);

    int code = 0, places = 0;
    MUST(cudaMemcpy(&code, err, 4, cudaMemcpyDeviceToHost) == cudaSuccess);
    MUST(code == glc::kDevTimeoutEmpty);
    MUST(cudaMemcpy(&places, work + glc::kRowsWorkBytes, 4, cudaMemcpyDeviceToHost) == cudaSuccess);
    MUST(places > 2 * glc::kItemBufs * ctas && places <= slots);   // more than the CTAs could hand out
    std::vector<uint8_t> host((size_t)places * glc::kTileUnitBytes);
    MUST(cudaMemcpy(host.data(), work + glc::kRowsWorkBytes + glc::kTileUnitBytes, host.size(), cudaMemcpyDeviceToHost) ==
         cudaSuccess);
    int units = 0;
    for (int s = 0; s < places; ++s) {
        const glc::TileUnit& u = *reinterpret_cast<const glc::TileUnit*>(host.data() + (size_t)s * glc::kTileUnitBytes);
        MUST(u.parts >= 0 && u.parts <= glc::kMaxParts && s + u.parts <= places);
        if (!u.parts) continue;
        ++units;
        MUST(u.g >= 0 && u.g < n_kv && u.row0 >= 0 && u.ntok[0] >= 0 && u.ntok[0] <= tpt && u.ntok[1] >= 0 && u.ntok[1] <= tpt);
        MUST(u.row0 + u.ntok[0] + u.ntok[1] <= T);
    }
    MUST(units == 5 * n_kv);
    std::printf("ok: %d units in %d places\n", units, places);
    return 0;
}
