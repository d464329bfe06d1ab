// The device error word of the paged entry points: a wait that gave up stays
// recorded when a bad argument comes after it, since the caller has to clear a
// captured call's workspace then.  The word is written from the host here.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <cstdlib>

#include "glacier_b200.h"
#include "paged.cuh"

#define MUST(x)                                                                       \
    do {                                                                              \
        if (!(x)) {                                                                   \
            std::printf("line %d: %s (%s)\n", __LINE__, #x, glc_last_error());        \
            std::exit(1);                                                             \
        }                                                                             \
    } while (0)

int main() {
    float* row = nullptr;
    __half* page = nullptr;
    int32_t* pos = nullptr;
    int64_t* slot = nullptr;
    MUST(cudaMalloc(&row, 128 * sizeof(float)) == cudaSuccess && cudaMalloc(&page, 16 * 128 * sizeof(__half)) == cudaSuccess);
    MUST(cudaMalloc(&pos, sizeof(int32_t)) == cudaSuccess && cudaMalloc(&slot, sizeof(int64_t)) == cudaSuccess);
    MUST(cudaMemset(row, 0, 128 * sizeof(float)) == cudaSuccess && cudaMemset(pos, 0, sizeof(int32_t)) == cudaSuccess);
    const int64_t past = 77;
    MUST(cudaMemcpy(slot, &past, sizeof(past), cudaMemcpyHostToDevice) == cudaSuccess);
    const glc_kv_pages cache{page, page, 16 * 128, 16 * 128, 128, 1, 16, 1, 128};
    int* word = nullptr;
    MUST(glc::paged_error_word(&word) == GLC_OK);
    cudaStream_t st = nullptr;
    MUST(cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking) == cudaSuccess);
    const auto bad = [&] {
        return glc_rope_append_dev(nullptr, 0, row, row, 128, 1, 0, 1, pos, slot, 1e6f, &cache, nullptr, GLC_GGUF_F32,
                                   nullptr, nullptr, st);
    };
    MUST(glc_paged_poll_error() == GLC_OK);
    for (const int code : {(int)glc::kDevTimeoutFull, (int)glc::kDevTimeoutEmpty, (int)glc::kDevTimeoutGrid}) {
        MUST(cudaMemcpy(word, &code, sizeof(code), cudaMemcpyHostToDevice) == cudaSuccess);
        MUST(bad() == GLC_OK);
        MUST(glc_paged_poll_error() == GLC_ERR_TIMEOUT);
        MUST(glc_paged_poll_error() == GLC_OK);
        MUST(bad() == GLC_OK);
        MUST(glc_paged_poll_error() == GLC_ERR_INVALID_ARG);
        MUST(glc_paged_poll_error() == GLC_OK);
    }
    std::printf("ok\n");
    return 0;
}
