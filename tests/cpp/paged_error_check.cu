// The device error word of the paged entry points.
//   order: a wait that gave up stays recorded when a bad argument comes after it,
//     since the caller has to clear a captured call's workspace then.  The word is
//     written from the host here.
//   lost: what a call records while another host thread polls is in that poll or in
//     the next, also while the default stream has work queued.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <thread>

#include "glacier_b200.h"
#include "paged.cuh"

#define MUST(x)                                                                       \
    do {                                                                              \
        if (!(x)) {                                                                   \
            std::printf("line %d: %s (%s)\n", __LINE__, #x, glc_last_error());        \
            std::exit(1);                                                             \
        }                                                                             \
    } while (0)

__global__ void busy(long long cycles) {
    const long long t0 = clock64();
    while (clock64() - t0 < cycles) __nanosleep(200);
}

__global__ void record(int* word, int code) { atomicExch(word, code); }

int main(int argc, char** argv) {
    MUST(argc == 2);
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
    if (!std::strcmp(argv[1], "order")) {
        for (const int code : {(int)glc::kDevTimeoutFull, (int)glc::kDevTimeoutEmpty, (int)glc::kDevTimeoutGrid}) {
            MUST(cudaMemcpy(word, &code, sizeof(code), cudaMemcpyHostToDevice) == cudaSuccess);
            MUST(bad() == GLC_OK);
            MUST(glc_paged_poll_error() == GLC_ERR_TIMEOUT);
            MUST(glc_paged_poll_error() == GLC_OK);
            MUST(bad() == GLC_OK);
            MUST(glc_paged_poll_error() == GLC_ERR_INVALID_ARG);
            MUST(glc_paged_poll_error() == GLC_OK);
        }
    } else {
        std::atomic<bool> stop{false};
        std::thread other([&] {   // the default stream always has up to four kernels of 0.1 ms queued
            cudaEvent_t done[4];
            for (auto& e : done) cudaEventCreateWithFlags(&e, cudaEventDisableTiming);
            for (int i = 0; !stop; ++i) {
                cudaEventSynchronize(done[i % 4]);
                busy<<<1, 32>>>(180000);
                cudaEventRecord(done[i % 4], cudaStreamLegacy);
            }
            cudaStreamSynchronize(cudaStreamLegacy);
        });
        // bad arguments and fake timeouts from this thread, polls from a third one
        std::atomic<int> begun{0}, ended{0}, timeouts{0};
        std::thread poller([&] {
            while (!stop) {
                ++begun;
                timeouts += glc_paged_poll_error() == GLC_ERR_TIMEOUT;
                ++ended;
            }
        });
        int lost = 0;
        for (int i = 0; i < 200; ++i) {
            const int before = timeouts;
            MUST(bad() == GLC_OK);
            std::this_thread::sleep_for(std::chrono::microseconds(37 * i % 1500));
            record<<<1, 1, 0, st>>>(word, glc::kDevTimeoutFull);
            MUST(cudaStreamSynchronize(st) == cudaSuccess);
            const int due = begun + 1;   // a poll that begins from here on reads the word afterwards
            while (ended < due) std::this_thread::yield();
            lost += timeouts == before;
        }
        stop = true;
        other.join();
        poller.join();
        if (lost) std::printf("%d of 200 timeouts lost\n", lost);
        MUST(lost == 0);
    }
    std::printf("ok\n");
    return 0;
}
