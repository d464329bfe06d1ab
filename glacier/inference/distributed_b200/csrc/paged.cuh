// paged.cuh -- what the paged-cache entry points share: argument errors with a
// formatted message, the device error word, the checks of a glc_kv_pages and
// the TMA descriptors of its pages.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "../../../../include/glacier_b200.h"
#include "kernels.h"

namespace glc {

// Records the formatted message for glc_last_error() and returns `code`.
int paged_fail(int code, const char* fmt, ...);

// Device error word of the current device (GLC_OK and *err set, or the status
// of the failure).  A fixed device word of the library: nothing is allocated.
int paged_error_word(int** err);

// Records a bad page id, slot or length.  A wait that gave up is never hidden by one:
// the caller has to clear the workspace of captured calls after it (and that code is
// recorded over this one).
__device__ __forceinline__ void record_bad_arg(int* err) { atomicCAS(err, kDevOk, kDevBadArg); }

// GLC_OK when every pointer that is not null is memory the current device owns or can
// be handed without faulting (managed and pinned host memory included).
struct DevicePtr {
    const void* p;
    const char* what;
};
int paged_check_devices(std::initializer_list<DevicePtr> ptrs);

// The shape, strides and alignment rules of a page set.
int paged_check_pages(const glc_kv_pages* c);

// A 128-byte swizzled fp16 descriptor (strides in bytes, one less than the rank).
int paged_encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                 const cuuint32_t* box);

// A descriptor of 128-wide fp16 rows as [pages][heads][2 halves][rows][64]:
// a box is `box_rows` rows of `box_halves` 64-element halves of one head of
// one page, 128-byte swizzled.  Rows and pages past the end read as zeros.
int paged_tensor_map(CUtensorMap* map, const void* base, int64_t rows, int64_t row_stride, int64_t heads,
                     int64_t head_stride, int64_t pages, int64_t page_stride, int box_rows, int box_halves);

}  // namespace glc
