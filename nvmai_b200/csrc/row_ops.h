// Between the row operators' translation units: element types, checks of arguments, the quantisation launcher.
#pragma once
#include <cuda_runtime.h>
#include <initializer_list>
#include <stddef.h>
#include <stdint.h>

namespace nvmai {

enum : uint32_t { ELEM_F16 = 0, ELEM_F32 = 1, ELEM_BF16 = 2, ELEM_I8 = 3 };
constexpr uint32_t kRowMaxExperts = 1024, kRowMaxTopK = 64;
constexpr uint32_t kRowMaxLength = 1u << 30;       // elements of a row: counts of pieces and their steps stay in 32 bits

inline size_t elem_size(uint32_t e) { return e == ELEM_F32 ? 4 : e == ELEM_I8 ? 1 : 2; }
inline bool aligned_to(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Every pointer given (null ones aside) is memory of the current device, or managed memory: a buffer of another device or of the
// host would be an illegal address in the kernel.  An error is cleared: the call is refused, the context is as it was.
// 0.05 us a pointer.
inline bool on_current_device(std::initializer_list<const void *> ptrs, int *device = nullptr) {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return false; }
    if (device != nullptr) *device = dev;
    for (const void *p : ptrs) {
        if (p == nullptr) continue;
        cudaPointerAttributes a;
        if (cudaPointerGetAttributes(&a, p) != cudaSuccess) { cudaGetLastError(); return false; }
        if (a.type != cudaMemoryTypeManaged && (a.type != cudaMemoryTypeDevice || a.device != dev)) return false;
    }
    return true;
}

// The body of a C entry point: no exception (a failed allocation on the host) leaves it.
template <typename F>
int without_exceptions(F &&f) noexcept {
    try {
        return f();
    } catch (...) {
        return 12;           // NVMAI_CUDA_ENOMEM
    }
}

// the longest a device-side wait of the products lasts
cudaError_t int8_set_wait_limit(unsigned long long ns);

// rows of `n` elements -> codes and scales; arguments checked by the caller
cudaError_t launch_quantize(const void *x, uint32_t elem, uint32_t x_stride, uint32_t rows, uint32_t n, int8_t *q, uint32_t q_stride,
                            float *scales, cudaStream_t st);

}  // namespace nvmai
