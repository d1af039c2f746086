// Products of rows with matrices of 8-bit codes: kernels and entry points.
#include "../../include/nvmai_cuda_moe.h"

#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "int8_gemm.cuh"
#include "launch.h"
#include "row_elem.cuh"
#include "tensor_map.h"
#include "tma.cuh"

using namespace nvmai;

namespace {

static_assert(kActNone == NVMAI_ACT_NONE && ACT_SILU == NVMAI_ACT_SILU && ACT_GELU == NVMAI_ACT_GELU_TANH, "activations of the header");

struct MatmulParams {
    const int8_t *a; size_t a_stride; const float *a_scales;
    uint32_t rows, k;
    const int8_t *b; size_t b_stride; const float *b_scales;
    uint32_t n, channels, E;
    const uint32_t *begin;          // or nullptr: one matrix
    uint32_t act;
    void *out; uint32_t out_elem; size_t out_stride;
};

// The expert of a row: the last e with begin[e] <= row; E where the row is nobody's.
__device__ __forceinline__ uint32_t expert_of_row(const uint32_t *begin, uint32_t E, uint32_t row) {
    if (begin == nullptr) return 0;
    if (row < begin[0] || row >= begin[E]) return E;
    uint32_t lo = 0, hi = E;                     // begin[lo] <= row < begin[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (begin[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void store_elem(void *out, uint32_t elem, size_t i, float v) {
    if (elem == ELEM_F16) static_cast<__half *>(out)[i] = __float2half_rn(v);
    else if (elem == ELEM_BF16) static_cast<__nv_bfloat16 *>(out)[i] = __float2bfloat16_rn(v);
    else static_cast<float *>(out)[i] = v;
}

// sum over a row's codes, by one warp
__device__ __forceinline__ int warp_dot(const int8_t *a, const int8_t *b, uint32_t k) {
    const uint32_t lane = threadIdx.x & 31u;
    int acc = 0;
    const uint32_t whole = k & ~15u;
    for (uint32_t i = lane * 16u; i < whole; i += 512u) {
        const int4 x = *reinterpret_cast<const int4 *>(a + i), y = *reinterpret_cast<const int4 *>(b + i);
        acc = __dp4a(x.x, y.x, acc); acc = __dp4a(x.y, y.y, acc);
        acc = __dp4a(x.z, y.z, acc); acc = __dp4a(x.w, y.w, acc);
    }
    if (lane < (k & 15u)) acc += (int)a[whole + lane] * (int)b[whole + lane];
    return __reduce_add_sync(0xffffffffu, acc);
}

// One warp per output.
__global__ void __launch_bounds__(256) int8_matmul_kernel(MatmulParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t j = blockIdx.y * 8u + (threadIdx.x >> 5), r = blockIdx.x;
    const uint32_t e = expert_of_row(p.begin, p.E, r);
    if (j >= p.n || e >= p.E) return;
    const int8_t *a = p.a + (size_t)r * p.a_stride;
    const size_t ch = (size_t)e * p.channels + j;
    const float sa = p.a_scales[r];
    float v = (sa * p.b_scales[ch]) * (float)warp_dot(a, p.b + ch * p.b_stride, p.k);
    if (p.act != kActNone) {
        const float u = (sa * p.b_scales[ch + p.n]) * (float)warp_dot(a, p.b + (ch + p.n) * p.b_stride, p.k);
        v = hidden_act(v, p.act) * u;
    }
    if ((threadIdx.x & 31u) == 0) store_elem(p.out, p.out_elem, (size_t)r * p.out_stride + j, v);
}

// codes and scales of rows that come as 16- or 32-bit elements
size_t code_stride(uint32_t k) { return ((size_t)k + 15) & ~(size_t)15; }
size_t scales_offset(uint32_t rows, uint32_t k) { return ((size_t)rows * code_stride(k) + 255) & ~(size_t)255; }

static __device__ unsigned int g_int8_status;      // a bounded wait gave up (nvmai_cuda_moe_int8_matmul_status)

// One tensor map of rows of codes in boxes of `box_rows` rows x 128 bytes, 128-byte swizzle; bytes outside read as zeros.
bool code_map(CUtensorMap *map, const void *base, uint64_t rows, uint32_t k, uint64_t stride, uint32_t box_rows) {
    const EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return false;
    const cuuint64_t dim[2] = {k, rows}, str[1] = {stride};
    const cuuint32_t box[2] = {128, box_rows}, one[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dim, str, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

unsigned int *status_word() {
    static unsigned int *at[64] = {};
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    if (at[dev] == nullptr) {
        void *p = nullptr;
        if (cudaGetSymbolAddress(&p, g_int8_status) != cudaSuccess) { cudaGetLastError(); return nullptr; }
        at[dev] = static_cast<unsigned int *>(p);
    }
    return at[dev];
}

constexpr uint32_t kSms = 148;

cudaError_t launch_gemm(const MatmulParams &m, cudaStream_t st) {
    IgArgs args;
    IgParams &p = args.p;
    p = IgParams{};
    const bool gated = m.act != kActNone;
    p.rows = m.rows; p.k = m.k; p.n = m.n; p.channels = m.channels; p.E = m.E; p.begin = m.begin;
    p.a_scales = m.a_scales; p.b_scales = m.b_scales; p.act = m.act; p.out = m.out; p.out_stride = m.out_stride;
    p.status = status_word();
    if (!p.status || !code_map(&args.a, m.a, m.rows, m.k, m.a_stride, kIgBoxRows) ||
        !code_map(&args.b, m.b, (uint64_t)m.E * m.channels, m.k, m.b_stride, 128)) return cudaErrorInvalidValue;
    const uint32_t average = (m.rows + m.E - 1) / m.E;
    p.nt = std::min(128u, std::max(32u, (average + 31) / 32 * 32));
    p.subs = gated || (uint64_t)((m.n + 255) / 256) * ((m.rows + p.nt - 1) / p.nt) >= kSms ? 2 : 1;
    p.channel_tiles = (m.n + (gated ? 128 : p.subs * 128) - 1) / (gated ? 128 : p.subs * 128);
    const size_t stage = p.subs * kIgTileBytes + (size_t)p.nt * 128;
    p.stages = (uint32_t)std::min<size_t>(kIgMaxStages, (227 * 1024 - sizeof(IgShared) - 2048) / stage);
    const size_t smem = 1024 + p.stages * stage;
    // units: at most a row tile for each expert that has rows and one for each nt rows
    const uint64_t tiles = m.begin ? std::min<uint64_t>(m.rows, (uint64_t)m.E + m.rows / p.nt) : (m.rows + p.nt - 1) / p.nt;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(kSms, tiles * p.channel_tiles);
    auto go = [&](auto T) {
        if (gated) return launch_pdl(int8_gemm_kernel<decltype(T), true>, dim3(blocks), dim3(kIgThreads), smem, st, true, args);
        return launch_pdl(int8_gemm_kernel<decltype(T), false>, dim3(blocks), dim3(kIgThreads), smem, st, true, args);
    };
    return m.out_elem == ELEM_F16 ? go(__half{}) : m.out_elem == ELEM_BF16 ? go(__nv_bfloat16{}) : go(float{});
}

}  // namespace

extern "C" {

uint64_t nvmai_cuda_moe_int8_matmul_workspace(uint32_t rows, uint32_t k, uint32_t a_elem) {
    return a_elem == NVMAI_ELEM_I8 ? 0 : scales_offset(rows, k) + (size_t)rows * 4;
}

int nvmai_cuda_moe_int8_matmul(const void *a, uint32_t a_elem, uint32_t a_stride, const float *a_scales, uint32_t rows, uint32_t k,
                               const void *b, uint32_t b_stride, const float *b_scales, uint32_t n, uint32_t num_experts,
                               const uint32_t *expert_begin, uint32_t activation, void *out, uint32_t out_elem, uint32_t out_stride,
                               void *workspace, uint64_t workspace_bytes, void *stream) {
    if (!b || !b_scales || (rows != 0 && (!a || !out))) return NVMAI_CUDA_EINVAL;
    if (a_elem > ELEM_I8 || out_elem > ELEM_BF16 || activation > NVMAI_ACT_NONE) return NVMAI_CUDA_EINVAL;
    if (k == 0 || n == 0 || a_stride < k || b_stride < k || out_stride < n) return NVMAI_CUDA_EINVAL;
    if (num_experts == 0 || (!expert_begin && num_experts != 1)) return NVMAI_CUDA_EINVAL;
    const uint64_t channels = activation == NVMAI_ACT_NONE ? n : 2ull * n;
    if (k >= 131072 || num_experts > kRowMaxExperts || rows >= (1u << 31) || channels * num_experts >= (1ull << 31)) return NVMAI_CUDA_ERANGE;
    if (!aligned_to(b, 16) || b_stride % 16 != 0 || !aligned_to(b_scales, 4) || !aligned_to(out, elem_size(out_elem)) || !aligned_to(expert_begin, 4))
        return NVMAI_CUDA_EINVAL;
    const bool coded = a_elem == ELEM_I8;
    if (coded != (a_scales != nullptr) && rows != 0) return NVMAI_CUDA_EINVAL;
    if (coded ? !aligned_to(a, 16) || a_stride % 16 != 0 || !aligned_to(a_scales, 4) : !aligned_to(a, elem_size(a_elem))) return NVMAI_CUDA_EINVAL;
    if (rows == 0) return NVMAI_CUDA_OK;
    if (!coded) {
        if (workspace_bytes < nvmai_cuda_moe_int8_matmul_workspace(rows, k, a_elem)) return NVMAI_CUDA_ERANGE;
        if (!workspace || !aligned_to(workspace, 16)) return NVMAI_CUDA_EINVAL;
    }
    if (!on_current_device({a, a_scales, b, b_scales, expert_begin, out, coded ? nullptr : workspace})) return NVMAI_CUDA_EINVAL;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    MatmulParams p{};
    p.rows = rows; p.k = k;
    p.b = static_cast<const int8_t *>(b); p.b_stride = b_stride; p.b_scales = b_scales;
    p.n = n; p.channels = (uint32_t)channels; p.E = num_experts; p.begin = expert_begin; p.act = activation;
    p.out = out; p.out_elem = out_elem; p.out_stride = out_stride;
    if (coded) {
        p.a = static_cast<const int8_t *>(a); p.a_stride = a_stride; p.a_scales = a_scales;
    } else {
        int8_t *q = static_cast<int8_t *>(workspace);
        float *scales = reinterpret_cast<float *>(q + scales_offset(rows, k));
        const cudaError_t e = launch_quantize(a, a_elem, a_stride, rows, k, q, (uint32_t)code_stride(k), scales, st);
        count_launches(1);
        if (e != cudaSuccess) { cudaGetLastError(); return NVMAI_CUDA_ECUDA; }
        p.a = q; p.a_stride = code_stride(k); p.a_scales = scales;
    }
    const cudaError_t e = rows > 8 ? launch_gemm(p, st) : launch_pdl(int8_matmul_kernel, dim3(rows, (n + 7) / 8), dim3(256), 0, st, true, p);
    count_launches(1);
    if (e != cudaSuccess) { cudaGetLastError(); return NVMAI_CUDA_ECUDA; }
    return NVMAI_CUDA_OK;
}

int nvmai_cuda_moe_int8_matmul_status(void *stream) {
    unsigned int status = 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cudaMemcpyFromSymbolAsync(&status, g_int8_status, sizeof(status), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
        cudaStreamSynchronize(st) != cudaSuccess) {
        cudaGetLastError();
        return NVMAI_CUDA_ECUDA;
    }
    if (status == 0) return NVMAI_CUDA_OK;
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbolAsync(g_int8_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st) != cudaSuccess) {
        cudaGetLastError();
        return NVMAI_CUDA_ECUDA;
    }
    return NVMAI_CUDA_ETIMEOUT;
}

}  // extern "C"
