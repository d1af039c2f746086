// Products of rows with matrices of 8-bit codes: kernels and entry points.
#include "../../include/nvmai_cuda_moe.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "give_ups.h"
#include "int8_gemm.cuh"
#include "int8_stream.cuh"
#include "launch.h"
#include "row_elem.cuh"
#include "tensor_map.h"
#include "tma.cuh"

using namespace nvmai;

namespace {

static_assert(kActNone == NVMAI_ACT_NONE && ACT_SILU == NVMAI_ACT_SILU && ACT_GELU == NVMAI_ACT_GELU_TANH, "activations of the header");

struct Matmul {
    const void *a; uint32_t a_elem; size_t a_stride; const float *a_scales;
    uint32_t rows, k;
    const int8_t *b; size_t b_stride; const float *b_scales;
    uint32_t n, channels, E;
    const uint32_t *begin;          // or nullptr: one matrix
    uint32_t act;
    void *out; uint32_t out_elem; size_t out_stride;
    bool ready;                     // the call's own quantisation is the kernel in front
};

// codes and scales of rows that come as 16- or 32-bit elements
size_t code_stride(uint32_t k) { return ((size_t)k + 15) & ~(size_t)15; }
size_t scales_offset(uint32_t rows, uint32_t k) { return ((size_t)rows * code_stride(k) + 255) & ~(size_t)255; }

// One tensor map of rows of codes in boxes of `box_rows` rows x 128 bytes, 128-byte swizzle; bytes outside read as zeros.
bool code_map(CUtensorMap *map, const void *base, uint64_t rows, uint32_t k, uint64_t stride, uint32_t box_rows) {
    const EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return false;
    const cuuint64_t dim[2] = {k, rows}, str[1] = {stride};
    const cuuint32_t box[2] = {128, box_rows}, one[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dim, str, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

std::atomic<bool> g_drop_copy{false};      // test hook, see nvmai_cuda_moe_debug_drop_int8_copy

// made with the first call and never destroyed: threads may still ask while the process ends
GiveUps &give_ups() {
    static GiveUps *all = new GiveUps;
    return *all;
}

constexpr uint32_t kSms = 148;

struct IgTile { uint32_t subs, nt; };

// Features of a unit.
uint32_t unit_features(const Matmul &m, uint32_t subs) { return m.act != kActNone ? 128 : 128 * subs; }

// The cheapest tile for `experts` runs of `rows` rows by a model of the time, in ns, fitted to 16 shapes of one matrix (40 to 16384
// rows, 512 to 2048 codes, 300 to 2048 channels): a K block costs 104 and 4.1 for each KB of it, the last epilogue of a block 10 for
// each row and tile of its unit (an activation counts double), earlier ones 6.5 beside the next unit or, with one set of
// accumulators, 10 in its way.  The tile it picks took at most 9 % longer than the best one in those shapes, 128 rows of two
// tiles up to 80 %.
IgTile cheapest_tile(const Matmul &m, uint32_t experts, float rows) {
    const bool gated = m.act != kActNone;
    const float blocks = (float)((m.k + 127) / 128);
    IgTile best{};
    float best_ns = INFINITY;
    for (uint32_t subs = gated ? 2 : 1; subs <= 2; ++subs)
        for (uint32_t nt = 32; nt * subs <= 512 && nt <= 256; nt += 32) {
            const float tiles = std::ceil(rows / (float)nt), units = tiles * (float)experts * (float)((m.n + unit_features(m, subs) - 1) / unit_features(m, subs));
            const float waves = std::ceil(units / (float)kSms), per = std::ceil(rows / tiles / 16.0f) * 16.0f;
            const float kb = (float)(16 * subs) + std::ceil(per / 32.0f) * 4.0f, outs = per * (float)(subs * (gated ? 2 : 1));
            const float epilogues = 2 * subs * nt <= 512 ? 10.4f + 6.5f * (waves - 1.0f) : 10.4f * waves;
            const float ns = waves * blocks * (104.0f + 4.1f * kb) + outs * epilogues;
            if (ns < best_ns) { best_ns = ns; best = IgTile{subs, nt}; }
            if ((float)nt >= rows) break;
        }
    return best;
}

// One matrix, or one for each expert.  With three units an SM or more (counted for all experts, those without rows too), the rule is
// made for many experts, where HBM is the limit: the codes come once for each unit of an expert (past the first from the L2), so a
// unit holds the average expert and 2.5 times the spread of an even routing around it.  Past 128 rows that leaves one set of
// accumulators; 256 experts of 128 rows on average, 2048 -> 2 x 512: 128 rows a unit 114.1 us, 160 106.0, 192 106.6 (three ring slots
// instead of four); 512 -> 2048: 76.2, 70.0, 69.6.  Two channel tiles a unit read the rows half as often: 201 tokens, 512 -> 2048,
// 52.6 us with one, 45.4 with two.  Below three units an SM the model picks, for the average and twice the spread: 41 tokens x 8
// through 8 experts of 1711 -> 596 10.9 us with the rule above, 7.4 to 8.1 with the model; 201 x 8 through 16 of 2048 -> 2 x 512
// 13.4 / 12.0; 1000 x 8 through 64 of those 34.8 / 35.4.  Few large experts are bound by the operations, which the rule does not
// know: 4096 x 8 through 8 of those 66.2 us with it, 61.4 with the model, 512 -> 2048 51 / 48; through 64 75.9 / 74.1 and 53.8 / 55.5.
IgTile row_tile(const Matmul &m) {
    if (m.begin == nullptr) return cheapest_tile(m, 1, (float)m.rows);
    const float average = (float)m.rows / (float)m.E;
    const uint32_t want = (uint32_t)std::ceil((average + 2.5f * std::sqrt(average)) / 32.0f) * 32u;
    const IgTile tile{m.act != kActNone || m.n > 128 ? 2u : 1u, std::min(160u, std::max(32u, want))};
    const float units = std::ceil(average / (float)tile.nt) * (float)m.E * (float)((m.n + unit_features(m, tile.subs) - 1) / unit_features(m, tile.subs));
    return units >= 3.0f * (float)kSms ? tile : cheapest_tile(m, m.E, std::max(1.0f, average + 2.0f * std::sqrt(average)));
}

cudaError_t launch_gemm(const Matmul &m, cudaStream_t st) {
    IgArgs args;
    IgParams &p = args.p;
    p = IgParams{};
    const bool gated = m.act != kActNone;
    p.rows = m.rows; p.k = m.k; p.n = m.n; p.channels = m.channels; p.E = m.E; p.begin = m.begin;
    p.a_scales = m.a_scales; p.b_scales = m.b_scales; p.act = m.act; p.out = m.out; p.out_stride = m.out_stride;
    // a matrix of fewer than 128 features fetches no more rows than it has: 176 rows of 1161 -> 2 x 21 by 83 experts 9.6 -> 8.2 us
    p.box_channels = std::min(128u, (m.n + 7) / 8 * 8);
    if (!code_map(&args.a, m.a, m.rows, m.k, m.a_stride, kIgBoxRows) ||
        !code_map(&args.b, m.b, (uint64_t)m.E * m.channels, m.k, m.b_stride, p.box_channels)) return cudaErrorInvalidValue;
    const IgTile tile = row_tile(m);
    const uint32_t subs = tile.subs;
    p.nt = tile.nt;
    p.channel_tiles = (m.n + unit_features(m, subs) - 1) / unit_features(m, subs);
    const size_t stage = subs * kIgTileBytes + (size_t)p.nt * 128;
    p.accs = 2 * subs * p.nt <= 512 ? 2 : 1;
    p.ready = m.ready;
    p.debug_drop_rows = g_drop_copy.exchange(false) ? 1 : 0;
    // A small output stays in the L2 for its reader if the codes, read once, make room first; a larger one is in the way of the rows
    // then.  By expert, 512 -> 2048 fp16 out, three sets of buffers in turn, without / with on a B200: 201 tokens (7 MB) 46.2 / 45.2 us,
    // 512 (17 MB) 48.1 / 48.3, 800 (26 MB) 49.7 / 52.7, 2500 (82 MB) 59.3 / 65.3; 2048 -> 2 x 512, 201 tokens 86.9 / 85.0.
    p.evict_first = m.begin != nullptr && (uint64_t)m.rows * m.n * elem_size(m.out_elem) <= (16u << 20) ? 1 : 0;
    p.paired = m.n % 2 == 0 && m.out_stride % 2 == 0 && aligned_to(m.out, 4);
    p.stages = (uint32_t)std::min<size_t>(kIgMaxStages, (227 * 1024 - sizeof(IgShared) - 2048) / stage);
    const size_t smem = 1024 + p.stages * stage;
    // units: at most a row tile for each expert that has rows and one for each nt rows
    const uint64_t tiles = m.begin ? std::min<uint64_t>(m.rows, (uint64_t)m.E + m.rows / p.nt) : (m.rows + p.nt - 1) / p.nt;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(kSms, tiles * p.channel_tiles);
    auto go = [&](auto T) {
        if (gated) return launch_pdl(int8_gemm_kernel<decltype(T), true, 2>, dim3(blocks), dim3(kIgThreads), smem, st, true, args);
        if (subs == 2) return launch_pdl(int8_gemm_kernel<decltype(T), false, 2>, dim3(blocks), dim3(kIgThreads), smem, st, true, args);
        return launch_pdl(int8_gemm_kernel<decltype(T), false, 1>, dim3(blocks), dim3(kIgThreads), smem, st, true, args);
    };
    return m.out_elem == ELEM_F16 ? go(__half{}) : m.out_elem == ELEM_BF16 ? go(__nv_bfloat16{}) : go(float{});
}

// The streaming kernel's tiles of 8 rows, 0: the tcgen05 kernel's.  One matrix: up to 16 rows, up to 32 where the tcgen05 kernel would
// go through eight K blocks or more one after the other (codes on a B200, streaming / tcgen05: 2048 -> 2 x 512, 1 row 2.9 / 8.1 us,
// 16 rows 4.2 / 8.1, 32 rows 5.9 / 8.3; 512 -> 2048, 16 rows 3.2 / 4.1, 32 rows 4.2 / 4.2; 1024 -> 1024, 32 rows 4.3 / 4.9).  By
// expert a block has the rows of one, and every one fetches its codes anew: while rows x k is below 2^15 (8 rows of 2048: 5.4 /
// 9.8 us, 16 rows 10.9 / 10.4, 24 rows 15.4 / 12.4; 16 rows of 512 4.9 / 6.1, 32 rows 9.9 / 9.7, 64 rows 16.3 / 14.0).
uint32_t stream_tiles(const Matmul &m) {
    if (m.begin != nullptr ? (uint64_t)m.rows * m.k >= 32768 || m.rows > 64 : m.rows > (m.k >= 1024 ? 32u : 16u)) return 0;
    const uint32_t nt = m.begin != nullptr || m.rows <= 8 ? 1 : m.rows <= 16 ? 2 : 4;
    return is_smem(m.k, nt) <= 200 * 1024 ? nt : 0;
}
// Does it quantise the rows itself?  Each of its blocks then does, 0.3 us a row of 2048 in front of the product; a launch for all of
// them runs beside the fetching of the codes, and costs the host 2.4 us (2048 -> 2 x 512, one launch / two: 1 row 3.6 / 4.4 us, 3
// rows 4.2 / 4.2, 4 rows 4.9 / 4.2; 3 rows of 4096 6.2 / 4.9; one token through eight experts 6.2 / 6.3).
bool stream_quantizes(const Matmul &m) { return m.begin != nullptr || (m.rows <= 4 && m.rows * m.k <= 6144); }

cudaError_t launch_stream(const Matmul &m, uint32_t nt, cudaStream_t st) {
    using std::integral_constant;
    const bool gated = m.act != kActNone;
    IsParams p{m.a, m.a_stride, m.a_scales, m.rows, m.k, m.b, m.b_stride, m.b_scales, m.n, m.channels, m.E, m.begin, m.act,
               m.out, m.out_elem, m.out_stride, m.ready, is_row_bytes(m.k), 1};
    const uint32_t steps = (m.k + kIsStep - 1) / kIsStep, columns = m.begin != nullptr ? m.rows : (m.rows + 8 * nt - 1) / (8 * nt);
    const uint32_t features = (gated ? 8 : 16) * kIsWarps;                // of a block whose warps do not split K
    auto blocks = [&] { return (uint32_t)(((uint64_t)m.n * p.parts + features - 1) / features); };
    const uint64_t resident = nt == 1 ? 2 * kSms : kSms;                 // blocks
    while (p.parts < kIsWarps && p.parts < steps && (steps > p.parts * kIsAhead || 2ull * blocks() * columns <= resident)) p.parts *= 2;
    const dim3 grid(blocks(), columns);
    auto go = [&](auto T, auto V, auto G, auto N) {
        return launch_pdl(int8_stream_kernel<decltype(T), decltype(V)::value, decltype(G)::value, decltype(N)::value>, grid,
                          dim3(kIsThreads), is_smem(m.k, nt), st, true, p);
    };
    // rows that the kernel quantises itself are eight a block at most (stream_quantizes)
    auto with_tiles = [&](auto T, auto V, auto G) {
        if constexpr (sizeof(T) == 1) {
            if (nt == 2) return go(T, V, G, integral_constant<int, 2>{});
            if (nt == 4) return go(T, V, G, integral_constant<int, 4>{});
        }
        return go(T, V, G, integral_constant<int, 1>{});
    };
    auto with_gate = [&](auto T, auto V) {
        return gated ? with_tiles(T, V, integral_constant<bool, true>{}) : with_tiles(T, V, integral_constant<bool, false>{});
    };
    if (m.a_elem == ELEM_I8) return with_gate(int8_t{}, integral_constant<int, 16>{});
    const bool wide = m.k % 4 == 0 && m.a_stride % 4 == 0 && aligned_to(m.a, 4 * elem_size(m.a_elem));     // four elements at once
    auto with_pieces = [&](auto T, auto V) { return wide ? with_gate(T, V) : with_gate(T, integral_constant<int, 1>{}); };
    return m.a_elem == ELEM_F32 ? with_pieces(float{}, integral_constant<int, 4>{})
           : m.a_elem == ELEM_BF16 ? with_pieces(__nv_bfloat16{}, integral_constant<int, 4>{}) : with_pieces(__half{}, integral_constant<int, 4>{});
}

}  // namespace

cudaError_t nvmai::int8_set_wait_limit(unsigned long long ns) { return cudaMemcpyToSymbol(g_wait_limit_ns, &ns, sizeof(ns)); }

extern "C" {

uint64_t nvmai_cuda_moe_int8_matmul_workspace(uint32_t rows, uint32_t k, uint32_t a_elem) {
    return a_elem == NVMAI_ELEM_I8 ? 0 : scales_offset(rows, k) + (size_t)rows * 4;
}

int nvmai_cuda_moe_int8_matmul(const void *a, uint32_t a_elem, uint32_t a_stride, const float *a_scales, uint32_t rows, uint32_t k,
                               const void *b, uint32_t b_stride, const float *b_scales, uint32_t n, uint32_t num_experts,
                               const uint32_t *expert_begin, uint32_t activation, void *out, uint32_t out_elem, uint32_t out_stride,
                               void *workspace, uint64_t workspace_bytes, void *stream) {
    return without_exceptions([&]() -> int {
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
        int dev = -1;
        if (!on_current_device({a, a_scales, b, b_scales, expert_begin, out, coded ? nullptr : workspace}, &dev)) return NVMAI_CUDA_EINVAL;
        give_ups().product(dev, stream);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        Matmul m{a, a_elem, a_stride, a_scales, rows, k, static_cast<const int8_t *>(b), b_stride, b_scales, n, (uint32_t)channels,
                 num_experts, expert_begin, activation, out, out_elem, out_stride, false};
        auto launched = [](cudaError_t e) {
            count_launches(1);
            if (e != cudaSuccess) cudaGetLastError();
            return e == cudaSuccess ? NVMAI_CUDA_OK : NVMAI_CUDA_ECUDA;
        };
        const uint32_t nt = stream_tiles(m);
        if (!coded && !(nt && stream_quantizes(m))) {
            int8_t *q = static_cast<int8_t *>(workspace);
            float *scales = reinterpret_cast<float *>(q + scales_offset(rows, k));
            const int rc = launched(launch_quantize(a, a_elem, a_stride, rows, k, q, (uint32_t)code_stride(k), scales, st));
            if (rc) return rc;
            m.a = q; m.a_elem = ELEM_I8; m.a_stride = code_stride(k); m.a_scales = scales; m.ready = true;
        }
        return launched(nt ? launch_stream(m, nt, st) : launch_gemm(m, st));
    });
}

int nvmai_cuda_moe_int8_matmul_status(void *stream) {
    return without_exceptions([&]() -> int {
        unsigned int count = 0;
        int dev = -1;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaStreamIsCapturing(st, &capturing) != cudaSuccess) { cudaGetLastError(); return NVMAI_CUDA_ECUDA; }
        if (capturing != cudaStreamCaptureStatusNone) return NVMAI_CUDA_EINVAL;        // a capture has nothing to wait for
        if (cudaMemcpyFromSymbolAsync(&count, g_int8_give_ups, sizeof(count), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
            cudaStreamSynchronize(st) != cudaSuccess) {
            cudaGetLastError();
            return NVMAI_CUDA_ECUDA;
        }
        return give_ups().news(dev, stream, count) ? NVMAI_CUDA_ETIMEOUT : NVMAI_CUDA_OK;
    });
}

int nvmai_cuda_moe_debug_drop_int8_copy(void) {
    g_drop_copy.store(true);
    return NVMAI_CUDA_OK;
}

}  // extern "C"
