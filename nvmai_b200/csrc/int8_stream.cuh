// Products of a few rows with matrices of 8-bit codes: the codes go from HBM to the registers of mma.sync, once.
//
// A warp has 16 channels (with an activation: 8 gate rows and the 8 up rows of the same features, so that one thread has
// both sums of an output) of one matrix, up to 8 NT rows and a part of K: the block's sixteen warps split K until a part is short
// (kIsAhead steps, all requested at once; shorter where that still gives no SM a second round) and have different channels
// beyond that.  A lane fetches 16 neighbouring codes of two channels at a time and uses them as two K steps of m16n8k32: the order
// of K inside a step is free as long as both operands share it.  Few rows of 16- or 32-bit elements are quantised by every
// block that needs them.  The sums are whole numbers, so neither the split nor the order changes a bit.  Latency bounds it: one row
// 2048 -> 2 x 512 takes 2.9 us on a B200 from codes (2 MB) and 3.6 from fp16, eight experts' 16.8 MB 5.5 and 6.2.
#pragma once
#include "common.cuh"
#include "int8_gemm.cuh"
#include "row_elem.cuh"
#include "tma.cuh"

namespace nvmai {

constexpr int kIsThreads = 512, kIsWarps = 16;
constexpr uint32_t kIsStep = 64;             // codes of a row that a warp uses at a time
constexpr uint32_t kIsAhead = 4;             // steps whose codes are requested together

struct IsParams {
    const void *a; size_t a_stride; const float *a_scales;
    uint32_t rows, k;
    const int8_t *b; size_t b_stride; const float *b_scales;
    uint32_t n, channels, E;
    const uint32_t *begin;
    uint32_t act;
    void *out; uint32_t out_elem; size_t out_stride;
    uint32_t ready;                          // the kernel in front made the rows' codes and nothing else that is read here
    uint32_t row_bytes;                      // a row of codes in shared memory
    uint32_t parts;                          // of K: a power of two up to 16 warps
};

// Codes are zero from k to the end of the last step.  64 bytes more than a multiple of 128: two rows of a fragment
// load cover all banks.
__host__ __device__ constexpr uint32_t is_row_bytes(uint32_t k) {
    const uint32_t steps = (k + kIsStep - 1) / kIsStep * kIsStep;
    return steps % 128 == 0 ? steps + 64 : steps;
}
__host__ __device__ constexpr size_t is_smem(uint32_t k, uint32_t nt) { return (size_t)is_row_bytes(k) * 8 * nt + (size_t)kIsWarps * nt * 512; }

__device__ __forceinline__ void mma_i8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 codes past the L1, by an ordinary load: rows, and a matrix that was just quantised too, may come from the kernel in front, which
// still runs when the first blocks here start, and the non-coherent load is for memory that nobody writes while its kernel lives.
__device__ __forceinline__ uint4 load_codes(const int8_t *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// 16 codes of a row from position i < k on, those behind k as zeros.  Rows start on 16-byte boundaries and are readable to the next one,
// so a row's last piece is fetched whole.
__device__ __forceinline__ uint4 codes16(const int8_t *row, uint32_t i, uint32_t k) {
    uint4 v = load_codes(row + i);
    if (i + 16u > k) {
        const uint32_t n = k - i;                              // 1 .. 15 of them
        auto keep = [n](uint32_t w, uint32_t at) { return n >= at + 4u ? w : n <= at ? 0u : w & (0xffffffffu >> (32u - 8u * (n - at))); };
        v = make_uint4(keep(v.x, 0u), keep(v.y, 4u), keep(v.z, 8u), keep(v.w, 12u));
    }
    return v;
}

// T: type of the rows (int8_t: codes with a_scales).  V: elements of a row read at once.
template <typename T, int V, bool GATED, int NT>
__global__ void __launch_bounds__(kIsThreads, NT == 1 ? 2 : 1) int8_stream_kernel(IsParams p) {
    constexpr bool kCoded = sizeof(T) == 1;
    constexpr uint32_t kRows = 8 * NT, kFeatures = GATED ? 8 : 16;
    extern __shared__ __align__(16) unsigned char is_smem_raw[];
    __shared__ float scale[kRows], inverse[kRows];
    __shared__ uint32_t top[kRows], found[3];
    unsigned char *codes = is_smem_raw;
    int *partial = reinterpret_cast<int *>(is_smem_raw + (size_t)p.row_bytes * kRows);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    using P = Piece<T, V>;
    using Q = Piece<int8_t, V>;
    if (tid < kRows) top[tid] = 0u;
    if (tid == 0) found[0] = p.E;
    __syncthreads();
    auto wait_in_front = [&]() {
        pdl_wait();
        pdl_launch_dependents();
    };
    const bool ready = kCoded && p.ready != 0u;
    if (!ready) wait_in_front();

    // the rows: every kRows-th one of an expert has a block column of its own
    uint32_t row0 = blockIdx.y * kRows, e = 0, end = p.rows;
    const uint32_t pieces = p.k / V;
    if (p.begin != nullptr) row0 = blockIdx.y;
    const T *a = static_cast<const T *>(p.a) + (size_t)row0 * p.a_stride;
    P early;                                                   // of the first row, on its way while the expert is looked up
    if (!kCoded && tid < pieces) early = reinterpret_cast<const P *>(a)[tid];
    if (p.begin != nullptr) {
        for (uint32_t i = tid; i < p.E; i += kIsThreads) {
            const uint32_t from = p.begin[i], to = p.begin[i + 1];
            if (from <= row0 && row0 < to) { found[0] = i; found[1] = from; found[2] = to; }
        }
        __syncthreads();
        e = found[0];
        if (e >= p.E || (row0 - found[1]) % kRows != 0u) {
            if (ready) wait_in_front();
            return;
        }
        end = min(found[2], p.rows);
    }
    const uint32_t count = min(end - row0, kRows);

    // channels g and g + 8 of the warp's sixteen, and its part of K: every parts-th step
    const uint32_t parts = p.parts, part = warp % parts, group = warp / parts, groups = kIsWarps / parts;
    const uint32_t j0 = (blockIdx.x * groups + group) * kFeatures, j = j0 + g;
    const uint32_t c0 = j, c1 = GATED ? p.n + j : j + 8u;
    const bool live0 = j < p.n, live1 = GATED ? live0 : j + 8u < p.n;
    const int8_t *b0 = p.b + ((size_t)e * p.channels + (live0 ? c0 : 0u)) * p.b_stride;
    const int8_t *b1 = p.b + ((size_t)e * p.channels + (live1 ? c1 : 0u)) * p.b_stride;
    const uint32_t steps = (p.k + kIsStep - 1u) / kIsStep;
    uint4 w0[kIsAhead], w1[kIsAhead];
    auto request = [&](uint32_t s0) {
#pragma unroll
        for (uint32_t i = 0; i < kIsAhead; ++i) {
            const uint32_t s = s0 + i * parts, at = s * kIsStep + t * 16u;
            // behind k a channel's codes meet zeros of the rows, so its last piece needs no mask
            w0[i] = w1[i] = make_uint4(0, 0, 0, 0);
            if (at < p.k && live0) w0[i] = load_codes(b0 + at);
            if (at < p.k && live1) w1[i] = load_codes(b1 + at);
        }
    };
    request(part);
    if (ready) wait_in_front();

    // the rows' codes to shared memory, zeros behind k; rows that are not there stay what they are (their columns are not stored)
    const uint32_t padded = steps * kIsStep;
    if constexpr (kCoded) {
        const uint32_t each = padded / 16u;
        for (uint32_t i = tid; i < each * count; i += kIsThreads) {
            const uint32_t r = i / each, c = (i - r * each) * 16u;
            *reinterpret_cast<uint4 *>(codes + r * p.row_bytes + c) =
                c < p.k ? codes16(reinterpret_cast<const int8_t *>(a) + (size_t)r * p.a_stride, c, p.k) : make_uint4(0, 0, 0, 0);
        }
        if (tid < count) scale[tid] = p.a_scales[row0 + tid];
    } else {
        auto largest = [&](const P &v, uint32_t m) {
#pragma unroll
            for (int x = 0; x < V; ++x) m = max(m, magnitude_bits(elem_to_float(v.v[x])));
            return m;
        };
        // The first piece of up to three rows, or of one row of 16-byte pieces, is held between the two passes; what else there is comes
        // twice, the second time from the L1.  As many as 64 registers leave room for beside the requested codes: with four rows held
        // fp32 went through 64 bytes of local memory and bf16 through 14 (one row 2048 -> 2 x 512, four held / this: fp32 3.80 / 3.47 us,
        // bf16 4.02 / 3.62, fp16 3.72 / 3.63; three rows of bf16 4.83 / 4.19; with two held one row 3.52, three rows of fp16 4.50 for 4.23).
        // What is left of it: 16 to 32 bytes with fp32, 2 with bf16.
        auto piece = [&](uint32_t r, uint32_t i) { return reinterpret_cast<const P *>(a + (size_t)r * p.a_stride)[i]; };
        constexpr uint32_t kHeld = sizeof(P) > 8 ? 1 : 3;
        P held[kHeld];
        held[0] = early;
#pragma unroll
        for (uint32_t r = 1; r < kHeld; ++r)
            if (r < count && tid < pieces) held[r] = piece(r, tid);
        auto maximum = [&](uint32_t r, uint32_t m, uint32_t from) {
            for (uint32_t i = from; i < pieces; i += kIsThreads) m = largest(piece(r, i), m);
            m = __reduce_max_sync(0xffffffffu, m);
            if (lane == 0) atomicMax(&top[r], m);
        };
#pragma unroll
        for (uint32_t r = 0; r < kHeld; ++r)
            if (r < count) maximum(r, tid < pieces ? largest(held[r], 0u) : 0u, tid + kIsThreads);
        for (uint32_t r = kHeld; r < count; ++r) maximum(r, 0u, tid);
        __syncthreads();
        if (tid < count) {
            const RowScale rs = row_scale_bits(top[tid]);
            scale[tid] = rs.scale;
            inverse[tid] = rs.inverse;
        }
        __syncthreads();
        auto store_codes = [&](uint32_t r, uint32_t i, const P &v) {
            const RowScale rs{0.0f, inverse[r]};
            Q q;
#pragma unroll
            for (int x = 0; x < V; ++x) q.v[x] = i < pieces ? row_code(elem_to_float(v.v[x]), rs) : (int8_t)0;
            *reinterpret_cast<Q *>(codes + r * p.row_bytes + i * V) = q;
        };
        auto rest = [&](uint32_t r, uint32_t from) {
            for (uint32_t i = from; i < padded / V; i += kIsThreads) store_codes(r, i, i < pieces ? piece(r, i) : P{});
        };
#pragma unroll
        for (uint32_t r = 0; r < kHeld; ++r)
            if (r < count) {
                if (tid < padded / V) store_codes(r, tid, held[r]);
                rest(r, tid + kIsThreads);
            }
        for (uint32_t r = kHeld; r < count; ++r) rest(r, tid);
    }
    __syncthreads();

    int acc[NT][4];
#pragma unroll
    for (int x = 0; x < NT; ++x) acc[x][0] = acc[x][1] = acc[x][2] = acc[x][3] = 0;
    for (uint32_t s0 = part; s0 < steps; s0 += kIsAhead * parts) {
#pragma unroll
        for (uint32_t i = 0; i < kIsAhead; ++i) {
            const uint32_t s = s0 + i * parts;
            if (s < steps) {
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    const uint4 y = *reinterpret_cast<const uint4 *>(codes + (8u * x + g) * p.row_bytes + s * kIsStep + t * 16u);
                    mma_i8(acc[x], w0[i].x, w1[i].x, w0[i].y, w1[i].y, y.x, y.y);
                    mma_i8(acc[x], w0[i].z, w1[i].z, w0[i].w, w1[i].w, y.z, y.w);
                }
            }
        }
        if (s0 + kIsAhead * parts < steps) request(s0 + kIsAhead * parts);
    }
    // the warps' parts of the sums: [warp][tile of 8 rows][lane][4]
#pragma unroll
    for (int x = 0; x < NT; ++x)
        *reinterpret_cast<int4 *>(partial + ((warp * NT + x) * 32u + lane) * 4u) = make_int4(acc[x][0], acc[x][1], acc[x][2], acc[x][3]);
    __syncthreads();
    // out: consecutive threads take consecutive features of a row
    const uint32_t across = kFeatures * groups, first = blockIdx.x * across;
    const float *bs = p.b_scales + (size_t)e * p.channels;
    for (uint32_t i = tid; i < across * count; i += kIsThreads) {
        const uint32_t r = i / across, f = i - r * across, jf = first + f;
        if (jf >= p.n) continue;
        // row r is column r % 8 of tile r / 8: lane 4 (f % 8) + (r % 8) / 2, values r % 2 (channel f) and 2 + r % 2 (f + 8)
        const uint32_t in = f % kFeatures;
        const uint32_t at = ((f / kFeatures * parts * NT + r / 8u) * 32u + 4u * (in % 8u) + (r % 8u) / 2u) * 4u + (r % 2u) + (!GATED && in >= 8u ? 2u : 0u);
        int v = 0, u = 0;
        for (uint32_t w = 0; w < parts; ++w) {
            v += partial[w * NT * 128u + at];
            if (GATED) u += partial[w * NT * 128u + at + 2u];
        }
        float x = scaled(scale[r], bs[jf], v);
        if (GATED) x = (p.out_elem == ELEM_F32 ? gate_act<false>(x, p.act) : gate_act<true>(x, p.act)) * scaled(scale[r], bs[p.n + jf], u);
        store_elem(p.out, p.out_elem, (size_t)(row0 + r) * p.out_stride + jf, x);
    }
}

}  // namespace nvmai
