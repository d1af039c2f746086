// Products of many rows with matrices of 8-bit codes: tcgen05.mma kind::i8 (32-bit integer sums) from TMA-fed shared memory.
//
// The matrix is the M operand (128 channels a tile), the rows are N: a tile takes any multiple of 16 rows, so an expert with
// few rows costs few columns.  Two tiles of channels share a block of rows (with an activation: the gate rows and the up rows
// of the same 128 features, so that one thread has both accumulators of an output).  Persistent: one block per SM, units in
// the order (expert, channel tile, row tile), so that the row tiles that read the same codes run beside each other and the
// codes cross HBM once.  Warps: 16 epilogue, 1 for the copies, 1 for the MMAs; the accumulators are double-buffered where two sets
// fit.  By expert HBM bounds it: on a B200, 4096 tokens x 8 through 256 experts of 2048 -> 2 x 512 take 110 us (5.8 TB/s; 116 to 126
// in loops of seconds under the power cap, where leaving out three MMAs of four gave 109), 201 tokens of 512 -> 2048 45 us (6.2 TB/s).
// One matrix of 2048 -> 2 x 1024 and 16384 rows: 55 us, 2.5 x 10^15 operations a second (59 with three sets of rows in turn).
#pragma once
#include <type_traits>

#include "common.cuh"
#include "row_elem.cuh"
#include "tcgen05.cuh"

namespace nvmai {

constexpr int kIgEpilogueWarps = 16, kIgCopyWarp = 16, kIgMmaWarp = 17, kIgThreads = 576;
constexpr uint32_t kIgMaxStages = 8, kIgBoxRows = 32;
constexpr uint32_t kIgTileBytes = 128 * 128;           // 128 channels x 128 codes
constexpr uint32_t kActNone = 2;

static __device__ unsigned int g_int8_give_ups;    // bounded waits that ran out, never cleared (give_ups.h)

struct IgParams {
    uint32_t rows, k, n, channels, E;
    const uint32_t *begin;               // first row of each expert, or nullptr: one matrix
    const float *a_scales, *b_scales;
    uint32_t act;
    void *out; size_t out_stride;
    uint32_t nt, stages;                 // most rows of a unit (a multiple of 32), ring slots
    uint32_t evict_first;                // the matrix's lines leave the L2 before others
    uint32_t accs;                       // sets of accumulators (2, or 1 where two do not fit)
    uint32_t ready;                      // the kernel in front made the rows' codes and nothing else that is read here
    uint32_t paired;                     // 16-bit outputs: two neighbouring channels go out in one store
    uint32_t channel_tiles;              // units across the channels
    uint32_t box_channels;               // rows of a box of the matrix: 128, or what a narrower matrix has (lanes past it are not stored)
    uint32_t debug_drop_rows;            // test hook: block 0 leaves out the rows of its second K block, so waits run out
};
struct alignas(64) IgArgs {
    CUtensorMap a, b;                    // [rows][k], [E * channels][k] bytes; boxes of 32 and of box_channels rows x 128 bytes
    IgParams p;
};

__device__ __forceinline__ void umma_i8_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor, kind::i8: 32-bit integer accumulator (2 in bits 4-5), A and B signed (1 in bits 7-9 and 10-12),
// both K-major, N >> 3 in bits 17-22, M >> 4 in bits 24-28.
__device__ __forceinline__ uint32_t umma_idesc_i8(uint32_t m, uint32_t n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
// The gate's activation: g / (1 + e^-z), which for SiLU has z = g, and for the tanh form of GELU, 0.5 g (1 + tanh y), z = 2 y (1 + tanh
// itself keeps no digit of a value near 0: below g = -5.2 the result would be 0).  Below z = 0 as g / (1 + e^z) e^z, so that no e^
// overflows: with the first form alone everything below -88.7 would be 0, and times a large up row it is not.
// The hardware's exp2 and reciprocal have an error of (2 |z| + 9) 2^-24 (the argument's roundings, 2 ulp, 1 ulp and three more
// roundings), at most 0.013 of fp16's rounding and 0.002 of bf16's up to |z| = 50, 0.021 and 0.003 up to 80; GELU's z is off by
// 6 |z| 2^-24 before that.  So 16-bit outputs (HALF) and GELU take them; SiLU for fp32 outputs takes expf and the exact division,
// which cost more than the rest of an output (GELU with them, 4096 tokens, fp32 out: 128 us).
// Roundings are named where the compiler could fuse a product and a sum in one kernel and not in another: a row's bits
// do not depend on the kernel.
template <bool HALF>
__device__ __forceinline__ float gate_act(float g, uint32_t act) {
    const float z = act == ACT_SILU ? g : __fmul_rn(2.0f * 0.7978845608028654f, __fmaf_rn(0.044715f, __fmul_rn(__fmul_rn(g, g), g), g));
    float e, q;
    if (HALF || act != ACT_SILU) {
        asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(fabsf(z), -1.4426950408889634f)));
        asm("rcp.approx.f32 %0, %1;" : "=f"(q) : "f"(__fadd_rn(1.0f, e)));
        q *= g;
    } else {
        e = expf(-fabsf(z));
        q = g / __fadd_rn(1.0f, e);
    }
    return z < 0.0f ? q * e : q;
}
// value of a whole-number sum
__device__ __forceinline__ float scaled(float sa, float sb, int sum) { return __fmul_rn(__fmul_rn(sa, sb), (float)sum); }

// A box of the matrix whose lines are the first to leave the L2.
__device__ __forceinline__ uint64_t evict_first_policy() {
    uint64_t v;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(v));
    return v;
}
__device__ __forceinline__ void tma_load_2d_once(uint32_t dst_smem, const CUtensorMap *map, uint32_t c0, uint32_t c1, uint64_t *bar, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;"
                 ::"r"(dst_smem), "l"(map), "r"(c0), "r"(c1), "r"(smem_addr(bar)), "l"(policy)
                 : "memory");
}

struct IgShared {
    uint64_t full[kIgMaxStages], empty[kIgMaxStages], acc_full[2], acc_empty[2], drained;
    uint32_t tmem_slot, warp_sums[8];
    uint32_t gave_up;
    uint32_t tiles[kRowMaxExperts + 1];       // row tiles of the experts in front
    uint32_t first[kRowMaxExperts + 1];       // first row of each expert
    float4 row_scales[kIgEpilogueWarps][16];  // of the columns of an epilogue warp
};

struct IgUnit { uint32_t e, row, count, ch; };       // rows row .. row + count - 1 of expert e, channel tile ch

__device__ __forceinline__ IgUnit ig_unit(const IgShared &s, const IgParams &p, uint32_t u) {
    uint32_t lo = 0, hi = p.E;                        // tiles[lo] * C <= u < tiles[hi] * C
    const uint32_t tile = u / p.channel_tiles;        // a row tile of the same expert
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s.tiles[mid] <= tile) lo = mid; else hi = mid;
    }
    const uint32_t t_e = s.tiles[lo + 1] - s.tiles[lo], r = u - s.tiles[lo] * p.channel_tiles;
    const uint32_t n_e = s.first[lo + 1] - s.first[lo];
    const uint32_t per = ((n_e + t_e - 1) / t_e + 15u) & ~15u;      // even tiles; the last one keeps at least a row
    IgUnit un;
    un.e = lo;
    un.ch = r / t_e;
    const uint32_t at = (r - un.ch * t_e) * per;
    un.row = s.first[lo] + at;
    un.count = min(per, n_e - at);
    return un;
}

// SUBS: channel tiles of a unit (2 with an activation).
template <typename OUT, bool GATED, uint32_t SUBS>
__global__ void __launch_bounds__(kIgThreads, 1) int8_gemm_kernel(const __grid_constant__ IgArgs args) {
    const IgParams &p = args.p;
    __shared__ IgShared s;
    extern __shared__ unsigned char ig_ring_raw[];
    const uint32_t ring = (smem_addr(ig_ring_raw) + 1023u) & ~1023u;
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;

    if (tid == 0) {
        for (uint32_t i = 0; i < p.stages; ++i) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 1); }
        for (uint32_t i = 0; i < 2; ++i) { mbar_init(&s.acc_full[i], 1); mbar_init(&s.acc_empty[i], kIgEpilogueWarps); }
        mbar_init(&s.drained, 1);
        mbar_fence_init();
        s.gave_up = 0u;
    }
    if (warp == kIgMmaWarp) {
        tmem_alloc(&s.tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == kIgCopyWarp && lane == 0) { tma_prefetch_map(&args.a); tma_prefetch_map(&args.b); }
    auto wait_in_front = [&]() {
        pdl_wait();
        pdl_launch_dependents();
    };
    if (!p.ready) wait_in_front();
    // Row tiles in front of each expert: a thread adds up to four experts, the warps' sums are put together.  Begins behind
    // the last row or out of order give an expert fewer rows or none, never rows outside.
    {
        const uint32_t per = (p.E + 255u) / 256u, e0 = tid * per;
        uint32_t mine[4] = {0, 0, 0, 0}, sum = 0;
        if (tid < 256u) {
            for (uint32_t i = 0; i < per && e0 + i < p.E; ++i) {
                const uint32_t a = p.begin ? min(p.begin[e0 + i], p.rows) : 0u, b = p.begin ? min(p.begin[e0 + i + 1], p.rows) : p.rows;
                mine[i] = b > a ? (b - a + p.nt - 1u) / p.nt : 0u;
                s.first[e0 + i] = a;
                sum += mine[i];
            }
            uint32_t run = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= (uint32_t)o) run += up;
            }
            if (lane == 31u) s.warp_sums[warp] = run;
            sum = run - sum;
        }
        if (tid == 0) s.first[p.E] = p.begin ? min(p.begin[p.E], p.rows) : p.rows;
        tc_fence_before_sync();
        __syncthreads();
        tc_fence_after_sync();
        if (tid < 256u) {
            for (uint32_t w = 0; w < warp; ++w) sum += s.warp_sums[w];
            for (uint32_t i = 0; i < per && e0 + i < p.E; ++i) {
                s.tiles[e0 + i] = sum;
                sum += mine[i];
                if (e0 + i + 1 == p.E) s.tiles[p.E] = sum;
            }
        }
        __syncthreads();
    }
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&s.tmem_slot);
    const uint32_t total = s.tiles[p.E] * p.channel_tiles;
    const uint32_t n_kb = (p.k + 127u) / 128u;
    const uint32_t stage_bytes = SUBS * kIgTileBytes + p.nt * 128u;

    // bounded by the GPU's nanosecond timer; a role that gives up tells the others
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (mbar_try_wait_short(bar, parity)) return true;
        const unsigned long long t0 = global_timer_ns(), limit = g_wait_limit_ns;
        for (;;) {
#pragma unroll 1
            for (int it = 0; it < 16; ++it)
                if (mbar_try_wait_short(bar, parity)) return true;
            if (*reinterpret_cast<volatile uint32_t *>(&s.gave_up) != 0u) return false;
            if (global_timer_ns() - t0 > limit) break;
        }
        *reinterpret_cast<volatile uint32_t *>(&s.gave_up) = 1u;
        atomicAdd(&g_int8_give_ups, 1u);
        return false;
    };

    if (warp == kIgCopyWarp) {
        if (elect_one()) {
            uint32_t stage = 0, parity = 1, filled = 0;         // the first pass finds every slot empty
            bool ok = true;
            const uint64_t policy = evict_first_policy();
            // channel tiles of a unit's K block; a unit's bytes are announced with them
            auto load_channels = [&](const IgUnit &un, uint32_t kb, uint32_t at) {
                const uint32_t boxes = (un.count + kIgBoxRows - 1u) / kIgBoxRows, slot = ring + at * stage_bytes;
                const uint32_t ch0 = un.e * p.channels + un.ch * (GATED ? 128u : SUBS * 128u);
                mbar_expect_tx(&s.full[at], (SUBS * p.box_channels + boxes * kIgBoxRows) * 128u);
#pragma unroll
                for (uint32_t t = 0; t < SUBS; ++t) {
                    const uint32_t ch = ch0 + t * (GATED ? p.n : 128u);
                    if (p.evict_first) tma_load_2d_once(slot + t * kIgTileBytes, &args.b, kb * 128u, ch, &s.full[at], policy);
                    else tma_load_2d(slot + t * kIgTileBytes, &args.b, kb * 128u, ch, &s.full[at]);
                }
            };
            uint32_t early = 0;                                  // K blocks whose channels are on their way before the rows can be
            if (p.ready && blockIdx.x < total) {
                const IgUnit un = ig_unit(s, p, blockIdx.x);
                for (early = 0; early < min(n_kb, p.stages); ++early) load_channels(un, early, early);
            }
            if (p.ready) wait_in_front();
            for (uint32_t u = blockIdx.x; ok && u < total; u += gridDim.x) {
                const IgUnit un = ig_unit(s, p, u);
                const uint32_t boxes = (un.count + kIgBoxRows - 1u) / kIgBoxRows;
                for (uint32_t kb = 0; kb < n_kb; ++kb) {
                    const uint32_t slot = ring + stage * stage_bytes;
                    if (early != 0u) {
                        --early;
                    } else {
                        if (!(ok = wait(&s.empty[stage], parity))) break;
                        load_channels(un, kb, stage);
                    }
                    const bool drop = p.debug_drop_rows != 0u && u == 0u && kb == 1u;
                    for (uint32_t i = 0; i < boxes && !drop; ++i)
                        tma_load_2d(slot + SUBS * kIgTileBytes + i * kIgBoxRows * 128u, &args.a, kb * 128u, un.row + i * kIgBoxRows, &s.full[stage]);
                    ++filled;
                    if (++stage == p.stages) { stage = 0; parity ^= 1u; }
                }
            }
            if (!ok) {      // copies in flight end before the block does
                const unsigned long long t0 = global_timer_ns(), limit = g_wait_limit_ns;
                for (uint32_t i = 0; i < min(filled, p.stages); ++i) {
                    const uint32_t at = (stage + p.stages - 1u - i) % p.stages, lap = (filled - 1u - i) / p.stages;
                    while (!mbar_try_wait_short(&s.full[at], lap & 1u) && global_timer_ns() - t0 < limit) {}
                }
            }
        }
    } else if (warp == kIgMmaWarp) {
        if (elect_one()) {
            uint32_t stage = 0, parity = 0, it = 0;
            const uint64_t ring_desc = umma_desc_sw128(ring);
            bool ok = true;
            for (uint32_t u = blockIdx.x; ok && u < total; u += gridDim.x, ++it) {
                const IgUnit un = ig_unit(s, p, u);
                const uint32_t idesc = umma_idesc_i8(128u, (un.count + 15u) & ~15u);
                const uint32_t buf = p.accs == 2u ? it & 1u : 0u, turn = p.accs == 2u ? it >> 1 : it, acc = tmem + buf * SUBS * p.nt;
                if (!(ok = wait(&s.acc_empty[buf], (turn & 1u) ^ 1u))) break;
                tc_fence_after_sync();
                for (uint32_t kb = 0; kb < n_kb; ++kb) {
                    if (!(ok = wait(&s.full[stage], parity))) break;
                    tc_fence_after_sync();
                    const uint64_t a = ring_desc + stage * (stage_bytes >> 4), b = a + (SUBS * kIgTileBytes >> 4);
#pragma unroll
                    for (uint32_t t = 0; t < SUBS; ++t) {
#pragma unroll
                        for (uint32_t kk = 0; kk < 4u; ++kk)           // 32 codes = 32 bytes = 2 units of the descriptor's address
                            umma_i8_ss(acc + t * p.nt, a + t * (kIgTileBytes >> 4) + 2u * kk, b + 2u * kk, idesc, kk ? 1u : kb);
                    }
                    umma_commit(&s.empty[stage]);
                    if (++stage == p.stages) { stage = 0; parity ^= 1u; }
                }
                if (ok) umma_commit(&s.acc_full[buf]);
            }
            if (!ok) {      // MMAs in flight end before their operands and accumulators go
                umma_commit(&s.drained);
                const unsigned long long t0 = global_timer_ns(), limit = g_wait_limit_ns;
                while (!mbar_try_wait_short(&s.drained, 0u) && global_timer_ns() - t0 < limit) {}
            }
        }
    } else {
        // A warp has a quarter of the channels and every fourth run of 16 rows.  A lane has a channel, so two lanes exchange
        // halves of two rows' values and each stores both channels of one row: half the stores.
        constexpr bool kHalf = sizeof(OUT) == 2;
        const uint32_t quarter = warp & 3u, part = warp >> 2, odd = lane & 1u;
        const bool paired = kHalf && p.paired != 0u;
        float4 *scales = s.row_scales[warp];
        uint32_t it = 0;
        if (p.ready) wait_in_front();
        for (uint32_t u = blockIdx.x; u < total; u += gridDim.x, ++it) {
            const IgUnit un = ig_unit(s, p, u);
            const uint32_t buf = p.accs == 2u ? it & 1u : 0u, turn = p.accs == 2u ? it >> 1 : it;
            const uint32_t acc = tmem + buf * SUBS * p.nt + ((quarter * 32u) << 16);
            const uint32_t j0 = un.ch * (GATED ? 128u : SUBS * 128u) + quarter * 32u + lane;
            const bool live0 = j0 < p.n, live1 = !GATED && SUBS == 2 && j0 + 128u < p.n;
            const float *bs = p.b_scales + (size_t)un.e * p.channels + j0;
            const float sb0 = live0 ? bs[0] : 0.0f, sb1 = GATED ? (live0 ? bs[p.n] : 0.0f) : (live1 ? bs[128] : 0.0f);
#pragma unroll
            for (uint32_t i = 0; i < 2u; ++i) {                   // runs 2 i and 2 i + 1 of this warp
                const uint32_t run = 2u * i + (lane >> 4), c = (part + 4u * run) * 16u + (lane & 15u);
                reinterpret_cast<float *>(scales)[run * 16u + (lane & 15u)] = c < un.count ? p.a_scales[un.row + c] : 0.0f;
            }
            __syncwarp();
            if (!__all_sync(0xffffffffu, wait(&s.acc_full[buf], turn & 1u))) break;
            tc_fence_after_sync();
            auto store = [&](const float (&x)[16], OUT *o, uint32_t live, bool mine) {
                if constexpr (kHalf) {
                    if (paired) {
                        const uint32_t pick = odd ? 0x3276u : 0x5410u;
                        o += odd ? p.out_stride - 1 : 0;
#pragma unroll
                        for (uint32_t c = 0; c < 8u; ++c, o += 2 * p.out_stride) {
                            const uint32_t own = pack2<OUT>(x[2 * c], x[2 * c + 1]);
                            const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
                            if (mine && 2u * c + odd < live) *reinterpret_cast<uint32_t *>(o) = __byte_perm(own, other, pick);
                        }
                        return;
                    }
                }
#pragma unroll
                for (uint32_t c = 0; c < 16u; ++c, o += p.out_stride)
                    if (mine && c < live) *o = elem_from_float<OUT>(x[c]);
            };
            // Some runs at a time: the accumulators are free for the next unit's MMAs as soon as the last ones are in registers, not when
            // they are stored.
            constexpr uint32_t kRuns = GATED ? 2 : 2 / SUBS;
            for (uint32_t i = 0;; i += kRuns) {
                const uint32_t c0 = (part + 4u * i) * 16u;
                uint32_t v[kRuns][SUBS][16];
#pragma unroll
                for (uint32_t r = 0; r < kRuns; ++r)
                    if (c0 + 64u * r < un.count)
#pragma unroll
                        for (uint32_t t = 0; t < SUBS; ++t) tmem_ld16(acc + t * p.nt + c0 + 64u * r, v[r][t]);
                tmem_ld_wait();
                if (c0 + 64u * kRuns >= un.count) {
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s.acc_empty[buf]);
                }
#pragma unroll
                for (uint32_t r = 0; r < kRuns; ++r) {
                    const uint32_t c = c0 + 64u * r;
                    if (c >= un.count) break;
                    OUT *out = static_cast<OUT *>(p.out) + (size_t)(un.row + c) * p.out_stride + j0;
                    const float *sa = reinterpret_cast<const float *>(scales) + (i + r) * 16u;
                    float x[16];
                    if constexpr (GATED) {
                        // the activation is asked for once in sixteen outputs: asked for each, 16384 rows of one matrix took 60.0 us for 58.9
                        auto gate = [&](auto act) {
#pragma unroll
                            for (uint32_t k = 0; k < 16u; ++k)
                                x[k] = gate_act<kHalf>(scaled(sa[k], sb0, (int)v[r][0][k]), decltype(act)::value) * scaled(sa[k], sb1, (int)v[r][1][k]);
                        };
                        if (p.act == ACT_SILU) gate(std::integral_constant<uint32_t, ACT_SILU>{});
                        else gate(std::integral_constant<uint32_t, ACT_GELU>{});
                        store(x, out, un.count - c, live0);
                    } else {
#pragma unroll
                        for (uint32_t t = 0; t < SUBS; ++t) {
#pragma unroll
                            for (uint32_t k = 0; k < 16u; ++k) x[k] = scaled(sa[k], t ? sb1 : sb0, (int)v[r][t][k]);
                            store(x, out + 128u * t, un.count - c, t ? live1 : live0);
                        }
                    }
                }
                if (c0 + 64u * kRuns >= un.count) break;
            }
            __syncwarp();                                          // before the next unit's scales
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == kIgMmaWarp) tmem_dealloc(tmem, 512);
}

}  // namespace nvmai
