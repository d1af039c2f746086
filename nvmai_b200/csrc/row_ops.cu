// Rows sorted by expert and back, their gradients, and 8-bit codes of rows: kernels and entry points.
#include "../../include/nvmai_cuda_moe.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "launch.h"
#include "row_elem.cuh"
#include "tma.cuh"

using namespace nvmai;

namespace {

constexpr uint32_t kNoRow = 0xFFFFFFFFu;

// ---- sort_rows ------------------------------------------------------------------------------------------
// A stable counting sort: the row of a pair is (kept pairs of smaller experts) + (pairs of its expert in front of it).  Each
// block has a run of tokens; it counts the experts of all pairs, those in front of its run apart, and ranks its own pairs
// with one warp, 32 at a time (__match_any_sync gives the pairs of the same expert).  Then its warps move the tokens' rows.  Writing
// bounds it: 4096 tokens of 4 KB to eight experts each take 33.2 us on a B200, 5.9 of them for the order (the same 134 MB written in order
// take 24.6); one token 3.1.
constexpr uint32_t kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr uint32_t kSms = 148, kSortBlocks = kSms;
constexpr uint32_t kSortOwn = 4096;          // most pairs of a block: their experts and rows are in shared memory
// From this many pairs on the blocks' counts come from a kernel in front (the order alone on a B200, top-8 of 256: 8192 tokens 10.0
// us with all pairs counted by every block, 9.5 with that kernel; 16384 tokens 18.2 / 13.9; 65536 tokens 66.6 / 34.0).
constexpr uint32_t kSortCounted = 65536;

struct SortParams {
    const uint32_t *idx; uint32_t tokens, top_k, E;
    uint32_t *position, *source, *begin;
    const void *x; size_t x_stride; uint32_t d;
    void *rows; size_t rows_stride;
    float *row_scales;
    uint32_t *counts;        // [blocks][sort_columns(E)], or nullptr: every block counts all pairs
};
__host__ __device__ constexpr uint32_t sort_columns(uint32_t E) { return (E + 3u) & ~3u; }

__device__ __forceinline__ uint32_t sort_first_token(const SortParams &p, uint32_t block) {
    return (uint32_t)((uint64_t)p.tokens * block / gridDim.x);
}

// Kept pairs of each expert in a block's run.
__global__ void __launch_bounds__(512) sort_count_kernel(SortParams p) {
    __shared__ uint32_t count[kRowMaxExperts];
    const uint32_t lo = sort_first_token(p, blockIdx.x) * p.top_k, hi = sort_first_token(p, blockIdx.x + 1) * p.top_k;
    const uint32_t columns = sort_columns(p.E);
    for (uint32_t e = threadIdx.x; e < columns; e += blockDim.x) count[e] = 0u;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    for (uint32_t i = lo + threadIdx.x; i < hi; i += blockDim.x) {
        const uint32_t e = p.idx[i];
        if (e < p.E) atomicAdd(&count[e], 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < columns; e += blockDim.x) p.counts[(size_t)blockIdx.x * columns + e] = count[e];
}

// sum over the threads in front of this one (1024 threads); *total gets the sum over all
__device__ __forceinline__ uint32_t block_exclusive_sum(uint32_t v, uint32_t *warp_sums, uint32_t *total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= (uint32_t)o) s += up;
    }
    if (lane == 31u) warp_sums[warp] = s;
    __syncthreads();
    if (warp == 0) {
        uint32_t w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= (uint32_t)o) w += up;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    *total = warp_sums[31];
    return s - v + (warp ? warp_sums[warp - 1] : 0u);
}

// MOVE: 0 the order alone, 1 rows as they are, 2 as codes.  T: what a row is read as (MOVE 1: bits of that size), V at a time.
template <typename T, int V, int MOVE>
__global__ void __launch_bounds__(kSortThreads) sort_rows_kernel(SortParams p) {
    using P = Piece<T, V>;
    using Q = Piece<int8_t, V>;
    __shared__ uint32_t before[kRowMaxExperts + 1], rest[kRowMaxExperts + 1], warp_sums[32];
    __shared__ uint32_t own[kSortOwn], unkept;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t first = sort_first_token(p, blockIdx.x), last = sort_first_token(p, blockIdx.x + 1);
    const uint32_t pairs = p.tokens * p.top_k, lo = first * p.top_k, hi = last * p.top_k;
    for (uint32_t e = tid; e <= p.E; e += kSortThreads) before[e] = rest[e] = 0u;
    if (tid == 0) unkept = lo;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    for (uint32_t i = lo + tid; i < hi; i += kSortThreads) own[i - lo] = min(p.idx[i], p.E);
    if (p.counts == nullptr) {
        auto count = [&](uint32_t i, uint32_t e) { atomicAdd(i < lo ? &before[min(e, p.E)] : &rest[min(e, p.E)], 1u); };
        const uint32_t fours = (reinterpret_cast<uintptr_t>(p.idx) & 15u) == 0u ? pairs / 4u : 0u;
#pragma unroll 4
        for (uint32_t i = tid; i < fours; i += kSortThreads) {
            const uint4 e = reinterpret_cast<const uint4 *>(p.idx)[i];
            count(4u * i, e.x); count(4u * i + 1u, e.y); count(4u * i + 2u, e.z); count(4u * i + 3u, e.w);
        }
        for (uint32_t i = 4u * fours + tid; i < pairs; i += kSortThreads) count(i, p.idx[i]);
    } else {
        // 128 neighbouring experts a warp, the blocks spread over the warps that share them
        const uint32_t columns = sort_columns(p.E), across = (columns + 127u) / 128u, shares = kSortWarps / across;
        const uint32_t e = warp % across * 128u + lane * 4u;
        if (warp < across * shares && e < columns) {
            uint4 in_front = make_uint4(0, 0, 0, 0), behind = make_uint4(0, 0, 0, 0);
#pragma unroll 8
            for (uint32_t b = warp / across; b < gridDim.x; b += shares) {
                const uint4 n = *reinterpret_cast<const uint4 *>(p.counts + (size_t)b * columns + e);
                if (b < blockIdx.x) { in_front.x += n.x; in_front.y += n.y; in_front.z += n.z; in_front.w += n.w; }
                else { behind.x += n.x; behind.y += n.y; behind.z += n.z; behind.w += n.w; }
            }
            const uint32_t f[4] = {in_front.x, in_front.y, in_front.z, in_front.w}, r[4] = {behind.x, behind.y, behind.z, behind.w};
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                if (e + i < p.E) { atomicAdd(&before[e + i], f[i]); atomicAdd(&rest[e + i], r[i]); }
        }
    }
    __syncthreads();
    const uint32_t ahead = tid < p.E ? before[tid] : 0u;
    uint32_t kept;
    const uint32_t base = block_exclusive_sum(tid < p.E ? ahead + rest[tid] : 0u, warp_sums, &kept);
    if (tid < p.E) {
        before[tid] = base + ahead;              // row of the next pair of this expert
        if (blockIdx.x == 0) p.begin[tid] = base;
    }
    if (tid == 0 && blockIdx.x == 0) p.begin[p.E] = kept;
    // pairs that are not kept name the rows behind: those in front of the run are lo less the kept ones in front of it
    const uint32_t kept_ahead = __reduce_add_sync(0xffffffffu, ahead);
    if (lane == 0) atomicSub(&unkept, kept_ahead);
    __syncthreads();
    if (tid == 0) before[p.E] = unkept + kept;
    __syncthreads();
    if (warp == 0) {
        for (uint32_t i0 = lo; i0 < hi; i0 += 32u) {
            const uint32_t i = i0 + lane;
            const uint32_t e = i < hi ? own[i - lo] : 0xFFFFFFFFu;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            uint32_t row = 0;
            if (i < hi) row = before[e] + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
            if (i < hi) {
                if ((same >> lane) == 1u) before[e] = row + 1u;          // the last of them
                const uint32_t at = e < p.E ? row : kNoRow;
                p.source[row] = e < p.E ? i : kNoRow;
                p.position[i] = at;
                own[i - lo] = at;
            }
            __syncwarp();
        }
    }
    if constexpr (MOVE != 0) {
        __syncthreads();
        auto code = [](const P &v, const RowScale &rs) {
            Q q;
#pragma unroll
            for (int x = 0; x < V; ++x) q.v[x] = row_code(elem_to_float(v.v[x]), rs);
            return q;
        };
        auto scale_out = [&](const uint32_t *place, float scale) {
            for (uint32_t k = lane; k < p.top_k; k += 32u)
                if (place[k] != kNoRow) p.row_scales[place[k]] = scale;
        };
        // a warp takes a token's row, or a part of it (a piece a lane at least) where the block has fewer tokens than warps
        const uint32_t mine = last - first, pieces = p.d / V;
        const uint32_t parts = mine == 0 || mine >= kSortWarps ? 1u : min(kSortWarps / mine, (pieces + 31u) / 32u);
        const uint32_t each = (pieces + parts - 1u) / parts;
        for (uint32_t u = warp; u < mine * parts; u += kSortWarps) {
            const uint32_t t = first + u / parts, part = u % parts;
            const uint32_t c0 = part * each, c1 = min(pieces, c0 + each);
            const P *src = reinterpret_cast<const P *>(static_cast<const T *>(p.x) + (size_t)t * p.x_stride);
            const uint32_t *place = own + (t - first) * p.top_k;
            if constexpr (MOVE == 1) {
                // four pieces are requested before any is stored
                for (uint32_t c = c0 + lane; c < c1; c += 128u) {
                    P v[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i)
                        if (c + 32u * i < c1) v[i] = src[c + 32u * i];
                    for (uint32_t k = 0; k < p.top_k; ++k) {
                        const uint32_t row = place[k];
                        if (row == kNoRow) continue;
                        P *dst = reinterpret_cast<P *>(static_cast<T *>(p.rows) + (size_t)row * p.rows_stride) + c;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; ++i)
                            if (c + 32u * i < c1) dst[32u * i] = v[i];
                    }
                }
            } else {
                uint32_t m = 0;
#pragma unroll 4
                for (uint32_t c = lane; c < pieces; c += 32u) {
                    const P v = src[c];
#pragma unroll
                    for (int i = 0; i < V; ++i) m = max(m, magnitude_bits(elem_to_float(v.v[i])));
                }
                m = __reduce_max_sync(0xffffffffu, m);
                const RowScale rs = row_scale_bits(m);
                for (uint32_t c = c0 + lane; c < c1; c += 128u) {
                    Q q[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i)
                        if (c + 32u * i < c1) q[i] = code(src[c + 32u * i], rs);
                    for (uint32_t k = 0; k < p.top_k; ++k) {
                        const uint32_t row = place[k];
                        if (row == kNoRow) continue;
                        Q *dst = reinterpret_cast<Q *>(static_cast<int8_t *>(p.rows) + (size_t)row * p.rows_stride) + c;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; ++i)
                            if (c + 32u * i < c1) dst[32u * i] = q[i];
                    }
                }
                if (part == 0) scale_out(place, rs.scale);
            }
        }
    }
}

// ---- merge_rows -----------------------------------------------------------------------------------------
struct MergeParams {
    const void *rows; uint32_t rows_stride, n_rows;
    const uint32_t *position; const void *w; uint32_t w_elem;
    uint32_t tokens, top_k, d;
    const void *base; size_t base_stride;
    void *y; size_t y_stride;
};

__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, int bytes) {
    if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// A warp sums a run of 32 R pieces of V neighbouring elements of a token and goes on to the next run, as many warps further as
// there are.  A step is a run's pieces of up to eight slots; a step is copied into shared memory while the one before is
// added, each lane its own pieces, so that a lane waits for its own copies alone (cp.async groups) and no registers hold what is
// in flight: 24 warps an SM with a step of 4 KB each.  4096 tokens of eight 4 KB rows on a B200: 25.1 us, 6.0 TB/s; a thread per piece
// without the ring 35.2 (the rows' latency is exposed), a ring of four steps 56 (8 warps an SM, too few for the instructions).
constexpr uint32_t kMergeSlots = 8, kMergeAhead = 2;
__host__ __device__ constexpr uint32_t merge_stage_bytes(uint32_t top_k, uint32_t run_bytes) {
    return (top_k < kMergeSlots ? top_k : kMergeSlots) * run_bytes;
}

template <typename T, int V, int R>
__global__ void __launch_bounds__(256) merge_rows_kernel(MergeParams p) {
    using P = Piece<T, V>;
    constexpr int kPiece = sizeof(P);
    constexpr uint32_t kRun = 32u * R, kRunBytes = kRun * kPiece;
    extern __shared__ __align__(16) unsigned char merge_smem[];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t stage_bytes = merge_stage_bytes(p.top_k, kRunBytes);
    unsigned char *ring = merge_smem + warp * kMergeAhead * stage_bytes + lane * kPiece;
    const uint32_t ring_at = smem_addr(ring);
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t pieces = p.d / V, runs = (pieces + kRun - 1u) / kRun, groups = (p.top_k + kMergeSlots - 1u) / kMergeSlots;
    const uint32_t stride_t = gridDim.x * 8u / runs, stride_run = gridDim.x * 8u % runs;
    const T *rows = static_cast<const T *>(p.rows);
    struct At { uint32_t t, run, g; };
    auto next = [&](At &x) {
        if (++x.g < groups) return;
        x.g = 0u;
        x.t += stride_t;
        if ((x.run += stride_run) >= runs) { x.run -= runs; ++x.t; }
    };
    // lane k: position of the step's slot k
    auto position = [&](const At &x) {
        const uint32_t k = x.g * kMergeSlots + lane;
        return x.t < p.tokens && lane < kMergeSlots && k < p.top_k ? p.position[(size_t)x.t * p.top_k + k] : kNoRow;
    };
    // Held slots of a step.  All eight of a whole run, the common case, go without a question for each piece; else only those
    // that are held are gone through.
    constexpr uint32_t kAll = (1u << kMergeSlots) - 1u;
    auto held = [&](uint32_t pos) { return __ballot_sync(0xffffffffu, pos < p.n_rows); };
    auto whole = [&](const At &x, uint32_t mask) { return mask == kAll && (x.run + 1u) * kRun <= pieces; };
    auto request = [&](const At &x, uint32_t pos, uint32_t slot) {
        const uint32_t c = x.run * kRun + lane, to = ring_at + slot * stage_bytes, mask = held(pos);
        auto row = [&](uint32_t k, auto all) {
            const P *src = reinterpret_cast<const P *>(rows + (size_t)__shfl_sync(0xffffffffu, pos, k) * p.rows_stride) + c;
#pragma unroll
            for (uint32_t r = 0; r < R; ++r)
                if (decltype(all)::value || c + r * 32u < pieces) cp_async(to + k * kRunBytes + r * 32u * kPiece, src + r * 32u, kPiece);
        };
        if (whole(x, mask)) {
#pragma unroll
            for (uint32_t k = 0; k < kMergeSlots; ++k) row(k, std::true_type{});
        } else {
            for (uint32_t m = mask; m != 0u; m &= m - 1u) row(__ffs((int)m) - 1u, std::false_type{});
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const uint32_t first = blockIdx.x * 8u + warp;
    At now{first / runs, first % runs, 0u}, head = now;      // the step to add and the one to request
    next(head);
    uint32_t now_pos = position(now), head_pos = position(head);
    request(now, now_pos, 0u);
    float acc[R][V];
    for (uint32_t slot = 0; now.t < p.tokens; slot ^= 1u) {
        At then = head;
        next(then);
        const uint32_t then_pos = position(then);
        request(head, head_pos, slot ^ 1u);                  // into the slot that the last round emptied
        const uint32_t c = now.run * kRun + lane;
        if (now.g == 0u) {
#pragma unroll
            for (uint32_t r = 0; r < R; ++r) {
                P b;
                const bool has = p.base != nullptr && c + r * 32u < pieces;
                if (has) b = reinterpret_cast<const P *>(static_cast<const T *>(p.base) + (size_t)now.t * p.base_stride)[c + r * 32u];
#pragma unroll
                for (int i = 0; i < V; ++i) acc[r][i] = has ? elem_to_float(b.v[i]) : 0.0f;
            }
        }
        const bool weighs = p.w != nullptr && lane < kMergeSlots && now_pos < p.n_rows;
        const float mine = weighs ? load_elem(p.w, p.w_elem, (size_t)now.t * p.top_k + now.g * kMergeSlots + lane) : 1.0f;
        asm volatile("cp.async.wait_group %0;" ::"n"(kMergeAhead - 1) : "memory");
        auto add = [&](uint32_t k, auto all) {
            const float w = __shfl_sync(0xffffffffu, mine, k);
#pragma unroll
            for (uint32_t r = 0; r < R; ++r) {
                if (!decltype(all)::value && c + r * 32u >= pieces) continue;
                const P v = *reinterpret_cast<const P *>(ring + slot * stage_bytes + k * kRunBytes + r * 32u * kPiece);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[r][i] = fmaf(w, elem_to_float(v.v[i]), acc[r][i]);
            }
        };
        const uint32_t mask = held(now_pos);
        if (whole(now, mask)) {
#pragma unroll
            for (uint32_t k = 0; k < kMergeSlots; ++k) add(k, std::true_type{});
        } else {
            for (uint32_t m = mask; m != 0u; m &= m - 1u) add(__ffs((int)m) - 1u, std::false_type{});
        }
        if (now.g + 1u == groups) {
#pragma unroll
            for (uint32_t r = 0; r < R; ++r) {
                if (c + r * 32u >= pieces) continue;
                P o;
#pragma unroll
                for (int i = 0; i < V; ++i) o.v[i] = elem_from_float<T>(acc[r][i]);
                reinterpret_cast<P *>(static_cast<T *>(p.y) + (size_t)now.t * p.y_stride)[c + r * 32u] = o;
            }
        }
        now = head;
        now_pos = head_pos;
        head = then;
        head_pos = then_pos;
    }
}

// Rows of 16-bit elements that share no 4-byte boundary: a thread sums every 32nd element, four of them and four slots at a time
// (two-byte accesses bound it: 1531 tokens of eight rows of 999 elements 11.3 us on a B200, 2.4 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) merge_narrow_kernel(MergeParams p) {
    constexpr int U = 4, kAhead = 4;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t t = blockIdx.x * blockDim.y + threadIdx.y, lane = threadIdx.x & 31u;
    if (t >= p.tokens) return;                             // whole warps: a block row is a multiple of 32 threads
    const T *rows = static_cast<const T *>(p.rows);
    for (uint32_t c0 = threadIdx.x; c0 - lane < p.d; c0 += blockDim.x * U) {
        float acc[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t c = c0 + u * blockDim.x;
            acc[u] = p.base != nullptr && c < p.d ? elem_to_float(static_cast<const T *>(p.base)[(size_t)t * p.base_stride + c]) : 0.0f;
        }
        for (uint32_t k0 = 0; k0 < p.top_k; k0 += 32u) {
            const size_t pair = (size_t)t * p.top_k + k0 + lane;
            const uint32_t mine = k0 + lane < p.top_k ? p.position[pair] : kNoRow;
            const float mine_w = mine < p.n_rows && p.w != nullptr ? load_elem(p.w, p.w_elem, pair) : 1.0f;
            for (uint32_t s = 0; s < min(p.top_k - k0, 32u); s += kAhead) {
                T v[kAhead][U];
                uint32_t row[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    row[j] = s + j < 32u ? __shfl_sync(0xffffffffu, mine, s + j) : kNoRow;      // lanes past the slots hold kNoRow
                    if (row[j] < p.n_rows) {
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (c0 + u * blockDim.x < p.d) v[j][u] = rows[(size_t)row[j] * p.rows_stride + c0 + u * blockDim.x];
                    }
                }
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const float w = __shfl_sync(0xffffffffu, mine_w, (s + j) & 31u);
                    if (row[j] < p.n_rows) {
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (c0 + u * blockDim.x < p.d) acc[u] = fmaf(w, elem_to_float(v[j][u]), acc[u]);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * blockDim.x < p.d) static_cast<T *>(p.y)[(size_t)t * p.y_stride + c0 + u * blockDim.x] = elem_from_float<T>(acc[u]);
    }
}

struct MergeGradParams {
    const void *dy; size_t dy_stride;
    const void *rows; size_t rows_stride; uint32_t n_rows;
    const uint32_t *position; const void *w; uint32_t w_elem;
    uint32_t pairs, top_k, d;
    void *drows; size_t drows_stride;
    float *dw;
};

// A warp per pair; the eight warps of a block share the rows of dy in the L1.
template <typename T, int V>
__global__ void __launch_bounds__(256, 4) merge_rows_grad_kernel(MergeGradParams p) {
    using P = Piece<T, V>;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t pair = blockIdx.x * 8u + (threadIdx.x >> 5), lane = threadIdx.x & 31u;
    if (pair >= p.pairs) return;
    const uint32_t row = p.position[pair];
    if (row >= p.n_rows) {
        if (p.dw != nullptr && lane == 0) p.dw[pair] = 0.0f;
        return;
    }
    const float w = p.w != nullptr ? load_elem(p.w, p.w_elem, pair) : 1.0f;
    const P *dy = reinterpret_cast<const P *>(static_cast<const T *>(p.dy) + (size_t)(pair / p.top_k) * p.dy_stride);
    const P *v = reinterpret_cast<const P *>(static_cast<const T *>(p.rows) + (size_t)row * p.rows_stride);
    P *o = reinterpret_cast<P *>(static_cast<T *>(p.drows) + (size_t)row * p.drows_stride);
    // kAhead pieces of both rows are requested before any is stored: drows may be rows, so the compiler keeps loads behind stores.
    // 1531 tokens of 2048 bf16 elements on a B200: two pieces and 32 warps an SM 21.6 us, three and 24 warps 23.1, two and 40 24.7.
    constexpr int kAhead = V == 8 ? 2 : V == 4 ? 4 : 8;
    const uint32_t pieces = p.d / V;
    float dot = 0.0f;
    for (uint32_t c0 = lane; c0 < pieces; c0 += 32u * kAhead) {
        P gv[kAhead], rv[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (c0 + 32u * u < pieces) {
                gv[u] = dy[c0 + 32u * u];
                if (p.dw != nullptr) rv[u] = v[c0 + 32u * u];
            }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (c0 + 32u * u < pieces) {
                if (p.dw != nullptr) {
#pragma unroll
                    for (int i = 0; i < V; ++i) dot = fmaf(elem_to_float(gv[u].v[i]), elem_to_float(rv[u].v[i]), dot);
                }
                if (p.drows != nullptr) {
                    P s;
#pragma unroll
                    for (int i = 0; i < V; ++i) s.v[i] = elem_from_float<T>(w * elem_to_float(gv[u].v[i]));
                    o[c0 + 32u * u] = s;
                }
            }
    }
    if (p.dw != nullptr) {
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, k);
        if (lane == 0) p.dw[pair] = dot;
    }
}

// ---- quantize_rows --------------------------------------------------------------------------------------
struct QuantizeParams {
    const void *x; size_t x_stride; uint32_t rows, n;
    int8_t *q; size_t q_stride;
    float *scales;
};

// WARPS warps per row, which they hold in registers between the largest magnitude and the codes; a longer row is read twice.
// Reading bounds it: 4096 rows of 2048 fp16 elements 5.2 us on a B200, 4.8 TB/s.
constexpr int kQuantizeHeld = 8;             // pieces of a row that a lane holds
template <typename T, int V, int WARPS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantizeParams p) {
    using P = Piece<T, V>;
    using Q = Piece<int8_t, V>;
    __shared__ uint32_t top[8];
    pdl_wait();
    pdl_launch_dependents();
    constexpr uint32_t kAcross = 32u * WARPS;
    const uint32_t warp = threadIdx.x >> 5, in = threadIdx.x % kAcross;
    const uint32_t row = blockIdx.x * (8u / WARPS) + threadIdx.x / kAcross;
    if (row >= p.rows) return;               // whole warps, with WARPS = 8 the whole block
    const P *src = reinterpret_cast<const P *>(static_cast<const T *>(p.x) + (size_t)row * p.x_stride);
    Q *dst = reinterpret_cast<Q *>(p.q + (size_t)row * p.q_stride);
    const uint32_t pieces = p.n / V;
    auto largest = [](const P &v, uint32_t m) {
#pragma unroll
        for (int i = 0; i < V; ++i) m = max(m, magnitude_bits(elem_to_float(v.v[i])));
        return m;
    };
    P held[kQuantizeHeld];
    uint32_t m = 0;
#pragma unroll
    for (uint32_t i = 0; i < kQuantizeHeld; ++i)
        if (in + i * kAcross < pieces) held[i] = src[in + i * kAcross];
#pragma unroll
    for (uint32_t i = 0; i < kQuantizeHeld; ++i)
        if (in + i * kAcross < pieces) m = largest(held[i], m);
#pragma unroll 4
    for (uint32_t c = in + kQuantizeHeld * kAcross; c < pieces; c += kAcross) m = largest(src[c], m);
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (WARPS > 1) {
        if ((threadIdx.x & 31u) == 0u) top[warp] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WARPS; ++i) m = max(m, top[i]);
    }
    const RowScale rs = row_scale_bits(m);
    auto code = [&](const P &v) {
        Q q;
#pragma unroll
        for (int i = 0; i < V; ++i) q.v[i] = row_code(elem_to_float(v.v[i]), rs);
        return q;
    };
#pragma unroll
    for (uint32_t i = 0; i < kQuantizeHeld; ++i)
        if (in + i * kAcross < pieces) dst[in + i * kAcross] = code(held[i]);
#pragma unroll 4
    for (uint32_t c = in + kQuantizeHeld * kAcross; c < pieces; c += kAcross) dst[c] = code(src[c]);
    if (in == 0u) p.scales[row] = rs.scale;
}

// ---- launches -------------------------------------------------------------------------------------------

int launched(cudaError_t e) {
    count_launches(1);
    if (e != cudaSuccess) cudaGetLastError();
    return e == cudaSuccess ? NVMAI_CUDA_OK : NVMAI_CUDA_ECUDA;
}

// Elements a thread moves at once: as many as make 16 bytes where every buffer starts on such a boundary, its rows are that far
// apart and a row is a whole number of them; two of 16 bits by the same rule; else one.
struct Rows { const void *p; size_t stride, size; };
bool on_boundary(std::initializer_list<Rows> rows, size_t v) {
    for (const Rows &r : rows)
        if (r.p != nullptr && (r.stride % v != 0 || !aligned_to(r.p, v * r.size))) return false;
    return true;
}
template <typename F>
auto with_pieces(uint32_t elem, uint32_t d, std::initializer_list<Rows> rows, F &&f) {
    const size_t most = 16 / elem_size(elem);
    const size_t v = d % most == 0 && on_boundary(rows, most) ? most : d % 2 == 0 && on_boundary(rows, 2) ? 2 : 1;
    using std::integral_constant;
    auto with_16 = [&](auto T) {
        return v == 8 ? f(T, integral_constant<int, 8>{}) : v == 2 ? f(T, integral_constant<int, 2>{}) : f(T, integral_constant<int, 1>{});
    };
    if (elem == ELEM_F32) return v == 4 ? f(float{}, integral_constant<int, 4>{}) : f(float{}, integral_constant<int, 1>{});
    return elem == ELEM_BF16 ? with_16(__nv_bfloat16{}) : with_16(__half{});
}

}  // namespace

cudaError_t nvmai::launch_quantize(const void *x, uint32_t elem, uint32_t x_stride, uint32_t rows, uint32_t n, int8_t *q, uint32_t q_stride,
                                   float *scales, cudaStream_t st) {
    const QuantizeParams p{x, x_stride, rows, n, q, q_stride, scales};
    return with_pieces(elem, n, {{x, x_stride, elem_size(elem)}, {q, q_stride, 1}}, [&](auto T, auto V) {
        constexpr int v = decltype(V)::value;
        // Eight warps a row for few rows, and for rows that one warp cannot hold (fp16, one warp / eight: 1 x 2048 2.0 / 1.6 us,
        // 201 x 2048 2.5 / 2.0, 1000 x 2048 2.6 / 3.6, 32768 x 512 12.8 / 67.7, 300 x 8000 13.1 / 3.4)
        if (rows < 3 * kSms || n > 32u * kQuantizeHeld * v)
            return launch_pdl(quantize_rows_kernel<decltype(T), v, 8>, dim3(rows), dim3(256), 0, st, true, p);
        return launch_pdl(quantize_rows_kernel<decltype(T), v, 1>, dim3(rows / 8 + (rows % 8 != 0)), dim3(256), 0, st, true, p);
    });
}

// every block has at least a token and at most kSortOwn pairs
static uint32_t sort_blocks(uint32_t tokens, uint32_t top_k) {
    const uint32_t most = kSortOwn / top_k;
    return std::max({1u, std::min(tokens, kSortBlocks), (uint32_t)(((uint64_t)tokens + most - 1) / most)});
}

extern "C" {

uint64_t nvmai_cuda_moe_sort_rows_workspace(uint32_t tokens, uint32_t top_k, uint32_t num_experts) {
    if ((uint64_t)tokens * top_k < kSortCounted || top_k > kRowMaxTopK) return 0;
    return (uint64_t)sort_blocks(tokens, top_k) * sort_columns(num_experts) * 4;
}

int nvmai_cuda_moe_sort_rows(const uint32_t *idx, uint32_t tokens, uint32_t top_k, uint32_t num_experts, uint32_t *position,
                             uint32_t *source, uint32_t *expert_begin, const void *x, uint32_t x_elem, uint32_t x_stride, uint32_t d,
                             void *rows, uint32_t rows_elem, uint32_t rows_stride, float *row_scales, void *workspace,
                             uint64_t workspace_bytes, void *stream) {
    return without_exceptions([&]() -> int {
        if (tokens == 0) x = rows = row_scales = nullptr;            // buffers of no rows have no address, whatever the others are
        if (!expert_begin || (tokens != 0 && (!idx || !position || !source))) return NVMAI_CUDA_EINVAL;
        if (top_k == 0 || top_k > kRowMaxTopK || num_experts == 0 || num_experts > kRowMaxExperts) return NVMAI_CUDA_ERANGE;
        if ((uint64_t)tokens * top_k >= (1ull << 26)) return NVMAI_CUDA_ERANGE;
        if (!aligned_to(idx, 4) || !aligned_to(position, 4) || !aligned_to(source, 4) || !aligned_to(expert_begin, 4)) return NVMAI_CUDA_EINVAL;
        if ((x == nullptr) != (rows == nullptr)) return NVMAI_CUDA_EINVAL;
        if (x != nullptr) {
            if (x_elem > ELEM_BF16 || (rows_elem != x_elem && rows_elem != ELEM_I8)) return NVMAI_CUDA_EINVAL;
            if (d == 0 || x_stride < d || rows_stride < d) return NVMAI_CUDA_EINVAL;
            if (d > kRowMaxLength) return NVMAI_CUDA_ERANGE;
            if (!aligned_to(x, elem_size(x_elem)) || !aligned_to(rows, elem_size(rows_elem))) return NVMAI_CUDA_EINVAL;
            if ((rows_elem == ELEM_I8) != (row_scales != nullptr) || !aligned_to(row_scales, 4)) return NVMAI_CUDA_EINVAL;
        }
        const uint64_t counts_bytes = nvmai_cuda_moe_sort_rows_workspace(tokens, top_k, num_experts);
        if (workspace_bytes < counts_bytes) return NVMAI_CUDA_ERANGE;
        if (counts_bytes != 0 && (!workspace || !aligned_to(workspace, 16))) return NVMAI_CUDA_EINVAL;
        if (!on_current_device({idx, position, source, expert_begin, x, rows, row_scales, counts_bytes != 0 ? workspace : nullptr})) return NVMAI_CUDA_EINVAL;
        const SortParams p{idx, tokens, top_k, num_experts, position, source, expert_begin, x, x_stride, d, rows, rows_stride, row_scales,
                           counts_bytes != 0 ? static_cast<uint32_t *>(workspace) : nullptr};
        const dim3 grid(sort_blocks(tokens, top_k)), block(kSortThreads);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (p.counts != nullptr)
            if (const int rc = launched(launch_pdl(sort_count_kernel, grid, dim3(512), 0, st, true, p))) return rc;
        if (x == nullptr) return launched(launch_pdl(sort_rows_kernel<float, 1, 0>, grid, block, 0, st, true, p));
        return with_pieces(x_elem, d, {{x, x_stride, elem_size(x_elem)}, {rows, rows_stride, elem_size(rows_elem)}}, [&](auto T, auto V) {
            constexpr int v = decltype(V)::value;
            if (rows_elem == ELEM_I8) return launched(launch_pdl(sort_rows_kernel<decltype(T), v, 2>, grid, block, 0, st, true, p));
            return launched(launch_pdl(sort_rows_kernel<decltype(T), v, 1>, grid, block, 0, st, true, p));
    });
    });
}

int nvmai_cuda_moe_merge_rows(const void *rows, uint32_t elem, uint32_t rows_stride, uint32_t n_rows, const uint32_t *position,
                              const void *w, uint32_t w_elem, uint32_t tokens, uint32_t top_k, uint32_t d, const void *base,
                              uint32_t base_stride, void *y, uint32_t y_stride, void *stream) {
    return without_exceptions([&]() -> int {
        if ((n_rows != 0 && !rows) || (tokens != 0 && (!position || !y))) return NVMAI_CUDA_EINVAL;
        if (elem > ELEM_BF16 || (w && w_elem > ELEM_BF16)) return NVMAI_CUDA_EINVAL;
        if (top_k == 0 || top_k > kRowMaxTopK || (uint64_t)tokens * top_k >= (1ull << 31) || d > kRowMaxLength) return NVMAI_CUDA_ERANGE;
        if (d == 0 || y_stride < d || (n_rows != 0 && rows_stride < d) || (base && base_stride < d)) return NVMAI_CUDA_EINVAL;
        const size_t size = elem_size(elem);
        if (!aligned_to(rows, size) || !aligned_to(y, size) || !aligned_to(base, size) || (w && !aligned_to(w, elem_size(w_elem))) ||
            !aligned_to(position, 4))
            return NVMAI_CUDA_EINVAL;
        if (tokens == 0) return NVMAI_CUDA_OK;
        if (!on_current_device({n_rows != 0 ? rows : nullptr, position, w, base, y})) return NVMAI_CUDA_EINVAL;
        const MergeParams p{rows, rows_stride, n_rows, position, w, w_elem, tokens, top_k, d, base, base_stride, y, y_stride};
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const std::initializer_list<Rows> all{{n_rows != 0 ? rows : nullptr, rows_stride, size}, {base, base_stride, size}, {y, y_stride, size}};
        auto narrow = [&](auto T) {
            uint32_t tx = 32;
            while (tx < 256 && tx * 4 < d) tx *= 2;
            const uint32_t ty = 256 / tx;
            return launched(launch_pdl(merge_narrow_kernel<decltype(T)>, dim3((tokens + ty - 1) / ty), dim3(tx, ty), 0, st, true, p));
        };
        auto go = [&](auto T, auto V) {
            using std::integral_constant;
            constexpr uint32_t piece = sizeof(T) * decltype(V)::value;
            if constexpr (piece < 4) {
                return narrow(T);
            } else {
                constexpr int r = piece == 16 ? 1 : 4;               // 4-byte pieces: four times as many of them a step
                const size_t smem = 8 * kMergeAhead * (size_t)merge_stage_bytes(top_k, 32 * r * piece);
                const uint64_t runs = (uint64_t)tokens * ((d / decltype(V)::value + 32 * r - 1) / (32 * r));
                const uint64_t resident = kSms * std::min<uint64_t>(8, 220 * 1024 / (smem + 1024));
                return launched(launch_pdl(merge_rows_kernel<decltype(T), decltype(V)::value, r>, dim3((unsigned)std::min<uint64_t>(resident, (runs + 7) / 8)),
                                           dim3(256), smem, st, true, p));
            }
        };
        return with_pieces(elem, d, all, go);
    });
}

int nvmai_cuda_moe_merge_rows_grad(const void *dy, uint32_t elem, uint32_t dy_stride, const void *rows, uint32_t rows_stride,
                                   uint32_t n_rows, const uint32_t *position, const void *w, uint32_t w_elem, uint32_t tokens,
                                   uint32_t top_k, uint32_t d, void *drows, uint32_t drows_stride, float *dw, void *stream) {
    return without_exceptions([&]() -> int {
        const bool nothing = tokens == 0 || (!dw && n_rows == 0);     // a buffer of no rows has no address
        if ((!drows && !dw && !nothing) || (tokens != 0 && (!dy || !position))) return NVMAI_CUDA_EINVAL;
        if (dw && n_rows != 0 && !rows) return NVMAI_CUDA_EINVAL;
        if (elem > ELEM_BF16 || (w && w_elem > ELEM_BF16)) return NVMAI_CUDA_EINVAL;
        if (top_k == 0 || top_k > kRowMaxTopK || (uint64_t)tokens * top_k >= (1ull << 31) || d > kRowMaxLength) return NVMAI_CUDA_ERANGE;
        if (d == 0 || dy_stride < d || (drows && drows_stride < d) || (dw && n_rows != 0 && rows_stride < d)) return NVMAI_CUDA_EINVAL;
        const size_t size = elem_size(elem);
        if (!aligned_to(dy, size) || !aligned_to(rows, size) || !aligned_to(drows, size) || (w && !aligned_to(w, elem_size(w_elem))) ||
            !aligned_to(dw, 4) || !aligned_to(position, 4))
            return NVMAI_CUDA_EINVAL;
        if (nothing) return NVMAI_CUDA_OK;
        const void *read = dw && n_rows != 0 ? rows : nullptr;       // the rows are read for dw alone
        if (!on_current_device({dy, read, position, w, n_rows != 0 ? drows : nullptr, dw})) return NVMAI_CUDA_EINVAL;
        const uint32_t pairs = tokens * top_k;
        const MergeGradParams p{dy, dy_stride, rows, rows_stride, n_rows, position, w, w_elem, pairs, top_k, d, drows, drows_stride, dw};
        return with_pieces(elem, d, {{dy, dy_stride, size}, {read, rows_stride, size}, {drows, drows_stride, size}}, [&](auto T, auto V) {
            return launched(launch_pdl(merge_rows_grad_kernel<decltype(T), decltype(V)::value>, dim3((pairs + 7) / 8), dim3(256), 0,
                                       static_cast<cudaStream_t>(stream), true, p));
    });
    });
}

int nvmai_cuda_moe_quantize_rows(const void *x, uint32_t elem, uint32_t x_stride, uint32_t rows, uint32_t n, void *q, uint32_t q_stride,
                                 float *scales, void *stream) {
    return without_exceptions([&]() -> int {
        if (rows != 0 && (!x || !q || !scales)) return NVMAI_CUDA_EINVAL;
        if (elem > ELEM_BF16 || n == 0 || x_stride < n || q_stride < n) return NVMAI_CUDA_EINVAL;
        if (n > kRowMaxLength) return NVMAI_CUDA_ERANGE;
        if (!aligned_to(x, elem_size(elem)) || !aligned_to(scales, 4)) return NVMAI_CUDA_EINVAL;
        if (rows == 0) return NVMAI_CUDA_OK;
        if (!on_current_device({x, q, scales})) return NVMAI_CUDA_EINVAL;
        return launched(launch_quantize(x, elem, x_stride, rows, n, static_cast<int8_t *>(q), q_stride, scales,
                                        static_cast<cudaStream_t>(stream)));
    });
}

}  // extern "C"
