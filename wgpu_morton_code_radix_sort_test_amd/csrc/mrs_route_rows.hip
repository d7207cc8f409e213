// Rows moved between token order and expert order: dispatch, combine and their gradients
// (mrs_route_* in include/mrs.h).  Every row is read once and written once in 16-byte pieces; what
// bounds these kernels is memory bandwidth, at a few tokens the latency of one dependent chain
// (slot's row number -> row -> store).
#include <type_traits>

#include "mrs_route.hpp"

namespace mrs {

namespace {

constexpr uint32_t kMoveThreads = 128;     // dispatch
constexpr uint32_t kSumThreads = 1024;     // combine and its gradient: a workgroup covers whole rows
constexpr uint32_t kShortThreads = 128;     // ... shorter than a wave's 64 vectors
constexpr uint32_t kMaxBlocks = 1u << 20;  // more work than that is looped over
constexpr uint32_t kPadWaves = 2048;       // waves for the rows that fill segments up, two on a SIMD
// combine's gradient: waves share a token's pieces evenly, but where that makes fewer waves than this, as many as there are pieces
// for.  Evenly and with as many as that: 3 tokens of 4 slots and 6368 f32 (25 pieces) 17.7 and 6.0 us, 300 of 8 and 1500
// bf16 (3 pieces) 13.7 and 11.2, 1000 of 4 and 2600 f32 (11 pieces) 24.2 and 18.8; but 3000 of 3 and 1109 f32 (5 pieces) 18.1 and
// 22.6.  A bound of 512 takes the even way for the third, one of 8192 the other for the last.
constexpr uint64_t kFewWaves = 2048;
// Rows that cannot stay in the 256 MiB memory-side cache until somebody reads them again are streamed past the caches.
constexpr uint64_t kStreamBytes = 256ull << 20;

// How a launch cuts its work.  A group of lanes -- a power of two up to a wave's 64, enough for the row if they can be --
// takes a piece of a row, a 16-byte vector a lane.  Where the last vector would reach behind the row it ends with it instead and
// repeats some columns of the one before: they are worked out alike and written twice.  Only rows shorter than a
// vector go element by element.
struct Cut {
    uint32_t lanes_log2;
    uint32_t vectors;      // 16-byte vectors of a row, 0 if it is shorter than one
    uint32_t last_column;  // where the last vector starts
    uint32_t pieces;       // of a row
    uint32_t items;        // what groups take: tokens * pieces, or tokens * token_waves
    uint32_t token_waves;  // combine's gradient: waves that share a token's pieces, a power of two
    uint32_t blocks;       // workgroups for the items
    uint32_t pad_blocks;   // workgroups before them that zero the rows that fill segments up
    uint32_t pad_split;    // waves that share an expert's
};

int cut_rows(const MoveArgs& a, uint32_t element_bytes, uint32_t threads, uint32_t short_threads, bool whole_tokens, bool pads, Cut* out)
{
    Cut c;
    const uint64_t row_bytes = static_cast<uint64_t>(a.hidden) * element_bytes;
    const uint32_t touched = static_cast<uint32_t>((row_bytes + 15) / 16);
    c.vectors = row_bytes < 16 ? 0 : touched;
    c.last_column = row_bytes < 16 ? 0 : a.hidden - 16 / element_bytes;
    c.lanes_log2 = 0;
    while (c.lanes_log2 < 6 && (1u << c.lanes_log2) < touched) ++c.lanes_log2;
    c.pieces = (touched + (1u << c.lanes_log2) - 1) >> c.lanes_log2;
    if (c.lanes_log2 < 6) threads = short_threads;
    c.token_waves = 1;
    while (c.pieces % (c.token_waves * 2) == 0 && c.token_waves < threads / 64) c.token_waves *= 2;
    if (a.tokens * c.token_waves < kFewWaves)
        while (c.token_waves * 2 <= c.pieces && c.token_waves < threads / 64) c.token_waves *= 2;
    const uint64_t items = a.tokens * (whole_tokens ? c.token_waves : c.pieces);
    const uint32_t per_block = threads >> c.lanes_log2;
    uint64_t blocks = (items + per_block - 1) / per_block;
    if (blocks > kMaxBlocks) blocks = kMaxBlocks;
    c.blocks = static_cast<uint32_t>(blocks);
    // item numbers, and one step beyond the last, fit 32 bits
    if (items + blocks * per_block > 0xFFFFFFFFull) return fail(MRS_ERR_UNSUPPORTED, "more than 2^32 pieces of rows in one call");
    c.items = static_cast<uint32_t>(items);
    c.pad_split = 0;
    c.pad_blocks = 0;
    if (pads && a.align > 1) {
        c.pad_split = kPadWaves / a.experts;
        if (c.pad_split > a.align - 1) c.pad_split = a.align - 1;
        if (c.pad_split == 0) c.pad_split = 1;
        c.pad_blocks = (a.experts * c.pad_split + threads / 64 - 1) / (threads / 64);
    }
    *out = c;
    return MRS_OK;
}

template <bool STREAM>
__device__ __forceinline__ RouteVec get(const void* p)
{
    if (STREAM) return __builtin_nontemporal_load(static_cast<const RouteVecLoose*>(p));
    return load_vec(p);
}
template <bool STREAM>
__device__ __forceinline__ void put(void* p, RouteVec v)
{
    if (STREAM)
        __builtin_nontemporal_store(v, static_cast<RouteVecLoose*>(p));
    else
        store_vec(p, v);
}

// A wave's share of the rows of one expert's segment that no slot has: zeros.
template <typename Elem, uint32_t THREADS>
__device__ void zero_padding(const MoveArgs& a, const Cut& c)
{
    const uint32_t item = __builtin_amdgcn_readfirstlane(blockIdx.x * (THREADS / 64) + threadIdx.x / 64);
    const uint32_t e = item / c.pad_split;
    if (e >= a.experts) return;
    const int64_t first = static_cast<int64_t>(a.offsets[e]) + a.counts[e];
    int64_t end = a.offsets[e + 1];
    if (end > a.rows) end = a.rows;
    if (first < 0) return;
    Elem* out = static_cast<Elem*>(a.rows_out);
    constexpr uint32_t N = 16 / sizeof(Elem);
    const uint32_t lane = threadIdx.x & 63u;
    const RouteVec zero = {0, 0, 0, 0};
    for (int64_t r = first + item % c.pad_split; r < end; r += c.pad_split) {
        Elem* row = out + static_cast<uint64_t>(r) * a.ld_rows_out;
        for (uint32_t v = lane; v < c.vectors; v += 64) store_vec(row + min(v * N, c.last_column), zero);
        if (c.vectors == 0 && lane < a.hidden) row[lane] = Elem(0);
    }
}

// This group's first item.  Whole waves on one item say so: what depends on the token alone then lives in
// scalar registers and comes through scalar loads.
template <uint32_t THREADS, bool WAVE>
__device__ __forceinline__ uint32_t first_item(const Cut& c)
{
    uint32_t in_block = threadIdx.x >> c.lanes_log2;
    if (WAVE) in_block = __builtin_amdgcn_readfirstlane(in_block);
    return (blockIdx.x - c.pad_blocks) * (THREADS >> c.lanes_log2) + in_block;
}

// The rows of slots j0 .. j0 + K - 1 of a token; `rows` (none) for slots without one and behind the last.
// The loads do not depend on how many slots there are (those behind the last repeat it): guarded one by one they
// would also be waited for one by one.
template <uint32_t K>
__device__ __forceinline__ void load_slots(const int32_t* __restrict__ row_of_slot, uint32_t t, uint32_t j0, const MoveArgs& a,
                                           uint32_t (&r)[K])
{
    const int32_t* slots = row_of_slot + static_cast<uint64_t>(t) * a.topk;
#pragma unroll
    for (uint32_t j = 0; j < K; ++j) r[j] = static_cast<uint32_t>(slots[min(j0 + j, a.topk - 1)]);
#pragma unroll
    for (uint32_t j = 0; j < K; ++j)
        if (j0 + j >= a.topk || r[j] > a.rows) r[j] = a.rows;
}
template <uint32_t K>
__device__ __forceinline__ void load_weights(const float* __restrict__ weights, uint32_t t, uint32_t j0, const MoveArgs& a,
                                             float (&w)[K])
{
    weights += static_cast<uint64_t>(t) * a.topk;
#pragma unroll
    for (uint32_t j = 0; j < K; ++j) w[j] = weights[min(j0 + j, a.topk - 1)];
}

// ---- dispatch: a row is read once and written `topk` times -----------------------------------
// Workgroups of two waves, rows written through the caches: 0.239 ms for 16384 tokens, 8 slots, 4096 bf16 (1.1 GB
// written, 5.3 TB/s in all; plain copies reach 4.9 to 5.6).  Larger workgroups or stores past the caches: 0.243 to 0.261; reading
// by row, so that the writes run through the buffer in order: 0.34, the reads no longer come from memory once.
template <typename Elem, uint32_t K, bool WAVE>
__global__ __launch_bounds__(kMoveThreads) void route_dispatch_kernel(const Elem* __restrict__ x, Elem* __restrict__ out,
                                                                      const int32_t* __restrict__ row_of_slot, const MoveArgs a,
                                                                      const Cut c)
{
    if (blockIdx.x < c.pad_blocks) {
        zero_padding<Elem, kMoveThreads>(a, c);
        return;
    }
    constexpr uint32_t N = 16 / sizeof(Elem);
    const uint32_t lane = threadIdx.x & ((1u << c.lanes_log2) - 1);
    const uint32_t step = c.blocks * (kMoveThreads >> c.lanes_log2);
    for (uint32_t item = first_item<kMoveThreads, WAVE>(c); item < c.items; item += step) {
        const uint32_t t = item / c.pieces, piece = item - t * c.pieces;
        const Elem* in = x + static_cast<uint64_t>(t) * a.ld_token_in;
        const uint32_t v = (piece << c.lanes_log2) + lane;
        const uint32_t column = min(v * N, c.last_column);
        RouteVec d = {0, 0, 0, 0};
        if (v < c.vectors) d = load_vec(in + column);
        for (uint32_t j0 = 0; j0 < a.topk; j0 += K) {
            uint32_t r[K];
            load_slots<K>(row_of_slot, t, j0, a, r);
            if (v < c.vectors) {
#pragma unroll
                for (uint32_t j = 0; j < K; ++j)
                    if (r[j] < a.rows) store_vec(out + r[j] * a.ld_rows_out + column, d);
            }
            for (uint32_t h = lane; c.vectors == 0 && h < a.hidden; h += 1u << c.lanes_log2) {
                const Elem e = in[h];
#pragma unroll
                for (uint32_t j = 0; j < K; ++j)
                    if (r[j] < a.rows) out[r[j] * a.ld_rows_out + h] = e;
            }
        }
    }
}

// ---- combine: `topk` rows are read, one is written --------------------------------------------
// Up to eight rows' pieces are loaded before the first is used.  The sum is held in 32 bits and runs in the
// order of the slots, one fused multiply-add each.  Workgroups of 16 waves, which read whole rows of up to 16 KiB
// at about the same time, and loads past the caches: 0.205 ms for 16384 tokens, 8 slots, 4096 bf16 (5.9 TB/s); with
// workgroups of 4 waves 0.214, with ordinary loads 0.231, with neither 0.24.  Where the rows fit the memory-side
// cache ordinary loads win: 64 MiB of them 13.5 against 14 us.
template <typename T, uint32_t K, bool MORE, bool WEIGHTED, bool WAVE, bool STREAM>
__global__ __launch_bounds__(WAVE ? kSumThreads : kShortThreads) void route_combine_kernel(
    const T* __restrict__ rows, T* __restrict__ out, const int32_t* __restrict__ row_of_slot, const float* __restrict__ weights,
    const MoveArgs a, const Cut c)
{
    constexpr uint32_t N = 16 / sizeof(T), THREADS = WAVE ? kSumThreads : kShortThreads;
    const uint32_t lane = threadIdx.x & ((1u << c.lanes_log2) - 1);
    const uint32_t step = c.blocks * (THREADS >> c.lanes_log2);
    for (uint32_t item = first_item<THREADS, WAVE>(c); item < c.items; item += step) {
        const uint32_t t = item / c.pieces, piece = item - t * c.pieces;
        T* to = out + static_cast<uint64_t>(t) * a.ld_token_out;
        const uint32_t v = (piece << c.lanes_log2) + lane;
        const uint32_t column = min(v * N, c.last_column);
        uint32_t r[K];
        float w[K];
        load_slots<K>(row_of_slot, t, 0, a, r);
        if (WEIGHTED) load_weights<K>(weights, t, 0, a, w);
        if (v < c.vectors) {
            float acc[N];
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) acc[i] = 0.0f;
            for (uint32_t j0 = 0;;) {
                RouteVec d[K];
#pragma unroll
                for (uint32_t j = 0; j < K; ++j) {
                    d[j] = RouteVec{0, 0, 0, 0};
                    if (r[j] < a.rows) d[j] = get<STREAM>(rows + r[j] * a.ld_rows_in + column);
                }
#pragma unroll
                for (uint32_t j = 0; j < K; ++j) {
                    if (r[j] >= a.rows) continue;
                    const RouteElems<T> e = as_elems<T>(d[j]);
#pragma unroll
                    for (uint32_t i = 0; i < N; ++i) acc[i] = WEIGHTED ? fmaf(w[j], to_f32(e.e[i]), acc[i]) : acc[i] + to_f32(e.e[i]);
                }
                j0 += K;
                if (!MORE || j0 >= a.topk) break;
                load_slots<K>(row_of_slot, t, j0, a, r);
                if (WEIGHTED) load_weights<K>(weights, t, j0, a, w);
            }
            RouteElems<T> o;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) o.e[i] = static_cast<T>(acc[i]);
            put<STREAM>(to + column, as_vec(o));
        }
        for (uint32_t h = lane; c.vectors == 0 && h < a.hidden; h += 1u << c.lanes_log2) {
            float acc = 0.0f;
            for (uint32_t j = 0; j < a.topk; ++j) {
                uint32_t r[1];
                load_slots<1>(row_of_slot, t, j, a, r);
                if (r[0] >= a.rows) continue;
                const float x = to_f32(rows[r[0] * a.ld_rows_in + h]);
                acc = WEIGHTED ? fmaf(weights[static_cast<uint64_t>(t) * a.topk + j], x, acc) : acc + x;
            }
            to[h] = static_cast<T>(acc);
        }
    }
}

// ---- combine's gradient ----------------------------------------------------------------------
// For K slots at a time: a piece of out_grad is read, and for every slot the piece of its row is read for the dot
// product and the weighted piece written.  token_waves waves of a workgroup share a token; the lanes' partial dot
// products are added by a fixed tree, the waves' in order, so results are the same every time.  Reads and writes
// come in equal parts, past the caches where they are large: 0.445 ms for 16384 tokens, 8 slots, 4096 bf16 (5.3 TB/s; a
// plain copy 4.9 to 5.6).  One wave for each token: 0.463; through the caches: 0.468.

// Sums of K values over a wave, M = 32.  While there are several values left, a step hands half of them to the
// other half of the lanes.  Lane l returns the sum of value l / (64 / K).
template <uint32_t K, uint32_t M>
__device__ __forceinline__ float sums_over_wave(const float (&v)[K])
{
    if constexpr (M == 0) {
        return v[0];
    } else if constexpr (K == 1) {
        const float both[1] = {v[0] + __shfl_xor(v[0], static_cast<int>(M))};
        return sums_over_wave<1, M / 2>(both);
    } else {
        const bool upper = threadIdx.x & M;
        float half[K / 2];
#pragma unroll
        for (uint32_t j = 0; j < K / 2; ++j) {
            const float give = upper ? v[j] : v[j + K / 2];
            const float keep = upper ? v[j + K / 2] : v[j];
            half[j] = keep + __shfl_xor(give, static_cast<int>(M));
        }
        return sums_over_wave<K / 2, M / 2>(half);
    }
}

template <typename T, uint32_t K, bool WAVE, bool STREAM>
__global__ __launch_bounds__(WAVE ? kSumThreads : kShortThreads) void route_combine_backward_kernel(
    const T* __restrict__ rows, const T* __restrict__ out_grad, T* __restrict__ rows_grad, const int32_t* __restrict__ row_of_slot,
    const float* __restrict__ weights, const MoveArgs a, const Cut c)
{
    constexpr uint32_t THREADS = WAVE ? kSumThreads : kShortThreads;
    if (blockIdx.x < c.pad_blocks) {
        zero_padding<T, THREADS>(a, c);
        return;
    }
    constexpr uint32_t N = 16 / sizeof(T);
    __shared__ float partial[2][THREADS / 64][K];
    const uint32_t lanes = 1u << c.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const uint32_t per_block = THREADS >> c.lanes_log2;
    uint32_t item = first_item<THREADS, WAVE>(c);
    uint32_t half = 0;
    // the whole workgroup leaves together: its first item is what counts
    for (uint32_t base = (blockIdx.x - c.pad_blocks) * per_block; base < c.items; base += c.blocks * per_block, item += c.blocks * per_block) {
        const uint32_t t = item / c.token_waves, share = item - t * c.token_waves;
        for (uint32_t j0 = 0; j0 < a.topk; j0 += K) {
            float dot[K];
#pragma unroll
            for (uint32_t j = 0; j < K; ++j) dot[j] = 0.0f;
            if (item < c.items) {
                uint32_t r[K];
                float w[K];
                load_slots<K>(row_of_slot, t, j0, a, r);
                load_weights<K>(weights, t, j0, a, w);
                const T* grad = out_grad + static_cast<uint64_t>(t) * a.ld_token_in;
                // LAST: the piece holds a vector that repeats columns of the one before; they count once
                const auto walk = [&](uint32_t v, auto last) {
                    constexpr bool LAST = decltype(last)::value;
                    const uint32_t column = LAST ? min(v * N, c.last_column) : v * N;
                    const uint32_t repeated = LAST ? v * N - column : 0;
                    const RouteElems<T> ge = as_elems<T>(get<STREAM>(grad + column));
                    RouteVec d[K];
#pragma unroll
                    for (uint32_t j = 0; j < K; ++j) {
                        d[j] = RouteVec{0, 0, 0, 0};
                        if (r[j] < a.rows) d[j] = get<STREAM>(rows + r[j] * a.ld_rows_in + column);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < K; ++j) {
                        if (r[j] >= a.rows) continue;
                        const RouteElems<T> e = as_elems<T>(d[j]);
                        RouteElems<T> o;
#pragma unroll
                        for (uint32_t i = 0; i < N; ++i) {
                            const float g = to_f32(ge.e[i]);
                            const float sum = fmaf(g, to_f32(e.e[i]), dot[j]);
                            dot[j] = LAST && i < repeated ? dot[j] : sum;
                            o.e[i] = static_cast<T>(w[j] * g);
                        }
                        put<STREAM>(rows_grad + r[j] * a.ld_rows_out + column, as_vec(o));
                    }
                };
                for (uint32_t v = (share << c.lanes_log2) + lane; v < c.vectors; v += c.token_waves << c.lanes_log2) {
                    if ((v - lane + lanes) * N > a.hidden)
                        walk(v, std::true_type{});
                    else
                        walk(v, std::false_type{});
                }
                for (uint32_t h = lane; c.vectors == 0 && h < a.hidden; h += lanes) {
                    const float g = to_f32(grad[h]);
#pragma unroll
                    for (uint32_t j = 0; j < K; ++j) {
                        if (r[j] >= a.rows) continue;
                        dot[j] = fmaf(g, to_f32(rows[r[j] * a.ld_rows_in + h]), dot[j]);
                        rows_grad[r[j] * a.ld_rows_out + h] = static_cast<T>(w[j] * g);
                    }
                }
            }
            float* sums = a.weights_grad + static_cast<uint64_t>(t) * a.topk + j0;
            if (WAVE) {
                constexpr uint32_t kLanesPerSlot = 64 / K;
                const float d = sums_over_wave<K, 32>(dot);
                const uint32_t j = lane / kLanesPerSlot;
                const bool first_lane = lane % kLanesPerSlot == 0;
                const bool writes = first_lane && j0 + j < a.topk && item < c.items;
                if (c.token_waves == 1) {
                    if (writes) sums[j] = d;
                } else {
                    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
                    if (first_lane) partial[half][wave][j] = d;
                    __syncthreads();
                    if (share == 0 && writes) {
                        float sum = d;
                        for (uint32_t i = 1; i < c.token_waves; ++i) sum += partial[half][wave + i][j];
                        sums[j] = sum;
                    }
                    half ^= 1;  // the next round writes the other half: one barrier a round is enough
                }
            } else {
                for (uint32_t m = lanes >> 1; m > 0; m >>= 1)
#pragma unroll
                    for (uint32_t j = 0; j < K; ++j) dot[j] += __shfl_xor(dot[j], static_cast<int>(m), static_cast<int>(lanes));
#pragma unroll
                for (uint32_t j = 0; j < K; ++j)
                    if (item < c.items && j0 + j < a.topk && lane == (j & (lanes - 1))) sums[j] = dot[j];
            }
        }
    }
}

// Calls f with the number of slots a kernel takes at a time, and whether there are more.
template <typename F>
void with_slots(uint32_t topk, F&& f)
{
    if (topk <= 4)
        f(std::integral_constant<uint32_t, 4>{}, std::false_type{});
    else if (topk <= 8)
        f(std::integral_constant<uint32_t, 8>{}, std::false_type{});
    else
        f(std::integral_constant<uint32_t, 8>{}, std::true_type{});
}

template <typename E>
int start_dispatch(const MoveArgs& a, hipStream_t s)
{
    Cut c;
    if (int rc = cut_rows(a, sizeof(E), kMoveThreads, kMoveThreads, false, true, &c)) return rc;
    const dim3 grid(c.blocks + c.pad_blocks), block(kMoveThreads);
    with_slots(a.topk, [&](auto k, auto) {
        constexpr uint32_t K = decltype(k)::value;
        const E* x = static_cast<const E*>(a.token_in);
        E* rows = static_cast<E*>(a.rows_out);
        if (c.lanes_log2 == 6)
            hipLaunchKernelGGL((route_dispatch_kernel<E, K, true>), grid, block, 0, s, x, rows, a.row_of_slot, a, c);
        else
            hipLaunchKernelGGL((route_dispatch_kernel<E, K, false>), grid, block, 0, s, x, rows, a.row_of_slot, a, c);
    });
    MRS_CHECK_LAUNCH("route_dispatch_kernel");
    return MRS_OK;
}

template <typename T, bool WEIGHTED>
int start_combine(const MoveArgs& a, hipStream_t s)
{
    Cut c;
    if (int rc = cut_rows(a, sizeof(T), kSumThreads, kShortThreads, false, false, &c)) return rc;
    const dim3 grid(c.blocks), block(c.lanes_log2 == 6 ? kSumThreads : kShortThreads);
    const bool stream = a.tokens * a.topk * a.hidden * sizeof(T) >= kStreamBytes;
    // a loop for more than eight slots costs the others 1 %
    with_slots(a.topk, [&](auto k, auto more) {
        constexpr uint32_t K = decltype(k)::value;
        constexpr bool MORE = decltype(more)::value;
        const T* rows = static_cast<const T*>(a.rows_in);
        T* out = static_cast<T*>(a.token_out);
        if (c.lanes_log2 < 6)
            hipLaunchKernelGGL((route_combine_kernel<T, K, MORE, WEIGHTED, false, false>), grid, block, 0, s, rows, out, a.row_of_slot, a.weights,
                               a, c);
        else if (!stream)
            hipLaunchKernelGGL((route_combine_kernel<T, K, MORE, WEIGHTED, true, false>), grid, block, 0, s, rows, out, a.row_of_slot, a.weights,
                               a, c);
        else
            hipLaunchKernelGGL((route_combine_kernel<T, K, MORE, WEIGHTED, true, true>), grid, block, 0, s, rows, out, a.row_of_slot, a.weights,
                               a, c);
    });
    MRS_CHECK_LAUNCH("route_combine_kernel");
    return MRS_OK;
}

template <typename T>
int start_combine_backward(const MoveArgs& a, hipStream_t s)
{
    Cut c;
    if (int rc = cut_rows(a, sizeof(T), kSumThreads, kShortThreads, true, true, &c)) return rc;
    const dim3 grid(c.blocks + c.pad_blocks), block(c.lanes_log2 == 6 ? kSumThreads : kShortThreads);
    const bool stream = 2 * a.tokens * a.topk * a.hidden * sizeof(T) >= kStreamBytes;  // read and written
    with_slots(a.topk, [&](auto k, auto) {
        constexpr uint32_t K = decltype(k)::value;
        const T* rows = static_cast<const T*>(a.rows_in);
        const T* grad = static_cast<const T*>(a.token_in);
        T* out = static_cast<T*>(a.rows_out);
        if (c.lanes_log2 < 6)
            hipLaunchKernelGGL((route_combine_backward_kernel<T, K, false, false>), grid, block, 0, s, rows, grad, out, a.row_of_slot, a.weights,
                               a, c);
        else if (!stream)
            hipLaunchKernelGGL((route_combine_backward_kernel<T, K, true, false>), grid, block, 0, s, rows, grad, out, a.row_of_slot, a.weights,
                               a, c);
        else
            hipLaunchKernelGGL((route_combine_backward_kernel<T, K, true, true>), grid, block, 0, s, rows, grad, out, a.row_of_slot, a.weights,
                               a, c);
    });
    MRS_CHECK_LAUNCH("route_combine_backward_kernel");
    return MRS_OK;
}

}  // namespace

int launch_route_dispatch(int element_bytes, const MoveArgs& a, hipStream_t s)
{
    if (element_bytes == 1) return start_dispatch<uint8_t>(a, s);
    if (element_bytes == 2) return start_dispatch<uint16_t>(a, s);
    return start_dispatch<uint32_t>(a, s);
}

int launch_route_combine(int type, const MoveArgs& a, hipStream_t s)
{
    if (type == MRS_TYPE_F32) return a.weights ? start_combine<float, true>(a, s) : start_combine<float, false>(a, s);
    if (type == MRS_TYPE_F16) return a.weights ? start_combine<_Float16, true>(a, s) : start_combine<_Float16, false>(a, s);
    return a.weights ? start_combine<__bf16, true>(a, s) : start_combine<__bf16, false>(a, s);
}

int launch_route_combine_backward(int type, const MoveArgs& a, hipStream_t s)
{
    if (type == MRS_TYPE_F32) return start_combine_backward<float>(a, s);
    if (type == MRS_TYPE_F16) return start_combine_backward<_Float16>(a, s);
    return start_combine_backward<__bf16>(a, s);
}

}  // namespace mrs
