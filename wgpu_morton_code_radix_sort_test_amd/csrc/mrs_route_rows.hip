// Rows moved between token order and expert order: dispatch, combine and their gradients
// (mrs_route_* in include/mrs.h).  Every row is read once and written once in 16-byte pieces; what
// bounds these kernels is memory bandwidth, at a few tokens the latency of one dependent chain
// (slot's row number -> row -> store).
#include <type_traits>

#include "mrs_route.hpp"

namespace mrs {

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint64_t kMaxBlocks = 1u << 22;  // more work than that is looped over

// How a launch cuts its work: a token's row in pieces of `lanes` 16-byte vectors (a power of two up
// to a wave's 64), one item per (token, piece), 256 / lanes items per workgroup.
struct Cut {
    uint32_t lanes_log2;
    uint32_t vectors;  // vectors of a row, the last one possibly cut short
    uint32_t pieces;   // ceil(vectors / lanes)
    uint64_t items;
    uint32_t blocks;      // workgroups for the items
    uint32_t pad_blocks;  // workgroups behind them that zero the rows between segments' ends
    uint32_t pad_split;   // of these, how many share an expert
};

Cut cut_rows(const MoveArgs& a, uint32_t element_bytes, bool one_item_per_token, bool pads)
{
    Cut c;
    c.vectors = static_cast<uint32_t>((static_cast<uint64_t>(a.hidden) * element_bytes + 15) / 16);
    c.lanes_log2 = 0;
    while (c.lanes_log2 < 6 && (1u << c.lanes_log2) < c.vectors) ++c.lanes_log2;
    c.pieces = one_item_per_token ? 1 : (c.vectors + (1u << c.lanes_log2) - 1) >> c.lanes_log2;
    c.items = a.tokens * c.pieces;
    const uint64_t per_block = kThreads >> c.lanes_log2;
    uint64_t blocks = (c.items + per_block - 1) / per_block;
    if (blocks > kMaxBlocks) blocks = kMaxBlocks;
    c.blocks = static_cast<uint32_t>(blocks);
    c.pad_split = 0;
    c.pad_blocks = 0;
    if (pads && a.align > 1) {
        c.pad_split = a.align - 1 < 8 ? a.align - 1 : 8;
        c.pad_blocks = a.experts * c.pad_split;
    }
    return c;
}

// Zeroes the rows of one expert's segment that no slot has.
template <typename Elem>
__device__ void zero_padding(const MoveArgs& a, const Cut& c, uint32_t block)
{
    const uint32_t e = block / c.pad_split;
    const uint32_t part = block % c.pad_split;
    const int64_t first = static_cast<int64_t>(a.offsets[e]) + a.counts[e];
    int64_t end = a.offsets[e + 1];
    if (end > a.rows) end = a.rows;
    if (first < 0) return;
    Elem* out = static_cast<Elem*>(a.rows_out);
    constexpr uint32_t N = 16 / sizeof(Elem);
    const uint32_t whole = a.hidden / N;
    const RouteVec zero = {0, 0, 0, 0};
    for (int64_t r = first + part; r < end; r += c.pad_split) {
        Elem* row = out + static_cast<uint64_t>(r) * a.ld_rows_out;
        for (uint32_t v = threadIdx.x; v < whole; v += kThreads) store_vec(row + static_cast<uint64_t>(v) * N, zero);
        for (uint32_t h = whole * N + threadIdx.x; h < a.hidden; h += kThreads) row[h] = Elem(0);
    }
}

// The item of this thread: token, piece.  With whole waves on one item the token is the same for all
// lanes and said to be (its slots' row numbers then come through scalar loads).
template <bool WAVE>
__device__ __forceinline__ uint64_t first_item(const Cut& c)
{
    uint32_t in_block = threadIdx.x >> c.lanes_log2;
    if (WAVE) in_block = __builtin_amdgcn_readfirstlane(in_block);
    return static_cast<uint64_t>(blockIdx.x) * (kThreads >> c.lanes_log2) + in_block;
}

__device__ __forceinline__ uint64_t token_of(const Cut& c, uint64_t item, uint32_t* piece)
{
    if (c.pieces == 1) {
        *piece = 0;
        return item;
    }
    if (item >> 32) {
        const uint64_t t = item / c.pieces;
        *piece = static_cast<uint32_t>(item - t * c.pieces);
        return t;
    }
    const uint32_t t = static_cast<uint32_t>(item) / c.pieces;
    *piece = static_cast<uint32_t>(item) - t * c.pieces;
    return t;
}

// ---- dispatch: a row is read once and written `topk` times -----------------------------------
template <typename Elem, bool WAVE>
__global__ __launch_bounds__(kThreads) void route_dispatch_kernel(const MoveArgs a, const Cut c)
{
    if (blockIdx.x >= c.blocks) {
        zero_padding<Elem>(a, c, blockIdx.x - c.blocks);
        return;
    }
    constexpr uint32_t N = 16 / sizeof(Elem);
    const uint32_t lane = threadIdx.x & ((1u << c.lanes_log2) - 1);
    const uint64_t step = static_cast<uint64_t>(c.blocks) * (kThreads >> c.lanes_log2);
    for (uint64_t item = first_item<WAVE>(c); item < c.items; item += step) {
        uint32_t piece;
        const uint64_t t = token_of(c, item, &piece);
        const uint32_t h = ((piece << c.lanes_log2) + lane) * N;
        if (h >= a.hidden) continue;
        const Elem* in = static_cast<const Elem*>(a.token_in) + t * a.ld_token_in + h;
        Elem* out = static_cast<Elem*>(a.rows_out) + h;
        const int32_t* slots = a.row_of_slot + t * a.topk;
        if (h + N <= a.hidden) {
            const RouteVec v = load_vec(in);
            for (uint32_t j = 0; j < a.topk; ++j) {
                const uint32_t r = static_cast<uint32_t>(slots[j]);
                if (r < a.rows) store_vec(out + static_cast<uint64_t>(r) * a.ld_rows_out, v);
            }
        } else {
            for (uint32_t j = 0; j < a.topk; ++j) {
                const uint32_t r = static_cast<uint32_t>(slots[j]);
                if (r >= a.rows) continue;
                for (uint32_t i = 0; h + i < a.hidden; ++i) out[static_cast<uint64_t>(r) * a.ld_rows_out + i] = in[i];
            }
        }
    }
}

// ---- combine: `topk` rows are read, one is written --------------------------------------------
// Rows are loaded eight at a time before the first is used.  The sum is held in 32 bits and runs in
// the order of the slots, one fused multiply-add each.
template <typename T, bool WEIGHTED, bool WAVE>
__global__ __launch_bounds__(kThreads) void route_combine_kernel(const MoveArgs a, const Cut c)
{
    constexpr uint32_t N = 16 / sizeof(T);
    constexpr uint32_t B = 8;
    const uint32_t lane = threadIdx.x & ((1u << c.lanes_log2) - 1);
    const uint64_t step = static_cast<uint64_t>(c.blocks) * (kThreads >> c.lanes_log2);
    for (uint64_t item = first_item<WAVE>(c); item < c.items; item += step) {
        uint32_t piece;
        const uint64_t t = token_of(c, item, &piece);
        const uint32_t h = ((piece << c.lanes_log2) + lane) * N;
        if (h >= a.hidden) continue;
        const T* in = static_cast<const T*>(a.rows_in) + h;
        T* out = static_cast<T*>(a.token_out) + t * a.ld_token_out + h;
        const int32_t* slots = a.row_of_slot + t * a.topk;
        const float* weights = WEIGHTED ? a.weights + t * a.topk : nullptr;
        if (h + N <= a.hidden) {
            float acc[N];
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) acc[i] = 0.0f;
            for (uint32_t j0 = 0; j0 < a.topk; j0 += B) {
                RouteVec v[B];
                uint32_t r[B];
#pragma unroll
                for (uint32_t j = 0; j < B; ++j) r[j] = j0 + j < a.topk ? static_cast<uint32_t>(slots[j0 + j]) : 0xFFFFFFFFu;
#pragma unroll
                for (uint32_t j = 0; j < B; ++j) {
                    v[j] = RouteVec{0, 0, 0, 0};
                    if (r[j] < a.rows) v[j] = load_vec(in + static_cast<uint64_t>(r[j]) * a.ld_rows_in);
                }
#pragma unroll
                for (uint32_t j = 0; j < B; ++j) {
                    if (r[j] >= a.rows) continue;
                    const float w = WEIGHTED ? weights[j0 + j] : 1.0f;
                    const RouteElems<T> e = as_elems<T>(v[j]);
#pragma unroll
                    for (uint32_t i = 0; i < N; ++i) acc[i] = WEIGHTED ? fmaf(w, to_f32(e.e[i]), acc[i]) : acc[i] + to_f32(e.e[i]);
                }
            }
            RouteElems<T> o;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) o.e[i] = static_cast<T>(acc[i]);
            store_vec(out, as_vec(o));
        } else {
            for (uint32_t i = 0; h + i < a.hidden; ++i) {
                float acc = 0.0f;
                for (uint32_t j = 0; j < a.topk; ++j) {
                    const uint32_t r = static_cast<uint32_t>(slots[j]);
                    if (r >= a.rows) continue;
                    const float x = to_f32(in[static_cast<uint64_t>(r) * a.ld_rows_in + i]);
                    acc = WEIGHTED ? fmaf(weights[j], x, acc) : acc + x;
                }
                out[i] = static_cast<T>(acc);
            }
        }
    }
}

// ---- combine's gradient ----------------------------------------------------------------------
// One pass: a piece of out_grad is read once, and for every slot the piece of its row is read for the
// dot product and the weighted piece written.  A token belongs to one group of lanes, which walks
// its row; the lanes' partial dot products are added by a fixed tree at the end, so
// results are the same every time.
template <typename T, uint32_t K, bool WAVE>
__global__ __launch_bounds__(kThreads) void route_combine_backward_kernel(const MoveArgs a, const Cut c)
{
    if (blockIdx.x >= c.blocks) {
        zero_padding<T>(a, c, blockIdx.x - c.blocks);
        return;
    }
    constexpr uint32_t N = 16 / sizeof(T);
    constexpr uint32_t B = K < 8 ? K : 8;
    const uint32_t lanes = 1u << c.lanes_log2;
    const uint32_t lane = threadIdx.x & (lanes - 1);
    const uint64_t step = static_cast<uint64_t>(c.blocks) * (kThreads >> c.lanes_log2);
    for (uint64_t t = first_item<WAVE>(c); t < c.items; t += step) {
        const int32_t* slots = a.row_of_slot + t * a.topk;
        const float* weights = a.weights + t * a.topk;
        const T* grad = static_cast<const T*>(a.token_in) + t * a.ld_token_in;
        float dot[K];
#pragma unroll
        for (uint32_t j = 0; j < K; ++j) dot[j] = 0.0f;
        for (uint32_t h = lane * N; h < a.hidden; h += lanes * N) {
            const T* in = static_cast<const T*>(a.rows_in) + h;
            T* out = static_cast<T*>(a.rows_out) + h;
            if (h + N <= a.hidden) {
                const RouteElems<T> ge = as_elems<T>(load_vec(grad + h));
#pragma unroll
                for (uint32_t j0 = 0; j0 < K; j0 += B) {
                    RouteVec v[B];
                    uint32_t r[B];
#pragma unroll
                    for (uint32_t j = 0; j < B; ++j) r[j] = j0 + j < a.topk ? static_cast<uint32_t>(slots[j0 + j]) : 0xFFFFFFFFu;
#pragma unroll
                    for (uint32_t j = 0; j < B; ++j) {
                        v[j] = RouteVec{0, 0, 0, 0};
                        if (r[j] < a.rows) v[j] = load_vec(in + static_cast<uint64_t>(r[j]) * a.ld_rows_in);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < B; ++j) {
                        if (r[j] >= a.rows) continue;
                        const float w = weights[j0 + j];
                        const RouteElems<T> e = as_elems<T>(v[j]);
                        RouteElems<T> o;
#pragma unroll
                        for (uint32_t i = 0; i < N; ++i) {
                            const float g = to_f32(ge.e[i]);
                            dot[j0 + j] = fmaf(g, to_f32(e.e[i]), dot[j0 + j]);
                            o.e[i] = static_cast<T>(w * g);
                        }
                        store_vec(out + static_cast<uint64_t>(r[j]) * a.ld_rows_out, as_vec(o));
                    }
                }
            } else {
#pragma unroll
                for (uint32_t j = 0; j < K; ++j) {
                    const uint32_t r = j < a.topk ? static_cast<uint32_t>(slots[j]) : 0xFFFFFFFFu;
                    if (r >= a.rows) continue;
                    const float w = weights[j];
                    for (uint32_t i = 0; h + i < a.hidden; ++i) {
                        const float g = to_f32(grad[h + i]);
                        dot[j] = fmaf(g, to_f32(in[static_cast<uint64_t>(r) * a.ld_rows_in + i]), dot[j]);
                        out[static_cast<uint64_t>(r) * a.ld_rows_out + i] = static_cast<T>(w * g);
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < K; ++j) {
            float d = dot[j];
            for (uint32_t m = lanes >> 1; m > 0; m >>= 1) d += __shfl_xor(d, static_cast<int>(m), static_cast<int>(lanes));
            if (j < a.topk && lane == (j & (lanes - 1))) a.weights_grad[t * a.topk + j] = d;
        }
    }
}

}  // namespace

int launch_route_dispatch(int element_bytes, const MoveArgs& a, int num_cus, hipStream_t s)
{
    (void)num_cus;
    const Cut c = cut_rows(a, element_bytes, false, true);
    const dim3 grid(c.blocks + c.pad_blocks), block(kThreads);
    if (grid.x == 0) return MRS_OK;
    const auto go = [&](auto elem) {
        using E = decltype(elem);
        if (c.lanes_log2 == 6)
            hipLaunchKernelGGL((route_dispatch_kernel<E, true>), grid, block, 0, s, a, c);
        else
            hipLaunchKernelGGL((route_dispatch_kernel<E, false>), grid, block, 0, s, a, c);
    };
    if (element_bytes == 1)
        go(uint8_t{});
    else if (element_bytes == 2)
        go(uint16_t{});
    else
        go(uint32_t{});
    MRS_CHECK_LAUNCH("route_dispatch_kernel");
    return MRS_OK;
}

template <typename T>
static void start_combine(const MoveArgs& a, hipStream_t s)
{
    const Cut c = cut_rows(a, sizeof(T), false, false);
    const dim3 grid(c.blocks), block(kThreads);
    if (grid.x == 0) return;
    const bool wave = c.lanes_log2 == 6;
    if (a.weights) {
        if (wave)
            hipLaunchKernelGGL((route_combine_kernel<T, true, true>), grid, block, 0, s, a, c);
        else
            hipLaunchKernelGGL((route_combine_kernel<T, true, false>), grid, block, 0, s, a, c);
    } else {
        if (wave)
            hipLaunchKernelGGL((route_combine_kernel<T, false, true>), grid, block, 0, s, a, c);
        else
            hipLaunchKernelGGL((route_combine_kernel<T, false, false>), grid, block, 0, s, a, c);
    }
}

int launch_route_combine(int type, const MoveArgs& a, int num_cus, hipStream_t s)
{
    (void)num_cus;
    if (type == MRS_TYPE_F32)
        start_combine<float>(a, s);
    else if (type == MRS_TYPE_F16)
        start_combine<_Float16>(a, s);
    else
        start_combine<__bf16>(a, s);
    MRS_CHECK_LAUNCH("route_combine_kernel");
    return MRS_OK;
}

template <typename T>
static void start_combine_backward(const MoveArgs& a, hipStream_t s)
{
    const Cut c = cut_rows(a, sizeof(T), true, true);
    const dim3 grid(c.blocks + c.pad_blocks), block(kThreads);
    if (grid.x == 0) return;
    const auto go = [&](auto k) {
        constexpr uint32_t K = decltype(k)::value;
        if (c.lanes_log2 == 6)
            hipLaunchKernelGGL((route_combine_backward_kernel<T, K, true>), grid, block, 0, s, a, c);
        else
            hipLaunchKernelGGL((route_combine_backward_kernel<T, K, false>), grid, block, 0, s, a, c);
    };
    if (a.topk <= 2)
        go(std::integral_constant<uint32_t, 2>{});
    else if (a.topk <= 4)
        go(std::integral_constant<uint32_t, 4>{});
    else if (a.topk <= 8)
        go(std::integral_constant<uint32_t, 8>{});
    else if (a.topk <= 16)
        go(std::integral_constant<uint32_t, 16>{});
    else
        go(std::integral_constant<uint32_t, 32>{});
}

int launch_route_combine_backward(int type, const MoveArgs& a, int num_cus, hipStream_t s)
{
    (void)num_cus;
    if (type == MRS_TYPE_F32)
        start_combine_backward<float>(a, s);
    else if (type == MRS_TYPE_F16)
        start_combine_backward<_Float16>(a, s);
    else
        start_combine_backward<__bf16>(a, s);
    MRS_CHECK_LAUNCH("route_combine_backward_kernel");
    return MRS_OK;
}

}  // namespace mrs
