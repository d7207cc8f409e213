// The topk largest of every row of scores, the weights they give, and the scores' gradient
// (mrs_route_select, mrs_route_select_backward in include/mrs.h).
//
// A row belongs to a group of L lanes, V elements a lane.  A key and its column travel together in the
// 52 mantissa bits of a double in [1, 2) -- the key mapped to an unsigned number of the same order in
// the upper 32, the complement of the column below -- so that one 64-bit maximum picks the larger key and, of
// equal keys, the lower column.  Every lane sorts its V elements once; a step takes the largest
// head of the group's lists.
#include "mrs_route.hpp"

namespace mrs {

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxBlocks = 1u << 20;
constexpr uint32_t kColumnMask = 0x3FFu;  // MRS_ROUTE_MAX_EXPERTS - 1
constexpr uint32_t kLowestKey = 0x007FFFFFu;  // -infinity; keys that take part are above
static_assert(MRS_ROUTE_MAX_EXPERTS <= kColumnMask + 1, "a column fits its bits");

// The order of floats as an order of unsigned numbers; 0 for what does not take part.
__device__ __forceinline__ uint32_t ordered_key(float key)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, key + 0.0f);  // -0 and +0 are equal keys
    const uint32_t o = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
    return key > -__builtin_inff() ? o : 0u;
}
__device__ __forceinline__ double pack(uint32_t ordered, uint32_t column)
{
    const uint64_t bits = 0x3FF0000000000000ull | (static_cast<uint64_t>(ordered) << 20) | (kColumnMask - column);
    return __builtin_bit_cast(double, bits);
}
__device__ __forceinline__ uint32_t packed_key(double p) { return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, p) >> 20); }
__device__ __forceinline__ uint32_t packed_column(double p)
{
    return kColumnMask - (static_cast<uint32_t>(__builtin_bit_cast(uint64_t, p)) & kColumnMask);
}

template <uint32_t L>
__device__ __forceinline__ double group_max(double v)
{
#pragma unroll
    for (uint32_t m = L / 2; m > 0; m /= 2) v = fmax(v, __shfl_xor(v, static_cast<int>(m), static_cast<int>(L)));
    return v;
}
template <uint32_t L>
__device__ __forceinline__ float group_max(float v)
{
#pragma unroll
    for (uint32_t m = L / 2; m > 0; m /= 2) v = fmaxf(v, __shfl_xor(v, static_cast<int>(m), static_cast<int>(L)));
    return v;
}
template <uint32_t L>
__device__ __forceinline__ float group_sum(float v)
{
#pragma unroll
    for (uint32_t m = L / 2; m > 0; m /= 2) v += __shfl_xor(v, static_cast<int>(m), static_cast<int>(L));
    return v;
}

// log(1 / (1 + exp(-s))), without overflow on either side
__device__ __forceinline__ float log_sigmoid(float s) { return fminf(s, 0.0f) - log1pf(expf(-fabsf(s))); }
__device__ __forceinline__ float sigmoid(float s)
{
    const float x = expf(-fabsf(s));
    return (s >= 0.0f ? 1.0f : x) / (1.0f + x);
}

// Maximum and sum of exponentials of the row's scores that take part.  NaN if one is +infinity.
template <typename T, uint32_t L, uint32_t V>
__device__ __forceinline__ void softmax_of_row(const float (&s)[V], const bool (&part)[V], float* m, float* sum)
{
    float top = -__builtin_inff();
#pragma unroll
    for (uint32_t i = 0; i < V; ++i)
        if (part[i]) top = fmaxf(top, s[i]);
    *m = group_max<L>(top);
    float total = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i)
        if (part[i]) total += expf(s[i] - *m);
    *sum = group_sum<L>(total);
}

// The row's scores, and which of them take part.  Lane l holds the columns i * L + l.
template <typename T, uint32_t L, uint32_t V>
__device__ __forceinline__ void load_row(const SelectArgs& a, uint64_t t, uint32_t lane, float (&s)[V], float (&key)[V])
{
    const T* row = static_cast<const T*>(a.scores) + t * a.ld_scores;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) {
        const uint32_t e = i * L + lane;
        s[i] = -__builtin_inff();
        key[i] = -__builtin_inff();
        if (e < a.experts) {
            s[i] = to_f32(row[e]);
            key[i] = a.bias ? s[i] + a.bias[e] : s[i];
        }
    }
}

template <typename T, uint32_t L, uint32_t V>
__global__ __launch_bounds__(kThreads) void route_select_kernel(const SelectArgs a)
{
    constexpr uint32_t kGroups = kThreads / L;
    const uint32_t lane = threadIdx.x & (L - 1);
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kGroups + threadIdx.x / L; t < a.tokens;
         t += static_cast<uint64_t>(gridDim.x) * kGroups) {
        float s[V], key[V];
        load_row<T, L, V>(a, t, lane, s, key);
        float m = 0.0f, sum = 1.0f;
        if (a.gate == MRS_GATE_SOFTMAX && !a.normalize) {
            bool part[V];
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) part[i] = key[i] > -__builtin_inff();
            softmax_of_row<T, L, V>(s, part, &m, &sum);
        }
        double list[V];
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) list[i] = pack(ordered_key(key[i]), i * L + lane);
        // odd-even merge sort, largest first
#pragma unroll
        for (uint32_t p = 1; p < V; p *= 2)
#pragma unroll
            for (uint32_t k = p; k >= 1; k /= 2)
#pragma unroll
                for (uint32_t j = k % p; j + k < V; j += 2 * k)
#pragma unroll
                    for (uint32_t i = 0; i < k; ++i)
                        if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                            const double hi = fmax(list[i + j], list[i + j + k]);
                            const double lo = fmin(list[i + j], list[i + j + k]);
                            list[i + j] = hi;
                            list[i + j + k] = lo;
                        }
        double mine = 1.0;  // lane j keeps the j-th largest
        for (uint32_t j = 0; j < a.topk; ++j) {
            const double top = group_max<L>(list[0]);
            if (lane == j) mine = top;
            if (list[0] == top) {
#pragma unroll
                for (uint32_t i = 0; i + 1 < V; ++i) list[i] = list[i + 1];
                list[V - 1] = 1.0;
            }
        }
        const bool used = lane < a.topk;
        const bool chosen = used && packed_key(mine) > kLowestKey;
        const uint32_t e = packed_column(mine);
        float w = 0.0f;
        const float score = chosen ? to_f32(static_cast<const T*>(a.scores)[t * a.ld_scores + e]) : -__builtin_inff();
        if (a.normalize) {
            // p[id] / sum of p over the slots, as a softmax over the slots of log p
            const float x = a.gate == MRS_GATE_SOFTMAX ? score : chosen ? log_sigmoid(score) : score;
            const float top = group_max<L>(x);
            w = chosen ? expf(x - top) : 0.0f;
            w = w / group_sum<L>(w);
        } else if (a.gate == MRS_GATE_SOFTMAX) {
            w = expf(score - m) / sum;
        } else {
            w = sigmoid(score);
        }
        if (used) {
            a.ids_out[t * a.topk + lane] = chosen ? static_cast<int32_t>(e) : -1;
            a.weights_out[t * a.topk + lane] = chosen ? w * a.scale : 0.0f;
        }
    }
}

// The gradient: the slots' derivatives are worked out by the first lanes of the group, laid into a row in LDS and
// written out with the rest of the row.
template <typename T, uint32_t L, uint32_t V>
__global__ __launch_bounds__(kThreads) void route_select_backward_kernel(const SelectArgs a)
{
    constexpr uint32_t kGroups = kThreads / L;
    __shared__ float grads[kGroups][L * V];
    const uint32_t lane = threadIdx.x & (L - 1);
    volatile float* grad = grads[threadIdx.x / L];
    const bool whole_row = a.gate == MRS_GATE_SOFTMAX && !a.normalize;
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kGroups + threadIdx.x / L; t < a.tokens;
         t += static_cast<uint64_t>(gridDim.x) * kGroups) {
        float s[V], key[V];
        float m = 0.0f, sum = 1.0f;
        bool part[V];
        if (whole_row) {
            load_row<T, L, V>(a, t, lane, s, key);
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) part[i] = key[i] > -__builtin_inff();
            softmax_of_row<T, L, V>(s, part, &m, &sum);
        }
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) grad[i * L + lane] = 0.0f;
        const bool used = lane < a.topk;
        const uint32_t id = used ? static_cast<uint32_t>(a.ids[t * a.topk + lane]) : 0xFFFFFFFFu;
        float score = -__builtin_inff();
        bool chosen = id < a.experts;
        if (chosen) {
            score = to_f32(static_cast<const T*>(a.scores)[t * a.ld_scores + id]);
            chosen = (a.bias ? score + a.bias[id] : score) > -__builtin_inff();
        }
        const float g = chosen ? a.weights_grad[t * a.topk + lane] * a.scale : 0.0f;
        float d;
        float all = 0.0f;
        if (a.normalize) {
            const float x = !chosen ? -__builtin_inff() : a.gate == MRS_GATE_SOFTMAX ? score : log_sigmoid(score);
            const float top = group_max<L>(x);
            float q = chosen ? expf(x - top) : 0.0f;
            q = q / group_sum<L>(q);
            const float mean = group_sum<L>(chosen ? q * g : 0.0f);
            d = q * (g - mean);
            if (a.gate == MRS_GATE_SIGMOID) d *= sigmoid(-score);
        } else if (a.gate == MRS_GATE_SOFTMAX) {
            d = expf(score - m) / sum * g;
            all = group_sum<L>(chosen ? d : 0.0f);
        } else {
            d = sigmoid(score) * sigmoid(-score) * g;
        }
        // a repeated id: all its slots hold the sum, added in the order of the slots
        float total = 0.0f;
        for (uint32_t j = 0; j < a.topk; ++j) {
            const uint32_t other = __shfl(id, static_cast<int>(j), static_cast<int>(L));
            const float x = __shfl(d, static_cast<int>(j), static_cast<int>(L));
            if (other == id) total += x;
        }
        if (chosen) grad[id] = total;
        T* out = static_cast<T*>(a.scores_grad) + t * a.ld_scores_grad;
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) {
            const uint32_t e = i * L + lane;
            if (e >= a.experts) continue;
            float x = grad[e];
            if (whole_row && part[i]) x -= expf(s[i] - m) / sum * all;
            out[e] = static_cast<T>(x);
        }
    }
}

template <typename T, uint32_t L, uint32_t V>
void start(const SelectArgs& a, bool backward, hipStream_t s)
{
    constexpr uint32_t kGroups = kThreads / L;
    uint64_t blocks = (a.tokens + kGroups - 1) / kGroups;
    if (blocks > kMaxBlocks) blocks = kMaxBlocks;
    const dim3 grid(static_cast<uint32_t>(blocks)), block(kThreads);
    if (backward)
        hipLaunchKernelGGL((route_select_backward_kernel<T, L, V>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((route_select_kernel<T, L, V>), grid, block, 0, s, a);
}

// Lanes of a row: 16, more where topk (a slot per lane at the end) or 16 columns a lane ask for it.
template <typename T>
void choose(const SelectArgs& a, bool backward, hipStream_t s)
{
    if (a.experts <= 256 && a.topk <= 16) {
        if (a.experts <= 16)
            start<T, 16, 1>(a, backward, s);
        else if (a.experts <= 64)
            start<T, 16, 4>(a, backward, s);
        else if (a.experts <= 128)
            start<T, 16, 8>(a, backward, s);
        else
            start<T, 16, 16>(a, backward, s);
    } else if (a.experts <= 128) {
        start<T, 32, 4>(a, backward, s);
    } else if (a.experts <= 512) {
        start<T, 32, 16>(a, backward, s);
    } else {
        start<T, 64, 16>(a, backward, s);
    }
}

int launch(int type, const SelectArgs& a, bool backward, hipStream_t s)
{
    if (a.tokens == 0) return MRS_OK;
    if (type == MRS_TYPE_F32)
        choose<float>(a, backward, s);
    else if (type == MRS_TYPE_F16)
        choose<_Float16>(a, backward, s);
    else
        choose<__bf16>(a, backward, s);
    MRS_CHECK_LAUNCH(backward ? "route_select_backward_kernel" : "route_select_kernel");
    return MRS_OK;
}

}  // namespace

int launch_route_select(int type, const SelectArgs& a, int, hipStream_t s) { return launch(type, a, false, s); }
int launch_route_select_backward(int type, const SelectArgs& a, int, hipStream_t s) { return launch(type, a, true, s); }

}  // namespace mrs
