// The topk largest of every row of scores, the weights they give, and the scores' gradient
// (mrs_route_select, mrs_route_select_backward in include/mrs.h).
//
// A row belongs to a group of L lanes, V columns a lane in runs of up to 16 bytes.  A key and its column travel together
// in the 52 mantissa bits of a double in [1, 2) -- the key mapped to an unsigned number of the same order in the upper
// 32, the complement of the column below -- so that one 64-bit maximum picks the larger key and, of equal keys, the
// lower column.  Every lane sorts its V columns once by a network of such maxima and minima; a step then takes the largest head
// of the group's lists, found by rotations inside a row of 16 lanes.  For few slots the steps are unrolled, and only
// as much of a list is kept and moved up as later steps can ask for.
#include "mrs_route.hpp"

namespace mrs {

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxBlocks = 1u << 20;
constexpr uint32_t kColumnMask = 0x3FFu;      // MRS_ROUTE_MAX_EXPERTS - 1
constexpr uint32_t kLowestKey = 0x007FFFFFu;  // -infinity; keys that take part are above
constexpr float kLog2E = 1.44269504088896340736f;
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

// The value M lanes on: inside a row of 16 lanes by a rotation, which after steps of 8, 4, 2 and 1 has combined all of them like an
// exchange does; across rows by an exchange.
template <uint32_t M>
__device__ __forceinline__ uint32_t neighbour(uint32_t v)
{
    if constexpr (M < 16)
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x120 + M, 0xF, 0xF, false));  // row_ror
    else if constexpr (M == 16)
        return static_cast<uint32_t>(__builtin_amdgcn_ds_swizzle(static_cast<int>(v), 0x401F));  // lane ^ 16
    else
        return __shfl_xor(v, static_cast<int>(M));
}
template <uint32_t M>
__device__ __forceinline__ float neighbour(float v)
{
    return __builtin_bit_cast(float, neighbour<M>(__builtin_bit_cast(uint32_t, v)));
}
template <uint32_t M>
__device__ __forceinline__ double neighbour(double v)
{
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint64_t low = neighbour<M>(static_cast<uint32_t>(bits)), high = neighbour<M>(static_cast<uint32_t>(bits >> 32));
    return __builtin_bit_cast(double, low | high << 32);
}
template <uint32_t M>
__device__ __forceinline__ double max_of_group(double v)
{
    if constexpr (M == 0)
        return v;
    else
        return max_of_group<M / 2>(fmax(v, neighbour<M>(v)));
}
template <uint32_t M>
__device__ __forceinline__ float max_of_group(float v)
{
    if constexpr (M == 0)
        return v;
    else
        return max_of_group<M / 2>(fmaxf(v, neighbour<M>(v)));
}
// Every lane adds the same numbers, in an order of its own inside a row of 16; what matters is that it is fixed.  The first
// lane's sum is given to all.
template <uint32_t M>
__device__ __forceinline__ float add_group(float v)
{
    if constexpr (M == 0)
        return v;
    else
        return add_group<M / 2>(v + neighbour<M>(v));
}

// log(1 / (1 + exp(-s))), without overflow on either side
__device__ __forceinline__ float log_sigmoid(float s) { return fminf(s, 0.0f) - log1pf(expf(-fabsf(s))); }
__device__ __forceinline__ float sigmoid(float s)
{
    const float x = expf(-fabsf(s));
    return (s >= 0.0f ? 1.0f : x) / (1.0f + x);
}

// How a group of L lanes shares a row: V columns a lane, in runs of W.
template <typename T, uint32_t L, uint32_t V>
struct Share {
    static constexpr uint32_t W = V * sizeof(T) < 16 ? V : 16 / sizeof(T);
    static_assert(V % W == 0);
    struct __attribute__((packed, aligned(sizeof(T)))) Run {
        T e[W];
    };
    __device__ static uint32_t column(uint32_t lane, uint32_t i) { return (i / W * L + lane) * W + i % W; }

    // -infinity behind the last column
    __device__ static void load(const T* row, uint32_t experts, uint32_t lane, float (&s)[V])
    {
#pragma unroll
        for (uint32_t c = 0; c < V / W; ++c) {
            const uint32_t e = (c * L + lane) * W;
            if (e + W <= experts) {
                const Run run = *reinterpret_cast<const Run*>(row + e);
#pragma unroll
                for (uint32_t i = 0; i < W; ++i) s[c * W + i] = to_f32(run.e[i]);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < W; ++i) s[c * W + i] = e + i < experts ? to_f32(row[e + i]) : -__builtin_inff();
            }
        }
    }
    __device__ static void store(T* row, uint32_t experts, uint32_t lane, const float (&s)[V])
    {
#pragma unroll
        for (uint32_t c = 0; c < V / W; ++c) {
            const uint32_t e = (c * L + lane) * W;
            if (e + W <= experts) {
                Run run;
#pragma unroll
                for (uint32_t i = 0; i < W; ++i) run.e[i] = static_cast<T>(s[c * W + i]);
                *reinterpret_cast<Run*>(row + e) = run;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < W; ++i)
                    if (e + i < experts) row[e + i] = static_cast<T>(s[c * W + i]);
            }
        }
    }
    // the keys choices are made by
    __device__ static void keys(const float* __restrict__ bias, uint32_t experts, uint32_t lane, const float (&s)[V], float (&key)[V])
    {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) key[i] = s[i];
        if (!bias) return;
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) key[i] += bias[min(column(lane, i), experts - 1)];
    }
};

// Maximum m of the row's scores that take part and sum of exp(s - m); the others become -infinity, whose exponential is 0
// (a row of them: NaN that nobody reads).  exp(s - m) is 2^(s log2 e - m log2 e), off by 2 |s - m| + 2 roundings at most.
template <uint32_t L, uint32_t V>
__device__ __forceinline__ void softmax_of_row(float (&s)[V], const float (&key)[V], float* m, float* sum)
{
    float top = -__builtin_inff();
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) {
        if (!(key[i] > -__builtin_inff())) s[i] = -__builtin_inff();
        top = fmaxf(top, s[i]);
    }
    *m = max_of_group<L / 2>(top);
    float total = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) total += __builtin_amdgcn_exp2f((s[i] - *m) * kLog2E);
    *sum = __shfl(add_group<L / 2>(total), 0, static_cast<int>(L));
}

// Step J of the unrolled form: lane J keeps the largest head, and the list it came from moves up -- as far as the steps
// still to come can reach.
template <uint32_t L, uint32_t J, uint32_t D>
__device__ __forceinline__ void take_largest(double (&list)[D], uint32_t topk, uint32_t lane, double* mine)
{
    constexpr uint32_t kSteps = 8;
    if constexpr (J < kSteps) {
        if (J >= topk) return;
        const double top = max_of_group<L / 2>(list[0]);
        if (lane == J) *mine = top;
        const bool taken = list[0] == top;
        constexpr uint32_t kLeft = kSteps - 1 - J < D ? kSteps - 1 - J : D;
#pragma unroll
        for (uint32_t i = 0; i < kLeft; ++i) {
            if constexpr (D > 1)
                list[i] = taken ? (i + 1 < D ? list[i + 1 < D ? i + 1 : i] : 1.0) : list[i];
            else
                list[i] = taken ? 1.0 : list[i];
        }
        take_largest<L, J + 1, D>(list, topk, lane, mine);
    }
}

template <typename T, uint32_t L, uint32_t V, bool FEW>
__global__ __launch_bounds__(kThreads) void route_select_kernel(const T* __restrict__ scores, const float* __restrict__ bias,
                                                                const SelectArgs a)
{
    using S = Share<T, L, V>;
    constexpr uint32_t kGroups = kThreads / L;
    const uint32_t lane = threadIdx.x & (L - 1);
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kGroups + threadIdx.x / L; t < a.tokens;
         t += static_cast<uint64_t>(gridDim.x) * kGroups) {
        const T* row = scores + t * a.ld_scores;
        float s[V], key[V];
        S::load(row, a.experts, lane, s);
        S::keys(bias, a.experts, lane, s, key);
        double list[V];
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) list[i] = pack(ordered_key(key[i]), S::column(lane, i));
        float m = 0.0f, sum = 1.0f;
        if (a.gate == MRS_GATE_SOFTMAX && !a.normalize) softmax_of_row<L, V>(s, key, &m, &sum);
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
                            const double high = fmax(list[i + j], list[i + j + k]);
                            const double low = fmin(list[i + j], list[i + j + k]);
                            list[i + j] = high;
                            list[i + j + k] = low;
                        }
        double mine = 1.0;  // lane j keeps the j-th largest
        if constexpr (FEW) {
            constexpr uint32_t kDepth = V < 8 ? V : 8;
            double heads[kDepth];
#pragma unroll
            for (uint32_t i = 0; i < kDepth; ++i) heads[i] = list[i];
            take_largest<L, 0, kDepth>(heads, a.topk, lane, &mine);
        } else {
            for (uint32_t j = 0; j < a.topk; ++j) {
                const double top = max_of_group<L / 2>(list[0]);
                if (lane == j) mine = top;
                if (list[0] == top) {
#pragma unroll
                    for (uint32_t i = 0; i + 1 < V; ++i) list[i] = list[i + 1];
                    list[V - 1] = 1.0;
                }
            }
        }
        const bool used = lane < a.topk;
        const bool chosen = used && packed_key(mine) > kLowestKey;
        const uint32_t e = packed_column(mine);
        const float score = chosen ? to_f32(row[e]) : -__builtin_inff();
        float w;
        if (a.normalize) {
            // p[id] / sum of p over the slots, as a softmax over the slots of log p
            const float x = a.gate == MRS_GATE_SOFTMAX ? score : chosen ? log_sigmoid(score) : score;
            const float top = max_of_group<L / 2>(x);
            w = chosen ? expf(x - top) : 0.0f;
            w = w / __shfl(add_group<L / 2>(w), 0, static_cast<int>(L));
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

// The gradient.  The slots' derivatives are worked out by the first lanes of the group and laid into a row in LDS, which is written
// out, less p[e] times their sum where the softmax runs over the whole row.
template <typename T, uint32_t L, uint32_t V>
__global__ __launch_bounds__(kThreads) void route_select_backward_kernel(const T* __restrict__ scores, const float* __restrict__ bias,
                                                                         T* __restrict__ scores_grad, const SelectArgs a)
{
    using S = Share<T, L, V>;
    constexpr uint32_t kGroups = kThreads / L;
    __shared__ float grads[kGroups][L * V];
    const uint32_t lane = threadIdx.x & (L - 1), group = threadIdx.x / L;
    const bool whole_row = a.gate == MRS_GATE_SOFTMAX && !a.normalize;
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kGroups + group; t < a.tokens;
         t += static_cast<uint64_t>(gridDim.x) * kGroups) {
        const T* row = scores + t * a.ld_scores;
        const bool used = lane < a.topk;
        const uint32_t id = used ? static_cast<uint32_t>(a.ids[t * a.topk + lane]) : 0xFFFFFFFFu;
        const float dw = used ? a.weights_grad[t * a.topk + lane] : 0.0f;
        float m = 0.0f, sum = 1.0f;
        float s[V];
        if (whole_row) {
            float key[V];
            S::load(row, a.experts, lane, s);
            S::keys(bias, a.experts, lane, s, key);
            softmax_of_row<L, V>(s, key, &m, &sum);
        }
        float score = -__builtin_inff();
        bool chosen = id < a.experts;
        if (chosen) {
            score = to_f32(row[id]);
            chosen = (bias ? score + bias[id] : score) > -__builtin_inff();
        }
        const float g = chosen ? dw * a.scale : 0.0f;
        float d;
        float all = 0.0f;
        if (a.normalize) {
            const float x = !chosen ? -__builtin_inff() : a.gate == MRS_GATE_SOFTMAX ? score : log_sigmoid(score);
            const float top = max_of_group<L / 2>(x);
            float q = chosen ? expf(x - top) : 0.0f;
            q = q / __shfl(add_group<L / 2>(q), 0, static_cast<int>(L));
            const float mean = __shfl(add_group<L / 2>(chosen ? q * g : 0.0f), 0, static_cast<int>(L));
            d = q * (g - mean);
            if (a.gate == MRS_GATE_SIGMOID) d *= sigmoid(-score);
        } else if (a.gate == MRS_GATE_SOFTMAX) {
            d = expf(score - m) / sum * g;
            all = __shfl(add_group<L / 2>(chosen ? d : 0.0f), 0, static_cast<int>(L));
        } else {
            d = sigmoid(score) * sigmoid(-score) * g;
        }
        // ids that repeat show by a lane not finding its own mark; their slots are then added one after the other
        if (chosen) grads[group][id] = static_cast<float>(lane);
        wave_lds_sync();
        const bool repeated = chosen && grads[group][id] != static_cast<float>(lane);
        wave_lds_sync();
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) grads[group][i * L + lane] = 0.0f;
        wave_lds_sync();
        if (__ballot(repeated)) {
            for (uint32_t j = 0; j < a.topk; ++j) {
                if (lane == j && chosen) grads[group][id] = grads[group][id] + d;
                wave_lds_sync();
            }
        } else if (chosen) {
            grads[group][id] = d;
        }
        wave_lds_sync();
        const float share = all / sum;
        float out[V];
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) out[i] = grads[group][S::column(lane, i)];
        wave_lds_sync();
        if (whole_row) {
#pragma unroll
            for (uint32_t i = 0; i < V; ++i)
                if (s[i] > -__builtin_inff()) out[i] -= __builtin_amdgcn_exp2f((s[i] - m) * kLog2E) * share;
        }
        S::store(scores_grad + t * a.ld_scores_grad, a.experts, lane, out);
    }
}

template <typename T, uint32_t L, uint32_t V>
void start(const SelectArgs& a, bool backward, hipStream_t s)
{
    constexpr uint32_t kGroups = kThreads / L;
    uint64_t blocks = (a.tokens + kGroups - 1) / kGroups;
    if (blocks > kMaxBlocks) blocks = kMaxBlocks;
    const dim3 grid(static_cast<uint32_t>(blocks)), block(kThreads);
    const T* scores = static_cast<const T*>(a.scores);
    if (backward)
        hipLaunchKernelGGL((route_select_backward_kernel<T, L, V>), grid, block, 0, s, scores, a.bias, static_cast<T*>(a.scores_grad), a);
    else if (a.topk <= 8)
        hipLaunchKernelGGL((route_select_kernel<T, L, V, true>), grid, block, 0, s, scores, a.bias, a);
    else
        hipLaunchKernelGGL((route_select_kernel<T, L, V, false>), grid, block, 0, s, scores, a.bias, a);
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
