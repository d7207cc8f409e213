// The topk largest of every row of scores, the weights they give, and the scores' gradient
// (mrs_route_select, mrs_route_select_backward in include/mrs.h).
//
// A row belongs to a group of L lanes, V columns a lane in runs of up to 16 bytes.  A key and its column travel together
// in the 52 mantissa bits of a double in [1, 2) -- the key mapped to an unsigned number of the same order in the upper
// 32, the complement of the column below -- so that one 64-bit maximum picks the larger key and, of equal keys, the
// lower column.  Every lane sorts its columns once by networks of such maxima and minima; a step then takes the largest head
// of the group's lists, found by exchanges inside a row of 16 lanes.
//
// The work is arithmetic, not memory: few lanes with many columns each make the steps, which run once for all rows of a
// wave, cheaper.  Up to eight slots a row has 8 lanes (to 256 experts), the lists keep eight entries and the steps
// are unrolled, each moving up only what later ones can reach.
#include "mrs_route.hpp"

namespace mrs {

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxBlocks = 1u << 20;
constexpr uint32_t kColumnMask = 0x3FFu;      // MRS_ROUTE_MAX_EXPERTS - 1
constexpr uint32_t kLowestKey = 0x007FFFFFu;  // what -infinity maps to; keys that take part are above
constexpr float kLog2E = 1.44269504088896340736f;
static_assert(MRS_ROUTE_MAX_EXPERTS <= kColumnMask + 1, "a column fits its bits");

// The order of floats as an order of unsigned numbers; what does not take part -- -infinity, NaN -- maps to kLowestKey.
__device__ __forceinline__ uint32_t ordered_key(float key)
{
    // + 0: -0 and +0 are equal keys
    const uint32_t u = __builtin_bit_cast(uint32_t, fmaxf(key + 0.0f, -__builtin_inff()));
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
// `rest` are the low bits: the complement of the column
__device__ __forceinline__ double pack(uint32_t ordered, uint32_t rest)
{
    const uint32_t low = ordered << 20 | rest, high = __builtin_amdgcn_alignbit(0x3FF, ordered, 12);
    return __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
}
__device__ __forceinline__ uint32_t packed_key(double p) { return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, p) >> 20); }
__device__ __forceinline__ uint32_t packed_column(double p)
{
    return kColumnMask - (static_cast<uint32_t>(__builtin_bit_cast(uint64_t, p)) & kColumnMask);
}
constexpr double kNothing = 1.0;  // below every key

// The other lane of a pair, for M = 1, 2, 4, ...: after the step for M, groups of 2 M lanes hold the same.
template <uint32_t M>
__device__ __forceinline__ uint32_t partner(uint32_t v)
{
    if constexpr (M < 16) {
        // quad_perm [1,0,3,2], quad_perm [2,3,0,1], row_half_mirror, row_mirror
        constexpr int kControl = M == 1 ? 0xB1 : M == 2 ? 0x4E : M == 4 ? 0x141 : 0x140;
        return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), kControl, 0xF, 0xF, true));
    } else if constexpr (M == 16) {
        return static_cast<uint32_t>(__builtin_amdgcn_ds_swizzle(static_cast<int>(v), 0x401F));  // lane ^ 16
    } else {
        return __shfl_xor(v, static_cast<int>(M));
    }
}
template <uint32_t M>
__device__ __forceinline__ float partner(float v)
{
    return __builtin_bit_cast(float, partner<M>(__builtin_bit_cast(uint32_t, v)));
}
template <uint32_t M>
__device__ __forceinline__ double partner(double v)
{
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint64_t low = partner<M>(static_cast<uint32_t>(bits)), high = partner<M>(static_cast<uint32_t>(bits >> 32));
    return __builtin_bit_cast(double, low | high << 32);
}
// Over a group of L lanes; all of them get the same, sums included (a pair adds the same two numbers).
template <uint32_t L, uint32_t M = 1>
__device__ __forceinline__ double max_of_group(double v)
{
    if constexpr (M == L)
        return v;
    else
        return max_of_group<L, 2 * M>(fmax(v, partner<M>(v)));
}
template <uint32_t L, uint32_t M = 1>
__device__ __forceinline__ float max_of_group(float v)
{
    if constexpr (M == L)
        return v;
    else
        return max_of_group<L, 2 * M>(fmaxf(v, partner<M>(v)));
}
template <uint32_t L, uint32_t M = 1>
__device__ __forceinline__ float sum_of_group(float v)
{
    if constexpr (M == L)
        return v;
    else
        return sum_of_group<L, 2 * M>(v + partner<M>(v));
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
    // column = run i / W of the lane, then the lane, then the element: three fields that do not meet
    __device__ static uint32_t column(uint32_t lane, uint32_t i) { return (i / W * L + lane) * W + i % W; }

    // -infinity behind the last column
    __device__ static void fetch(const T* row, uint32_t experts, uint32_t lane, Run (&runs)[V / W])
    {
#pragma unroll
        for (uint32_t c = 0; c < V / W; ++c) {
            const uint32_t e = (c * L + lane) * W;
            if (e + W <= experts) {
                runs[c] = *reinterpret_cast<const Run*>(row + e);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < W; ++i) runs[c].e[i] = e + i < experts ? row[e + i] : static_cast<T>(-__builtin_inff());
            }
        }
    }
    __device__ static void convert(const Run (&runs)[V / W], float (&s)[V])
    {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) s[i] = to_f32(runs[i / W].e[i % W]);
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
        if (!bias) {
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) key[i] = s[i];
            return;
        }
#pragma unroll
        for (uint32_t c = 0; c < V / W; ++c) {
            const uint32_t e = (c * L + lane) * W;
            struct __attribute__((packed, aligned(4))) Biases {
                float e[W];
            };
            if (e + W <= experts) {
                const Biases run = *reinterpret_cast<const Biases*>(bias + e);
#pragma unroll
                for (uint32_t i = 0; i < W; ++i) key[c * W + i] = s[c * W + i] + run.e[i];
            } else {
#pragma unroll
                for (uint32_t i = 0; i < W; ++i) key[c * W + i] = s[c * W + i] + (e + i < experts ? bias[e + i] : 0.0f);
            }
        }
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
    *m = max_of_group<L>(top);
    float total = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) total += __builtin_amdgcn_exp2f((s[i] - *m) * kLog2E);
    *sum = sum_of_group<L>(total);
}

__device__ __forceinline__ void exchange(double& a, double& b)
{
    const double high = fmax(a, b), low = fmin(a, b);
    a = high;
    b = low;
}
// Odd-even merge sort, largest first.
template <uint32_t N>
__device__ __forceinline__ void sort_list(double (&list)[N])
{
#pragma unroll
    for (uint32_t p = 1; p < N; p *= 2)
#pragma unroll
        for (uint32_t k = p; k >= 1; k /= 2)
#pragma unroll
            for (uint32_t j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (uint32_t i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) exchange(list[i + j], list[i + j + k]);
}
// The eight largest of two sorted lists of eight, sorted: one of each opposite pair, a bitonic sequence.
__device__ __forceinline__ void merge_largest(double (&list)[8], const double (&other)[8])
{
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) list[i] = fmax(list[i], other[7 - i]);
#pragma unroll
    for (uint32_t d = 4; d >= 1; d /= 2)
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if ((i & d) == 0) exchange(list[i], list[i + d]);
}

// Step J of the unrolled form: lane J keeps the largest head, and the list it came from moves up -- as far as the steps
// still to come can reach.
template <uint32_t L, uint32_t J>
__device__ __forceinline__ void take_largest(double (&list)[8], uint32_t topk, uint32_t lane, double* mine)
{
    if constexpr (J < 8) {
        if (J >= topk) return;
        const double top = max_of_group<L>(list[0]);
        if (lane == J) *mine = top;
        const bool taken = list[0] == top;
#pragma unroll
        for (uint32_t i = 0; i < 7 - J; ++i) list[i] = taken ? list[i + 1] : list[i];
        take_largest<L, J + 1>(list, topk, lane, mine);
    }
}

// WHOLE: the weights need a softmax over the whole row.  Four waves on a SIMD (the second bound) leave 128 registers each.
// 8 of 256 scores for 65536 tokens: 20 us, of 128 for 16384 tokens 5 us; about 1100 vector instructions for eight tokens, half
// of the time.  16 lanes a row and 16 columns a lane take 35 us; reading the next row ahead gains nothing.
template <typename T, uint32_t L, uint32_t V, bool FEW, bool WHOLE>
__global__ __launch_bounds__(kThreads, 4) void route_select_kernel(const T* __restrict__ scores, const float* __restrict__ bias,
                                                                   const SelectArgs a)
{
    using S = Share<T, L, V>;
    constexpr uint32_t kGroups = kThreads / L;
    const uint32_t lane = threadIdx.x & (L - 1);
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kGroups + threadIdx.x / L; t < a.tokens;
         t += static_cast<uint64_t>(gridDim.x) * kGroups) {
        const T* row = scores + t * a.ld_scores;
        typename S::Run runs[V / S::W];
        float s[V], key[V];
        S::fetch(row, a.experts, lane, runs);
        S::convert(runs, s);
        S::keys(bias, a.experts, lane, s, key);
        float m = 0.0f, sum = 1.0f;
        if constexpr (WHOLE) softmax_of_row<L, V>(s, key, &m, &sum);
        // A lane's columns share its own bits, which are left out until the lists of different lanes meet.
        const uint32_t lane_bits = S::column(lane, 0);
        double mine = kNothing;  // lane j keeps the j-th largest
        if constexpr (FEW) {
            double list[8];
#pragma unroll
            for (uint32_t c = 0; c < V; c += 8) {
                double part[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) part[i] = pack(ordered_key(key[c + i]), kColumnMask - S::column(0, c + i));
                sort_list<8>(part);
                if (c == 0) {
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) list[i] = part[i];
                } else {
                    merge_largest(list, part);
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                list[i] = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, list[i]) - lane_bits);
            take_largest<L, 0>(list, a.topk, lane, &mine);
        } else {
            double list[V];
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) list[i] = pack(ordered_key(key[i]), kColumnMask - S::column(0, i) - lane_bits);
            sort_list<V>(list);
            for (uint32_t j = 0; j < a.topk; ++j) {
                const double top = max_of_group<L>(list[0]);
                if (lane == j) mine = top;
                if (list[0] == top) {
#pragma unroll
                    for (uint32_t i = 0; i + 1 < V; ++i) list[i] = list[i + 1];
                    list[V - 1] = kNothing;
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
            const float top = max_of_group<L>(x);
            w = chosen ? expf(x - top) : 0.0f;
            w = w / sum_of_group<L>(w);
        } else if (WHOLE) {
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

// The gradient: 18.5 us for 65536 tokens, 8 of 256 scores.  It writes whole rows (64 MiB) and reads the chosen scores,
// which lie in most of a row's cache lines; 8 to 32 lanes a row take the same.  The slots' derivatives are worked out
// by the first lanes of the group and laid into a row in LDS, which is written out, less p[e] times their sum where the
// softmax runs over the whole row.
template <typename T, uint32_t L, uint32_t V, bool WHOLE>
__global__ __launch_bounds__(kThreads) void route_select_backward_kernel(const T* __restrict__ scores, const float* __restrict__ bias,
                                                                         T* __restrict__ scores_grad, const SelectArgs a)
{
    using S = Share<T, L, V>;
    constexpr uint32_t kGroups = kThreads / L;
    __shared__ float grads[kGroups][L * V];
    const uint32_t lane = threadIdx.x & (L - 1), group = threadIdx.x / L;
    for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kGroups + group; t < a.tokens;
         t += static_cast<uint64_t>(gridDim.x) * kGroups) {
        const T* row = scores + t * a.ld_scores;
        const bool used = lane < a.topk;
        const uint32_t id = used ? static_cast<uint32_t>(a.ids[t * a.topk + lane]) : 0xFFFFFFFFu;
        const float dw = used ? a.weights_grad[t * a.topk + lane] : 0.0f;
        float m = 0.0f, sum = 1.0f;
        float s[V];
        if constexpr (WHOLE) {
            float key[V];
            typename S::Run runs[V / S::W];
            S::fetch(row, a.experts, lane, runs);
            S::convert(runs, s);
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
            const float top = max_of_group<L>(x);
            float q = chosen ? expf(x - top) : 0.0f;
            q = q / sum_of_group<L>(q);
            const float mean = sum_of_group<L>(chosen ? q * g : 0.0f);
            d = q * (g - mean);
            if (a.gate == MRS_GATE_SIGMOID) d *= sigmoid(-score);
        } else if (WHOLE) {
            d = expf(score - m) / sum * g;
            all = sum_of_group<L>(chosen ? d : 0.0f);
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
        if constexpr (WHOLE) {
#pragma unroll
            for (uint32_t i = 0; i < V; ++i)
                if (s[i] > -__builtin_inff()) out[i] -= __builtin_amdgcn_exp2f((s[i] - m) * kLog2E) * share;
        }
        S::store(scores_grad + t * a.ld_scores_grad, a.experts, lane, out);
    }
}

template <uint32_t L>
dim3 grid_for(const SelectArgs& a)
{
    constexpr uint32_t kGroups = kThreads / L;
    const uint64_t blocks = (a.tokens + kGroups - 1) / kGroups;
    return dim3(blocks > kMaxBlocks ? kMaxBlocks : static_cast<uint32_t>(blocks));
}

template <typename T, uint32_t L, uint32_t V, bool FEW>
void start(const SelectArgs& a, hipStream_t s)
{
    const T* scores = static_cast<const T*>(a.scores);
    if (a.gate == MRS_GATE_SOFTMAX && !a.normalize)
        hipLaunchKernelGGL((route_select_kernel<T, L, V, FEW, true>), grid_for<L>(a), dim3(kThreads), 0, s, scores, a.bias, a);
    else
        hipLaunchKernelGGL((route_select_kernel<T, L, V, FEW, false>), grid_for<L>(a), dim3(kThreads), 0, s, scores, a.bias, a);
}

template <typename T, uint32_t L, uint32_t V>
void start_backward(const SelectArgs& a, hipStream_t s)
{
    const T* scores = static_cast<const T*>(a.scores);
    T* grad = static_cast<T*>(a.scores_grad);
    if (a.gate == MRS_GATE_SOFTMAX && !a.normalize)
        hipLaunchKernelGGL((route_select_backward_kernel<T, L, V, true>), grid_for<L>(a), dim3(kThreads), 0, s, scores, a.bias, grad, a);
    else
        hipLaunchKernelGGL((route_select_backward_kernel<T, L, V, false>), grid_for<L>(a), dim3(kThreads), 0, s, scores, a.bias, grad, a);
}

template <typename T>
void choose(const SelectArgs& a, hipStream_t s)
{
    if (a.topk <= 8) {
        if (a.experts <= 64)
            start<T, 8, 8, true>(a, s);
        else if (a.experts <= 128)
            start<T, 8, 16, true>(a, s);
        else if (a.experts <= 256)
            start<T, 8, 32, true>(a, s);
        else if (a.experts <= 512)
            start<T, 16, 32, true>(a, s);
        else
            start<T, 32, 32, true>(a, s);
    } else if (a.experts <= 256 && a.topk <= 16) {  // a lane for every slot
        if (a.experts <= 16)
            start<T, 16, 1, false>(a, s);
        else if (a.experts <= 64)
            start<T, 16, 4, false>(a, s);
        else if (a.experts <= 128)
            start<T, 16, 8, false>(a, s);
        else
            start<T, 16, 16, false>(a, s);
    } else if (a.experts <= 512) {
        start<T, 32, 16, false>(a, s);
    } else {
        start<T, 64, 16, false>(a, s);
    }
}

template <typename T>
void choose_backward(const SelectArgs& a, hipStream_t s)
{
    if (a.experts <= 256 && a.topk <= 16) {
        if (a.experts <= 64)
            start_backward<T, 16, 4>(a, s);
        else if (a.experts <= 128)
            start_backward<T, 16, 8>(a, s);
        else
            start_backward<T, 16, 16>(a, s);
    } else if (a.experts <= 512) {
        start_backward<T, 32, 16>(a, s);
    } else {
        start_backward<T, 64, 16>(a, s);
    }
}

}  // namespace

int launch_route_select(int type, const SelectArgs& a, hipStream_t s)
{
    if (type == MRS_TYPE_F32)
        choose<float>(a, s);
    else if (type == MRS_TYPE_F16)
        choose<_Float16>(a, s);
    else
        choose<__bf16>(a, s);
    MRS_CHECK_LAUNCH("route_select_kernel");
    return MRS_OK;
}

int launch_route_select_backward(int type, const SelectArgs& a, hipStream_t s)
{
    if (type == MRS_TYPE_F32)
        choose_backward<float>(a, s);
    else if (type == MRS_TYPE_F16)
        choose_backward<_Float16>(a, s);
    else
        choose_backward<__bf16>(a, s);
    MRS_CHECK_LAUNCH("route_select_backward_kernel");
    return MRS_OK;
}

}  // namespace mrs
