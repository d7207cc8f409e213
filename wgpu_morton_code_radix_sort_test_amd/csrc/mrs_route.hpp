// Shared by the translation units of token routing (mrs_route*.hip): rows ordered by a small integer
// key and back.  The definitions are in include/mrs.h.
#ifndef MRS_ROUTE_HPP
#define MRS_ROUTE_HPP

#include "mrs_internal.h"

struct mrs_route {
    mrs_context* ctx;
    mrs_route_desc desc;
    uint32_t* tile_counts;  // [kRouteMaxTiles][experts]: what every workgroup of an ordering counted
};

namespace mrs {

constexpr uint32_t kRouteMaxTiles = 256;  // workgroups of a large ordering: one per compute unit

struct SelectArgs {
    const void* scores;
    uint64_t ld_scores;
    const float* bias;  // may be null
    uint64_t tokens;
    uint32_t experts;
    uint32_t topk;
    int32_t gate;
    int32_t normalize;
    float scale;
    // forward
    int32_t* ids_out;
    float* weights_out;
    // backward
    const int32_t* ids;
    const float* weights_grad;
    void* scores_grad;
    uint64_t ld_scores_grad;
};

struct OrderArgs {
    const int32_t* ids;
    uint64_t slots;
    uint32_t experts;
    uint32_t align;
    uint32_t capacity;  // 0xFFFFFFFF: no limit
    int32_t* row_of_slot;
    int32_t* slot_of_row;
    int32_t* counts;
    int32_t* offsets;
    uint32_t rows;
    uint32_t* tile_counts;
};

// One side of a move between tokens and rows.  Strides and lengths in elements of the type.
struct MoveArgs {
    uint64_t tokens;
    uint32_t topk;
    uint32_t rows;
    uint32_t hidden;
    const int32_t* row_of_slot;
    // segments, for the rows that only fill them up: null when align is 1
    const int32_t* counts;
    const int32_t* offsets;
    uint32_t experts;
    uint32_t align;
    const void* token_in;  // x, out_grad
    uint64_t ld_token_in;
    const void* rows_in;  // rows, rows_grad
    uint64_t ld_rows_in;
    void* token_out;  // out, x_grad
    uint64_t ld_token_out;
    void* rows_out;  // rows, rows_grad
    uint64_t ld_rows_out;
    const float* weights;
    float* weights_grad;
};

int launch_route_select(int type, const SelectArgs& a, hipStream_t s);
int launch_route_select_backward(int type, const SelectArgs& a, hipStream_t s);
int launch_route_order(const OrderArgs& a, hipStream_t s);
int launch_route_dispatch(int element_bytes, const MoveArgs& a, hipStream_t s);
int launch_route_combine(int type, const MoveArgs& a, hipStream_t s);  // weights null: all 1
int launch_route_combine_backward(int type, const MoveArgs& a, hipStream_t s);

// ---- device side ------------------------------------------------------------------------------

typedef uint32_t RouteVec __attribute__((ext_vector_type(4)));
// 16 bytes at the alignment of an element: gfx950 takes such loads and stores as they are
typedef RouteVec RouteVecLoose __attribute__((aligned(1)));

__device__ __forceinline__ RouteVec load_vec(const void* p) { return *static_cast<const RouteVecLoose*>(p); }
__device__ __forceinline__ void store_vec(void* p, RouteVec v) { *static_cast<RouteVecLoose*>(p) = v; }

// LDS written by some lanes of a wave is read by others: the accesses stay in order on the device, and this keeps the
// compiler from moving them across.
__device__ __forceinline__ void wave_lds_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Conversions; to fewer bits round to nearest even.
template <typename T>
__device__ __forceinline__ float to_f32(T v)
{
    return static_cast<float>(v);
}

template <typename T>
struct RouteElems {
    static constexpr int N = 16 / static_cast<int>(sizeof(T));
    T e[N];
};

template <typename T>
__device__ __forceinline__ RouteElems<T> as_elems(RouteVec v)
{
    return __builtin_bit_cast(RouteElems<T>, v);
}
template <typename T>
__device__ __forceinline__ RouteVec as_vec(const RouteElems<T>& e)
{
    return __builtin_bit_cast(RouteVec, e);
}

}  // namespace mrs

#endif
