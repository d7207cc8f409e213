// Stable counting sort of token slots by expert (mrs_route_order in include/mrs.h).
//
// row(slot) = offset of its expert + how many earlier kept slots have the same expert.  A workgroup
// ranks `16 waves x 64 lanes x R` consecutive slots at a time: a wave takes 64 neighbouring slots, finds
// the lanes with the same expert by one ballot per bit of its number, and adds their count to its own
// counter of that expert, so that a slot's rank inside the wave's stretch is the counter before plus
// the equal lanes below; a scan over the waves' counters gives the rank inside the tile.  No
// atomics decide an order, so rows are the same every time.
//
// Up to kSmallSlots slots one workgroup does everything (512 slots, 256 experts: 4.0 us); what bounds it is the launch and
// the chain of LDS accesses and barriers.  Up to kDirectSlots one launch of several workgroups, a slot a thread, each of
// which counts all slots by itself (4096 slots 5.3 us, 16384 6.3, 32768 8.0, where two launches take 7.3, 7.9 and 7.9;
// one workgroup alone 7.3 for 4096).  Above, a first launch counts tiles of 1, 2 or 4 slots a thread, and in a second one
// every workgroup adds up the counts of the tiles before its own by itself (read from L2) instead of waiting for a scan
// launch between the two (65536 slots 7.9 us, with four slots a thread 11.0).  2^20 slots: 16.7 us, 4 of them for the counts,
// about 3 each for adding them up and for the writes to slot_of_row in runs of some 16 rows.
#include <algorithm>

#include "mrs_route.hpp"

namespace mrs {

namespace {

constexpr uint32_t kWaves = 16;
constexpr uint32_t kThreads = kWaves * 64;
constexpr uint32_t kMaxExperts = MRS_ROUTE_MAX_EXPERTS;
static_assert(kMaxExperts <= kThreads, "one thread per expert in the scans");
constexpr uint32_t kSmallSlots = kThreads;
constexpr uint32_t kDirectSlots = 24576;

struct OrderShared {
    alignas(4) uint16_t wave_count[kWaves][kMaxExperts];  // slots per wave, then those of the waves before
    uint32_t row[kMaxExperts];                            // first row of the expert in this tile
    uint32_t room[kMaxExperts];                           // rows it may still take
    uint32_t fill[kMaxExperts];                           // first row of its segment without a slot
    uint32_t fill_end[kMaxExperts];
    uint32_t wave_sum[kWaves];
};

// Lanes of the wave that hold the same value; `bits` significant bits.
__device__ __forceinline__ uint64_t same_value(uint32_t v, uint32_t bits)
{
    uint64_t same = ~0ull;
    for (uint32_t b = 0; b < bits; ++b) {
        const bool set = (v >> b) & 1u;
        const uint64_t with = __ballot(set);
        same &= set ? with : ~with;
    }
    return same;
}

// Exclusive scan of one value per thread over the workgroup; *total is the sum of all.
__device__ __forceinline__ uint32_t block_exclusive_scan(uint32_t v, uint32_t* wave_sum, uint32_t* total)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t incl = v;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(incl, d);
        if (lane >= d) incl += up;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    uint32_t before = 0, sum = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        const uint32_t x = wave_sum[w];
        if (w < wave) before += x;
        sum += x;
    }
    *total = sum;
    return before + incl - v;
}

__device__ __forceinline__ uint32_t round_up_to(uint32_t v, uint32_t a) { return (v + a - 1) / a * a; }

// The experts of a tile's slots, `experts` where a slot has none.  A wave takes 64 * R neighbouring slots.
template <uint32_t R>
__device__ __forceinline__ void load_experts(const OrderArgs& a, uint64_t first, uint32_t (&expert)[R])
{
    const uint64_t mine = first + (threadIdx.x >> 6) * (64u * R) + (threadIdx.x & 63u);
#pragma unroll
    for (uint32_t i = 0; i < R; ++i) {
        const uint64_t slot = mine + i * 64u;
        expert[i] = slot < a.slots ? static_cast<uint32_t>(a.ids[slot]) : a.experts;
    }
#pragma unroll
    for (uint32_t i = 0; i < R; ++i)
        if (expert[i] > a.experts) expert[i] = a.experts;
}

// Ranks slots inside their wave's stretch, and leaves its counts in the wave's row of counters.  Only the wave itself
// touches that row, and its LDS accesses stay in order: no barrier here.
template <uint32_t R>
__device__ __forceinline__ void rank_in_waves(const OrderArgs& a, OrderShared& sh, uint32_t bits, const uint32_t (&expert)[R],
                                              uint32_t (&rank)[R])
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t* words = reinterpret_cast<uint32_t*>(sh.wave_count[wave]);
    for (uint32_t w = lane; w < (a.experts + 1) / 2; w += 64) words[w] = 0;
    wave_lds_sync();
#pragma unroll
    for (uint32_t i = 0; i < R; ++i) {
        const uint64_t same = same_value(expert[i], bits);
        const uint32_t below = __popcll(same & ((1ull << lane) - 1ull));
        rank[i] = below;
        uint32_t before = 0;
        if (expert[i] < a.experts) before = sh.wave_count[wave][expert[i]];
        rank[i] += before;
        wave_lds_sync();
        if (expert[i] < a.experts && below == 0) sh.wave_count[wave][expert[i]] = static_cast<uint16_t>(before + __popcll(same));
        wave_lds_sync();
    }
}

// Turns thread e's column of counters into those of the waves before; returns the tile's sum.
__device__ __forceinline__ uint32_t scan_waves(OrderShared& sh, uint32_t e)
{
    uint32_t c[kWaves];
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) c[w] = sh.wave_count[w][e];
    uint32_t run = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        sh.wave_count[w][e] = static_cast<uint16_t>(run);
        run += c[w];
    }
    return run;
}

template <uint32_t R>
__device__ __forceinline__ void write_rows(const OrderArgs& a, const OrderShared& sh, uint64_t first,
                                           const uint32_t (&expert)[R], const uint32_t (&rank)[R])
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint64_t mine = first + wave * (64u * R) + lane;
#pragma unroll
    for (uint32_t i = 0; i < R; ++i) {
        const uint64_t slot = mine + i * 64u;
        if (slot >= a.slots) continue;
        int32_t row = -1;
        if (expert[i] < a.experts) {
            const uint32_t in_tile = sh.wave_count[wave][expert[i]] + rank[i];
            if (in_tile < sh.room[expert[i]]) {
                row = static_cast<int32_t>(sh.row[expert[i]] + in_tile);
                if (static_cast<uint32_t>(row) < a.rows) a.slot_of_row[row] = static_cast<int32_t>(slot);
            }
        }
        a.row_of_slot[slot] = row;
    }
}

// Rows without a slot: what fills the segments up, shared out by expert among `blocks` workgroups and inside one among
// groups of lanes as wide as a segment can need, and everything behind the last segment.
__device__ __forceinline__ void mark_empty_rows(const OrderArgs& a, const OrderShared& sh, uint32_t end, uint32_t block,
                                                uint32_t blocks)
{
    if (a.align > 1) {
        uint32_t lanes = 64;
        while (lanes > 1 && lanes / 2 >= a.align - 1) lanes /= 2;
        for (uint32_t e = block + threadIdx.x / lanes * blocks; e < a.experts; e += kThreads / lanes * blocks) {
            const uint32_t last = sh.fill_end[e] < a.rows ? sh.fill_end[e] : a.rows;
            for (uint32_t r = sh.fill[e] + threadIdx.x % lanes; r < last; r += lanes) a.slot_of_row[r] = -1;
        }
    }
    for (uint64_t r = static_cast<uint64_t>(end) + static_cast<uint64_t>(block) * kThreads + threadIdx.x; r < a.rows;
         r += static_cast<uint64_t>(blocks) * kThreads)
        a.slot_of_row[r] = -1;
}

// A slot a thread, all in one workgroup.
__global__ __launch_bounds__(kThreads) void route_order_small_kernel(const OrderArgs a, uint32_t bits)
{
    __shared__ OrderShared sh;
    const uint32_t tid = threadIdx.x;
    uint32_t expert[1], rank[1];
    load_experts<1>(a, 0, expert);
    rank_in_waves<1>(a, sh, bits, expert, rank);
    __syncthreads();
    uint32_t kept = 0;
    if (tid < a.experts) {
        kept = scan_waves(sh, tid);
        if (kept > a.capacity) kept = a.capacity;
    }
    const uint32_t padded = round_up_to(kept, a.align);
    uint32_t end;
    const uint32_t offset = block_exclusive_scan(padded, sh.wave_sum, &end);
    if (tid < a.experts) {
        sh.row[tid] = offset;
        sh.room[tid] = a.capacity;
        sh.fill[tid] = offset + kept;
        sh.fill_end[tid] = offset + padded;
        a.counts[tid] = static_cast<int32_t>(kept);
        a.offsets[tid] = static_cast<int32_t>(offset);
        if (tid == a.experts - 1) a.offsets[a.experts] = static_cast<int32_t>(end);
    }
    __syncthreads();
    write_rows<1>(a, sh, 0, expert, rank);
    mark_empty_rows(a, sh, end, 0, 1);
}

// tile_counts[block][e] = slots of expert e in the block's stretch of `per_block` slots
__global__ __launch_bounds__(kThreads) void route_order_count_kernel(const OrderArgs a, uint64_t per_block, uint32_t stride)
{
    __shared__ uint32_t count[kMaxExperts];
    const uint32_t tid = threadIdx.x;
    if (tid < a.experts) count[tid] = 0;
    __syncthreads();
    const uint64_t first = blockIdx.x * per_block;
    uint64_t last = first + per_block;
    if (last > a.slots) last = a.slots;
    for (uint64_t slot = first + tid; slot < last; slot += kThreads) {
        const uint32_t e = static_cast<uint32_t>(a.ids[slot]);
        if (e < a.experts) atomicAdd(&count[e], 1u);
    }
    __syncthreads();
    if (tid < a.experts) a.tile_counts[static_cast<uint64_t>(blockIdx.x) * stride + tid] = count[tid];
}

__device__ __forceinline__ void add_tile_counts(const OrderArgs& a, uint32_t stride, uint32_t* before_me, uint32_t* of_all)
{
    // The counts of all tiles, four experts a thread, the tiles shared out among groups of threads.  Every workgroup
    // begins with its own: all of them reading the same tile at a time took 3 us longer.  Four loads at a time; a thread
    // that has fewer tiles left reads one again.
    const uint32_t tid = threadIdx.x;
    const uint32_t quads = stride / 4;
    const uint32_t groups = kThreads / quads;
    const uint32_t group = tid / quads;
    if (group < groups) {
        const uint32_t e = (tid - group * quads) * 4;
        uint32_t before[4] = {0, 0, 0, 0}, all[4] = {0, 0, 0, 0};
        for (uint32_t i0 = group; i0 < gridDim.x; i0 += 4 * groups) {
            uint4 c[4];
            uint32_t t[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t i = i0 + k * groups;
                t[k] = (i < gridDim.x ? i : i0) + blockIdx.x;
                if (t[k] >= gridDim.x) t[k] -= gridDim.x;
                c[k] = *reinterpret_cast<const uint4*>(a.tile_counts + static_cast<uint64_t>(t[k]) * stride + e);
                if (i >= gridDim.x) c[k] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t mask = t[k] < blockIdx.x ? 0xFFFFFFFFu : 0u;
                all[0] += c[k].x, all[1] += c[k].y, all[2] += c[k].z, all[3] += c[k].w;
                before[0] += c[k].x & mask, before[1] += c[k].y & mask, before[2] += c[k].z & mask, before[3] += c[k].w & mask;
            }
        }
        // whole numbers: the order of these additions does not matter
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (e + i < a.experts) {
                atomicAdd(&of_all[e + i], all[i]);
                atomicAdd(&before_me[e + i], before[i]);
            }
    }
}

// DIRECT: a workgroup counts all slots itself, into kCopies counters an expert that neighbouring lanes use in turn (equal
// experts in one instruction wait for each other).  Otherwise the counts of tiles are there from
// route_order_count_kernel.
template <bool DIRECT, uint32_t R>
__global__ __launch_bounds__(kThreads) void route_order_kernel(const OrderArgs a, uint64_t per_block, uint32_t stride, uint32_t bits)
{
    constexpr uint32_t kCopies = DIRECT ? 4 : 1;
    __shared__ OrderShared sh;
    __shared__ uint32_t before_me[kMaxExperts * kCopies];
    __shared__ uint32_t of_all[kMaxExperts * kCopies];  // DIRECT: of this tile and those behind
    const uint32_t tid = threadIdx.x;
    const uint64_t first = blockIdx.x * per_block;
    uint64_t last = first + per_block;
    if (last > a.slots) last = a.slots;
    uint32_t expert[R], rank[R];
    load_experts<R>(a, first, expert);
    for (uint32_t i = tid; i < a.experts * kCopies; i += kThreads) {
        before_me[i] = 0;
        of_all[i] = 0;
    }
    rank_in_waves<R>(a, sh, bits, expert, rank);
    __syncthreads();
    if constexpr (DIRECT) {
        for (uint64_t at = 0; at < a.slots; at += 8 * kThreads) {
            uint32_t e[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint64_t slot = at + i * kThreads + tid;
                e[i] = slot < a.slots ? static_cast<uint32_t>(a.ids[slot]) : a.experts;
            }
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                uint32_t* count = at + i * kThreads < first ? before_me : of_all;
                if (e[i] < a.experts) atomicAdd(&count[e[i] * kCopies + tid % kCopies], 1u);
            }
        }
    } else {
        add_tile_counts(a, stride, before_me, of_all);
    }
    __syncthreads();
    uint32_t kept = 0, taken = 0, in_tile = 0;
    if (tid < a.experts) {
        in_tile = scan_waves(sh, tid);
#pragma unroll
        for (uint32_t i = 0; i < kCopies; ++i) {
            taken += before_me[tid * kCopies + i];
            kept += of_all[tid * kCopies + i];
        }
        if (DIRECT) kept += taken;
        if (kept > a.capacity) kept = a.capacity;
        if (taken > a.capacity) taken = a.capacity;
    }
    const uint32_t padded = round_up_to(kept, a.align);
    uint32_t end;
    const uint32_t offset = block_exclusive_scan(padded, sh.wave_sum, &end);
    if (tid < a.experts) {
        sh.row[tid] = offset + taken;
        sh.room[tid] = a.capacity - taken;
        sh.fill[tid] = offset + kept;
        sh.fill_end[tid] = offset + padded;
        if (blockIdx.x == 0) {
            a.counts[tid] = static_cast<int32_t>(kept);
            a.offsets[tid] = static_cast<int32_t>(offset);
            if (tid == a.experts - 1) a.offsets[a.experts] = static_cast<int32_t>(end);
        }
    }
    __syncthreads();
    for (uint64_t at = first;;) {
        write_rows<R>(a, sh, at, expert, rank);
        at += kThreads * R;
        if (at >= last) break;
        load_experts<R>(a, at, expert);
        __syncthreads();
        if (tid < a.experts) {
            const uint32_t room = sh.room[tid];
            const uint32_t took = in_tile < room ? in_tile : room;
            sh.row[tid] += took;
            sh.room[tid] = room - took;
        }
        rank_in_waves<R>(a, sh, bits, expert, rank);
        __syncthreads();
        if (tid < a.experts) in_tile = scan_waves(sh, tid);
        __syncthreads();
    }
    mark_empty_rows(a, sh, end, blockIdx.x, gridDim.x);
}

}  // namespace

int launch_route_order(const OrderArgs& a, hipStream_t s)
{
    uint32_t bits = 0;
    while ((a.experts >> bits) != 0) ++bits;  // the values 0 .. experts
    if (a.slots <= kSmallSlots) {
        hipLaunchKernelGGL(route_order_small_kernel, dim3(1), dim3(kThreads), 0, s, a, bits);
        MRS_CHECK_LAUNCH("route_order_small_kernel");
        return MRS_OK;
    }
    const uint32_t stride = (a.experts + 3) / 4 * 4;
    if (a.slots <= kDirectSlots) {
        const uint32_t blocks = (static_cast<uint32_t>(a.slots) + kThreads - 1) / kThreads;
        hipLaunchKernelGGL((route_order_kernel<true, 1>), dim3(blocks), dim3(kThreads), 0, s, a, static_cast<uint64_t>(kThreads), stride, bits);
        MRS_CHECK_LAUNCH("route_order_kernel");
        return MRS_OK;
    }
    // Small tiles are ranked sooner, but every workgroup reads the counts of all of them.  So threads take more slots, up to
    // four, before tiles are more than `most`: 2^16 counts in all or 64 tiles (2^18 slots, 1024 experts: 256 tiles
    // 20.7 us, 64 tiles 15.1).  From there on tiles do get more, up to kRouteMaxTiles: held at `most`, with several stretches
    // each, 2^19 slots of 1024 experts take 23.1 us and not 20.2, 2^20 39 and not 30, of 512 23.3 and not 21.6.
    const uint64_t most = std::max(64u, std::min(kRouteMaxTiles, 65536u / a.experts));
    const uint32_t r = a.slots <= most * kThreads ? 1 : a.slots <= most * kThreads * 2 ? 2 : 4;
    const uint64_t tile = static_cast<uint64_t>(kThreads) * r;
    const uint64_t per_block = ((a.slots + tile - 1) / tile + kRouteMaxTiles - 1) / kRouteMaxTiles * tile;
    const dim3 grid(static_cast<uint32_t>((a.slots + per_block - 1) / per_block)), block(kThreads);
    hipLaunchKernelGGL(route_order_count_kernel, grid, block, 0, s, a, per_block, stride);
    MRS_CHECK_LAUNCH("route_order_count_kernel");
    if (r == 1)
        hipLaunchKernelGGL((route_order_kernel<false, 1>), grid, block, 0, s, a, per_block, stride, bits);
    else if (r == 2)
        hipLaunchKernelGGL((route_order_kernel<false, 2>), grid, block, 0, s, a, per_block, stride, bits);
    else
        hipLaunchKernelGGL((route_order_kernel<false, 4>), grid, block, 0, s, a, per_block, stride, bits);
    MRS_CHECK_LAUNCH("route_order_kernel");
    return MRS_OK;
}

}  // namespace mrs
