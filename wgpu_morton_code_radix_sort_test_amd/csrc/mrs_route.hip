// C ABI of token routing: argument checks and launches (mrs_route_* in include/mrs.h).
#include "mrs_route.hpp"

#include <cmath>
#include <new>

using namespace mrs;

namespace {

constexpr uint64_t kMaxRows = 0x7FFFFFFFull;       // row numbers are int32
constexpr uint64_t kMaxHidden = 1ull << 24;        // column arithmetic in 32 bits
constexpr uint64_t kMaxStride = 1ull << 40;        // stride * bytes of an element: 64-bit arithmetic has room
constexpr uint64_t kMaxBytes = 1ull << 56;         // from a matrix's first byte to its last: so have row * stride and addresses

int element_bytes(int32_t type) { return type == MRS_TYPE_F32 ? 4 : type == MRS_TYPE_8BIT ? 1 : 2; }

uint64_t max_rows_of(const mrs_route_desc& d, uint64_t tokens)
{
    const uint64_t n = tokens * static_cast<uint64_t>(d.topk);
    const uint64_t experts = static_cast<uint64_t>(d.experts), align = static_cast<uint64_t>(d.align);
    const uint64_t rows = n + (n < experts ? n : experts) * (align - 1);
    // Both bounds hold for any n and neither falls as n grows, so nor does their minimum: buffers for `tokens` tokens hold
    // fewer as well.  A capacity of 2^31 limits nothing and would overflow the product.
    if (d.capacity == 0 || d.capacity > kMaxRows) return rows;
    const uint64_t limited = experts * ((d.capacity + align - 1) / align * align);
    return limited < rows ? limited : rows;
}

int check_desc(const mrs_route_desc* d, const char* who)
{
    if (d->experts < 1 || d->experts > MRS_ROUTE_MAX_EXPERTS)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: experts = %d is not in [1, %d]", who, d->experts, MRS_ROUTE_MAX_EXPERTS);
    if (d->topk < 1 || d->topk > MRS_ROUTE_MAX_TOPK)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: topk = %d is not in [1, %d]", who, d->topk, MRS_ROUTE_MAX_TOPK);
    if (d->align < 1 || d->align > 1024) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: align = %d is not in [1, 1024]", who, d->align);
    if (d->gate != MRS_GATE_SOFTMAX && d->gate != MRS_GATE_SIGMOID)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: unknown gate %d", who, d->gate);
    if (d->normalize != 0 && d->normalize != 1) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: normalize must be 0 or 1", who);
    if (!std::isfinite(d->scale)) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: scale is not finite", who);
    if (d->tokens > kMaxRows ||
        d->tokens * static_cast<uint64_t>(d->topk) + static_cast<uint64_t>(d->experts) * static_cast<uint64_t>(d->align) > kMaxRows)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: tokens * topk + experts * align must stay below 2^31", who);
    return MRS_OK;
}

int check_call(const mrs_route* r, uint64_t tokens, const char* who)
{
    if (!r) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: null handle", who);
    if (tokens > r->desc.tokens)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %llu tokens exceed the handle's %llu", who, (unsigned long long)tokens,
                    (unsigned long long)r->desc.tokens);
    return check_device(r->ctx, who);
}

bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// A matrix of `rows` rows of `columns` elements, `stride` elements apart.
struct Matrix {
    const void* p;
    uint64_t rows, columns, stride;
    int bytes;  // of an element
};

int check_matrix(const Matrix& m, const char* who, const char* name)
{
    if (m.rows == 0) return MRS_OK;
    if (!m.p) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %s is null", who, name);
    if (!aligned_to(m.p, m.bytes)) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %s is not aligned to its elements", who, name);
    if (m.stride < m.columns || m.stride > kMaxStride)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: the rows of %s are %llu elements long but %llu apart", who, name,
                    (unsigned long long)m.columns, (unsigned long long)m.stride);
    if (m.rows > 1 && m.stride > (kMaxBytes / m.bytes - m.columns) / (m.rows - 1))
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %s reaches over more than 2^56 bytes: %llu rows, %llu elements apart", who, name,
                    (unsigned long long)m.rows, (unsigned long long)m.stride);
    return MRS_OK;
}

// Whether two matrices share an element.  Column blocks of one buffer (same stride, disjoint columns) do not.
bool overlap(const Matrix& a, const Matrix& b)
{
    if (!a.p || !b.p || a.rows == 0 || b.rows == 0 || a.columns == 0 || b.columns == 0) return false;
    const uint64_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    const uint64_t ea = pa + ((a.rows - 1) * a.stride + a.columns) * a.bytes;
    const uint64_t eb = pb + ((b.rows - 1) * b.stride + b.columns) * b.bytes;
    if (ea <= pb || eb <= pa) return false;
    const uint64_t pitch = a.stride * a.bytes;
    if (pitch != b.stride * b.bytes) return true;
    const uint64_t shift = pa <= pb ? (pb - pa) % pitch : pitch - 1 - (pa - pb - 1) % pitch;  // of b's columns behind a's
    return shift < a.columns * a.bytes || shift + b.columns * b.bytes > pitch;
}

// An array without rows of its own.
Matrix flat(const void* p, uint64_t count) { return {p, 1, count, count, 4}; }

// No output may share memory with an input or another output.
struct Named {
    Matrix m;
    const char* name;
};
template <size_t OUT, size_t IN>
int check_outputs(const Named (&out)[OUT], const Named (&in)[IN], const char* who)
{
    for (size_t i = 0; i < OUT; ++i) {
        for (size_t j = 0; j < IN; ++j)
            if (overlap(out[i].m, in[j].m)) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %s and %s overlap", who, out[i].name, in[j].name);
        for (size_t j = i + 1; j < OUT; ++j)
            if (overlap(out[i].m, out[j].m)) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %s and %s overlap", who, out[i].name, out[j].name);
    }
    return MRS_OK;
}

int check_ints(const void* p, const char* who, const char* name)
{
    if (!p) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %s is null", who, name);
    if (!aligned_to(p, 4)) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %s is not aligned to its elements", who, name);
    return MRS_OK;
}

// What a move reads of the map.
int check_map(const mrs_route* r, uint64_t tokens, const mrs_route_map* m, bool segments, const char* who)
{
    if (!m) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: null map", who);
    if (m->rows > kMaxRows) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: more than 2^31 - 1 rows", who);
    if (tokens == 0) return MRS_OK;
    if (int rc = check_ints(m->row_of_slot, who, "row_of_slot")) return rc;
    if (segments && r->desc.align > 1) {
        if (int rc = check_ints(m->counts, who, "counts")) return rc;
        if (int rc = check_ints(m->offsets, who, "offsets")) return rc;
    }
    return MRS_OK;
}

int check_type(int32_t type, bool eight_bits, const char* who)
{
    if (type == MRS_TYPE_F32 || type == MRS_TYPE_F16 || type == MRS_TYPE_BF16 || (eight_bits && type == MRS_TYPE_8BIT)) return MRS_OK;
    return fail(MRS_ERR_INVALID_ARGUMENT, "%s: unsupported element type %d", who, type);
}

int check_hidden(uint64_t hidden, const char* who)
{
    if (hidden < 1 || hidden > kMaxHidden)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: hidden = %llu is not in [1, 2^24]", who, (unsigned long long)hidden);
    return MRS_OK;
}

MoveArgs move_args(const mrs_route* r, uint64_t tokens, const mrs_route_map* m, uint64_t hidden)
{
    MoveArgs a{};
    a.tokens = tokens;
    a.topk = static_cast<uint32_t>(r->desc.topk);
    a.rows = static_cast<uint32_t>(m->rows);
    a.hidden = static_cast<uint32_t>(hidden);
    a.row_of_slot = m->row_of_slot;
    a.counts = m->counts;
    a.offsets = m->offsets;
    a.experts = static_cast<uint32_t>(r->desc.experts);
    a.align = static_cast<uint32_t>(r->desc.align);
    return a;
}

SelectArgs select_args(const mrs_route* r, uint64_t tokens, const void* scores, uint64_t ld, const float* bias)
{
    SelectArgs a{};
    a.scores = scores;
    a.ld_scores = ld;
    a.bias = bias;
    a.tokens = tokens;
    a.experts = static_cast<uint32_t>(r->desc.experts);
    a.topk = static_cast<uint32_t>(r->desc.topk);
    a.gate = r->desc.gate;
    a.normalize = r->desc.normalize;
    a.scale = r->desc.scale;
    return a;
}

int check_select(const mrs_route* r, uint64_t tokens, const void* scores, uint64_t ld, int32_t type, const float* bias,
                 const char* who)
{
    if (int rc = check_call(r, tokens, who)) return rc;
    if (int rc = check_type(type, false, who)) return rc;
    if (r->desc.topk > r->desc.experts)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: topk = %d exceeds the %d experts", who, r->desc.topk, r->desc.experts);
    if (bias && !aligned_to(bias, 4)) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: bias is not aligned to its elements", who);
    return check_matrix({scores, tokens, static_cast<uint64_t>(r->desc.experts), ld, element_bytes(type)}, who, "scores");
}

}  // namespace

extern "C" int mrs_route_max_rows(const mrs_route_desc* desc, uint64_t* rows)
{
    clear_error();
    if (!desc || !rows) return fail(MRS_ERR_INVALID_ARGUMENT, "mrs_route_max_rows: null argument");
    if (int rc = check_desc(desc, "mrs_route_max_rows")) return rc;
    *rows = max_rows_of(*desc, desc->tokens);
    return MRS_OK;
}

extern "C" int mrs_route_create(mrs_context* ctx, const mrs_route_desc* desc, mrs_route** out)
{
    clear_error();
    const char* who = "mrs_route_create";
    if (!ctx || !desc || !out) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: null argument", who);
    *out = nullptr;
    if (int rc = check_desc(desc, who)) return rc;
    if (int rc = check_device(ctx, who)) return rc;
    mrs_route* r = new (std::nothrow) mrs_route();
    if (!r) return fail(MRS_ERR_OUT_OF_MEMORY, "%s: out of host memory", who);
    r->ctx = ctx;
    r->desc = *desc;
    const size_t bytes = static_cast<size_t>(kRouteMaxTiles) * ((desc->experts + 3) / 4 * 4) * sizeof(uint32_t);
    void* temp = nullptr;
    const hipError_t e = hipMalloc(&temp, bytes);
    if (e != hipSuccess) {
        delete r;
        return fail(MRS_ERR_OUT_OF_MEMORY, "%s: hipMalloc(%zu) failed: %s", who, bytes, hipGetErrorString(e));
    }
    r->tile_counts = static_cast<uint32_t*>(temp);
    ctx->live_plans++;
    *out = r;
    return MRS_OK;
}

extern "C" int mrs_route_destroy(mrs_route* route)
{
    clear_error();
    if (!route) return MRS_OK;
    MRS_TEARDOWN(hipFree(route->tile_counts));
    route->ctx->live_plans--;
    delete route;
    return MRS_OK;
}

extern "C" int mrs_route_select(mrs_route* route, uint64_t tokens, const void* scores_dev, uint64_t ld_scores, int32_t type,
                                const float* bias_dev, int32_t* ids_dev, float* weights_dev, void* stream)
{
    clear_error();
    const char* who = "mrs_route_select";
    if (int rc = check_select(route, tokens, scores_dev, ld_scores, type, bias_dev, who)) return rc;
    if (tokens == 0) return MRS_OK;
    if (int rc = check_ints(ids_dev, who, "ids")) return rc;
    if (int rc = check_ints(weights_dev, who, "weights")) return rc;
    const uint64_t experts = static_cast<uint64_t>(route->desc.experts), slots = tokens * static_cast<uint64_t>(route->desc.topk);
    const Named out[] = {{flat(ids_dev, slots), "ids"}, {flat(weights_dev, slots), "weights"}};
    const Named in[] = {{{scores_dev, tokens, experts, ld_scores, element_bytes(type)}, "scores"}, {flat(bias_dev, experts), "bias"}};
    if (int rc = check_outputs(out, in, who)) return rc;
    SelectArgs a = select_args(route, tokens, scores_dev, ld_scores, bias_dev);
    a.ids_out = ids_dev;
    a.weights_out = weights_dev;
    const ProfilerRange range("Select");
    return launch_route_select(type, a, static_cast<hipStream_t>(stream));
}

extern "C" int mrs_route_select_backward(mrs_route* route, uint64_t tokens, const void* scores_dev, uint64_t ld_scores,
                                         int32_t type, const float* bias_dev, const int32_t* ids_dev,
                                         const float* weights_grad_dev, void* scores_grad_dev, uint64_t ld_scores_grad,
                                         void* stream)
{
    clear_error();
    const char* who = "mrs_route_select_backward";
    if (int rc = check_select(route, tokens, scores_dev, ld_scores, type, bias_dev, who)) return rc;
    if (tokens == 0) return MRS_OK;
    if (int rc = check_ints(ids_dev, who, "ids")) return rc;
    if (int rc = check_ints(weights_grad_dev, who, "weights_grad")) return rc;
    const uint64_t experts = static_cast<uint64_t>(route->desc.experts), slots = tokens * static_cast<uint64_t>(route->desc.topk);
    const int bytes = element_bytes(type);
    const Named out[] = {{{scores_grad_dev, tokens, experts, ld_scores_grad, bytes}, "scores_grad"}};
    const Named in[] = {{{scores_dev, tokens, experts, ld_scores, bytes}, "scores"},
                        {flat(bias_dev, experts), "bias"},
                        {flat(ids_dev, slots), "ids"},
                        {flat(weights_grad_dev, slots), "weights_grad"}};
    if (int rc = check_matrix(out[0].m, who, "scores_grad")) return rc;
    if (int rc = check_outputs(out, in, who)) return rc;
    SelectArgs a = select_args(route, tokens, scores_dev, ld_scores, bias_dev);
    a.ids = ids_dev;
    a.weights_grad = weights_grad_dev;
    a.scores_grad = scores_grad_dev;
    a.ld_scores_grad = ld_scores_grad;
    const ProfilerRange range("Select backward");
    return launch_route_select_backward(type, a, static_cast<hipStream_t>(stream));
}

extern "C" int mrs_route_order(mrs_route* route, uint64_t tokens, const int32_t* ids_dev, const mrs_route_map* map, void* stream)
{
    clear_error();
    const char* who = "mrs_route_order";
    if (int rc = check_call(route, tokens, who)) return rc;
    if (!map) return fail(MRS_ERR_INVALID_ARGUMENT, "%s: null map", who);
    const uint64_t need = max_rows_of(route->desc, tokens);
    if (map->rows < need || map->rows > kMaxRows)
        return fail(MRS_ERR_INVALID_ARGUMENT, "%s: %llu rows, need at least %llu and at most 2^31 - 1", who,
                    (unsigned long long)map->rows, (unsigned long long)need);
    if (int rc = check_ints(map->counts, who, "counts")) return rc;
    if (int rc = check_ints(map->offsets, who, "offsets")) return rc;
    if (map->rows)
        if (int rc = check_ints(map->slot_of_row, who, "slot_of_row")) return rc;
    if (tokens) {
        if (int rc = check_ints(ids_dev, who, "ids")) return rc;
        if (int rc = check_ints(map->row_of_slot, who, "row_of_slot")) return rc;
    }
    const uint64_t experts = static_cast<uint64_t>(route->desc.experts), slots = tokens * static_cast<uint64_t>(route->desc.topk);
    const Named out[] = {{flat(map->row_of_slot, slots), "row_of_slot"},
                         {flat(map->slot_of_row, map->rows), "slot_of_row"},
                         {flat(map->counts, experts), "counts"},
                         {flat(map->offsets, experts + 1), "offsets"}};
    const Named in[] = {{flat(ids_dev, slots), "ids"}};
    if (int rc = check_outputs(out, in, who)) return rc;
    OrderArgs a{};
    a.ids = ids_dev;
    a.slots = slots;
    a.experts = static_cast<uint32_t>(route->desc.experts);
    a.align = static_cast<uint32_t>(route->desc.align);
    a.capacity = route->desc.capacity == 0 || route->desc.capacity > 0xFFFFFFFFull ? 0xFFFFFFFFu
                                                                                 : static_cast<uint32_t>(route->desc.capacity);
    a.row_of_slot = map->row_of_slot;
    a.slot_of_row = map->slot_of_row;
    a.counts = map->counts;
    a.offsets = map->offsets;
    a.rows = static_cast<uint32_t>(map->rows);
    a.tile_counts = route->tile_counts;
    const ProfilerRange range("Order");
    return launch_route_order(a, static_cast<hipStream_t>(stream));
}

extern "C" int mrs_route_dispatch(mrs_route* route, uint64_t tokens, const mrs_route_map* map, int32_t type, uint64_t hidden,
                                  const void* x_dev, uint64_t ld_x, void* rows_dev, uint64_t ld_rows, void* stream)
{
    clear_error();
    const char* who = "mrs_route_dispatch";
    if (int rc = check_call(route, tokens, who)) return rc;
    if (int rc = check_type(type, true, who)) return rc;
    if (int rc = check_hidden(hidden, who)) return rc;
    if (int rc = check_map(route, tokens, map, true, who)) return rc;
    if (tokens == 0) return MRS_OK;
    const int bytes = element_bytes(type);
    const uint64_t experts = static_cast<uint64_t>(route->desc.experts), slots = tokens * static_cast<uint64_t>(route->desc.topk);
    const Named out[] = {{{rows_dev, map->rows, hidden, ld_rows, bytes}, "rows"}};
    const Named in[] = {{{x_dev, tokens, hidden, ld_x, bytes}, "x"},
                        {flat(map->row_of_slot, slots), "row_of_slot"},
                        {flat(map->counts, experts), "counts"},
                        {flat(map->offsets, experts + 1), "offsets"}};
    if (int rc = check_matrix(in[0].m, who, "x")) return rc;
    if (int rc = check_matrix(out[0].m, who, "rows")) return rc;
    if (int rc = check_outputs(out, in, who)) return rc;
    MoveArgs a = move_args(route, tokens, map, hidden);
    a.token_in = x_dev;
    a.ld_token_in = ld_x;
    a.rows_out = rows_dev;
    a.ld_rows_out = ld_rows;
    const ProfilerRange range("Dispatch");
    return launch_route_dispatch(bytes, a, static_cast<hipStream_t>(stream));
}

// Token rows as sums of expert rows: combine, and dispatch's gradient (no weights).
static int gather_sum(mrs_route* route, uint64_t tokens, const mrs_route_map* map, int32_t type, uint64_t hidden,
                      const void* rows_dev, uint64_t ld_rows, const char* rows_name, const float* weights_dev, void* out_dev,
                      uint64_t ld_out, const char* out_name, const char* who, void* stream)
{
    const int bytes = element_bytes(type);
    const uint64_t slots = tokens * static_cast<uint64_t>(route->desc.topk);
    const Named out[] = {{{out_dev, tokens, hidden, ld_out, bytes}, out_name}};
    const Named in[] = {{{rows_dev, map->rows, hidden, ld_rows, bytes}, rows_name},
                        {flat(map->row_of_slot, slots), "row_of_slot"},
                        {flat(weights_dev, slots), "weights"}};
    if (int rc = check_matrix(in[0].m, who, rows_name)) return rc;
    if (int rc = check_matrix(out[0].m, who, out_name)) return rc;
    if (int rc = check_outputs(out, in, who)) return rc;
    MoveArgs a = move_args(route, tokens, map, hidden);
    a.rows_in = rows_dev;
    a.ld_rows_in = ld_rows;
    a.weights = weights_dev;
    a.token_out = out_dev;
    a.ld_token_out = ld_out;
    return launch_route_combine(type, a, static_cast<hipStream_t>(stream));
}

extern "C" int mrs_route_dispatch_backward(mrs_route* route, uint64_t tokens, const mrs_route_map* map, int32_t type,
                                           uint64_t hidden, const void* rows_grad_dev, uint64_t ld_rows_grad, void* x_grad_dev,
                                           uint64_t ld_x_grad, void* stream)
{
    clear_error();
    const char* who = "mrs_route_dispatch_backward";
    if (int rc = check_call(route, tokens, who)) return rc;
    if (int rc = check_type(type, false, who)) return rc;
    if (int rc = check_hidden(hidden, who)) return rc;
    if (int rc = check_map(route, tokens, map, false, who)) return rc;
    if (tokens == 0) return MRS_OK;
    const ProfilerRange range("Dispatch backward");
    return gather_sum(route, tokens, map, type, hidden, rows_grad_dev, ld_rows_grad, "rows_grad", nullptr, x_grad_dev, ld_x_grad,
                      "x_grad", who, stream);
}

extern "C" int mrs_route_combine(mrs_route* route, uint64_t tokens, const mrs_route_map* map, int32_t type, uint64_t hidden,
                                 const void* rows_dev, uint64_t ld_rows, const float* weights_dev, void* out_dev, uint64_t ld_out,
                                 void* stream)
{
    clear_error();
    const char* who = "mrs_route_combine";
    if (int rc = check_call(route, tokens, who)) return rc;
    if (int rc = check_type(type, false, who)) return rc;
    if (int rc = check_hidden(hidden, who)) return rc;
    if (int rc = check_map(route, tokens, map, false, who)) return rc;
    if (tokens == 0) return MRS_OK;
    if (int rc = check_ints(weights_dev, who, "weights")) return rc;
    const ProfilerRange range("Combine");
    return gather_sum(route, tokens, map, type, hidden, rows_dev, ld_rows, "rows", weights_dev, out_dev, ld_out, "out", who, stream);
}

extern "C" int mrs_route_combine_backward(mrs_route* route, uint64_t tokens, const mrs_route_map* map, int32_t type,
                                          uint64_t hidden, const void* out_grad_dev, uint64_t ld_out_grad, const void* rows_dev,
                                          uint64_t ld_rows, const float* weights_dev, void* rows_grad_dev, uint64_t ld_rows_grad,
                                          float* weights_grad_dev, void* stream)
{
    clear_error();
    const char* who = "mrs_route_combine_backward";
    if (int rc = check_call(route, tokens, who)) return rc;
    if (int rc = check_type(type, false, who)) return rc;
    if (int rc = check_hidden(hidden, who)) return rc;
    if (int rc = check_map(route, tokens, map, true, who)) return rc;
    if (tokens == 0) return MRS_OK;
    if (int rc = check_ints(weights_dev, who, "weights")) return rc;
    if (int rc = check_ints(weights_grad_dev, who, "weights_grad")) return rc;
    const int bytes = element_bytes(type);
    const uint64_t experts = static_cast<uint64_t>(route->desc.experts), slots = tokens * static_cast<uint64_t>(route->desc.topk);
    const Named out[] = {{{rows_grad_dev, map->rows, hidden, ld_rows_grad, bytes}, "rows_grad"},
                         {flat(weights_grad_dev, slots), "weights_grad"}};
    const Named in[] = {{{out_grad_dev, tokens, hidden, ld_out_grad, bytes}, "out_grad"},
                        {{rows_dev, map->rows, hidden, ld_rows, bytes}, "rows"},
                        {flat(weights_dev, slots), "weights"},
                        {flat(map->row_of_slot, slots), "row_of_slot"},
                        {flat(map->counts, experts), "counts"},
                        {flat(map->offsets, experts + 1), "offsets"}};
    if (int rc = check_matrix(in[0].m, who, "out_grad")) return rc;
    if (int rc = check_matrix(in[1].m, who, "rows")) return rc;
    if (int rc = check_matrix(out[0].m, who, "rows_grad")) return rc;
    if (int rc = check_outputs(out, in, who)) return rc;
    MoveArgs a = move_args(route, tokens, map, hidden);
    a.token_in = out_grad_dev;
    a.ld_token_in = ld_out_grad;
    a.rows_in = rows_dev;
    a.ld_rows_in = ld_rows;
    a.weights = weights_dev;
    a.rows_out = rows_grad_dev;
    a.ld_rows_out = ld_rows_grad;
    a.weights_grad = weights_grad_dev;
    const ProfilerRange range("Combine backward");
    return launch_route_combine_backward(type, a, static_cast<hipStream_t>(stream));
}
