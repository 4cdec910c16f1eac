// C ABI of the operators that serve a block from a paged cache, and of the
// norms of queries and keys (include/mtpx.h): argument checks, workspaces,
// launches on the caller's stream.
#include "ops_checks.hpp"
#include "ops_internal.hpp"

#include <algorithm>
#include <exception>

namespace mtpx {
namespace {

constexpr int kMaxHeadDim = 256, kMaxAxes = 8, kMaxSequences = 1 << 24;
constexpr int64_t kMaxRoom = int64_t(1) << 30;  // rows of one sequence

// No exception leaves a C entry point: a message takes memory.
template <class F>
int guarded(const F &f) noexcept
{
    try {
        return f();
    } catch (const std::exception &) {
        return MTPX_E_ALLOC;
    }
}

// The rotation's arguments, which two requests name alike.
template <class R>
int check_turn(mtpx_context *ctx, const R &r)
{
    if (r.rotated < 0 || r.rotated > r.dim || r.rotated % 2 != 0)
        return invalid(ctx, "rotated must be even and at most dim");
    if (r.axes < 1 || r.axes > kMaxAxes)
        return invalid(ctx, "axes must be 1 to 8");
    if (r.position_dtype != MTPX_F32 && r.position_dtype != MTPX_F64 && r.position_dtype != MTPX_I32 &&
        r.position_dtype != MTPX_I64)
        return invalid(ctx, "unknown position_dtype");
    if (r.position_row < 0 || r.position_axis < 0)
        return invalid(ctx, "negative position stride");
    if (r.rows == 0 || r.rotated == 0)
        return MTPX_OK;
    MTPX_TRY(check_flat(ctx, r.positions, r.position_dtype == MTPX_F32 || r.position_dtype == MTPX_I32 ? 4 : 8, "positions"));
    MTPX_TRY(check_flat(ctx, r.freq, 4, "freq"));
    return check_flat(ctx, r.axis, 4, "axis");
}
// And those of the norm, with the counts.
template <class R>
int check_norms(mtpx_context *ctx, const R &r, int last_kind)
{
    if (!is_dtype(r.dtype))
        return invalid(ctx, "dtype must be MTPX_F32, MTPX_BF16 or MTPX_F16");
    if (r.rows < 0 || r.dim < 1)
        return invalid(ctx, "rows must not be negative and dim positive");
    if (r.dim > kMaxHeadDim || r.rows > kMaxRows || r.heads > 65535 || r.kv_heads > 65535)
        return set_error(ctx, MTPX_E_CAPACITY, "dim beyond 256, more than 65535 heads or too many rows");
    if (r.kind < MTPX_NORM_RMS || r.kind > last_kind)
        return invalid(ctx, "unknown norm kind");
    if (!(r.eps >= 0.f) || !std::isfinite(r.eps))
        return invalid(ctx, "eps must not be negative");
    for (const void *w : {r.q_weight, r.k_weight})
        if (!aligned(w, dtype_bytes(r.dtype)))
            return invalid(ctx, "a weight is not aligned to its elements");
    return check_turn(ctx, r);
}
int check_place(mtpx_context *ctx, const mtpx_rows &x, const mtpx_rows &y, int maps, const char *name)
{
    if (x.data == y.data && (x.row != y.row || x.head != y.head || (maps > 1 && x.map != y.map)))
        return invalid(ctx, std::string(name) + " in the place of its input needs its strides");
    return MTPX_OK;
}

template <class R>
HeadArgs head_args(const R &r, int maps)
{
    HeadArgs a{};
    a.rows = r.rows;
    a.vectors[0] = r.heads * maps;
    a.vectors[1] = r.kv_heads * maps;
    a.maps = maps;
    a.dim = r.dim;
    a.rotated = r.rotated;
    a.interleaved = r.interleaved != 0;
    a.kind = r.kind;
    a.axes = r.axes;
    a.position_dtype = r.position_dtype;
    a.eps = r.eps;
    a.in[0] = r.q;
    a.in[1] = r.k;
    a.weight[0] = r.q_weight;
    a.weight[1] = r.k_weight;
    a.positions = r.positions;
    a.position_row = r.position_row;
    a.position_axis = r.position_axis;
    a.freq = r.freq;
    a.axis = r.axis;
    return a;
}

// Lanes of a row: a whole workgroup where there are few rows, as that takes the
// fewest steps one after the other (36 heads of two vectors of 64 in 16 bits: 64
// rows 5.1 us, 7.3 us with a wave each; 4,001 rows 21 us, 16 us with a wave each);
// else up to a wave, as few as leave the device full, since a row's cos and sin are
// formed by as many lanes and its vectors read ahead (160,000 rows of 16 and 16
// vectors of 64 in 16 bits: forward 303 us with 64 lanes, 235 us with 16; backward
// 479 us with 64, 382 us with 8).  The backward pass's workgroups have more to end
// with, which many rows pay for if they take few steps (those heads: 1 row 13.7 us
// with a wave, 11.1 us with a workgroup; 2,048 rows 21 and 28 us; 32 vectors of 128
// with a wave each: 1,024 rows 40 and 23 us).
constexpr int64_t kForwardThreads = int64_t(1) << 21, kBackwardThreads = int64_t(1) << 20;
void row_lanes(mtpx_context *ctx, HeadArgs &a, bool back)
{
    const int64_t wanted = (int64_t)std::max(a.vectors[0], a.vectors[1]) * a.group, few = 2 * (int64_t)ctx->num_cus;
    const int most = a.rows <= few || (a.rows <= 4 * few && (!back || wanted >= 16 * 64)) ? 256 : 64;
    a.lanes = a.group;
    while (a.lanes < most && a.lanes < wanted && a.rows * a.lanes < (back ? kBackwardThreads : kForwardThreads))
        a.lanes *= 2;
    if (back && a.lanes == 128)
        a.lanes = 64;  // the backward pass's workgroups have one row of more than a wave, or none
}

// The widest access that every piece of a vector allows (`fits`: the tensors'
// addresses and strides), and the lanes of a vector and of a row.
template <class Fits>
void shape_heads(mtpx_context *ctx, HeadArgs &a, int64_t size, bool back, const Fits &fits)
{
    const int half = a.rotated / 2;
    a.width = (int)(16 / size);
    while (a.width > 1 && !((a.interleaved ? a.rotated : half) % a.width == 0 && (a.dim - a.rotated) % a.width == 0 &&
                            aligned(a.weight[0], a.width * size) && aligned(a.weight[1], a.width * size) && fits(a.width)))
        a.width /= 2;
    const int unit = a.interleaved ? std::max(a.width / 2, 1) : a.width;
    const int units = half / unit + (a.dim - a.rotated) / a.width;
    a.group = 1;
    while (a.group < 64 && a.group < units)
        a.group *= 2;
    row_lanes(ctx, a, back);
}
bool fits_rows(const mtpx_rows &t, int width, int64_t size, int maps)
{
    return !t.data || (aligned(t.data, width * size) && t.row % width == 0 && t.head % width == 0 &&
                       (maps == 1 || t.map % width == 0));
}

// Workgroups of the backward pass: as many as the device holds of it, by the
// registers that a lane's elements take (160,000 rows of 8 and 8 heads of two
// vectors of 64 in 16 bits, pairs side by side: 389 us with 3 a compute unit, 441
// with 2 and 459 with 4; 4,001 rows with the halves apart: 22 us with 2, 28 with 3
// or 4; 160,000 rows of 10 and 5 heads of 40 in 32 bits: 560 us with 4, 623 with 3).
int head_parts(mtpx_context *ctx, const HeadArgs &a)
{
    const int64_t together = 256 / a.lanes, each = a.width < 8 ? 4 : a.interleaved ? 3 : 2;
    return (int)std::min<int64_t>((a.rows + together - 1) / together, each * (int64_t)ctx->num_cus);
}

int check_head_sizes(mtpx_context *ctx, const mtpx_head_norm_rotary_request &r)
{
    if (r.heads < 1 || r.kv_heads < 0)
        return invalid(ctx, "heads must be positive and kv_heads not negative");
    if (r.maps != 1 && r.maps != 2)
        return invalid(ctx, "maps must be 1 or 2");
    return MTPX_OK;
}

int head_request(mtpx_context *ctx, const mtpx_head_norm_rotary_request &r, bool back, HeadArgs &a)
{
    MTPX_TRY(check_head_sizes(ctx, r));
    MTPX_TRY(check_norms(ctx, r, MTPX_NORM_LAYER));
    a = head_args(r, r.maps);
    const size_t size = dtype_bytes(r.dtype);
    if (back) {
        if ((r.dq_weight && !r.q_weight) || (r.dk_weight && !r.k_weight))
            return invalid(ctx, "a weight's gradient without the weight");
        for (const void *p : {r.dq_weight, r.dk_weight})
            if (!aligned(p, size))
                return invalid(ctx, "a weight's gradient is not aligned to its elements");
        if (r.dpositions && r.position_dtype != MTPX_F32 && r.position_dtype != MTPX_F64)
            return invalid(ctx, "integer positions have no gradient");
        if (r.dpositions && !aligned(r.dpositions, r.position_dtype == MTPX_F64 ? 8 : 4))
            return invalid(ctx, "dpositions is not aligned to its elements");
    }
    a.out[0] = back ? r.dq : r.q_out;
    a.out[1] = back ? r.dk : r.k_out;
    if (back) {
        a.grad[0] = r.dq_out;
        a.grad[1] = r.dk_out;
        a.dweight[0] = r.dq_weight;
        a.dweight[1] = r.dk_weight;
        a.dpositions = r.dpositions;
    }
    const char *const names[2][4] = {{"q", "q_out", "dq_out", "dq"}, {"k", "k_out", "dk_out", "dk"}};
    for (int i = 0; i < 2 && r.rows > 0; ++i) {
        if (a.vectors[i] == 0)
            continue;
        MTPX_TRY(check_rows(ctx, a.in[i], r.dtype, names[i][0]));
        MTPX_TRY(check_rows(ctx, a.out[i], r.dtype, names[i][back ? 3 : 1]));
        if (back)
            MTPX_TRY(check_rows(ctx, a.grad[i], r.dtype, names[i][2]));
        MTPX_TRY(check_place(ctx, back ? a.grad[i] : a.in[i], a.out[i], r.maps, names[i][back ? 3 : 1]));
    }
    shape_heads(ctx, a, size, back, [&](int width) {
        for (int i = 0; i < 2; ++i)
            if (a.vectors[i] && !(fits_rows(a.in[i], width, size, r.maps) && fits_rows(a.out[i], width, size, r.maps) &&
                                  fits_rows(a.grad[i], width, size, r.maps)))
                return false;
        return true;
    });
    return MTPX_OK;
}

// Enough for any alignment of the tensors.
size_t head_bytes(mtpx_context *ctx, const mtpx_head_norm_rotary_request &r)
{
    const int64_t parts = std::min<int64_t>(r.rows, 4 * (int64_t)ctx->num_cus);
    return std::max<size_t>(sizeof(float) * 2 * (size_t)parts * r.dim, 16);
}

// A cache's pages: what the host can see of them.
int check_pages(mtpx_context *ctx, const mtpx_pages &c, int dtype)
{
    if (c.pages < 0 || c.page_rows < 1 || c.table_width < 0 || c.table_row < 0)
        return invalid(ctx, "pages, table_width and table_row must not be negative and page_rows positive");
    if (c.pages > INT32_MAX || c.page_rows > 1 << 20 || (int64_t)c.table_width * c.page_rows > kMaxRoom)
        return set_error(ctx, MTPX_E_CAPACITY, "too many pages, rows of a page or rows of a sequence");
    if (c.pages > 0) {
        MTPX_TRY(check_rows(ctx, c.k, dtype, "cache.k"));
        MTPX_TRY(check_rows(ctx, c.v, dtype, "cache.v"));
        if (c.k_page < 0 || c.v_page < 0)
            return invalid(ctx, "negative page stride");
    }
    return c.table_width > 0 ? check_flat(ctx, c.table, 4, "table") : MTPX_OK;
}
int check_batch(mtpx_context *ctx, int sequences, const int *offsets, const int *lengths)
{
    if (sequences < 0)
        return invalid(ctx, "negative count of sequences");
    if (sequences > kMaxSequences)
        return set_error(ctx, MTPX_E_CAPACITY, "more than 2^24 sequences");
    if (sequences == 0)
        return MTPX_OK;
    MTPX_TRY(check_flat(ctx, offsets, 4, "offsets"));
    return check_flat(ctx, lengths, 4, "lengths");
}
bool pages_fit(const mtpx_pages &c, int width, int64_t size)
{
    return fits_rows(c.k, width, size, 2) && fits_rows(c.v, width, size, 2) && c.k_page % width == 0 && c.v_page % width == 0;
}

// How the work of a call is split, from what the host knows: rows, sequences,
// the most new rows of one, and the room of the tables.
struct PagedPlan {
    int narrow_columns = 0;
    RoleArgs narrow{}, wide{};
    size_t narrow_bytes = 0, wide_bytes = 0;
    int64_t items = 0;
};
// Columns of a narrow tile (64 sequences of one row, 32 heads of 64 on 4: 152 us,
// 163 us on wide tiles; 8 heads of 32: 165 and 180 us).
constexpr int kNarrowColumns = 32;
// Sequences and tiles whose keys workgroups share.  Of so many a tile each is a
// little faster if they are alike (4,096 rows of 50 to 1,500 keys: 1,233 us, 1,346
// us shared), and a long one among them does not keep the device waiting (one of
// 32,000: 454 us, 31 us shared).
constexpr int64_t kMaxShared = 4096, kMaxUnits = 1 << 18;

PagedPlan paged_plan(mtpx_context *ctx, const mtpx_diff_attention_paged_request &r)
{
    PagedPlan p;
    const int64_t group = r.heads / r.kv_heads, n = r.sequences;
    const int64_t room = std::max<int64_t>((int64_t)r.cache.table_width * r.cache.page_rows, 1);
    const int64_t most = r.max_rows > 0 ? std::min<int64_t>(r.max_rows, r.rows) : r.rows;
    const int width = r.dim <= 32 ? 32 : r.dim <= 64 ? 64 : 128;
    const bool half = r.dtype != MTPX_F32;
    // workgroups that the device holds at once: by their 64 KiB of LDS, or 32
    const int64_t slots = 2 * (int64_t)ctx->num_cus;
    const bool both = group <= kNarrowColumns && most * group > kNarrowColumns;
    const int columns = half ? (width < 128 ? 128 : 64) : width < 128 ? 64 : 32;
    const int64_t all = r.rows * group / columns;  // whole wide tiles of a key head
    // A few long sequences among many short ones (by the average's share of the
    // longest): shares of both widths run beside each other, on less than all slots
    // each, as the ones read while the others multiply (46 single rows and chunks
    // of 727, heads of 128: 294 us, 334 us with all slots each, 398 us with half;
    // 30 rows and two chunks of 512, heads of 64: 161 us, 175 us).  Many wide tiles
    // of up to 64 need all (46 rows and a chunk of 2,048: 392 us, 464 us with half).
    const bool beside = both && half && r.rows * 4 <= n * most && (all + n) * r.kv_heads < (width == 128 ? 4 : 1) * slots;
    auto role = [&](RoleArgs &a, size_t &bytes, int tile, int64_t units, bool each) {
        // (costs are counted in 32 bits)
        a.each_unit = each || n > kMaxShared || units > kMaxUnits || units * ((room + r.rows) / 32 + 16) > INT32_MAX / 2;
        // (small calls of both widths share the slots, so that neither waits for the
        // other: 12 sequences of up to 700 rows in 32 bits, 52 us and 41 us a call)
        const bool small = both && units * ((room + 63) / 64) <= 8 * slots;
        const int64_t mine = small || (beside && (&a == &p.narrow || width < 128)) ? slots / 2 : beside ? slots / 4 * 3 : slots;
        const int64_t groups = a.each_unit ? units : std::min(mine, units * ((room + 63) / 64));
        a.groups = (int)std::min<int64_t>(groups, INT32_MAX);
        p.items += groups;
        if (!a.each_unit && a.groups > 1)
            bytes = sizeof(float) * 2 * (4 + 2 * width) * 2 * (size_t)tile * a.groups;
    };
    if (group <= kNarrowColumns) {
        p.narrow_columns = kNarrowColumns;
        role(p.narrow, p.narrow_bytes, kNarrowColumns, n * r.kv_heads, false);
    }
    if (p.narrow_columns == 0 || both) {
        // every sequence's tiles in one order where that leaves few without rows (8
        // sequences of 4,096 rows, 16 heads of 64: 926 us, 942 us sequence by
        // sequence; of 2,500 to 6,000 rows: 1,060 and 981 us)
        const int64_t level = (most * group + columns - 1) / columns * n;
        // A tile a workgroup, of more tiles than slots: about as long as the longest
        // tile over the even share, with tiles half as long as there is room on
        // average.  Shared, a slot and a tile have `split` steps' time of partial
        // results each (3 prompts of 1,024 rows, 32 heads of 64: 59 us and 89 us
        // shared; one of 8,192, 16 heads: 446 and 464 us; a chunk of 2,048 rows of
        // 32,000: 1,094 and 795 us).
        p.wide.split = half ? 8 : 3;
        const int64_t steps = (room - 1) / (2 * width * (half ? 2 : 4) <= 256 ? 64 : 32) + 1, units = all * r.kv_heads;
        const bool each = units >= 4 * slots || (units > slots && steps * slots <= 2 * p.wide.split * (units + slots));
        p.wide.level = each && level * 10 <= all * 11;
        const int64_t tiles = p.wide.level ? level : all + n;
        p.wide.tiles = (int)std::min<int64_t>(tiles, INT32_MAX);
        if (each && r.causal && !p.wide.level)
            p.wide.quarters = (int)std::min<int64_t>(all / 4 + n, INT32_MAX);
        role(p.wide, p.wide_bytes, columns, (tiles + p.wide.quarters) * r.kv_heads, each);
    }
    return p;
}

// magic = floor(2^(31 + shift) / d) + 1 with 2^shift >= d: n magic / 2^(31 + shift)
// is above n / d by less than n / 2^31 of 1 / d.
Divisor divisor(int d)
{
    int shift = 0;
    while ((1 << shift) < d)
        ++shift;
    return {(unsigned)((uint64_t(1) << (31 + shift)) / (uint64_t)d + 1), shift};
}

int check_paged(mtpx_context *ctx, const mtpx_diff_attention_paged_request &r)
{
    MTPX_TRY(check_heads(ctx, r.dtype, r.heads, r.kv_heads, r.dim, r.scale));
    if (r.rows < 0 || r.max_rows < 0 || r.sequences < 0)
        return invalid(ctx, "negative count");
    if (r.cache.page_rows < 1 || r.cache.table_width < 0)
        return invalid(ctx, "page_rows must be positive and table_width not negative");
    if (r.rows > kMaxRows || r.sequences > kMaxSequences || r.heads > 65535 || r.cache.page_rows > 1 << 20 ||
        (int64_t)r.cache.table_width * r.cache.page_rows > kMaxRoom)
        return set_error(ctx, MTPX_E_CAPACITY, "too many rows, sequences, heads or rows of a sequence");
    // (columns, of which there are rows times heads, and the costs of their tiles are
    // counted in 32 bits)
    if (r.rows * r.heads > kMaxGroups || paged_plan(ctx, r).items > kMaxGroups)
        return set_error(ctx, MTPX_E_CAPACITY, "too many rows and heads for one call");
    return MTPX_OK;
}

}  // namespace
}  // namespace mtpx

extern "C" {

int mtpx_head_norm_rotary(mtpx_context *ctx, const mtpx_head_norm_rotary_request *req)
{
    return guarded([&]() -> int {
        if (!ctx || !req)
            return set_error(ctx, MTPX_E_INVALID, "null argument");
        HeadArgs a;
        MTPX_TRY(head_request(ctx, *req, false, a));
        if (a.rows == 0)
            return MTPX_OK;
        OnDevice here(ctx->device);
        HIP_TRY(launch_head_forward(req->dtype, a, (hipStream_t)req->stream), "launch head norm");
        return MTPX_OK;
    });
}

int mtpx_head_norm_rotary_workspace(mtpx_context *ctx, const mtpx_head_norm_rotary_request *req, size_t *bytes)
{
    return guarded([&]() -> int {
        if (!ctx || !req || !bytes)
            return set_error(ctx, MTPX_E_INVALID, "null argument");
        if (req->rows < 0 || req->dim < 1)
            return invalid(ctx, "rows must not be negative and dim positive");
        if (req->dim > kMaxHeadDim || req->rows > kMaxRows)
            return set_error(ctx, MTPX_E_CAPACITY, "dim beyond 256 or too many rows");
        *bytes = head_bytes(ctx, *req);
        return MTPX_OK;
    });
}

int mtpx_head_norm_rotary_backward(mtpx_context *ctx, const mtpx_head_norm_rotary_request *req)
{
    return guarded([&]() -> int {
        if (!ctx || !req)
            return set_error(ctx, MTPX_E_INVALID, "null argument");
        HeadArgs a;
        MTPX_TRY(head_request(ctx, *req, true, a));
        MTPX_TRY(check_workspace(ctx, req->workspace, req->workspace_bytes, head_bytes(ctx, *req)));
        a.part = static_cast<float *>(req->workspace);
        a.parts = head_parts(ctx, a);
        OnDevice here(ctx->device);
        HIP_TRY(launch_head_backward(req->dtype, a, (hipStream_t)req->stream), "launch head norm gradient");
        return MTPX_OK;
    });
}

int mtpx_append_paged(mtpx_context *ctx, const mtpx_append_paged_request *req)
{
    return guarded([&]() -> int {
        if (!ctx || !req)
            return set_error(ctx, MTPX_E_INVALID, "null argument");
        const mtpx_append_paged_request &r = *req;
        if (r.heads < 0 || r.kv_heads < 1)
            return invalid(ctx, "heads must not be negative and kv_heads positive");
        MTPX_TRY(check_norms(ctx, r, MTPX_NORM_NONE));
        if (r.kind == MTPX_NORM_NONE && (r.q_weight || r.k_weight))
            return invalid(ctx, "weights without a norm");
        MTPX_TRY(check_batch(ctx, r.sequences, r.offsets, r.lengths));
        MTPX_TRY(check_pages(ctx, r.cache, r.dtype));
        if (r.rows == 0 || r.sequences == 0)
            return MTPX_OK;
        MTPX_TRY(check_rows(ctx, r.k, r.dtype, "k"));
        MTPX_TRY(check_rows(ctx, r.v, r.dtype, "v"));
        HeadArgs a = head_args(r, 2);
        a.cache = r.cache;
        a.v = r.v;
        a.offsets = r.offsets;
        a.lengths = r.lengths;
        a.sequences = r.sequences;
        if (r.heads > 0) {
            MTPX_TRY(check_rows(ctx, r.q, r.dtype, "q"));
            MTPX_TRY(check_rows(ctx, r.q_out, r.dtype, "q_out"));
            MTPX_TRY(check_place(ctx, r.q, r.q_out, 2, "q_out"));
            a.out[0] = r.q_out;
        }
        const int64_t size = (int64_t)dtype_bytes(r.dtype);
        shape_heads(ctx, a, size, false, [&](int width) {
            return fits_rows(a.in[1], width, size, 2) && fits_rows(a.v, width, size, 2) && pages_fit(r.cache, width, size) &&
                   (r.heads == 0 || (fits_rows(a.in[0], width, size, 2) && fits_rows(a.out[0], width, size, 2)));
        });
        OnDevice here(ctx->device);
        HIP_TRY(launch_head_append(r.dtype, a, (hipStream_t)r.stream), "launch append");
        return MTPX_OK;
    });
}

int mtpx_diff_attention_paged_workspace(mtpx_context *ctx, const mtpx_diff_attention_paged_request *req, size_t *bytes)
{
    return guarded([&]() -> int {
        if (!ctx || !req || !bytes)
            return set_error(ctx, MTPX_E_INVALID, "null argument");
        mtpx_diff_attention_paged_request r = *req;
        r.scale = 1.f;
        MTPX_TRY(check_paged(ctx, r));
        const PagedPlan p = paged_plan(ctx, r);
        *bytes = p.narrow_bytes + p.wide_bytes;
        return MTPX_OK;
    });
}

int mtpx_diff_attention_paged(mtpx_context *ctx, const mtpx_diff_attention_paged_request *req)
{
    return guarded([&]() -> int {
        if (!ctx || !req)
            return set_error(ctx, MTPX_E_INVALID, "null argument");
        const mtpx_diff_attention_paged_request &r = *req;
        MTPX_TRY(check_paged(ctx, r));
        MTPX_TRY(check_pages(ctx, r.cache, r.dtype));
        MTPX_TRY(check_batch(ctx, r.sequences, r.offsets, r.lengths));
        if (r.rows == 0 || r.sequences == 0)
            return MTPX_OK;
        MTPX_TRY(check_rows(ctx, r.q, r.dtype, "q"));
        MTPX_TRY(check_rows(ctx, r.out, r.dtype, "out"));
        MTPX_TRY(check_flat(ctx, r.lambda, 4, "lambda"));
        const PagedPlan p = paged_plan(ctx, r);
        MTPX_TRY(check_workspace(ctx, r.workspace, r.workspace_bytes, p.narrow_bytes + p.wide_bytes));
        const int64_t size = (int64_t)dtype_bytes(r.dtype);
        PagedArgs a{};
        a.rows = r.rows;
        a.sequences = r.sequences;
        a.heads = r.heads;
        a.kv_heads = r.kv_heads;
        a.dim = r.dim;
        a.causal = r.causal != 0;
        a.scale = r.scale;
        a.q = r.q;
        a.out = r.out;
        a.cache = r.cache;
        a.offsets = r.offsets;
        a.lengths = r.lengths;
        a.lambda = r.lambda;
        a.vec = r.dim * size % 16 == 0 && whole_pieces(r.q, size) && whole_pieces(r.out, size) &&
                pages_fit(r.cache, (int)(16 / size), size);
        const mtpx_pages &c = r.cache;
        const int64_t limit = int64_t(1) << 26;  // elements: eight rows and two maps stay within 32 bits of bytes
        a.alike = a.vec && c.k.row == c.v.row && c.k.map == c.v.map && c.k_page == c.v_page && c.k.row < limit && c.k.map < limit;
        a.heads_each = r.heads / r.kv_heads;
        a.page = divisor(c.page_rows);
        a.group = divisor(a.heads_each);
        a.narrow_columns = p.narrow_columns;
        a.narrow = p.narrow;
        a.wide = p.wide;
        float *part = static_cast<float *>(r.workspace);
        if (p.narrow_bytes)
            a.narrow.part = part;
        if (p.wide_bytes)
            a.wide.part = part + p.narrow_bytes / sizeof(float);
        OnDevice here(ctx->device);
        HIP_TRY(launch_paged(r.dtype, a, (hipStream_t)r.stream), "launch paged attention");
        return MTPX_OK;
    });
}

}  // extern "C"
