// C ABI of the operators on device tensors (include/mtpx.h): argument checks,
// workspaces, launches on the caller's stream.
#include "context.hpp"
#include "ops_internal.hpp"

#include <algorithm>
#include <cmath>
#include <exception>
#include <mutex>
#include <new>
#include <utility>

struct mtpx_sequences {
    int device = 0, n = 0;
    int64_t total_q = 0, total_k = 0;
    DBuf tiles;
    TileTable table{};
    ~mtpx_sequences() { tiles.release(); }
};

namespace mtpx {
namespace {

// Tables of destroyed handles, freed by the next creation: a handle may be
// destroyed at any time (by a garbage collector, say), also while a graph is
// recorded, which no free may happen in, and while queued work reads it.
struct Retired {
    std::mutex lock;
    std::vector<std::pair<int, void *>> tables;  // by device

    void add(int device, void *p)
    {
        std::lock_guard<std::mutex> held(lock);
        tables.emplace_back(device, p);
    }
    // Those of the current device; waits for its work.
    void free(int device)
    {
        std::vector<void *> mine;
        {
            std::lock_guard<std::mutex> held(lock);
            mine.reserve(tables.size());
            auto end = std::remove_if(tables.begin(), tables.end(), [&](const std::pair<int, void *> &t) {
                if (t.first == device)
                    mine.push_back(t.second);
                return t.first == device;
            });
            tables.erase(end, tables.end());
        }
        if (!mine.empty())
            (void)hipDeviceSynchronize();
        for (void *p : mine)
            (void)hipFree(p);
    }
};
Retired &retired()
{
    static Retired *r = new Retired;  // kept: handles may be destroyed as the process ends
    return *r;
}

constexpr int64_t kMaxLength = int64_t(1) << 30;  // rows of one sequence
// a launch's threads are counted in 32 bits: workgroups of 512, rows of 64
constexpr int64_t kMaxGroups = UINT32_MAX / 512, kMaxRows = UINT32_MAX / 64;

int invalid(mtpx_context *ctx, const std::string &msg) { return set_error(ctx, MTPX_E_INVALID, msg); }

size_t dtype_bytes(int dtype) { return dtype == MTPX_F32 ? 4 : 2; }
bool is_dtype(int d) { return d == MTPX_F32 || d == MTPX_BF16 || d == MTPX_F16; }
bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A tensor of rows: present, element-aligned, strides that count forward.
int check_rows(mtpx_context *ctx, const mtpx_rows &r, int dtype, const char *name)
{
    if (!r.data)
        return invalid(ctx, std::string("null ") + name);
    if (!aligned(r.data, dtype_bytes(dtype)))
        return invalid(ctx, std::string(name) + " is not aligned to its elements");
    if (r.row < 0 || r.head < 0 || r.map < 0)
        return invalid(ctx, std::string(name) + " has a negative stride");
    return MTPX_OK;
}
int check_flat(mtpx_context *ctx, const void *p, size_t align, const char *name)
{
    if (!p)
        return invalid(ctx, std::string("null ") + name);
    if (!aligned(p, align))
        return invalid(ctx, std::string(name) + " is not aligned to its elements");
    return MTPX_OK;
}

// The context's device while a call queues its work, then the caller's again:
// these calls run inside programs that keep a current device of their own.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device)
    {
        int d = -1;
        if (hipGetDevice(&d) == hipSuccess && d == device)
            return;
        before = d;
        (void)hipSetDevice(device);
    }
    ~OnDevice()
    {
        if (before >= 0)
            (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

bool whole_pieces(const mtpx_rows &r, size_t size)
{
    return aligned(r.data, 16) && r.row * size % 16 == 0 && r.head * size % 16 == 0 &&
           r.map * size % 16 == 0;
}

#define MTPX_TRY(expr)                                                                     \
    do {                                                                                   \
        if (int rc_ = (expr))                                                              \
            return rc_;                                                                    \
    } while (0)

int check_heads(mtpx_context *ctx, int dtype, int heads, int kv_heads, int dim, float scale)
{
    if (!is_dtype(dtype))
        return invalid(ctx, "dtype must be MTPX_F32, MTPX_BF16 or MTPX_F16");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0)
        return invalid(ctx, "heads must be a positive multiple of kv_heads");
    if (dim < 1)
        return invalid(ctx, "dim must be positive");
    if (dim > 128)
        return set_error(ctx, MTPX_E_CAPACITY, "dim beyond 128");
    if (!(scale > 0.f) || !std::isfinite(scale))
        return invalid(ctx, "scale must be positive and finite");
    return MTPX_OK;
}

// Parts of the key pass's walk over the rows of every head that shares a key:
// one where tiles of 64 keys give each CU two workgroups or more, else enough
// to do that, each with four tiles of rows at least (14,488 causal rows, 16
// heads over 2, 16 wide: a training step of 2.23 ms with one part, 1.31 ms so).
int key_parts(mtpx_context *ctx, const mtpx_diff_attention_request &r)
{
    const TileTable &t = r.sequences->table;
    const int64_t groups = std::max<int64_t>((int64_t)t.nk[0] * r.kv_heads, 1), full = 2 * (int64_t)ctx->num_cus;
    if (groups >= full)
        return 1;
    const int64_t walk = (int64_t)((t.longest_q + 63) / 64) * (r.heads / r.kv_heads);
    return (int)std::max<int64_t>(1, std::min<int64_t>({(2 * full + groups - 1) / groups, walk / 4, 16}));
}

struct AttnSizes {
    size_t delta, part, kv, total;
};
AttnSizes attn_workspace(mtpx_context *ctx, const mtpx_diff_attention_request &r)
{
    const mtpx_sequences &q = *r.sequences;
    const int parts = key_parts(ctx, r);
    auto pad = [](size_t n) { return (n + 15) / 16 * 16; };
    AttnSizes s;
    // D of both maps, and in float16 the largest of |dO|
    const size_t planes = r.dtype == MTPX_F16 ? 3 : 2;
    s.delta = pad(sizeof(float) * planes * (size_t)r.heads * (size_t)q.total_q);
    s.part = pad(sizeof(float) * (size_t)r.heads *
                 (size_t)attn_backward_tiles(r.dtype, r.dim, r.heads, q.table));
    s.kv = parts == 1 ? 0 : sizeof(float) * 4 * (size_t)r.dim * parts * r.kv_heads * (size_t)q.total_k;
    s.total = std::max<size_t>(s.delta + s.part + s.kv, 16);
    return s;
}

// Checks of both passes and the launch arguments they share.
int attn_args(mtpx_context *ctx, const mtpx_diff_attention_request &r, bool back, AttnArgs &a)
{
    MTPX_TRY(check_heads(ctx, r.dtype, r.heads, r.kv_heads, r.dim, r.scale));
    if (!r.sequences)
        return invalid(ctx, "null sequences");
    const mtpx_sequences &sq = *r.sequences;
    if (sq.device != ctx->device)
        return invalid(ctx, "the sequences belong to another device");
    for (int i = 0; i < 2; ++i)
        if ((int64_t)std::max(sq.table.nq[i], sq.table.nk[i]) * r.heads > kMaxGroups)
            return set_error(ctx, MTPX_E_CAPACITY, "too many rows and heads for one launch");
    const size_t size = dtype_bytes(r.dtype);
    const bool q = sq.total_q > 0, k = sq.total_k > 0;
    if (q) {
        MTPX_TRY(check_rows(ctx, r.q, r.dtype, "q"));
        MTPX_TRY(check_rows(ctx, r.out, r.dtype, "out"));
    }
    if (k) {
        MTPX_TRY(check_rows(ctx, r.k, r.dtype, "k"));
        MTPX_TRY(check_rows(ctx, r.v, r.dtype, "v"));
    }
    MTPX_TRY(check_flat(ctx, r.lambda, 4, "lambda"));
    if ((r.lse != nullptr) != (r.out1 != nullptr))
        return invalid(ctx, "lse and out1 are kept together");
    if (r.lse) {
        MTPX_TRY(check_flat(ctx, r.lse, 4, "lse"));
        MTPX_TRY(check_flat(ctx, r.out1, size, "out1"));
    }
    bool vec = r.dim * size % 16 == 0 && (!r.out1 || aligned(r.out1, 16));
    auto also = [&](const mtpx_rows &t) { vec = vec && (!t.data || whole_pieces(t, size)); };
    for (const mtpx_rows *t : {&r.q, &r.k, &r.v, &r.out})
        also(*t);
    if (back) {
        if (q) {
            MTPX_TRY(check_rows(ctx, r.dout, r.dtype, "dout"));
            MTPX_TRY(check_rows(ctx, r.dq, r.dtype, "dq"));
            if (!r.lse)
                return invalid(ctx, "null lse and out1");
        }
        if (k) {
            MTPX_TRY(check_rows(ctx, r.dk, r.dtype, "dk"));
            MTPX_TRY(check_rows(ctx, r.dv, r.dtype, "dv"));
        }
        MTPX_TRY(check_flat(ctx, r.dlambda, 4, "dlambda"));
        for (const mtpx_rows *t : {&r.dout, &r.dq, &r.dk, &r.dv})
            also(*t);
    }
    a.tiles = sq.table;
    a.heads = r.heads;
    a.kv_heads = r.kv_heads;
    a.dim = r.dim;
    a.causal = r.causal != 0;
    a.total_q = sq.total_q;
    a.total_k = sq.total_k;
    a.scale = r.scale;
    a.q = r.q;
    a.k = r.k;
    a.v = r.v;
    a.out = r.out;
    a.dout = r.dout;
    a.dq = r.dq;
    a.dk = r.dk;
    a.dv = r.dv;
    a.mask = r.key_mask;
    a.lambda = r.lambda;
    a.out1 = r.out1;
    a.lse = r.lse;
    a.delta = a.dlam_part = nullptr;
    a.dlambda = r.dlambda;
    a.vec = vec;
    return MTPX_OK;
}

// Workgroups that share one sequence's keys: one where its waves (eight, or as
// many as their tiles of V leave room for) have no more than four steps of 32
// keys each, as a second launch costs as much, or not many more and every CU
// has two workgroups (200 caches of 1,000 rows of 8 heads, 128 wide, in 16
// bits: 295 us so, 349 us in two splits); else enough to fill the device, each
// with a step per wave at least (2 caches of 946 rows of 8 heads, 40 wide, in
// 32 bits: 18 us, 59 us in one).
int cache_splits(mtpx_context *ctx, const mtpx_diff_attention_cache_request &r)
{
    const int width = r.dim <= 32 ? 32 : r.dim <= 64 ? 64 : 128, group = r.heads / r.kv_heads;
    const int64_t base = std::max<int64_t>((int64_t)r.sequences * r.kv_heads * ((group + 15) / 16), 1);
    const int waves = std::min(8, 1024 / (width * (r.dtype == MTPX_F32 ? 4 : 2)));
    if (r.capacity <= (base >= 2 * (int64_t)ctx->num_cus ? 8 : waves) * 4 * 32)
        return 1;
    const int64_t most = (r.capacity + 127) / 128;
    const int64_t want = (8 * (int64_t)ctx->num_cus + base - 1) / base;
    return (int)std::min<int64_t>({want, most, (int64_t)kMaxSplits});
}

int check_cache(mtpx_context *ctx, const mtpx_diff_attention_cache_request &r)
{
    MTPX_TRY(check_heads(ctx, r.dtype, r.heads, r.kv_heads, r.dim, r.scale));
    if (r.sequences < 0 || r.capacity < 0)
        return invalid(ctx, "negative count");
    if (r.sequences > 65535 || r.heads > 65535)
        return set_error(ctx, MTPX_E_CAPACITY, "more than 65535 sequences or heads");
    return MTPX_OK;
}
size_t cache_bytes(mtpx_context *ctx, const mtpx_diff_attention_cache_request &r)
{
    const int width = r.dim <= 32 ? 32 : r.dim <= 64 ? 64 : 128, splits = cache_splits(ctx, r);
    return splits == 1 ? 0 : sizeof(float) * 2 * (size_t)r.sequences * r.heads * splits * (2 + 2 * width);
}

int check_norm(mtpx_context *ctx, const mtpx_norm_block_request &r)
{
    if (!is_dtype(r.dtype))
        return invalid(ctx, "dtype must be MTPX_F32, MTPX_BF16 or MTPX_F16");
    if (r.rows < 0 || r.width < 1)
        return invalid(ctx, "rows must not be negative and width positive");
    if (r.width > 16384 || r.rows > kMaxRows)
        return set_error(ctx, MTPX_E_CAPACITY, "width beyond 16384 or too many rows");
    if (r.kind != MTPX_NORM_RMS && r.kind != MTPX_NORM_LAYER)
        return invalid(ctx, "unknown norm kind");
    if (r.gate_act < MTPX_GATE_NONE || r.gate_act > MTPX_GATE_TANH)
        return invalid(ctx, "unknown gate activation");
    if (!(r.eps >= 0.f) || !std::isfinite(r.residual_scale) || !std::isfinite(r.block_scale))
        return invalid(ctx, "eps must not be negative and the scales finite");
    for (int64_t s : {r.x_row, r.y_row, r.gate_row, r.s_row, r.n_row, r.ds_row, r.dn_row, r.dx_row,
                      r.dy_row, r.dgate_row})
        if (s < 0)
            return invalid(ctx, "negative row stride");
    return MTPX_OK;
}

int norm_args(mtpx_context *ctx, const mtpx_norm_block_request &r, bool back, NormArgs &a)
{
    MTPX_TRY(check_norm(ctx, r));
    const size_t size = dtype_bytes(r.dtype);
    bool vec = r.width * size % 16 == 0;
    auto tensor = [&](const void *p, int64_t row, bool need, const char *name) -> int {
        if (!p)
            return need ? invalid(ctx, std::string("null ") + name) : MTPX_OK;
        if (!aligned(p, size))
            return invalid(ctx, std::string(name) + " is not aligned to its elements");
        vec = vec && aligned(p, 16) && row * size % 16 == 0;
        return MTPX_OK;
    };
    const bool rows = r.rows > 0;
    MTPX_TRY(tensor(r.x, r.x_row, false, "x"));
    MTPX_TRY(tensor(r.y, r.y_row, rows, "y"));
    MTPX_TRY(tensor(r.gate, r.gate_row, false, "gate"));
    MTPX_TRY(tensor(r.post_weight, 0, false, "post_weight"));
    MTPX_TRY(tensor(r.pre_weight, 0, false, "pre_weight"));
    if (r.stats && !aligned(r.stats, 16))
        return invalid(ctx, "stats are not aligned to 16 bytes");
    if (!back) {
        MTPX_TRY(tensor(r.s, r.s_row, rows, "s"));
        MTPX_TRY(tensor(r.n, r.n_row, false, "n"));
    } else {
        if (rows && !r.stats)
            return invalid(ctx, "null stats");
        if (r.dgate && !r.gate)
            return invalid(ctx, "dgate without a gate");
        if (r.dx && !r.x)
            return invalid(ctx, "dx without x");
        if (r.dpost_weight && !r.post_weight)
            return invalid(ctx, "dpost_weight without post_weight");
        if (r.dpre_weight && !r.pre_weight)
            return invalid(ctx, "dpre_weight without pre_weight");
        MTPX_TRY(tensor(r.ds, r.ds_row, false, "ds"));
        MTPX_TRY(tensor(r.dn, r.dn_row, false, "dn"));
        MTPX_TRY(tensor(r.dx, r.dx_row, false, "dx"));
        MTPX_TRY(tensor(r.dy, r.dy_row, false, "dy"));
        MTPX_TRY(tensor(r.dgate, r.dgate_row, false, "dgate"));
        for (const void *p : {r.dpost_weight, r.dpre_weight})
            if (!aligned(p, size))
                return invalid(ctx, "a weight gradient is not aligned to its elements");
    }
    a = NormArgs{r.rows, r.width, r.kind, r.gate_act, r.residual_scale, r.block_scale, r.eps,
                 r.x, r.y, r.gate, r.post_weight, r.pre_weight, r.x_row, r.y_row, r.gate_row,
                 r.s, r.n, r.s_row, r.n_row, r.stats, r.ds, r.dn, r.ds_row, r.dn_row,
                 r.dx, r.dy, r.dgate, r.dpost_weight, r.dpre_weight, r.dx_row, r.dy_row,
                 r.dgate_row, nullptr, norm_backward_parts(r.rows, r.width), vec};
    return MTPX_OK;
}

size_t norm_bytes(const mtpx_norm_block_request &r)
{
    return std::max<size_t>(sizeof(float) * 3 * (size_t)norm_backward_parts(r.rows, r.width) * r.width, 16);
}

int check_workspace(mtpx_context *ctx, const void *p, size_t have, size_t need)
{
    if (need == 0)
        return MTPX_OK;
    if (have < need || !p)
        return invalid(ctx, "the workspace holds " + std::to_string(p ? have : 0) + " bytes, " +
                                std::to_string(need) + " are needed");
    if (!aligned(p, 16))
        return invalid(ctx, "the workspace is not aligned to 16 bytes");
    return MTPX_OK;
}

}  // namespace
}  // namespace mtpx

extern "C" {

int mtpx_rotary(mtpx_context *ctx, const mtpx_rotary_request *req)
{
    if (!ctx || !req)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    const mtpx_rotary_request &r = *req;
    if (!is_dtype(r.dtype))
        return invalid(ctx, "dtype must be MTPX_F32, MTPX_BF16 or MTPX_F16");
    if (r.rows < 0 || r.heads < 1 || r.dim < 1)
        return invalid(ctx, "rows must not be negative, heads and dim positive");
    if (r.dim > 1024 || r.rows > kMaxRows)
        return set_error(ctx, MTPX_E_CAPACITY, "dim beyond 1024 or too many rows");
    if (r.rotated < 0 || r.rotated > r.dim || r.rotated % 2 != 0)
        return invalid(ctx, "rotated must be even and at most dim");
    if (r.axes < 1 || r.axes > 8)
        return invalid(ctx, "axes must be 1 to 8");
    if (r.position_dtype != MTPX_F32 && r.position_dtype != MTPX_F64 &&
        r.position_dtype != MTPX_I32 && r.position_dtype != MTPX_I64)
        return invalid(ctx, "unknown position_dtype");
    if (r.position_row < 0 || r.position_axis < 0)
        return invalid(ctx, "negative position stride");
    const size_t psize = r.position_dtype == MTPX_F32 || r.position_dtype == MTPX_I32 ? 4 : 8;
    if (r.dpositions) {
        if (!r.inverse)
            return invalid(ctx, "dpositions needs inverse");
        if (r.position_dtype != MTPX_F32 && r.position_dtype != MTPX_F64)
            return invalid(ctx, "integer positions have no gradient");
    }
    if (r.rows == 0)
        return MTPX_OK;
    MTPX_TRY(check_rows(ctx, r.x, r.dtype, "x"));
    MTPX_TRY(check_rows(ctx, r.y, r.dtype, "y"));
    MTPX_TRY(check_flat(ctx, r.positions, psize, "positions"));
    if (r.rotated > 0) {
        MTPX_TRY(check_flat(ctx, r.freq, 4, "freq"));
        MTPX_TRY(check_flat(ctx, r.axis, 4, "axis"));
    }
    if (r.dpositions) {
        MTPX_TRY(check_rows(ctx, r.forward, r.dtype, "forward"));
        MTPX_TRY(check_flat(ctx, r.dpositions, psize, "dpositions"));
    }
    if (r.y.data == r.x.data && (r.y.row != r.x.row || r.y.head != r.x.head))
        return invalid(ctx, "y in the place of x needs its strides");
    // the widest access that every piece of a row allows
    const int64_t size = (int64_t)dtype_bytes(r.dtype), half = r.rotated / 2;
    int width = (int)(16 / size);
    auto fits = [&](const mtpx_rows &t) {
        return aligned(t.data, width * size) && t.row % width == 0 && t.head % width == 0;
    };
    while (width > 1 && !((r.interleaved ? r.rotated : half) % width == 0 &&
                          (r.dim - r.rotated) % width == 0 && fits(r.x) && fits(r.y) &&
                          (!r.dpositions || fits(r.forward))))
        width /= 2;
    RotaryArgs a{r.rows, r.heads, r.dim, r.rotated, r.interleaved != 0, r.inverse != 0, r.axes,
                 r.position_dtype, r.x, r.y, r.forward, r.positions, r.position_row,
                 r.position_axis, r.freq, r.axis, r.dpositions, width, 0};
    // a row gets a lane per piece, or as few as its pairs' table allows
    const int64_t unit = r.interleaved && width > 1 ? width / 2 : width;
    const int64_t pieces = (half / unit + (r.dim - r.rotated) / width) * r.heads;
    a.lanes = 64;
    while (a.lanes > 4 && a.lanes / 2 >= pieces && half * (128 / a.lanes) <= 512)
        a.lanes /= 2;
    OnDevice here(ctx->device);
    HIP_TRY(launch_rotary(r.dtype, a, (hipStream_t)r.stream), "launch rotary");
    return MTPX_OK;
}

int mtpx_sequences_create(mtpx_context *ctx, int n, const int64_t *q_offsets,
                          const int64_t *k_offsets, mtpx_sequences **out)
{
    if (!ctx || !out)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    *out = nullptr;
    if (n < 0 || !q_offsets)
        return invalid(ctx, "sequences need a count and offsets");
    const int64_t *ko = k_offsets ? k_offsets : q_offsets;
    if (q_offsets[0] != 0 || ko[0] != 0)
        return invalid(ctx, "offsets start at 0");
    for (int i = 0; i < n; ++i) {
        if (q_offsets[i + 1] < q_offsets[i] || ko[i + 1] < ko[i])
            return invalid(ctx, "offsets must ascend");
        if (q_offsets[i + 1] - q_offsets[i] > kMaxLength || ko[i + 1] - ko[i] > kMaxLength)
            return set_error(ctx, MTPX_E_CAPACITY, "a sequence of more than 2^30 rows");
    }
    // what a launch cannot take is refused before its tables are built
    for (const int64_t *o : {q_offsets, ko})
        for (int64_t rows : kTileRows) {
            int64_t tiles = 0;
            for (int i = 0; i < n; ++i)
                tiles += (o[i + 1] - o[i] + rows - 1) / rows;
            if (tiles > kMaxGroups)
                return set_error(ctx, MTPX_E_CAPACITY, "too many rows for one launch");
        }
    mtpx_sequences *sq = nullptr;
    try {
        sq = new mtpx_sequences;
        sq->device = ctx->device;
        sq->n = n;
        sq->total_q = q_offsets[n];
        sq->total_k = ko[n];
        // the tiles with the most work first: they start while there is other
        // work to fill the device's last round with
        std::vector<SeqTile> all;
        size_t first[4], count[4];
        for (int side = 0; side < 2; ++side)
            for (int j = 0; j < 2; ++j) {
                std::vector<SeqTile> t;
                for (int i = 0; i < n; ++i) {
                    const int nq = (int)(q_offsets[i + 1] - q_offsets[i]), nk = (int)(ko[i + 1] - ko[i]);
                    for (int64_t s = 0; s < (side ? nk : nq); s += kTileRows[j])
                        t.push_back(SeqTile{q_offsets[i], ko[i], nq, nk, (int)s});
                }
                std::stable_sort(t.begin(), t.end(), [&](const SeqTile &a, const SeqTile &b) {
                    const int la = side ? a.nq : a.nk, lb = side ? b.nq : b.nk;
                    // with causal rows the last queries and the first keys have the most
                    return la != lb ? la > lb : side ? a.start < b.start : a.start > b.start;
                });
                first[2 * side + j] = all.size();
                count[2 * side + j] = t.size();
                all.insert(all.end(), t.begin(), t.end());
            }
        OnDevice here(ctx->device);
        retired().free(ctx->device);
        hipError_t e = upload(sq->tiles, all, ctx->stream);
        if (e == hipSuccess)
            e = hipStreamSynchronize(ctx->stream);
        if (e != hipSuccess) {
            delete sq;
            return hip_fail(ctx, e, "upload sequences");
        }
        for (int i = 0; i < n; ++i) {
            sq->table.longest_q = std::max(sq->table.longest_q, (int)(q_offsets[i + 1] - q_offsets[i]));
            sq->table.longest_k = std::max(sq->table.longest_k, (int)(ko[i + 1] - ko[i]));
        }
        for (int j = 0; j < 2; ++j) {
            sq->table.q[j] = sq->tiles.as<SeqTile>() + first[j];
            sq->table.k[j] = sq->tiles.as<SeqTile>() + first[2 + j];
            sq->table.nq[j] = (int)count[j];
            sq->table.nk[j] = (int)count[2 + j];
        }
    } catch (const std::exception &) {
        delete sq;
        return set_error(ctx, MTPX_E_ALLOC, "out of host memory");
    }
    *out = sq;
    return MTPX_OK;
}

void mtpx_sequences_destroy(mtpx_sequences *seqs)
{
    if (!seqs)
        return;
    try {
        if (seqs->tiles.p)
            retired().add(seqs->device, seqs->tiles.p);
    } catch (const std::exception &) {  // no room to note it: left allocated
    }
    seqs->tiles.p = nullptr;
    delete seqs;
}

int mtpx_diff_attention(mtpx_context *ctx, const mtpx_diff_attention_request *req)
{
    if (!ctx || !req)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    AttnArgs a{};
    MTPX_TRY(attn_args(ctx, *req, false, a));
    if (a.total_q == 0)
        return MTPX_OK;
    OnDevice here(ctx->device);
    HIP_TRY(launch_attn_forward(req->dtype, a, (hipStream_t)req->stream), "launch attention");
    return MTPX_OK;
}

int mtpx_diff_attention_workspace(mtpx_context *ctx, const mtpx_diff_attention_request *req,
                                  size_t *bytes)
{
    if (!ctx || !req || !bytes)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    MTPX_TRY(check_heads(ctx, req->dtype, req->heads, req->kv_heads, req->dim, 1.f));
    if (!req->sequences)
        return invalid(ctx, "null sequences");
    *bytes = attn_workspace(ctx, *req).total;
    return MTPX_OK;
}

int mtpx_diff_attention_backward(mtpx_context *ctx, const mtpx_diff_attention_request *req)
{
    if (!ctx || !req)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    AttnArgs a{};
    MTPX_TRY(attn_args(ctx, *req, true, a));
    const AttnSizes w = attn_workspace(ctx, *req);
    MTPX_TRY(check_workspace(ctx, req->workspace, req->workspace_bytes, w.total));
    a.delta = static_cast<float *>(req->workspace);
    a.dlam_part = a.delta + w.delta / sizeof(float);
    a.kv_parts = key_parts(ctx, *req);
    a.kv_part = a.dlam_part + w.part / sizeof(float);
    OnDevice here(ctx->device);
    HIP_TRY(launch_attn_backward(req->dtype, a, (hipStream_t)req->stream), "launch attention gradient");
    return MTPX_OK;
}

int mtpx_diff_attention_cache_workspace(mtpx_context *ctx,
                                        const mtpx_diff_attention_cache_request *req, size_t *bytes)
{
    if (!ctx || !req || !bytes)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    mtpx_diff_attention_cache_request r = *req;
    r.scale = 1.f;
    MTPX_TRY(check_cache(ctx, r));
    *bytes = cache_bytes(ctx, r);
    return MTPX_OK;
}

int mtpx_diff_attention_cache(mtpx_context *ctx, const mtpx_diff_attention_cache_request *req)
{
    if (!ctx || !req)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    const mtpx_diff_attention_cache_request &r = *req;
    MTPX_TRY(check_cache(ctx, r));
    if (r.sequences == 0)
        return MTPX_OK;
    MTPX_TRY(check_rows(ctx, r.q, r.dtype, "q"));
    MTPX_TRY(check_rows(ctx, r.out, r.dtype, "out"));
    if (r.capacity > 0) {
        MTPX_TRY(check_rows(ctx, r.k, r.dtype, "k"));
        MTPX_TRY(check_rows(ctx, r.v, r.dtype, "v"));
        if (r.k_sequence < 0 || r.v_sequence < 0)
            return invalid(ctx, "negative sequence stride");
    }
    MTPX_TRY(check_flat(ctx, r.lengths, 4, "lengths"));
    MTPX_TRY(check_flat(ctx, r.lambda, 4, "lambda"));
    MTPX_TRY(check_workspace(ctx, r.workspace, r.workspace_bytes, cache_bytes(ctx, r)));
    const size_t size = dtype_bytes(r.dtype);
    const bool vec = r.dim * size % 16 == 0 && whole_pieces(r.q, size) && whole_pieces(r.k, size) &&
                     whole_pieces(r.v, size) && r.k_sequence * size % 16 == 0 &&
                     r.v_sequence * size % 16 == 0;
    CacheArgs a{r.sequences, r.heads, r.kv_heads, r.dim, cache_splits(ctx, r), r.capacity,
                r.k_sequence, r.v_sequence, r.scale, r.q, r.k, r.v, r.out, r.lengths, r.lambda,
                static_cast<float *>(r.workspace), vec};
    OnDevice here(ctx->device);
    HIP_TRY(launch_attn_cache(r.dtype, a, (hipStream_t)r.stream), "launch cache attention");
    return MTPX_OK;
}

int mtpx_norm_block(mtpx_context *ctx, const mtpx_norm_block_request *req)
{
    if (!ctx || !req)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    NormArgs a;
    MTPX_TRY(norm_args(ctx, *req, false, a));
    OnDevice here(ctx->device);
    HIP_TRY(launch_norm_forward(req->dtype, a, (hipStream_t)req->stream), "launch norm block");
    return MTPX_OK;
}

int mtpx_norm_block_workspace(mtpx_context *ctx, const mtpx_norm_block_request *req, size_t *bytes)
{
    if (!ctx || !req || !bytes)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    MTPX_TRY(check_norm(ctx, *req));
    *bytes = norm_bytes(*req);
    return MTPX_OK;
}

int mtpx_norm_block_backward(mtpx_context *ctx, const mtpx_norm_block_request *req)
{
    if (!ctx || !req)
        return set_error(ctx, MTPX_E_INVALID, "null argument");
    NormArgs a;
    MTPX_TRY(norm_args(ctx, *req, true, a));
    MTPX_TRY(check_workspace(ctx, req->workspace, req->workspace_bytes, norm_bytes(*req)));
    a.part = static_cast<float *>(req->workspace);
    OnDevice here(ctx->device);
    HIP_TRY(launch_norm_backward(req->dtype, a, (hipStream_t)req->stream), "launch norm block gradient");
    return MTPX_OK;
}

}  // extern "C"
