// Differential attention of each sequence's new rows over a paged cache
// (mtpx_diff_attention_paged),
//
//   out = (P_0 - lambda P_1) V,   P_m = softmax(scale Q_m K_m^T).
//
// The heads of a group read the same keys, so a sequence's m rows and the g
// heads of a group are m g columns of one product: column x is row x / g, head
// x % g.  A unit of the work is a tile of columns of one sequence and group,
// with the keys that they see.  A few columns (a decoding step) are bound by the
// reads of the cache, many (a prompt's chunk) by the matrix units: there are
// narrow and wide tiles.  Where units are many, a workgroup takes one; where they
// are few or unlike, the workgroups that the device holds at once share all
// units' keys evenly (Shares), and paged_join joins the runs of a unit that
// several of them have (one row of 997 keys, 8 heads of 32: 10 us, 18.5 us a unit
// each; of 32,000: 31 and 454 us).
//
// Compiled once per element type (MTPX_OPS_TYPE).
#include "paged_device.hpp"

namespace mtpx {

namespace {

#if MTPX_OPS_TYPE == 0
typedef float Type;
#define MTPX_OPS_NAME(f) f##_f32
#elif MTPX_OPS_TYPE == 1
typedef __bf16 Type;
#define MTPX_OPS_NAME(f) f##_bf16
#else
typedef _Float16 Type;
#define MTPX_OPS_NAME(f) f##_f16
#endif

// A row's exponentials are taken relative to a level (in powers of two) that
// is renewed, and the row's products rescaled, only when a score passes it by
// this much: exp2 then stays below 2^8, within every type's range.  kNoLevel,
// the level of a row that has seen no key, is passed by every finite score.
constexpr float kSlack = 8.f, kNoLevel = -3.0e38f;

// n / d for n below 2^31, by what the host has made of d.
__device__ inline int quotient(int n, const Divisor &d) { return (int)(__umulhi(2u * (unsigned)n, d.magic) >> d.shift); }

// One sequence's place in the batch and in the cache.
struct Sequence {
    int first, rows;    // of the batch (below 0: the offsets do not ascend here)
    int length, shift;  // keys; row j sees those up to shift + j (causal)

    __device__ inline Sequence() : first(0), rows(0), length(0), shift(0) {}
    __device__ inline Sequence(const PagedArgs &a, int i)
    {
        first = row_offset(a.offsets, i, a.rows);
        rows = row_offset(a.offsets, i + 1, a.rows) - first;
        const int given = max(0, a.lengths[i]);
        length = min(given, a.cache.table_width * a.cache.page_rows);
        shift = given - rows;
    }
    // Lane `lane`'s, in all lanes.
    __device__ inline Sequence of_lane(int lane) const
    {
        Sequence s;
        s.first = __builtin_amdgcn_readlane(first, lane);
        s.rows = __builtin_amdgcn_readlane(rows, lane);
        s.length = __builtin_amdgcn_readlane(length, lane);
        s.shift = __builtin_amdgcn_readlane(shift, lane);
        return s;
    }
    // Keys that columns up to `last` see.
    __device__ inline int keys(const PagedArgs &a, int last) const
    {
        return a.causal ? max(0, min(length, shift + quotient(last, a.group) + 1)) : length;
    }
};

// Floats of a partial result of one column and map: level, sum, -, -, product.
template <int D>
constexpr int kPart = 4 + 2 * D;

// What kernels of one width of tiles are told apart by: sequences of up to
// a.narrow_columns columns have one narrow tile, the others wide ones.  (Columns:
// below 2^23, as rows and heads are.)
template <int COLS, int KB>
struct Role {
    // what a unit takes to begin, in steps of KB keys
    static constexpr int kStart = 128 / KB;
    const RoleArgs &r;
    bool narrow;

    __device__ inline int tiles(const PagedArgs &a, const Sequence &sq) const
    {
        const int columns = sq.rows * a.heads_each;
        return columns > 0 && (columns <= a.narrow_columns) == narrow ? (columns + COLS - 1) / COLS : 0;
    }
    // The steps of tile t.
    __device__ inline int steps(const PagedArgs &a, const Sequence &sq, int t) const
    {
        return (sq.keys(a, min((t + 1) * COLS, sq.rows * a.heads_each) - 1) + KB - 1) / KB;
    }
    __device__ inline int cost(const PagedArgs &a, const Sequence &sq, int t) const
    {
        return tile_costs(a.causal, sq.length, sq.rows, sq.shift, a.heads_each, COLS, KB, kStart, t);
    }
};

// Inclusive sums, or the like, over a wave: shifts within rows of 16 lanes, then
// from row to row (0 comes in).
template <class Op>
__device__ inline int wave_scan(int v, const Op &op)
{
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // row_shr:1
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // row_bcast:15
    return op(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // row_bcast:31
}
__device__ inline int wave_scan(int v)
{
    return wave_scan(v, [](int x, int y) { return x + y; });
}

// The units of one key head lie one after the other on a line of costs, tile by
// tile and sequence by sequence, the key heads behind one another; workgroup w
// takes what lies from w `each` on.  Built by a whole workgroup, for up to 64 runs
// of 64 sequences (of more than one run, the sums before each lie in LDS).  Costs
// are 32-bit numbers, which the host has made sure of for offsets that ascend: of
// others the line is empty.
struct Line {
    int before[kWave];
};
// Where the tiles are no more than the workgroups and the longest takes no more
// than an even share with its part of writing and joining partial results, a
// workgroup takes a tile: a tile costs 1 then.
struct Costs {
    int head, total, each;  // of a key head, of all, of a workgroup
    bool whole;             // tiles
};
template <class R>
struct Shares {
    const PagedArgs &a;
    const R &role;
    Line &line;
    Costs costs{0, 0, 0, false};
    int lane;
    // the lane's sequence of a run of 64, and the costs up to its end and before the run
    int run = -1, upto = 0, own = 0;
    Sequence sq;

    __device__ inline bool single() const { return a.sequences <= kWave; }
    __device__ inline void read(int i)
    {
        if (i == run)
            return;
        run = i;
        const int at = i * kWave + lane;
        sq = Sequence();
        if (at < a.sequences)
            sq = Sequence(a, at);
        const int tiles = role.tiles(a, sq);
        own = costs.whole ? tiles : role.cost(a, sq, tiles);
        upto = wave_scan(own) + (single() ? 0 : line.before[i]);
    }
    // Where the line is there.
    __device__ inline Shares(const PagedArgs &args, const R &r, Line &l, const Costs &c)
        : a(args), role(r), line(l), costs(c), lane(threadIdx.x & (kWave - 1))
    {
    }
    __device__ inline Shares(const PagedArgs &args, const R &r, Line &l)
        : a(args), role(r), line(l), lane(threadIdx.x & (kWave - 1))
    {
        const int wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
        const int groups = role.r.groups;
        if (single()) {
            read(0);
            costs.head = __any(sq.rows < 0) ? 0 : __builtin_amdgcn_readlane(upto, kWave - 1);
            if (!role.narrow) {
                const int n = role.tiles(a, sq);
                const int units = __builtin_amdgcn_readlane(wave_scan(n), kWave - 1) * a.kv_heads;
                const int longest = wave_scan(n > 0 ? role.steps(a, sq, n - 1) : 0, [](int x, int y) { return max(x, y); });
                const int even = (costs.head * a.kv_heads + role.r.split * (units + groups)) / groups;
                if (costs.head > 0 && units <= groups && __builtin_amdgcn_readlane(longest, kWave - 1) + role.kStart <= even) {
                    costs = {units / a.kv_heads, units, 1, true};
                    return;
                }
            }
        } else {
            const int n = (a.sequences + kWave - 1) / kWave;
            for (int i = wave; i < n; i += waves) {
                const int at = i * kWave + lane;
                Sequence s;
                if (at < a.sequences)
                    s = Sequence(a, at);
                const int sum = wave_scan(role.cost(a, s, role.tiles(a, s)));
                const bool astray = __any(s.rows < 0);
                if (lane == kWave - 1)
                    line.before[i] = astray ? -1 : sum;
            }
            __syncthreads();
            const int mine = lane < n ? line.before[lane] : 0, all = wave_scan(mine);
            __syncthreads();
            if (wave == 0)
                line.before[lane] = all - mine;  // (runs beyond the last begin where it ends)
            __syncthreads();
            costs.head = __any(mine < 0) ? 0 : __builtin_amdgcn_readlane(all, kWave - 1);
        }
        costs.total = costs.head * a.kv_heads;
        costs.each = (costs.total + groups - 1) / groups;
    }
    // The sequence at cost p (below costs.head) of a key head, and the cost of those before it.
    __device__ inline int find(int p, Sequence &s, int &start)
    {
        read(single() ? 0 : __popcll(__ballot(line.before[lane] <= p)) - 1);
        const int l = __popcll(__ballot(upto <= p));
        start = __builtin_amdgcn_readlane(upto - own, l);
        s = sq.of_lane(l);
        return run * kWave + l;
    }
    // Sequence i, and the cost of those before it.
    __device__ inline void at(int i, Sequence &s, int &start)
    {
        read(i / kWave);
        start = __builtin_amdgcn_readlane(upto - own, i % kWave);
        s = sq.of_lane(i % kWave);
    }
};

__device__ inline int page_of(const PagedArgs &a, int key) { return quotient(key, a.page); }
__device__ inline bool there(const PagedArgs &a, int page) { return page >= 0 && page < a.cache.pages; }

// The way of a tile of keys and values from the pages straight into LDS, by W
// waves.  look_up() reads the table for a tile, one tile ahead of fetch().
// Any pages: lane l looks up key l of the tile, and every wave's instruction fills
// kGroup rows of it from where those lanes say.
template <class T, int D, int ROWS, int W, bool FAST>
struct TileLoader {
    using TL = Tile<T, D>;
    static constexpr int kGroup = 1024 / TL::kRowBytes;
    static constexpr int N = ROWS / (kGroup * W);
    static_assert(N * kGroup * W == ROWS, "rows of a tile");
    const PagedArgs &a;
    const int *table;
    int kv, lane, wave, page = -1, first = 0;

    __device__ inline TileLoader(const PagedArgs &args, const int *t, int head, int l, int w)
        : a(args), table(t), kv(head), lane(l), wave(w)
    {
    }
    __device__ inline void look_up(int k0, int end)
    {
        first = k0;
        page = k0 + lane < end ? table[page_of(a, k0 + lane)] : -1;
    }
    // Returns which of the tile's keys are there; the others become zeros.
    __device__ inline unsigned long long fetch(char *smem, int k_tile, int v_tile)
    {
        const unsigned long long seen = __ballot(there(a, page)) & ~0ull >> (64 - ROWS);
        const int slot = first + lane - page_of(a, first + lane) * a.cache.page_rows;
        auto half = [&](const mtpx_rows &s, int64_t stride, int tile) {
            const int64_t mine = there(a, page) ? (int64_t)(unsigned)page * stride + (int64_t)(unsigned)slot * s.row : 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r0 = (i * W + wave) * kGroup, r = r0 + lane / TL::kPieces;
                const int col = ((lane % TL::kPieces) ^ (r & 7)) * TL::E, c = col % D, to = tile + r0 * TL::kRowBytes;
                const T *p = (const T *)s.data + kv * s.head + (int64_t)__shfl((long long)mine, r) + col / D * s.map + c;
                const bool on = (seen >> r & 1) && c < a.dim;
                if (a.vec)
                    load_to_lds(on ? (const void *)p : (const void *)&kZeroPiece, to);
                else
                    *reinterpret_cast<u32x4 *>(smem + to + lane * 16) = load16(p, on ? a.dim - c : 0, 0);
            }
        };
        half(a.cache.k, a.cache.k_page, k_tile);
        half(a.cache.v, a.cache.v_page, v_tile);
        return seen;
    }
};

// 16 bytes per lane straight into LDS as load_to_lds(), from the same address in
// all lanes and an offset of each.
__device__ inline void load_lanes_to_lds(const void *p, unsigned lane_offset, unsigned offset)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane_offset), "s"(p), "{m0}"(offset) : "memory");
}

// FAST: rows of whole 16-byte pieces, keys and values laid out alike, pages of
// whole runs of kGroup rows, which one load of a wave brings.  Lane l forms the
// address of key l once for keys and values, a load begins where the first of its
// rows lies, and the lanes keep their offsets from there: the vector unit has the
// softmax to do (a chunk of 2,048 rows of 32,000, 16 heads of 64: 795 us, 920 us
// through the other loader; 46 single rows and two chunks of 727, heads of 128: 294
// and 391 us; a chunk of 1,024 rows of 8,192 in pages of 24, 32 heads of 64: 221 and
// 263 us.  Addresses of whole runs of a wave by the scalar unit alone take 1 to 2 %
// less, and leave such pages to the other loader).
template <class T, int D, int ROWS, int W>
struct TileLoader<T, D, ROWS, W, true> {
    using TL = Tile<T, D>;
    static constexpr int kGroup = 1024 / TL::kRowBytes, kRun = ROWS / W, N = kRun / kGroup;
    static_assert(N * kGroup == kRun && kRun % 8 == 0, "rows of a wave");
    static constexpr int kColumns = kGroup >= 8 ? 1 : 8 / kGroup < N ? 8 / kGroup : N;  // the permutation's phases
    const PagedArgs &a;
    const int *table;
    const char *k, *v;
    int lane, wave, first = 0, page = -1;
    unsigned offset[kColumns];

    __device__ inline int column(int i) const
    {
        return ((lane % TL::kPieces) ^ ((i * kGroup + lane / TL::kPieces) & 7)) * TL::E;
    }
    __device__ inline TileLoader(const PagedArgs &args, const int *t, int kv, int l, int w) : a(args), table(t), lane(l), wave(w)
    {
        k = (const char *)((const T *)a.cache.k.data + kv * a.cache.k.head);
        v = (const char *)((const T *)a.cache.v.data + kv * a.cache.v.head);
#pragma unroll
        for (int i = 0; i < kColumns; ++i)
            offset[i] = (unsigned)(lane / TL::kPieces * (int)a.cache.k.row + column(i) / D * (int)a.cache.k.map + column(i) % D) *
                        (unsigned)sizeof(T);
    }
    __device__ inline void look_up(int k0, int end)
    {
        first = k0;
        page = k0 + lane < end ? table[page_of(a, k0 + lane)] : -1;
    }
    __device__ inline unsigned long long fetch(char *, int k_tile, int v_tile)
    {
        const unsigned long long seen = __ballot(there(a, page)) & ~0ull >> (64 - ROWS);
        const int slot = first + lane - page_of(a, first + lane) * a.cache.page_rows;
        const uint64_t at = (uint64_t)(unsigned)page * (uint64_t)(a.cache.k_page * (int64_t)sizeof(T)) +
                            (uint64_t)(unsigned)slot * ((unsigned)a.cache.k.row * (unsigned)sizeof(T));
        uint64_t begins[N];  // of a load's rows
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int l = wave * kRun + i * kGroup;
            begins[i] = (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(at >> 32), l) << 32 |
                        (unsigned)__builtin_amdgcn_readlane((int)at, l);
        }
        const unsigned mine = (unsigned)(seen >> (wave * kRun)) & ~0u >> (32 - kRun);
        const bool all = mine == ~0u >> (32 - kRun) && a.dim == D;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const char *from = half ? v : k;
            const int to = (half ? v_tile : k_tile) + wave * kRun * TL::kRowBytes;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const char *p = from + begins[i];
                if (all) {
                    load_lanes_to_lds(p, offset[i % kColumns], to + i * 1024);
                    continue;
                }
                const bool on = (mine >> (i * kGroup + lane / TL::kPieces) & 1) && column(i % kColumns) % D < a.dim;
                load_to_lds(on ? (const void *)(p + offset[i % kColumns]) : (const void *)&kZeroPiece, to + i * 1024);
            }
        }
        return seen;
    }
};

// Rounds per-lane column results 16 t + 4 (l / 16) + r, of width 2 D, to the
// row that lane l % 16 stands for.
template <class T, int D>
__device__ inline void store_columns(T *row, int64_t map, int dim, int t, int lane, f32x4 v, int vec)
{
    const int m = t * 16 / D, c = t * 16 % D + 4 * (lane >> 4);
    store4(row + m * map, c, dim, v, vec);
}

// A run of a unit's keys: steps [begin, end) of `steps` of KB keys each; all of
// them give the result, others a partial one.
struct Segment {
    int kv, begin, end, steps;
    int x0;  // first column of the tile
    float *part;
    const int *table;
};

// Keys and values come in tiles of KB rows, the next one while the present one is
// worked on (BUF 2).  S^T = K Q^T leaves a column of the product per lane column:
// its running level and sum are per lane, and exp(S^T), rounded to T, is operand B
// of O^T += V^T P^T as it stands (in 16-bit types results are off by 0.0023 of their
// size in bf16 and 0.0003 in f16, where one rounding is 0.0017 and 0.0002; the sum
// is of the 32-bit exponentials).  The two maps keep their own level, sum and
// product.
//
// A wave has QT 16 columns and both maps, which share each fragment of V read
// from LDS (M 2); or two waves share the columns, a map each (M 1).  A wave of
// wide heads has registers for 16 columns of two maps or 32 of one: those read
// 24 KiB of LDS for what takes the former 32 KiB (D 128, 32 keys).
//
// Wide tiles are bound by the matrix units and what their waves wait for between
// products.  A pair of row and key takes 8 D operations by the formula, 12 D here,
// where each map has its own product with V, as its sum is known at the end only: 8
// prompts of 2,500 to 6,000 rows, 16 heads of 64, take 985 us (960 us on another
// card), 580 TFLOP/s of the former and 865 of the latter; a chunk of 2,048 rows of
// 32,000 takes 795 us, 655 and 980 TFLOP/s.  (A plain product of two large matrices reaches 1,140 TFLOP/s.)  Narrow tiles are bound by the reads of the cache: 64 rows
// against up to 8,192 keys each, 32 heads of 64 on 4, take 150 us, 5.2 TB/s.
template <class T, int D, int W, int M, int QT, int KB, int BUF, bool FAST>
__device__ inline void attend(const PagedArgs &a, const Sequence &sq, const Segment &sg, char *smem)
{
    using TL = Tile<T, D>;
    constexpr int kTile = KB * TL::kRowBytes, kCols = W * M / 2 * QT * 16;
    constexpr unsigned long long kFull = ~0ull >> (64 - KB);
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m0 = M == 2 ? 0 : wave & 1, part = M == 2 ? wave : wave >> 1;
    const int group = a.heads_each, kv = sg.kv, columns = sq.rows * group, x0 = sg.x0;
    const int nk = sq.keys(a, min(x0 + kCols, columns) - 1);
    const int run_begin = sg.begin * KB, run_end = min(nk, sg.end * KB);

    TileLoader<T, D, KB, W, FAST> tiles(a, sg.table, kv, lane, wave);
    tiles.look_up(run_begin, run_end);
    const float c = a.scale * kLog2e;
    Reader<T, D> rd;
    rd.init(lane);

    const int w0 = x0 + part * QT * 16;  // first column of the wave
    Frag<T> qf[M][QT][D / 32];
    int last[QT];  // key that the lane's column sees
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int x = w0 + t * 16 + (lane & 15), j = quotient(x, a.group);
        last[t] = a.causal ? sq.shift + j : nk;
        const T *qp = (const T *)a.q.data + (kv * group + x - j * group) * a.q.head + (int64_t)(sq.first + j) * a.q.row;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
                qf[m][t][kk] = load_frag(qp + (m0 + m) * a.q.map, kk * 32 + 8 * g, a.dim, x < columns, FAST || a.vec);
    }
    // keys that the wave's first and last columns see last
    const bool none = w0 >= columns;
    const int low = a.causal ? sq.shift + quotient(w0, a.group) : nk;
    const int high = a.causal ? sq.shift + quotient(max(min(w0 + QT * 16, columns) - 1, 0), a.group) : nk;
    f32x4 acc[M][QT][D / 8];
    float level[M][QT], sum[M][QT];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            level[m][t] = kNoLevel;
            sum[m][t] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                acc[m][t][i] = f32x4{0, 0, 0, 0};
        }

    unsigned long long bits = 0;
    auto load = [&](int k0, int to) {
        bits = tiles.fetch(smem, to * 2 * kTile, to * 2 * kTile + kTile);
        tiles.look_up(k0 + KB, run_end);
    };
    if (run_begin < run_end)
        load(run_begin, 0);
    int buf = 0;
    for (int k0 = run_begin; k0 < run_end; k0 += KB) {
        wait_loads();
        __syncthreads();
        const unsigned long long now = bits;
        const char *kt = smem + buf * 2 * kTile, *vt = kt + kTile;
        auto next = [&] {
            if (k0 + KB < run_end) {
                buf = BUF - 1 - buf;
                load(k0 + KB, buf);
            }
        };
        if constexpr (BUF == 2)
            next();
        const bool idle = now == 0 || none || k0 > high;
        const bool partly = now != kFull || k0 + KB - 1 > low;
        if (!idle) {
#pragma unroll 1
            for (int b = 0; b < KB / 32; ++b) {
                if ((unsigned)(now >> (32 * b)) == 0 || k0 + 32 * b > high)
                    continue;
                f32x4 s[M][2][QT];
                {
                    // u, then map, then columns: one K fragment ahead
                    constexpr int kEach = M * (D / 32), kSteps = 2 * kEach;
                    auto key_frag = [&](int x) {
                        const int r0 = b * 32 + x / kEach * 16, column = x / (D / 32) % M * D + x % (D / 32) * 32;
                        if constexpr (M == 2)
                            return rd.row_frag(kt, r0, column);
                        else if constexpr (D * sizeof(T) % 128 == 0)  // whole runs of 8 pieces
                            return rd.row_frag(kt + m0 * (D * sizeof(T)), r0, column);
                        else
                            return m0 ? rd.row_frag(kt, r0, D + column) : rd.row_frag(kt, r0, column);
                    };
                    Frag<T> kf = key_frag(0);
#pragma unroll
                    for (int x = 0; x < kSteps; ++x) {
                        const int u = x / kEach, m = x / (D / 32) % M, kk = x % (D / 32);
                        Frag<T> following;
                        if (x + 1 < kSteps)
                            following = key_frag(x + 1);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int t = 0; t < QT; ++t)
                            s[m][u][t] = mma(kf, qf[m][t][kk], kk ? s[m][u][t] : f32x4{0, 0, 0, 0});
                        __builtin_amdgcn_sched_barrier(0);
                        kf = following;
                    }
                }
                if (partly) {
                    const unsigned mine = (unsigned)(now >> (32 * b + 4 * g));
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        const int most = last[t] - k0 - 32 * b - 4 * g;
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const bool on = (mine >> (16 * u + r) & 1) && 16 * u + r <= most;
#pragma unroll
                                for (int m = 0; m < M; ++m)
                                    s[m][u][t][r] = on ? s[m][u][t][r] : -INFINITY;
                            }
                    }
                }
                float hi[M][QT];
                bool passed = false;
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        const f32x4 x = s[m][0][t], y = s[m][1][t];
                        hi[m][t] = max3(max3(x[0], x[1], x[2]), max3(x[3], y[0], y[1]), max3(y[2], y[3], y[3]));
                        passed |= fmaf(hi[m][t], c, -level[m][t]) > kSlack;
                    }
                if (__any(passed)) {
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int t = 0; t < QT; ++t) {
                            const float up = fmaxf(level[m][t], column_max(hi[m][t]) * c);
                            const float f = exp2_fast(level[m][t] - up);
                            level[m][t] = up;
                            sum[m][t] *= f;
#pragma unroll
                            for (int i = 0; i < D / 8; ++i)
                                acc[m][t][i] *= f;
                        }
                }
                Frag<T> pf[M][QT];
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        float sums[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float p = exp2_fast(fmaf(s[m][u][t][r], c, -level[m][t]));
                                s[m][u][t][r] = p;
                                sums[u] = r ? sums[u] + p : p;
                            }
                        sum[m][t] += sums[0] + sums[1];
                        pf[m][t] = pack<T>(s[m][0][t], s[m][1][t]);
                    }
                // one V fragment ahead of the products, so that none waits for LDS
                Frag<T> vf = rd.column_frag(vt, b * 32, 0);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    Frag<T> following;
                    if (i + 1 < D / 8)
                        following = rd.column_frag(vt, b * 32, (i + 1) * 16);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int t = 0; t < QT; ++t)
                            acc[m][t][i] = mma(vf, pf[m][t], acc[m][t][i]);
                    __builtin_amdgcn_sched_barrier(0);
                    vf = following;
                }
            }
        }
        if constexpr (BUF == 1) {
            __syncthreads();
            next();
        }
    }

    const bool whole = sg.begin == 0 && sg.end == sg.steps;
    __syncthreads();  // the last tile's reads, before its place takes results or another tile
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int x = w0 + t * 16 + (lane & 15), j = quotient(x, a.group), head = kv * group + x - j * group;
        const int64_t row = sq.first + j;
        float total[M];
#pragma unroll
        for (int m = 0; m < M; ++m)
            total[m] = column_sum(sum[m][t]);
        if (!whole) {
            if (x >= columns)
                continue;
#pragma unroll
            for (int m = 0; m < M; ++m) {
                float *p = sg.part + ((x - x0) * 2 + m0 + m) * kPart<D>;
                if (g == 0) {
                    p[0] = level[m][t];
                    p[1] = total[m];
                }
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    *reinterpret_cast<f32x4 *>(p + 4 + i * 16 + 4 * g) = acc[m][t][i];
            }
            continue;
        }
        float inv[M];
#pragma unroll
        for (int m = 0; m < M; ++m)
            inv[m] = total[m] == 0.f ? 0.f : 1.f / total[m];
        if constexpr (M == 1) {
            // the second map's wave hands its 16 columns to the first's
            float *hand = reinterpret_cast<float *>(smem) + part * (D / 8 * kWave * 4) + lane * 4;
            if (m0 == 1)
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    *reinterpret_cast<f32x4 *>(hand + i * kWave * 4) = acc[0][t][i] * inv[0];
            __syncthreads();
            if (m0 == 0 && x < columns) {
                const float lambda = a.lambda[head];
                T *op = (T *)a.out.data + head * a.out.head + row * a.out.row;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    store_columns<T, D>(op, a.out.map, a.dim, i, lane,
                                        acc[0][t][i] * inv[0] - lambda * *reinterpret_cast<f32x4 *>(hand + i * kWave * 4), FAST || a.vec);
            }
            __syncthreads();
        } else if (x < columns) {
            const float lambda = a.lambda[head];
            T *op = (T *)a.out.data + head * a.out.head + row * a.out.row;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                store_columns<T, D>(op, a.out.map, a.dim, i, lane, acc[0][t][i] * inv[0] - lambda * (acc[M - 1][t][i] * inv[M - 1]),
                                    FAST || a.vec);
        }
    }
}

// The number of the first tile of sequence i among all wide ones: tiles of
// different sequences have different numbers, some none.
template <int COLS>
__device__ inline int tile_number(const PagedArgs &a, int i)
{
    return row_offset(a.offsets, i, a.rows) * a.heads_each / COLS + i;
}

// The work of workgroup `item` of a role: one unit, or the runs of units that lie
// in its share.
template <class T, int D, int W, int M, int QT, int KB, int BUF, bool FAST, bool NARROW>
__device__ inline void work(const PagedArgs &a, int item, char *smem, Line &line)
{
    constexpr int kCols = W * M / 2 * QT * 16;
    const Role<kCols, KB> role{NARROW ? a.narrow : a.wide, NARROW};
    // neighbours on one XCD, whose L2 holds the keys that they share
    const int n = role.r.groups, w = n % 8 ? item : item % 8 * (n / 8) + item / 8;
    Costs costs{0, 0, 0, false};
    if (!role.r.each_unit)
        costs = Shares<Role<kCols, KB>>(a, role, line).costs;
    const int p0 = w * costs.each, p1 = min(p0 + costs.each, costs.total);
    // (one place that works on a unit: a second would cost the first its registers)
    for (int p = p0;;) {
        Segment sg;
        Sequence sq;
        int seq, tile = 0;
        bool any = true, wrong = false;
        if (!role.r.each_unit) {
            if (p >= p1)
                return;
            sg.kv = (int)((unsigned)p / (unsigned)costs.head);
            Shares<Role<kCols, KB>> shares(a, role, line, costs);
            int at;
            seq = shares.find(p - sg.kv * costs.head, sq, at);
            at += sg.kv * costs.head;
            if constexpr (!NARROW)
                tile = costs.whole ? p - at
                                   : __builtin_amdgcn_readfirstlane(last_true(
                                         [&](int t) { return at + role.cost(a, sq, t) <= p; }, role.tiles(a, sq), kWave));
            const int a0 = __builtin_amdgcn_readfirstlane(at + role.cost(a, sq, tile)), keys = a0 + role.kStart;
            sg.steps = role.steps(a, sq, tile);
            sg.begin = max(0, min(sg.steps, p0 - keys));
            sg.end = max(0, min(sg.steps, p1 - keys));
            // a run that begins a unit lies behind one that does not
            sg.part = role.r.part + ((int64_t)w * 2 + (sg.begin == 0)) * kCols * 2 * kPart<D>;
            // a unit without keys has its zeros written where it begins
            any = sg.begin < sg.end || (sg.steps == 0 && p0 <= a0);
            p = __builtin_amdgcn_readfirstlane(at + role.cost(a, sq, tile + 1));
            if (costs.whole) {
                sg.begin = 0;
                sg.end = sg.steps;
                any = true;
                p = p1;
            }
        } else {
            if constexpr (NARROW) {
                seq = item / a.kv_heads;
                sg.kv = item % a.kv_heads;
            } else {
                // the last rows of a causal sequence have the most keys: they go
                // first, of all sequences where those are alike (`level`); else
                // sequence by sequence, whose workgroups then share what L2 holds of
                // its keys, and the first quarter of each behind all others, to
                // fill the end
                const Work wk = work_item(item, role.r.tiles + role.r.quarters, a.kv_heads);
                sg.kv = wk.head;
                const bool late = wk.tile >= role.r.tiles;
                const int at = role.r.tiles - 1 - wk.tile + (late ? role.r.quarters : 0);
                if (role.r.level) {
                    seq = at % a.sequences;
                    tile = at / a.sequences;
                } else {
                    auto number = [&](int i) { return late ? tile_number<4 * kCols>(a, i) : tile_number<kCols>(a, i); };
                    seq = __builtin_amdgcn_readfirstlane(last_true([&](int i) { return number(i) <= at; }, a.sequences, kWave));
                    if (seq < 0)
                        return;
                    tile = at - number(seq);
                    wrong = role.r.quarters > 0 && (tile < (role.tiles(a, Sequence(a, seq)) + 3) / 4) != late;
                }
            }
            sq = Sequence(a, seq);
            if (wrong || tile >= role.tiles(a, sq))
                return;
            sg.begin = 0;
            sg.end = sg.steps = role.steps(a, sq, tile);
            sg.part = nullptr;
        }
        sg.x0 = tile * kCols;
        sg.table = a.cache.table + seq * a.cache.table_row;
        if (any)
            attend<T, D, W, M, QT, KB, BUF, FAST>(a, sq, sg, smem);
        if (role.r.each_unit)
            return;
    }
}

// Joins what several workgroups have left of a unit that begins at cost a0: those
// in whose shares its steps lie.  `pieces` workgroups join a unit.
constexpr int kJoin = 256;
template <class T, int D, class R, int COLS>
__device__ inline void join_unit(const PagedArgs &a, const R &role, const Shares<R> &shares, const Sequence &sq, int kv, int tile,
                                 int a0, int piece, int pieces)
{
    if (shares.costs.total == 0 || shares.costs.whole)
        return;
    const int steps = role.steps(a, sq, tile), keys = a0 + role.kStart;
    const int from = keys / shares.costs.each, upto = (keys + steps - 1) / shares.costs.each;
    if (steps == 0 || from == upto)
        return;  // written already
    const int group = a.heads_each, x0 = tile * COLS, count = min(COLS, sq.rows * group - x0);
    constexpr int kColumn = 2 * kPart<D>;
    constexpr int64_t kSlot = (int64_t)COLS * kColumn;
    for (int e = piece * kJoin + threadIdx.x; e < count * (D / 2); e += pieces * kJoin) {
        const int x = e / (D / 2), y = e % (D / 2) * 4;
        const float *p = role.r.part + from * 2 * kSlot + x * kColumn;
        float hi[2] = {kNoLevel, kNoLevel}, total[2] = {0.f, 0.f};
        f32x4 v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll 4
        for (int i = 0; i <= upto - from; ++i) {
            const float *q = p + (2 * i + (i == 0)) * kSlot;
#pragma unroll
            for (int m = 0; m < 2; ++m, q += kPart<D>) {
                const float level = q[0], up = fmaxf(hi[m], level);
                // (0 for what has seen no key)
                const float f = exp2_fast(hi[m] - up), g = exp2_fast(level - up);
                hi[m] = up;
                total[m] = fmaf(f, total[m], g * q[1]);
                v[m] = f * v[m] + g * *reinterpret_cast<const f32x4 *>(q + 4 + y);
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
            v[m] *= total[m] == 0.f ? 0.f : 1.f / total[m];
        const int j = quotient(x0 + x, a.group), head = kv * group + x0 + x - j * group;
        T *out = (T *)a.out.data + (int64_t)(sq.first + j) * a.out.row + head * a.out.head + y / D * a.out.map;
        store4(out, y % D, a.dim, v[0] - a.lambda[head] * v[1], a.vec);
    }
}

// Tile shapes by head width.
template <class T, int D>
struct Shape {
    static constexpr int kWaves = 4;
    static constexpr int kRows = 2 * D * (int)sizeof(T) <= 256 ? 64 : 32;
    static constexpr size_t kTiles = 2 * (size_t)kRows * 2 * D * sizeof(T);
    // two buffers of both tiles within the 64 KiB that loads into LDS address
    static constexpr int kBuffers = kTiles <= 32768 ? 2 : 1;
    static constexpr size_t kLds = kBuffers * kTiles;
    // maps of a wave and groups of 16 columns: narrow tiles have two waves that
    // work on 16 columns, which keeps them behind the reads of the cache
    static constexpr int kMaps = sizeof(T) == 2 && D <= 64 ? 2 : 1, kGroups = sizeof(T) == 4 && D == 128 ? 1 : 2;
    static constexpr int kNarrow = kWaves / 2 * 16, kWide = kWaves * kMaps / 2 * kGroups * 16;
    static constexpr int kPage = 1024 / (2 * D * (int)sizeof(T));  // rows of a wave's load
};

// Both roles in one launch, the wide tiles first, which take the longest.  (Eight
// workgroups of each in turn, for the reads of one and the products of the other to
// share the CUs, are slower: 48 sequences, two of them with chunks of 727 rows,
// 501 us; 294 us so.)
constexpr int kNarrowOnly = 1, kWideOnly = 2, kBoth = 3;
template <class T, int D, bool FAST, int ROLES>
__global__ __launch_bounds__((Shape<T, D>::kWaves * kWave), 2) void paged_kernel(PagedArgs a)
{
    using S = Shape<T, D>;
    // (the line behind the tiles: loads into LDS count from its start)
    extern __shared__ __align__(16) char smem[];
    Line &line = *reinterpret_cast<Line *>(smem + S::kLds);
    int item = blockIdx.x;
    bool narrow = ROLES == kNarrowOnly;
    if constexpr (ROLES == kBoth) {
        narrow = item >= a.wide.groups;
        if (narrow)
            item -= a.wide.groups;
    }
    if (ROLES != kNarrowOnly && !narrow)
        work<T, D, S::kWaves, S::kMaps, S::kGroups, S::kRows, S::kBuffers, FAST, false>(a, item, smem, line);
    if (ROLES != kWideOnly && narrow)
        work<T, D, S::kWaves, 1, 1, S::kRows, S::kBuffers, FAST, true>(a, item, smem, line);
}

// A workgroup per key head and sequence (narrow), or so many per wide tile.
template <class T, int D>
__global__ __launch_bounds__(kJoin) void paged_join(PagedArgs a, int narrow_items, int pieces)
{
    using S = Shape<T, D>;
    __shared__ Line line;
    int item = blockIdx.x, start;
    Sequence sq;
    if (item < narrow_items) {
        using R = Role<S::kNarrow, S::kRows>;
        const R role{a.narrow, true};
        if (role.tiles(a, Sequence(a, item / a.kv_heads)) == 0)
            return;
        Shares<R> shares(a, role, line);
        const int kv = item % a.kv_heads;
        shares.at(item / a.kv_heads, sq, start);
        join_unit<T, D, R, S::kNarrow>(a, role, shares, sq, kv, 0, kv * shares.costs.head + start, 0, 1);
        return;
    }
    item -= narrow_items;
    using R = Role<S::kWide, S::kRows>;
    const R role{a.wide, false};
    const int piece = item % pieces, kv = item / pieces % a.kv_heads, at = item / pieces / a.kv_heads;
    const int seq = __builtin_amdgcn_readfirstlane(
        last_true([&](int i) { return tile_number<S::kWide>(a, i) <= at; }, a.sequences, kWave));
    if (seq < 0)
        return;
    const int tile = at - tile_number<S::kWide>(a, seq);
    if (tile >= role.tiles(a, Sequence(a, seq)))
        return;
    Shares<R> shares(a, role, line);
    shares.at(seq, sq, start);
    join_unit<T, D, R, S::kWide>(a, role, shares, sq, kv, tile, kv * shares.costs.head + start + role.cost(a, sq, tile), piece, pieces);
}

template <int D, bool FAST>
hipError_t run(const PagedArgs &a, hipStream_t s)
{
    using S = Shape<Type, D>;
    const auto kernel = a.wide.groups == 0     ? paged_kernel<Type, D, FAST, kNarrowOnly>
                        : a.narrow.groups == 0 ? paged_kernel<Type, D, FAST, kWideOnly>
                                               : paged_kernel<Type, D, FAST, kBoth>;
    const hipError_t e = launch_kernel(kernel, dim3((unsigned)(a.narrow.groups + a.wide.groups)), dim3(S::kWaves * kWave),
                                       S::kLds + sizeof(Line), s, a);
    if (e != hipSuccess || (!a.narrow.part && !a.wide.part))
        return e;
    // a thread of a wide tile's join takes four columns of a result, or of two (12
    // sequences of up to 700 rows in 32 bits: 38 us, 41 us of four; of one: a chunk of
    // 128 rows of 4,000 of each of 16 sequences, 32 heads of 64, 218 us, 209 us so)
    constexpr int all = S::kWide * (D / 2) / kJoin, pieces = all < 8 ? all : 8;
    const int narrow_items = a.narrow.part ? a.sequences * a.kv_heads : 0;
    const int64_t wide_items = a.wide.part ? (int64_t)a.wide.tiles * a.kv_heads * pieces : 0;
    return launch_kernel(paged_join<Type, D>, dim3((unsigned)(narrow_items + wide_items)), dim3(kJoin), 0, s, a, narrow_items, pieces);
}
template <int D>
hipError_t by_pages(const PagedArgs &a, hipStream_t s)
{
    return a.alike && a.cache.page_rows % Shape<Type, D>::kPage == 0 ? run<D, true>(a, s) : run<D, false>(a, s);
}

}  // namespace

hipError_t MTPX_OPS_NAME(paged)(const PagedArgs &a, hipStream_t s)
{
    return a.dim <= 32 ? by_pages<32>(a, s) : a.dim <= 64 ? by_pages<64>(a, s) : by_pages<128>(a, s);
}

#if MTPX_OPS_TYPE == 0
hipError_t paged_bf16(const PagedArgs &, hipStream_t);
hipError_t paged_f16(const PagedArgs &, hipStream_t);

hipError_t launch_paged(int dtype, const PagedArgs &a, hipStream_t s)
{
    return dtype == MTPX_F32 ? paged_f32(a, s) : dtype == MTPX_BF16 ? paged_bf16(a, s) : paged_f16(a, s);
}
#endif

}  // namespace mtpx
