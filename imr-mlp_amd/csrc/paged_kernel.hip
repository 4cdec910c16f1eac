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
// several of them have.
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

// One sequence's place in the batch and in the cache.
struct Sequence {
    int first, rows;   // of the batch
    int length, shift; // keys; row j sees those up to shift + j (causal)
    const int *table;

    __device__ inline Sequence(const PagedArgs &a, int i)
    {
        first = row_offset(a.offsets, i, a.rows);
        rows = max(0, row_offset(a.offsets, i + 1, a.rows) - first);
        const int given = max(0, a.lengths[i]);
        length = min(given, a.cache.table_width * a.cache.page_rows);
        shift = given - rows;
        table = a.cache.table + i * a.cache.table_row;
    }
    // Keys that rows up to `last` see.
    __device__ inline int keys(const PagedArgs &a, int last) const
    {
        return a.causal ? max(0, min(length, shift + last + 1)) : length;
    }
};

// Floats of a partial result of one column and map: level, sum, -, -, product.
template <int D>
constexpr int kPart = 4 + 2 * D;

// What kernels of one width of tiles are told apart by: sequences of up to
// a.narrow columns have one narrow tile, the others wide ones.
template <int COLS>
struct Role {
    const RoleArgs &r;
    bool narrow;
    __device__ inline int tiles(const PagedArgs &a, const Sequence &sq) const
    {
        const int64_t columns = (int64_t)sq.rows * (a.heads / a.kv_heads);
        return columns > 0 && (columns <= a.narrow_columns) == narrow ? (int)((columns + COLS - 1) / COLS) : 0;
    }
    // What the first t tiles of a sequence cost: the keys that they see and
    // kStart for each, in units of 2^shift.  (Keys of causal tiles as a mean over
    // their rows: a cost need not be exact, only the same in every workgroup.)
    __device__ inline int cost(const PagedArgs &a, const Sequence &sq, int t) const
    {
        const int before = a.causal ? max(0, sq.length - sq.rows) : sq.length;
        const int64_t slope = a.causal ? (int64_t)t * (t + 1) * COLS / (2 * (a.heads / a.kv_heads)) : 0;
        return t * (start() + (before >> r.shift)) + (int)(slope >> r.shift);
    }
    __device__ inline int start() const { return max(1, 256 >> r.shift); }
};

// Inclusive sums over a wave: shifts within rows of 16 lanes, then from row to row.
__device__ inline int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
}

// The units of one key head lie one after the other on a line of costs, tile by
// tile and sequence by sequence, the key heads behind one another; workgroup w
// takes what lies from w `each` on.  Built by a whole workgroup, for up to 64 runs
// of 64 sequences.
struct Line {
    int before[kWave];  // cost of the sequences before each run of 64
};
template <int COLS>
struct Shares {
    const PagedArgs &a;
    Role<COLS> role;
    Line &line;
    int head, total, each;  // of a key head, of all, of a workgroup

    __device__ inline int sequence_cost(int i) const
    {
        if (i >= a.sequences)
            return 0;
        const Sequence sq(a, i);
        return role.cost(a, sq, role.tiles(a, sq));
    }
    __device__ inline int runs() const { return (a.sequences + kWave - 1) / kWave; }
    __device__ inline Shares(const PagedArgs &args, const Role<COLS> &r, Line &l) : a(args), role(r), line(l)
    {
        const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
        if (runs() == 1) {
            head = __builtin_amdgcn_readlane(wave_scan(sequence_cost(lane)), kWave - 1);
        } else {
            for (int i = wave; i < runs(); i += waves) {
                const int sum = wave_scan(sequence_cost(i * kWave + lane));
                if (lane == kWave - 1)
                    line.before[i] = sum;
            }
            __syncthreads();
            const int own = lane < runs() ? line.before[lane] : 0, upto = wave_scan(own);
            __syncthreads();
            if (wave == 0)
                line.before[lane] = upto - own;  // (runs beyond the last begin where it ends)
            __syncthreads();
            head = __builtin_amdgcn_readlane(upto, kWave - 1);
        }
        total = head * a.kv_heads;
        each = max((total + role.r.groups - 1) / role.r.groups, role.r.least);
    }
    // The sequence at cost p (below head) of a key head, and the cost of those before it.
    __device__ inline int find(int p, int &start) const
    {
        const int lane = threadIdx.x & (kWave - 1);
        const int run = runs() == 1 ? 0 : __popcll(__ballot(line.before[lane] <= p)) - 1;
        const int own = sequence_cost(run * kWave + lane);
        const int upto = wave_scan(own) + (runs() == 1 ? 0 : line.before[run]);
        const int l = __popcll(__ballot(upto <= p));
        start = __builtin_amdgcn_readlane(upto - own, l);
        return run * kWave + l;
    }
    // The cost of the sequences before i.
    __device__ inline int start(int i) const
    {
        const int lane = threadIdx.x & (kWave - 1), run = i / kWave;
        const int own = sequence_cost(run * kWave + lane);
        return __builtin_amdgcn_readlane(wave_scan(own) - own, i % kWave) + (runs() == 1 ? 0 : line.before[run]);
    }
};

// Where cost p falls into the n steps of a unit whose costs begin at a0, its keys'
// at `keys`, and end at a1.  (In 64-bit floats, whose quotient is the same
// wherever it is formed, and does not fall as p grows.)
__device__ inline int step_at(int p, int keys, int a1, int n)
{
    return p >= a1 ? n : p <= keys ? 0 : min(n, (int)((double)(p - keys) * n / (a1 - keys)));
}

__device__ inline int page_of(const PagedArgs &a, int key)
{
    return (int)(__umulhi(2u * (unsigned)key, a.page_magic) >> a.page_shift);
}
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
// whole runs of ROWS / W rows.  A wave's rows of a tile are one run, in one page,
// so that all addresses and the table are the scalar unit's work and the lanes
// keep their offsets (1,000 structures of 160 ... see launch): the vector unit has
// the softmax to do.
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
        const int of_run = __builtin_amdgcn_readlane(page, wave * kRun);
        const int key = first + wave * kRun, slot = key - page_of(a, key) * a.cache.page_rows;
        const unsigned row = (unsigned)a.cache.k.row * (unsigned)sizeof(T);
        const uint64_t at = (uint64_t)(unsigned)of_run * (uint64_t)(a.cache.k_page * (int64_t)sizeof(T)) + (uint64_t)(unsigned)slot * row;
        const unsigned mine = (unsigned)(seen >> (wave * kRun)) & ~0u >> (32 - kRun);
        const bool all = mine == ~0u >> (32 - kRun) && a.dim == D;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const char *from = (half ? v : k) + at;
            const int to = (half ? v_tile : k_tile) + wave * kRun * TL::kRowBytes;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const char *p = from + (uint64_t)(i * kGroup) * row;
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

// A run of a unit's keys: tiles of KB keys [begin, end) of `steps`; all of them
// give the result, others a partial one.
struct Segment {
    int kv, begin, end, steps;
    int64_t x0;  // first column of the tile
    float *part;
};

// Keys and values come in tiles of KB rows, the next one while the present one is
// worked on (BUF 2).  S^T = K Q^T leaves a column of the product per lane column:
// its running level and sum are per lane, and exp(S^T), rounded to T, is operand B
// of O^T += V^T P^T as it stands.  The two maps keep their own level, sum and
// product.
//
// A wave has QT 16 columns and both maps, which share each fragment of V read
// from LDS (M 2); or two waves share the columns, a map each (M 1).  A wave of
// wide heads has registers for 16 columns of two maps or 32 of one: those read
// 24 KiB of LDS for what takes the former 32 KiB (D 128, 32 keys).
template <class T, int D, int W, int M, int QT, int KB, int BUF, bool FAST>
__device__ inline void attend(const PagedArgs &a, const Sequence &sq, const Segment &sg, char *smem)
{
    using TL = Tile<T, D>;
    constexpr int kTile = KB * TL::kRowBytes, kCols = W * M / 2 * QT * 16;
    constexpr unsigned long long kFull = ~0ull >> (64 - KB);
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m0 = M == 2 ? 0 : wave & 1, part = M == 2 ? wave : wave >> 1;
    const int group = a.heads / a.kv_heads, kv = sg.kv;
    const int64_t columns = (int64_t)sq.rows * group, x0 = sg.x0;
    const int nk = sq.keys(a, (int)((min(x0 + kCols, columns) - 1) / group));
    const int run_begin = sg.begin * KB, run_end = min(nk, sg.end * KB);

    TileLoader<T, D, KB, W, FAST> tiles(a, sq.table, kv, lane, wave);
    tiles.look_up(run_begin, run_end);
    const float c = a.scale * kLog2e;
    Reader<T, D> rd;
    rd.init(lane);

    const int64_t w0 = x0 + part * QT * 16;  // first column of the wave
    Frag<T> qf[M][QT][D / 32];
    int last[QT];  // key that the lane's column sees
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int64_t x = w0 + t * 16 + (lane & 15);
        const int j = (int)(x / group);
        last[t] = a.causal ? sq.shift + j : nk;
        const T *qp = (const T *)a.q.data + (kv * group + x % group) * a.q.head + (int64_t)(sq.first + j) * a.q.row;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
                qf[m][t][kk] = load_frag(qp + (m0 + m) * a.q.map, kk * 32 + 8 * g, a.dim, x < columns, FAST || a.vec);
    }
    // keys that the wave's first and last columns see last
    const bool none = w0 >= columns;
    const int low = a.causal ? sq.shift + (int)(w0 / group) : nk;
    const int high = a.causal ? sq.shift + (int)((min(w0 + QT * 16, columns) - 1) / group) : nk;
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
        const int64_t x = w0 + t * 16 + (lane & 15);
        const int head = kv * group + (int)(x % group);
        const int64_t row = sq.first + x / group;
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

// The work of workgroup `item` of a role: one unit, or the runs of units that lie
// in its share.
template <class T, int D, int W, int M, int QT, int KB, int BUF, bool FAST, bool NARROW>
__device__ inline void work(const PagedArgs &a, int item, char *smem, Line &line)
{
    constexpr int kCols = W * M / 2 * QT * 16;
    const Role<kCols> role{NARROW ? a.narrow : a.wide, NARROW};
    const int group = a.heads / a.kv_heads, n = role.r.groups;
    // neighbours on one XCD, whose L2 holds the keys that they share
    const int w = n % 8 ? item : item % 8 * (n / 8) + item / 8;
    int p = 0, p0 = 0, p1 = 0;  // on the line: the next unit's, the share's
    for (bool begun = false;; begun = true) {
        int seq, kv, tile, a0 = 0, a1 = 0;
        if (!role.r.each_unit) {
            const Shares<kCols> shares(a, role, line);
            if (!begun) {
                p0 = p = w * shares.each;
                p1 = min(p0 + shares.each, shares.total);
            }
            if (p >= p1)
                return;
            kv = (int)((unsigned)p / (unsigned)shares.head);
            int at;
            seq = __builtin_amdgcn_readfirstlane(shares.find(p - kv * shares.head, at));
            at += kv * shares.head;
            const Sequence sq(a, seq);
            tile = __builtin_amdgcn_readfirstlane(
                last_true([&](int t) { return at + role.cost(a, sq, t) <= p; }, role.tiles(a, sq), kWave));
            a0 = __builtin_amdgcn_readfirstlane(at + role.cost(a, sq, tile));
            a1 = __builtin_amdgcn_readfirstlane(at + role.cost(a, sq, tile + 1));
        } else if (NARROW) {
            seq = item / a.kv_heads;
            kv = item % a.kv_heads;
            tile = 0;
        } else {
            const Work wk = work_item(item, role.r.tiles, a.kv_heads);
            // the last rows of a causal sequence have the most keys: they go first
            const int at = role.r.tiles - 1 - wk.tile;
            // (tile t of sequence i is number offsets[i] g / columns + i + t)
            auto start = [&](int i) { return (int64_t)row_offset(a.offsets, i, a.rows) * group / kCols + i; };
            seq = __builtin_amdgcn_readfirstlane(last_true([&](int i) { return start(i) <= at; }, a.sequences, kWave));
            if (seq < 0)
                return;
            kv = wk.head;
            tile = (int)(at - start(seq));
        }
        const Sequence sq(a, seq);
        if (tile >= role.tiles(a, sq))
            return;
        const int64_t columns = (int64_t)sq.rows * group, x0 = (int64_t)tile * kCols;
        const int nk = sq.keys(a, (int)((min(x0 + kCols, columns) - 1) / group)), steps = (nk + KB - 1) / KB;
        Segment sg{kv, 0, steps, steps, x0, nullptr};
        bool any = true;
        if (!role.r.each_unit) {
            sg.begin = __builtin_amdgcn_readfirstlane(step_at(p0, a0 + role.start(), a1, steps));
            sg.end = __builtin_amdgcn_readfirstlane(step_at(p1, a0 + role.start(), a1, steps));
            // a run that begins a unit and does not end it, or another
            sg.part = role.r.part + ((int64_t)w * 2 + (sg.begin == 0)) * kCols * 2 * kPart<D>;
            // a unit without keys has its zeros written where it begins
            any = sg.begin < sg.end || (steps == 0 && p0 <= a0);
        }
        if (any)
            attend<T, D, W, M, QT, KB, BUF, FAST>(a, sq, sg, smem);
        if (role.r.each_unit)
            return;
        p = a1;
    }
}

// Four columns from y on of a column x of a unit from the runs of both maps.
template <class T, int D, int COLS, int KB>
__device__ inline void join_unit(const PagedArgs &a, const Role<COLS> &role, const Sequence &sq, int kv, int tile, int a0, int a1,
                                 int each, int total, int piece, int pieces)
{
    const int group = a.heads / a.kv_heads;
    const int64_t columns = (int64_t)sq.rows * group, x0 = (int64_t)tile * COLS;
    const int nk = sq.keys(a, (int)((min(x0 + COLS, columns) - 1) / group)), steps = (nk + KB - 1) / KB;
    const int first = a0 / each, last = (a1 - 1) / each;
    auto part_at = [&](int w) { return step_at(min(w * each, total), a0 + role.start(), a1, steps); };
    // the workgroups that have a run of the unit: the first has its begin
    int from = -1, upto = -1;
    for (int w = first; w <= last; ++w) {
        const int b = part_at(w), e = part_at(w + 1);
        if (b == e)
            continue;
        if (b == 0 && e == steps)
            return;  // it has written the result
        from = from < 0 ? w : from;
        upto = w;
    }
    if (from < 0)
        return;
    const int count = (int)min((int64_t)COLS, columns - x0);
    for (int e = piece * blockDim.x + threadIdx.x; e < count * (D / 2); e += pieces * blockDim.x) {
        const int x = e / (D / 2), y = e % (D / 2) * 4;
        auto run = [&](int w, int m) {
            return role.r.part + (((int64_t)w * 2 + (w == from)) * COLS * 2 + x * 2 + m) * kPart<D>;
        };
        f32x4 v[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float hi = kNoLevel, total = 0.f;
#pragma unroll 4
            for (int w = from; w <= upto; ++w)
                if (part_at(w) != part_at(w + 1))
                    hi = fmaxf(hi, run(w, m)[0]);
            v[m] = f32x4{0, 0, 0, 0};
#pragma unroll 4
            for (int w = from; w <= upto; ++w) {
                if (part_at(w) == part_at(w + 1))
                    continue;
                const float *p = run(w, m);
                const float f = exp2_fast(p[0] - hi);  // 0 of an empty run
                total = fmaf(f, p[1], total);
                v[m] += f * *reinterpret_cast<const f32x4 *>(p + 4 + y);
            }
            v[m] *= total == 0.f ? 0.f : 1.f / total;
        }
        const int64_t row = sq.first + (x0 + x) / group;
        const int head = kv * group + (int)((x0 + x) % group);
        T *out = (T *)a.out.data + row * a.out.row + head * a.out.head + y / D * a.out.map;
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
    static constexpr int kPage = kRows / kWaves;  // rows of a wave
};

template <class T, int D, bool FAST>
__global__ __launch_bounds__((Shape<T, D>::kWaves * kWave), 2) void paged_narrow_kernel(PagedArgs a)
{
    using S = Shape<T, D>;
    // (behind the tiles: loads into LDS count from its start)
    extern __shared__ __align__(16) char smem[];
    Line &line = *reinterpret_cast<Line *>(smem + S::kLds);
    work<T, D, S::kWaves, 1, 1, S::kRows, S::kBuffers, FAST, true>(a, blockIdx.x, smem, line);
}
template <class T, int D, bool FAST>
__global__ __launch_bounds__((Shape<T, D>::kWaves * kWave), 2) void paged_wide_kernel(PagedArgs a)
{
    using S = Shape<T, D>;
    // (behind the tiles: loads into LDS count from its start)
    extern __shared__ __align__(16) char smem[];
    Line &line = *reinterpret_cast<Line *>(smem + S::kLds);
    work<T, D, S::kWaves, S::kMaps, S::kGroups, S::kRows, S::kBuffers, FAST, false>(a, blockIdx.x, smem, line);
}

constexpr int kJoin = 256;
template <class T, int D>
__global__ __launch_bounds__(kJoin) void paged_narrow_join(PagedArgs a)
{
    using S = Shape<T, D>;
    __shared__ Line line;
    const Role<S::kNarrow> role{a.narrow, true};
    const Shares<S::kNarrow> shares(a, role, line);
    const int kv = blockIdx.x % a.kv_heads, seq = blockIdx.x / a.kv_heads;
    const Sequence sq(a, seq);
    if (role.tiles(a, sq) == 0)
        return;
    const int at = kv * shares.head + shares.start(seq);
    join_unit<T, D, S::kNarrow, S::kRows>(a, role, sq, kv, 0, at, at + role.cost(a, sq, 1), shares.each, shares.total, 0, 1);
}
template <class T, int D>
__global__ __launch_bounds__(kJoin) void paged_wide_join(PagedArgs a, int pieces)
{
    using S = Shape<T, D>;
    __shared__ Line line;
    const Role<S::kWide> role{a.wide, false};
    const Shares<S::kWide> shares(a, role, line);
    const int piece = blockIdx.x % pieces, kv = blockIdx.x / pieces % a.kv_heads, at = blockIdx.x / pieces / a.kv_heads;
    const int group = a.heads / a.kv_heads;
    auto start = [&](int i) { return (int64_t)row_offset(a.offsets, i, a.rows) * group / S::kWide + i; };
    const int seq = last_true([&](int i) { return start(i) <= at; }, a.sequences, kWave);
    if (seq < 0)
        return;
    const Sequence sq(a, seq);
    const int tile = (int)(at - start(seq));
    if (tile >= role.tiles(a, sq))
        return;
    const int from = kv * shares.head + shares.start(seq);
    join_unit<T, D, S::kWide, S::kRows>(a, role, sq, kv, tile, from + role.cost(a, sq, tile), from + role.cost(a, sq, tile + 1),
                                        shares.each, shares.total, piece,
                                        pieces);
}

template <int D, bool FAST>
hipError_t run(const PagedArgs &a, hipStream_t s)
{
    using S = Shape<Type, D>;
    const dim3 block(S::kWaves * kWave);
    if (a.wide.groups > 0) {
        hipError_t e = launch_kernel(paged_wide_kernel<Type, D, FAST>, dim3((unsigned)a.wide.groups), block, S::kLds + sizeof(Line), s, a);
        if (e == hipSuccess && a.wide.part) {
            constexpr int pieces = S::kWide * (D / 2) / kJoin;
            e = launch_kernel(paged_wide_join<Type, D>, dim3((unsigned)((int64_t)a.wide.tiles * a.kv_heads * pieces)), dim3(kJoin), 0,
                              s, a, pieces);
        }
        if (e != hipSuccess)
            return e;
    }
    if (a.narrow.groups == 0)
        return hipSuccess;
    const hipError_t e = launch_kernel(paged_narrow_kernel<Type, D, FAST>, dim3((unsigned)a.narrow.groups), block, S::kLds + sizeof(Line), s, a);
    if (e != hipSuccess || !a.narrow.part)
        return e;
    return launch_kernel(paged_narrow_join<Type, D>, dim3((unsigned)((int64_t)a.sequences * a.kv_heads)), dim3(kJoin), 0, s, a);
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
