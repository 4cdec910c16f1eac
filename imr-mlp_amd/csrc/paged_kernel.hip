// Differential attention of each sequence's new rows over a paged cache
// (mtpx_diff_attention_paged),
//
//   out = (P_0 - lambda P_1) V,   P_m = softmax(scale Q_m K_m^T).
//
// The heads of a group read the same keys, so a sequence's m rows and the g
// heads of a group are m g columns of one product: column x is row x / g, head
// x % g.  A sequence of few columns goes to the deep part (its keys over waves
// and workgroups), one of many to the broad part (its columns over them);
// paged_join joins what workgroups that share a sequence's keys have left.
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

// The run of keys of one of the workgroups that share a sequence's keys:
// whole units, as even as they go, no fewer than `least` of them.
struct Run {
    int begin, end, used;
    __device__ inline Run(int keys, int split, int splits, int unit, int least)
    {
        const int units = (keys + unit - 1) / unit, each = max(least, (units + splits - 1) / splits);
        used = max(1, (units + each - 1) / each);
        begin = min(keys, split * each * unit);
        end = min(keys, begin + each * unit);
    }
};

// Floats of a partial result of one row, head and map: level, sum, -, -, product.
template <int D>
constexpr int kPart = 4 + 2 * D;
template <int D>
__device__ inline float *deep_result(const PagedArgs &a, int seq, int kv, int x, int m, int split)
{
    return a.deep_part + (((((int64_t)seq * a.kv_heads + kv) * a.deep_blocks * 16 + x) * 2 + m) * a.deep_splits + split) * kPart<D>;
}
template <int D>
__device__ inline float *broad_result(const PagedArgs &a, int64_t row, int head, int m, int split)
{
    return a.broad_part + (((row * a.heads + head) * 2 + m) * a.broad_splits + split) * kPart<D>;
}

// The page of the lane's key of a tile (lane l: key l of it), -1 where there is
// none: read a tile ahead of its use.
__device__ inline int page_of(const PagedArgs &a, int key)
{
    return (int)(__umulhi(2u * (unsigned)key, a.page_magic) >> a.page_shift);
}
__device__ inline int look_up(const PagedArgs &a, const Sequence &sq, int key, int end)
{
    return key < end ? sq.table[page_of(a, key)] : -1;
}
__device__ inline bool there(const PagedArgs &a, int page) { return page >= 0 && page < a.cache.pages; }
// Bytes from a pool's start to the row of the lane's key, whose page this is.
template <class T>
__device__ inline int64_t row_bytes(const PagedArgs &a, const mtpx_rows &s, int64_t stride, int page, int key)
{
    const int slot = key - page_of(a, key) * a.cache.page_rows;
    return there(a, page) ? (page * stride + slot * s.row) * (int64_t)sizeof(T) : 0;
}
// The same number in all lanes: lane `from`'s.
__device__ inline int64_t of_lane(int64_t v, int from)
{
    const unsigned lo = __builtin_amdgcn_readlane((int)v, from), hi = __builtin_amdgcn_readlane((int)(v >> 32), from);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// A tile's way from the pages straight into LDS, by W waves (wave `wave` of
// them): a wave's instruction fills kGroup rows of the tile.  FAST: rows are
// whole 16-byte pieces, and a page holds whole groups, so that a group's place
// is the same in all lanes.
template <class T, int D, int ROWS, int W, bool FAST>
struct PageLoader {
    using TL = Tile<T, D>;
    static constexpr int kGroup = 1024 / TL::kRowBytes;
    static constexpr int N = ROWS / (kGroup * W);
    static_assert(N * kGroup * W == ROWS, "rows of a tile");
    static constexpr bool kSame = W * kGroup % 8 == 0;
    const char *at;  // FAST: the lane's place in a group at the pool's start
    int64_t map;
    int lane, wave;

    __device__ inline int column(int i) const
    {
        const int r = (kSame ? 0 : i * W * kGroup) + wave * kGroup + lane / TL::kPieces;
        return ((lane % TL::kPieces) ^ (r & 7)) * TL::E;
    }
    __device__ inline int64_t column_bytes(int i) const
    {
        return (column(i) / D * map + column(i) % D) * (int64_t)sizeof(T);
    }
    __device__ inline void init(const mtpx_rows &s, int head, int l, int w)
    {
        map = s.map;
        lane = l;
        wave = w;
        at = (const char *)((const T *)s.data + head * s.head);
        if constexpr (FAST)
            at += lane / TL::kPieces * s.row * (int64_t)sizeof(T);
        if constexpr (kSame)
            at += column_bytes(0);
    }
    // bytes: of the lane's key; seen: the tile's rows that are there (all: every one).
    __device__ inline void load(const PagedArgs &a, char *smem, int tile, int64_t bytes, unsigned long long seen, bool all) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r0 = (i * W + wave) * kGroup, r = r0 + lane / TL::kPieces, to = tile + (i * W + wave) * 1024;
            const char *p = at + (FAST ? of_lane(bytes, r0) : (int64_t)__shfl((long long)bytes, r));
            if constexpr (!kSame)
                p += column_bytes(i);
            if (FAST && all && a.dim == D) {
                load_to_lds(p, to);
                continue;
            }
            const int c = column(i) % D;
            const bool on = (seen >> r & 1) && c < a.dim;
            if (FAST || a.vec)
                load_to_lds(on ? (const void *)p : (const void *)&kZeroPiece, to);
            else
                *reinterpret_cast<u32x4 *>(smem + to + lane * 16) = load16((const T *)p, on ? a.dim - c : 0, 0);
        }
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

// The broad part.  A workgroup takes columns of one sequence and group; keys and
// values come in tiles of KB rows, the next one while the present one is worked
// on (BUF 2).  S^T = K Q^T leaves a column of the product per lane column: its
// running level and sum are per lane, and exp(S^T), rounded to T, is operand B of
// O^T += V^T P^T as it stands.  The two maps keep their own level, sum and product.
//
// A wave has QT 16 columns and both maps, which share each fragment of V read
// from LDS (M 2); or two waves share the columns, a map each (M 1).  A wave of
// wide heads has registers for 16 columns of two maps or 32 of one: those read
// 24 KiB of LDS for what takes the former 32 KiB (D 128, 32 keys).
template <class T, int D, int W, int M, int QT, int KB, int BUF, bool FAST>
__device__ inline void broad_part(const PagedArgs &a, int item, char *smem)
{
    using TL = Tile<T, D>;
    constexpr int kTile = KB * TL::kRowBytes, kCols = W * M / 2 * QT * 16;
    constexpr unsigned long long kFull = ~0ull >> (64 - KB);
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m0 = M == 2 ? 0 : wave & 1, part = M == 2 ? wave : wave >> 1;
    const int group = a.heads / a.kv_heads;
    const Work wk = work_item(item, a.broad_tiles, a.kv_heads * a.broad_splits);
    const int kv = wk.head % a.kv_heads, split = wk.head / a.kv_heads;
    // the last rows of a causal sequence have the most keys: they go first
    const int tile = a.broad_tiles - 1 - wk.tile;
    auto start = [&](int i) { return (int64_t)row_offset(a.offsets, i, a.rows) * group / kCols + i; };
    const int seq = __builtin_amdgcn_readfirstlane(last_true([&](int i) { return start(i) <= tile; }, a.sequences, kWave));
    if (seq < 0)
        return;
    const Sequence sq(a, seq);
    const int64_t columns = (int64_t)sq.rows * group, x0 = (tile - start(seq)) * kCols;
    if (x0 >= columns || columns <= a.deep)
        return;
    const int nk = sq.keys(a, (int)((min(x0 + kCols, columns) - 1) / group));
    const Run run(nk, split, a.broad_splits, KB, a.broad_least / KB);
    if (split >= run.used)
        return;

    const float c = a.scale * kLog2e;
    Reader<T, D> rd;
    rd.init(lane);
    PageLoader<T, D, KB, W, FAST> lk, lv;
    lk.init(a.cache.k, kv, lane, wave);
    lv.init(a.cache.v, kv, lane, wave);

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
    int page = -1;
    auto load = [&](int k0, int to) {
        bits = __ballot(there(a, page)) & kFull;
        const int64_t kb = row_bytes<T>(a, a.cache.k, a.cache.k_page, page, k0 + lane);
        const int64_t vb = row_bytes<T>(a, a.cache.v, a.cache.v_page, page, k0 + lane);
        lk.load(a, smem, to * 2 * kTile, kb, bits, bits == kFull);
        lv.load(a, smem, to * 2 * kTile + kTile, vb, bits, bits == kFull);
        page = look_up(a, sq, k0 + KB + lane, run.end);
    };
    if (run.begin < run.end) {
        page = look_up(a, sq, run.begin + lane, run.end);
        load(run.begin, 0);
    }
    int buf = 0;
    for (int k0 = run.begin; k0 < run.end; k0 += KB) {
        wait_loads();
        __syncthreads();
        const unsigned long long now = bits;
        const char *kt = smem + buf * 2 * kTile, *vt = kt + kTile;
        auto next = [&] {
            if (k0 + KB < run.end) {
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
                        const int column = x / (D / 32) % M * D + x % (D / 32) * 32;
                        const char *of = M == 2 ? kt : kt + m0 * (2 * D * sizeof(T) / 2);
                        return rd.row_frag(of, b * 32 + x / kEach * 16, column);
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

    if constexpr (M == 1)
        __syncthreads();  // the last tile's reads, before its place takes results
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int64_t x = w0 + t * 16 + (lane & 15);
        const int head = kv * group + (int)(x % group);
        const int64_t row = sq.first + x / group;
        float total[M];
#pragma unroll
        for (int m = 0; m < M; ++m)
            total[m] = column_sum(sum[m][t]);
        if (run.used > 1) {
            if (x >= columns)
                continue;
#pragma unroll
            for (int m = 0; m < M; ++m) {
                float *p = broad_result<D>(a, row, head, m0 + m, split);
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

// Waits until no more than N of the loads that this wave has queued are under way.
template <int N>
__device__ inline void wait_all_but()
{
    static_assert(N < 64, "what the counter holds");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
    asm volatile("" ::: "memory");
}

// The deep part.  A workgroup takes 16 columns of one sequence and group (fewer
// leave columns of the product empty, which costs nothing, as the reads of the
// cache bound it) and one of the runs of their keys; its waves take steps of 32
// keys in turn, each with its own maxima and sums, and are joined through LDS at
// the end.  Keys and values go into LDS of the wave's own: those of the next step
// are queued as soon as the present one's have been read, so that a wave has a
// step's keys or values under way at any time.  FAST: nothing else is loaded in
// the loop (64 entries of the table lie in a register), so that a wait can leave
// the later loads under way.
template <class T, int D, int W, bool FAST>
__device__ inline void deep_part(const PagedArgs &a, int item, char *smem)
{
    using TL = Tile<T, D>;
    using PL = PageLoader<T, D, 32, 1, FAST>;
    constexpr int kTile = 32 * TL::kRowBytes;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = a.heads / a.kv_heads;
    const int block = item % a.deep_blocks, split = item / a.deep_blocks % a.deep_splits;
    const int kv = item / (a.deep_blocks * a.deep_splits) % a.kv_heads;
    const int seq = item / (a.deep_blocks * a.deep_splits) / a.kv_heads;
    const Sequence sq(a, seq);
    const int64_t columns = (int64_t)sq.rows * group;
    const int x0 = block * 16;
    if (columns > a.deep || x0 >= columns)
        return;
    const int count = min(16, (int)columns - x0);
    const int nk = sq.keys(a, (x0 + count - 1) / group);
    const Run run(nk, split, a.deep_splits, 32, a.deep_least / 32);
    if (split >= run.used)
        return;

    const float c = a.scale * kLog2e;
    const int kt = wave * 2 * kTile, vt = kt + kTile;
    Reader<T, D> rd;
    rd.init(lane);
    PL lk, lv;
    lk.init(a.cache.k, kv, lane, 0);
    lv.init(a.cache.v, kv, lane, 0);
    // entries of the table from `base` on
    int entries = -1, base = -64;
    const int pages = run.end > 0 ? page_of(a, run.end - 1) + 1 : 0;
    // the step's keys: whether they are there and where
    unsigned next_bits = 0;
    int64_t key_bytes = 0, value_bytes = 0;
    auto find = [&](int k0) {
        const int key = k0 + (lane & 31);
        int page;
        if constexpr (FAST) {
            const int first = page_of(a, k0), end = page_of(a, min(k0 + 32, run.end) - 1) + 1;
            if (end > base + 64) {
                base = first;
                entries = base + lane < pages ? sq.table[base + lane] : -1;
                wait_loads();
            }
            page = __shfl(entries, min(page_of(a, key) - base, 63));
            page = key < run.end ? page : -1;
        } else {
            page = look_up(a, sq, key, run.end);
        }
        next_bits = (unsigned)__ballot(there(a, page));
        key_bytes = row_bytes<T>(a, a.cache.k, a.cache.k_page, page, key);
        value_bytes = row_bytes<T>(a, a.cache.v, a.cache.v_page, page, key);
    };
    const int begin = run.begin + 32 * wave;
    if (begin < run.end) {
        find(begin);
        lk.load(a, smem, kt, key_bytes, next_bits, next_bits == ~0u);
        lv.load(a, smem, vt, value_bytes, next_bits, next_bits == ~0u);
    }
    const int x = x0 + col, j = x / group, head = kv * group + x % group;
    const int last = a.causal ? sq.shift + j : nk;
    const T *qp = (const T *)a.q.data + head * a.q.head + (int64_t)(sq.first + j) * a.q.row;
    Frag<T> qf[2][D / 32];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)
            qf[m][kk] = load_frag(qp + m * a.q.map, kk * 32 + 8 * g, a.dim, col < count, FAST || a.vec);

    f32x4 acc[2][D / 8];
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
        acc[0][i] = acc[1][i] = f32x4{0, 0, 0, 0};

    wait_loads();
    for (int k0 = begin; k0 < run.end; k0 += 32 * W) {
        const bool more = k0 + 32 * W < run.end;
        const unsigned bits = next_bits;
        if constexpr (FAST)
            wait_all_but<PL::N>();
        else
            wait_loads();
        f32x4 s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                s[m][u] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int kk = 0; kk < D / 32; ++kk)
                    s[m][u] = mma(rd.row_frag(smem + kt, 16 * u, m * D + kk * 32), qf[m][kk], s[m][u]);
            }
        wait_reads();
        if (more) {
            find(k0 + 32 * W);
            lk.load(a, smem, kt, key_bytes, next_bits, next_bits == ~0u);
        }
        if (bits != ~0u || k0 + 31 > last) {
            const unsigned mine = bits >> (4 * g);
            const int most = last - k0 - 4 * g;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool on = (mine >> (16 * u + r) & 1) && 16 * u + r <= most;
                    s[0][u][r] = on ? s[0][u][r] : -INFINITY;
                    s[1][u][r] = on ? s[1][u][r] : -INFINITY;
                }
        }
        Frag<T> pf[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float hi = s[m][0][0];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    hi = fmaxf(hi, s[m][u][r]);
            hi = fmaxf(top[m], column_max(hi) * c);
            if (__any(hi > top[m])) {
                const float f = top[m] == -INFINITY ? 0.f : exp2_fast(top[m] - hi);
                top[m] = hi;
                sum[m] *= f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    acc[m][i] *= f;
            }
            const float level = hi == -INFINITY ? 0.f : hi;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = exp2_fast(fmaf(s[m][u][r], c, -level));
                    s[m][u][r] = p;
                    sum[m] += p;
                }
            pf[m] = pack<T>(s[m][0], s[m][1]);
        }
        if (FAST && more)
            wait_all_but<PL::N>();
        else
            wait_loads();
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const Frag<T> vf = rd.column_frag(smem + vt, 0, i * 16);
            acc[0][i] = mma(vf, pf[0], acc[0][i]);
            acc[1][i] = mma(vf, pf[1], acc[1][i]);
        }
        wait_reads();
        if (more)
            lv.load(a, smem, vt, value_bytes, next_bits, next_bits == ~0u);
    }

    // Join the waves, one map at a time: column-major products in LDS, and the
    // first map's result beside them while the second's are joined.
    float *red = reinterpret_cast<float *>(smem);  // [W][16][kPart], [16][2 D]
    float *first = red + W * 16 * kPart<D>;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float total = column_sum(sum[m]);
        __syncthreads();
        float *mine = red + (wave * 16 + col) * kPart<D>;
        if (g == 0) {
            mine[0] = top[m];
            mine[1] = total;
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<f32x4 *>(mine + 4 + i * 16 + 4 * g) = acc[m][i];
        __syncthreads();
        for (int e = tid; e < count * 2 * D; e += W * kWave) {
            const int h = e / (2 * D), y = e % (2 * D);
            float hi = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w)
                hi = fmaxf(hi, red[(w * 16 + h) * kPart<D>]);
            float v = 0.f, l = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float *o = red + (w * 16 + h) * kPart<D>;
                const float f = o[0] == -INFINITY ? 0.f : exp2_fast(o[0] - hi);
                v = fmaf(f, o[4 + y], v);
                l = fmaf(f, o[1], l);
            }
            if (run.used > 1) {
                float *p = deep_result<D>(a, seq, kv, x0 + h, m, split);
                if (y == 0) {
                    p[0] = hi;
                    p[1] = l;
                }
                p[4 + y] = v;
                continue;
            }
            v = l == 0.f ? 0.f : v / l;
            if (m == 0) {
                first[e] = v;
            } else if (y % D < a.dim) {
                const int hd = kv * group + (x0 + h) % group, row = sq.first + (x0 + h) / group;
                ((T *)a.out.data)[(int64_t)row * a.out.row + hd * a.out.head + y / D * a.out.map + y % D] =
                    (T)(first[e] - a.lambda[hd] * v);
            }
        }
    }
}

template <class T, int D, int W, int M, int QT, int KB, int BUF, int OCC, bool FAST>
__global__ __launch_bounds__(W * kWave, OCC) void paged_broad_kernel(PagedArgs a)
{
    extern __shared__ __align__(16) char smem[];
    broad_part<T, D, W, M, QT, KB, BUF, FAST>(a, blockIdx.x, smem);
}
template <class T, int D, int W, int OCC, bool FAST>
__global__ __launch_bounds__(W * kWave, OCC) void paged_deep_kernel(PagedArgs a)
{
    extern __shared__ __align__(16) char smem[];
    deep_part<T, D, W, FAST>(a, blockIdx.x, smem);
}

// Four columns from y on of a row and head from the runs of both maps.
template <class T, int D>
__device__ inline void join_runs(const PagedArgs &a, const float *p0, const float *p1, int used, int64_t row, int head, int y)
{
    const float *from[2] = {p0, p1};
    f32x4 v[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float *p = from[m];
        float hi = kNoLevel;
#pragma unroll 4
        for (int i = 0; i < used; ++i)
            hi = fmaxf(hi, p[i * kPart<D>]);
        float total = 0.f;
        v[m] = f32x4{0, 0, 0, 0};
#pragma unroll 4
        for (int i = 0; i < used; ++i) {
            const float f = exp2_fast(p[i * kPart<D>] - hi);  // 0 of an empty run
            total = fmaf(f, p[i * kPart<D> + 1], total);
            v[m] += f * *reinterpret_cast<const f32x4 *>(p + i * kPart<D> + 4 + y);
        }
        v[m] *= total == 0.f ? 0.f : 1.f / total;
    }
    T *out = (T *)a.out.data + row * a.out.row + head * a.out.head + y / D * a.out.map;
    store4(out, y % D, a.dim, v[0] - a.lambda[head] * v[1], a.vec);
}
constexpr int kJoin = 256;

// A workgroup per sequence, group and block of 16 columns.
template <class T, int D>
__global__ __launch_bounds__(kJoin) void paged_join_deep(PagedArgs a)
{
    const int block = blockIdx.x % a.deep_blocks, kv = blockIdx.x / a.deep_blocks % a.kv_heads;
    const int seq = blockIdx.x / a.deep_blocks / a.kv_heads, group = a.heads / a.kv_heads;
    const Sequence sq(a, seq);
    const int64_t columns = (int64_t)sq.rows * group;
    const int x0 = block * 16;
    if (columns > a.deep || x0 >= columns)
        return;
    const int count = min(16, (int)columns - x0);
    const int used = Run(sq.keys(a, (x0 + count - 1) / group), 0, a.deep_splits, 32, a.deep_least / 32).used;
    if (used <= 1)
        return;
    for (int e = threadIdx.x; e < count * (D / 2); e += kJoin) {
        const int x = x0 + e / (D / 2), y = e % (D / 2) * 4;
        join_runs<T, D>(a, deep_result<D>(a, seq, kv, x, 0, 0), deep_result<D>(a, seq, kv, x, 1, 0), used,
                        sq.first + x / group, kv * group + x % group, y);
    }
}

// D / 2 lanes per row and head.
template <class T, int D>
__global__ __launch_bounds__(kJoin) void paged_join_broad(PagedArgs a, int unit)
{
    constexpr int kLanes = D / 2;
    const int64_t item = (int64_t)blockIdx.x * (kJoin / kLanes) + threadIdx.x / kLanes;
    const int64_t row = item / a.heads;
    const int head = item % a.heads, group = a.heads / a.kv_heads;
    const int seq = last_true([&](int i) { return row_offset(a.offsets, i, a.rows) <= row; }, a.sequences + 1, kLanes);
    if (row >= a.rows || seq < 0 || seq >= a.sequences)
        return;
    const Sequence sq(a, seq);
    const int64_t columns = (int64_t)sq.rows * group, x = (row - sq.first) * group + head % group;
    if (columns <= a.deep)
        return;
    const int64_t end = min(columns, x / a.broad_columns * a.broad_columns + a.broad_columns);
    const int used = Run(sq.keys(a, (int)((end - 1) / group)), 0, a.broad_splits, unit, a.broad_least / unit).used;
    if (used > 1)
        join_runs<T, D>(a, broad_result<D>(a, row, head, 0, 0), broad_result<D>(a, row, head, 1, 0), used, row, head,
                        threadIdx.x % kLanes * 4);
}

// Tile shapes by head width.
template <class T, int D>
struct Shape {
    static constexpr int kRows = 2 * D * (int)sizeof(T) <= 256 ? 64 : 32;
    // maps of a wave, and groups of 16 columns in broad tiles: two share the
    // reads from LDS that bound 16-bit products; 32-bit products take so long
    // that more waves serve them better
    static constexpr int kMaps = D == 128 && sizeof(T) == 2 ? 1 : 2;
    static constexpr int kWide = sizeof(T) == 2 ? 2 : 1;
    static constexpr size_t kLds = 2 * (size_t)kRows * 2 * D * sizeof(T);
    // two buffers of both tiles within the 64 KiB that loads into LDS address
    static constexpr int kBuffers = kLds <= 32768 ? 2 : 1;
    static constexpr int kOccupancy = kLds > 32768 ? 1 : 2;
    // waves whose keys and values of a step fit into that
    static constexpr int kDeepWaves = 512 / (D * (int)sizeof(T)) > 8 ? 8 : 512 / (D * (int)sizeof(T));
    static constexpr int kGroup = 32 / (D * (int)sizeof(T) / 16);  // rows of 1 KiB
};
constexpr int kWaves = 4;  // of the broad part

template <int D, bool FAST>
hipError_t deep(const PagedArgs &a, hipStream_t s)
{
    constexpr int W = Shape<Type, D>::kDeepWaves;
    constexpr size_t tiles = (size_t)W * 2 * 32 * 2 * D * sizeof(Type);
    static_assert(tiles <= 65536, "what loads into LDS address");
    constexpr size_t join = ((size_t)W * 16 * kPart<D> + 16 * 2 * D) * sizeof(float);
    constexpr int occ = W < 4 ? 1 : 2;  // waves per SIMD that LDS lets in
    const int64_t items = (int64_t)a.sequences * a.kv_heads * a.deep_blocks;
    const hipError_t e = launch_kernel(paged_deep_kernel<Type, D, W, occ, FAST>, dim3((unsigned)(items * a.deep_splits)),
                                       dim3(W * kWave), tiles > join ? tiles : join, s, a);
    if (e != hipSuccess || a.deep_splits == 1)
        return e;
    return launch_kernel(paged_join_deep<Type, D>, dim3((unsigned)items), dim3(kJoin), 0, s, a);
}
template <int D, int QT, bool FAST>
hipError_t broad(const PagedArgs &a, hipStream_t s)
{
    using S = Shape<Type, D>;
    const hipError_t e = launch_kernel(
        paged_broad_kernel<Type, D, kWaves, S::kMaps, QT, S::kRows, S::kBuffers, S::kOccupancy, FAST>,
        dim3((unsigned)((int64_t)a.broad_tiles * a.kv_heads * a.broad_splits)), dim3(kWaves * kWave), S::kBuffers * S::kLds, s, a);
    if (e != hipSuccess || a.broad_splits == 1)
        return e;
    constexpr int items = kJoin / (D / 2);
    return launch_kernel(paged_join_broad<Type, D>, dim3((unsigned)((a.rows * a.heads + items - 1) / items)), dim3(kJoin), 0, s, a,
                         S::kRows);
}

template <int D, bool FAST>
hipError_t run(const PagedArgs &a, hipStream_t s)
{
    using S = Shape<Type, D>;
    if (a.broad_tiles > 0)
        if (hipError_t e = a.broad_columns == kWaves * S::kMaps / 2 * 16 ? broad<D, 1, FAST>(a, s) : broad<D, S::kWide, FAST>(a, s))
            return e;
    return a.deep > 0 ? deep<D, FAST>(a, s) : hipSuccess;
}
template <int D>
hipError_t by_pages(const PagedArgs &a, hipStream_t s)
{
    return a.vec && a.cache.page_rows % Shape<Type, D>::kGroup == 0 ? run<D, true>(a, s) : run<D, false>(a, s);
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
