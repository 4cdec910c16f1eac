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
constexpr int kLeastKeys = 256;  // of one run

// Floats of a partial result of one row, head and map: level, sum, -, -, product.
template <int D>
constexpr int kPart = 4 + 2 * D;

// The lane's key of a run of 64 (or 32): where it stands.  The table is read
// one run ahead of the keys, these one tile ahead of their use.
struct Place {
    int page, slot;
};
__device__ inline Place place(const PagedArgs &a, const Sequence &sq, int key, int end)
{
    Place p;
    const int n = (int)(__umulhi(2u * (unsigned)key, a.page_magic) >> a.page_shift);
    p.slot = key - n * a.cache.page_rows;
    p.page = key < end ? sq.table[n] : -1;
    return p;
}
__device__ inline bool there(const PagedArgs &a, const Place &p) { return p.page >= 0 && p.page < a.cache.pages; }

// A tile's way from the pages straight into LDS, by W waves (wave `wave` of
// them): a wave's instruction fills kGroup rows of the tile.  Where a page
// holds a whole number of such groups, a group's page and row are the same in
// all lanes and its address is formed by the scalar unit.
template <class T, int D, int ROWS, int W>
struct PageLoader {
    using TL = Tile<T, D>;
    static constexpr int kGroup = 1024 / TL::kRowBytes;
    static constexpr int N = ROWS / (kGroup * W);
    static_assert(N * kGroup * W == ROWS, "rows of a tile");
    static constexpr bool kSame = W * kGroup % 8 == 0;
    const T *base;
    int64_t page, row, map;
    int lane, wave;

    __device__ inline int column(int i) const
    {
        const int r = (kSame ? 0 : i * W * kGroup) + wave * kGroup + lane / TL::kPieces;
        return ((lane % TL::kPieces) ^ (r & 7)) * TL::E;
    }
    __device__ inline void init(const mtpx_rows &s, int64_t page_stride, int head, int l, int w)
    {
        base = (const T *)s.data + head * s.head;
        page = page_stride;
        row = s.row;
        map = s.map;
        lane = l;
        wave = w;
    }
    __device__ inline void load(const PagedArgs &a, char *smem, int tile, const Place &pl, unsigned long long seen,
                                bool all) const
    {
        const bool even = a.cache.page_rows % kGroup == 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r0 = (i * W + wave) * kGroup, r = r0 + lane / TL::kPieces;
            const int col = column(i), c = col % D;
            const T *p = base + col / D * map + c;
            if (even) {
                const int pg = __builtin_amdgcn_readlane(pl.page, r0), sl = __builtin_amdgcn_readlane(pl.slot, r0);
                p += pg * page + sl * row + lane / TL::kPieces * row;
            } else {
                p += __shfl(pl.page, r) * page + __shfl(pl.slot, r) * row;
            }
            const int to = tile + (i * W + wave) * 1024;
            if (a.vec && all && a.dim == D) {
                load_to_lds(p, to);
                continue;
            }
            const bool on = (seen >> r & 1) && c < a.dim;
            if (a.vec)
                load_to_lds(on ? (const void *)p : (const void *)&kZeroPiece, to);
            else
                *reinterpret_cast<u32x4 *>(smem + to + lane * 16) = load16(p, on ? a.dim - c : 0, 0);
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

// The broad part.  A workgroup takes W QT 16 columns of one sequence and group,
// each wave QT 16 of them; the keys and values come in tiles of KB rows, the
// next one while the present one is worked on (BUF 2).  S^T = K Q^T leaves a
// column of the product per lane column: its running level and sum are per
// lane, and exp(S^T), rounded to T, is operand B of O^T += V^T P^T as it stands.
// The two maps keep their own level, sum and product.
template <class T, int D, int W, int QT, int KB, int BUF>
__device__ inline void broad_part(const PagedArgs &a, int item, char *smem)
{
    using TL = Tile<T, D>;
    constexpr int kTile = KB * TL::kRowBytes, kCols = W * QT * 16;
    constexpr unsigned long long kFull = ~0ull >> (64 - KB);
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
    const Run run(nk, split, a.broad_splits, KB, kLeastKeys / KB);
    if (split >= run.used)
        return;

    const float c = a.scale * kLog2e;
    Reader<T, D> rd;
    rd.init(lane);
    PageLoader<T, D, KB, W> lk, lv;
    lk.init(a.cache.k, a.cache.k_page, kv, lane, wave);
    lv.init(a.cache.v, a.cache.v_page, kv, lane, wave);

    const int64_t w0 = x0 + wave * QT * 16;  // first column of the wave
    Frag<T> qf[2][QT][D / 32];
    int last[QT];  // key that the lane's column sees
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int64_t x = w0 + t * 16 + (lane & 15);
        const int j = (int)(x / group);
        last[t] = a.causal ? sq.shift + j : nk;
        const T *qp = (const T *)a.q.data + (kv * group + x % group) * a.q.head + (int64_t)(sq.first + j) * a.q.row;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
                qf[m][t][kk] = load_frag(qp + m * a.q.map, kk * 32 + 8 * g, a.dim, x < columns, a.vec);
    }
    // keys that the wave's first and last columns see last
    const bool none = w0 >= columns;
    const int low = a.causal ? sq.shift + (int)(w0 / group) : nk;
    const int high = a.causal ? sq.shift + (int)((min(w0 + QT * 16, columns) - 1) / group) : nk;
    f32x4 acc[2][QT][D / 8];
    float level[2][QT], sum[2][QT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            level[m][t] = kNoLevel;
            sum[m][t] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                acc[m][t][i] = f32x4{0, 0, 0, 0};
        }

    unsigned long long bits = 0;
    Place ahead{-1, 0};
    auto load = [&](int k0, int to) {
        bits = __ballot(there(a, ahead)) & kFull;
        lk.load(a, smem, to * 2 * kTile, ahead, bits, bits == kFull);
        lv.load(a, smem, to * 2 * kTile + kTile, ahead, bits, bits == kFull);
        ahead = place(a, sq, k0 + KB + lane, run.end);
    };
    if (run.begin < run.end) {
        ahead = place(a, sq, run.begin + lane, run.end);
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
                f32x4 s[2][2][QT];
                {
                    // u, then map, then columns: one K fragment ahead
                    constexpr int kSteps = 2 * 2 * (D / 32);
                    Frag<T> kf = rd.row_frag(kt, b * 32, 0);
#pragma unroll
                    for (int x = 0; x < kSteps; ++x) {
                        const int u = x / (D / 16), m = x / (D / 32) % 2, kk = x % (D / 32);
                        Frag<T> following;
                        if (x + 1 < kSteps) {
                            const int y = x + 1, mc = y / (D / 32) % 2 * D + y % (D / 32) * 32;
                            following = rd.row_frag(kt, b * 32 + y / (D / 16) * 16, mc);
                        }
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
                                s[0][u][t][r] = on ? s[0][u][t][r] : -INFINITY;
                                s[1][u][t][r] = on ? s[1][u][t][r] : -INFINITY;
                            }
                    }
                }
                float hi[2][QT];
                bool passed = false;
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        const f32x4 x = s[m][0][t], y = s[m][1][t];
                        hi[m][t] = max3(max3(x[0], x[1], x[2]), max3(x[3], y[0], y[1]), max3(y[2], y[3], y[3]));
                        passed |= fmaf(hi[m][t], c, -level[m][t]) > kSlack;
                    }
                if (__any(passed)) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
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
                Frag<T> pf[2][QT];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        float part[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float p = exp2_fast(fmaf(s[m][u][t][r], c, -level[m][t]));
                                s[m][u][t][r] = p;
                                part[u] = r ? part[u] + p : p;
                            }
                        sum[m][t] += part[0] + part[1];
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
                    for (int m = 0; m < 2; ++m)
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

#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int64_t x = w0 + t * 16 + (lane & 15);
        const int head = kv * group + (int)(x % group);
        const int64_t row = sq.first + x / group;
        float total[2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
            total[m] = column_sum(sum[m][t]);
        if (x >= columns)
            continue;
        if (run.used > 1) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float *p = a.broad_part + (((row * a.heads + head) * 2 + m) * a.broad_splits + split) * kPart<D>;
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
        const float inv0 = total[0] == 0.f ? 0.f : 1.f / total[0], inv1 = total[1] == 0.f ? 0.f : 1.f / total[1];
        const float lambda = a.lambda[head];
        T *op = (T *)a.out.data + head * a.out.head + row * a.out.row;
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
            store_columns<T, D>(op, a.out.map, a.dim, i, lane, acc[0][t][i] * inv0 - lambda * (acc[1][t][i] * inv1), a.vec);
    }
}

// The deep part.  A workgroup takes 16 columns of one sequence and group (fewer
// leave columns of the product empty, which costs nothing, as the reads of the
// cache bound it) and one of the runs of their keys; its waves take steps of 32
// keys in turn, each with its own maxima and sums, and are joined through LDS at
// the end.  A wave reads K as operand A straight from the pages; V goes through
// LDS of its own to be read by columns.  The pages are looked up two steps, keys
// and values read one step ahead.  (WORK: the waves that LDS has room for; the
// others of the workgroup take part in the join only.)
template <class T, int D, int W, int WORK>
__device__ inline void deep_part(const PagedArgs &a, int item, char *smem)
{
    using TL = Tile<T, D>;
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
    const Run run(nk, split, a.deep_splits, 32, kLeastKeys / 32);
    if (split >= run.used)
        return;

    const float c = a.scale * kLog2e;
    char *tile = smem + wave * kTile;
    Reader<T, D> rd;
    rd.init(lane);
    const int x = x0 + col, j = x / group, head = kv * group + x % group;
    const int last = a.causal ? sq.shift + j : nk;
    const T *qp = (const T *)a.q.data + head * a.q.head + (int64_t)(sq.first + j) * a.q.row;
    Frag<T> qf[2][D / 32];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)
            qf[m][kk] = load_frag(qp + m * a.q.map, kk * 32 + 8 * g, a.dim, col < count, a.vec);

    f32x4 acc[2][D / 8];
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
        acc[0][i] = acc[1][i] = f32x4{0, 0, 0, 0};

    const T *kp = (const T *)a.cache.k.data + kv * a.cache.k.head;
    PageLoader<T, D, 32, 1> lv;
    lv.init(a.cache.v, a.cache.v_page, kv, lane, 0);
    Frag<T> kf[2][2][D / 32];
    Place ahead{-1, 0};
    unsigned bits = 0;
    auto fetch = [&](int k0) {
        bits = (unsigned)__ballot(there(a, ahead));
        lv.load(a, smem, wave * kTile, ahead, bits, bits == ~0u);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = 16 * u + col;
            const T *p = kp + __shfl(ahead.page, r) * a.cache.k_page + __shfl(ahead.slot, r) * a.cache.k.row;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int kk = 0; kk < D / 32; ++kk)
                    kf[u][m][kk] = load_frag(p + m * a.cache.k.map, kk * 32 + 8 * g, a.dim, bits >> r & 1, a.vec);
        }
        ahead = place(a, sq, k0 + 32 * WORK + (lane & 31), run.end);
    };
    const int begin = wave < WORK ? run.begin + 32 * wave : run.end;
    if (begin < run.end)
        ahead = place(a, sq, begin + (lane & 31), run.end);
    for (int k0 = begin; k0 < run.end; k0 += 32 * WORK) {
        wait_reads();
        fetch(k0);
        f32x4 s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                s[m][u] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int kk = 0; kk < D / 32; ++kk)
                    s[m][u] = mma(kf[u][m][kk], qf[m][kk], s[m][u]);
            }
        const unsigned mine = bits >> (4 * g);
        const int most = last - k0 - 4 * g;
        if (bits != ~0u || k0 + 31 > last) {
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
            const float base = hi == -INFINITY ? 0.f : hi;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = exp2_fast(fmaf(s[m][u][r], c, -base));
                    s[m][u][r] = p;
                    sum[m] += p;
                }
            pf[m] = pack<T>(s[m][0], s[m][1]);
        }
        wait_loads();
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const Frag<T> vf = rd.column_frag(tile, 0, i * 16);
            acc[0][i] = mma(vf, pf[0], acc[0][i]);
            acc[1][i] = mma(vf, pf[1], acc[1][i]);
        }
    }

    // Join the waves, one map at a time: column-major products in LDS, and the
    // first map's result beside them while the second's are joined.
    float *red = reinterpret_cast<float *>(smem);  // [WORK][16][kPart], [16][2 D]
    float *first = red + WORK * 16 * kPart<D>;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float total = column_sum(sum[m]);
        __syncthreads();
        if (wave < WORK) {
            float *mine = red + (wave * 16 + col) * kPart<D>;
            if (g == 0) {
                mine[0] = top[m];
                mine[1] = total;
            }
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<f32x4 *>(mine + 4 + i * 16 + 4 * g) = acc[m][i];
        }
        __syncthreads();
        for (int e = tid; e < count * 2 * D; e += W * kWave) {
            const int h = e / (2 * D), y = e % (2 * D);
            float hi = -INFINITY;
#pragma unroll
            for (int w = 0; w < WORK; ++w)
                hi = fmaxf(hi, red[(w * 16 + h) * kPart<D>]);
            float v = 0.f, l = 0.f;
#pragma unroll
            for (int w = 0; w < WORK; ++w) {
                const float *o = red + (w * 16 + h) * kPart<D>;
                const float f = o[0] == -INFINITY ? 0.f : exp2_fast(o[0] - hi);
                v = fmaf(f, o[4 + y], v);
                l = fmaf(f, o[1], l);
            }
            if (run.used > 1) {
                float *p = a.deep_part +
                           ((((int64_t)seq * a.kv_heads + kv) * a.deep_blocks * 16 + x0 + h) * 2 + m) * a.deep_splits * kPart<D> +
                           split * kPart<D>;
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

// Both parts in one launch: the broad tiles first, which take the longest.
template <class T, int D, int W, int WORK, int QT, int KB, int BUF, int OCC>
__global__ __launch_bounds__(W * kWave, OCC) void paged_kernel(PagedArgs a)
{
    extern __shared__ __align__(16) char smem[];
    const int broad = a.broad_tiles * a.kv_heads * a.broad_splits;
    if ((int)blockIdx.x < broad)
        broad_part<T, D, W, QT, KB, BUF>(a, blockIdx.x, smem);
    else
        deep_part<T, D, W, WORK>(a, blockIdx.x - broad, smem);
}
template <class T, int D, int W, int OCC>
__global__ __launch_bounds__(W * kWave, OCC) void paged_deep_kernel(PagedArgs a)
{
    extern __shared__ __align__(16) char smem[];
    deep_part<T, D, W, W>(a, blockIdx.x, smem);
}

// Joins the runs of one row and head: a thread per map and column.
template <class T, int D>
__global__ __launch_bounds__(4 * D) void paged_join(PagedArgs a, int broad_unit)
{
    __shared__ float joined[2 * D];
    const int tid = threadIdx.x, m = tid / (2 * D), y = tid % (2 * D), head = blockIdx.x % a.heads;
    const int64_t row = blockIdx.x / a.heads;
    const int seq = last_true([&](int i) { return row_offset(a.offsets, i, a.rows) <= row; }, a.sequences + 1, kWave);
    if (seq < 0 || seq >= a.sequences)
        return;
    const Sequence sq(a, seq);
    const int group = a.heads / a.kv_heads, kv = head / group;
    const int64_t columns = (int64_t)sq.rows * group, x = (row - sq.first) * group + head % group;
    const float *p;
    int used;
    if (columns <= a.deep) {
        const int end = min((int)columns, (int)x / 16 * 16 + 16);
        used = Run(sq.keys(a, (end - 1) / group), 0, a.deep_splits, 32, kLeastKeys / 32).used;
        p = a.deep_part + ((((int64_t)seq * a.kv_heads + kv) * a.deep_blocks * 16 + x) * 2 + m) * a.deep_splits * kPart<D>;
    } else {
        const int64_t end = min(columns, x / a.broad_columns * a.broad_columns + a.broad_columns);
        used = Run(sq.keys(a, (int)((end - 1) / group)), 0, a.broad_splits, broad_unit, kLeastKeys / broad_unit).used;
        p = a.broad_part + ((row * a.heads + head) * 2 + m) * a.broad_splits * kPart<D>;
    }
    if (used <= 1)
        return;
    float hi = -INFINITY;
    for (int i = 0; i < used; ++i)
        hi = fmaxf(hi, p[i * kPart<D>]);
    float total = 0.f, v = 0.f;
#pragma unroll 8
    for (int i = 0; i < used; ++i) {
        const float level = p[i * kPart<D>];
        const float f = level == -INFINITY ? 0.f : exp2_fast(level - hi);
        total = fmaf(f, p[i * kPart<D> + 1], total);
        v = fmaf(f, p[i * kPart<D> + 4 + y], v);
    }
    v = total == 0.f ? 0.f : v / total;
    if (m == 1)
        joined[y] = v;
    __syncthreads();
    if (m == 0 && y % D < a.dim)
        ((T *)a.out.data)[row * a.out.row + head * a.out.head + y / D * a.out.map + y % D] =
            (T)(v - a.lambda[head] * joined[y]);
}

// Tile shapes by head width.
template <class T, int D>
struct Shape {
    static constexpr int kRows = 2 * D * (int)sizeof(T) <= 256 ? 64 : 32;
    static constexpr int kWide = D <= 64 && sizeof(T) == 2 ? 2 : 1;
    static constexpr size_t kLds = 2 * (size_t)kRows * 2 * D * sizeof(T);
    // two buffers of both tiles within the 64 KiB that loads into LDS address
    static constexpr int kBuffers = kLds <= 32768 ? 2 : 1;
    static constexpr int kOccupancy = kLds > 32768 ? 1 : 2;
};

// LDS of the deep part with W waves.
template <int D, int W>
constexpr size_t deep_lds()
{
    constexpr size_t tiles = (size_t)W * 32 * 2 * D * sizeof(Type);
    static_assert(tiles <= 65536, "what loads into LDS address");
    constexpr size_t join = ((size_t)W * 16 * kPart<D> + 16 * 2 * D) * sizeof(float);
    return tiles > join ? tiles : join;
}
template <int D, int W>
hipError_t deep(const PagedArgs &a, int64_t items, hipStream_t s)
{
    constexpr int occ = D * sizeof(Type) < 256 ? 2 : 1;
    return launch_kernel(paged_deep_kernel<Type, D, W, occ>, dim3((unsigned)items), dim3(W * kWave), deep_lds<D, W>(), s, a);
}
// Waves of the broad part, and of the deep part that LDS has room for.
constexpr int kWaves = 4;
template <int D>
constexpr int kDeepWaves = D * sizeof(Type) > 256 ? 2 : 4;

template <int D, int QT>
hipError_t both(const PagedArgs &a, int64_t items, hipStream_t s)
{
    using S = Shape<Type, D>;
    constexpr size_t broad = S::kBuffers * S::kLds, lds = broad > deep_lds<D, kDeepWaves<D>>() ? broad : deep_lds<D, kDeepWaves<D>>();
    return launch_kernel(paged_kernel<Type, D, kWaves, kDeepWaves<D>, QT, S::kRows, S::kBuffers, S::kOccupancy>,
                         dim3((unsigned)items), dim3(kWaves * kWave), lds, s, a);
}

template <int D>
hipError_t run(const PagedArgs &a, hipStream_t s)
{
    using S = Shape<Type, D>;
    const int64_t deep_items = a.deep ? (int64_t)a.sequences * a.kv_heads * a.deep_blocks * a.deep_splits : 0;
    const int64_t items = deep_items + (int64_t)a.broad_tiles * a.kv_heads * a.broad_splits;
    hipError_t e;
    if (a.broad_tiles == 0)
        e = a.deep_splits == 1 ? deep<D, D * sizeof(Type) <= 128 ? 8 : kDeepWaves<D>>(a, items, s)
                               : deep<D, kDeepWaves<D>>(a, items, s);
    else
        e = a.broad_columns == kWaves * 16 ? both<D, 1>(a, items, s) : both<D, S::kWide>(a, items, s);
    if (e != hipSuccess || (a.deep_splits == 1 && a.broad_splits == 1))
        return e;
    return launch_kernel(paged_join<Type, D>, dim3((unsigned)(a.rows * a.heads)), dim3(4 * D), 0, s, a, S::kRows);
}

}  // namespace

hipError_t MTPX_OPS_NAME(paged)(const PagedArgs &a, hipStream_t s)
{
    return a.dim <= 32 ? run<32>(a, s) : a.dim <= 64 ? run<64>(a, s) : run<128>(a, s);
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
