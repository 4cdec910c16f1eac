// Norms of queries and keys for each head with their rotary positions
// (mtpx_head_norm_rotary and its backward pass), and the same on the way into
// a paged cache (mtpx_append_paged):
//
//   u = norm(x),  z = u w,  y = z turned by the row's positions.
//
// Every input is read once and every output written once; those bytes bound
// all three where rows are many (160,000 rows of 8 and 8 heads of two vectors of
// 64 in 16 bits: forward 1.3 GB in 235 us, 5.6 TB/s, backward 2.0 GB in 380 us, 5.2
// TB/s), a launch and the steps of a row where they are
// few (one row: 4.7 us).  Compiled once per element type (MTPX_OPS_TYPE).
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

constexpr int kThreads = 256, kMaxAxes = 8;

__device__ inline double position(const HeadArgs &a, int64_t row, int axis)
{
    const int64_t i = row * a.position_row + axis * a.position_axis;
    switch (a.position_dtype) {
    case MTPX_F32: return ((const float *)a.positions)[i];
    case MTPX_F64: return ((const double *)a.positions)[i];
    case MTPX_I32: return ((const int *)a.positions)[i];
    default: return (double)((const int64_t *)a.positions)[i];
    }
}
__device__ inline int pair_axis(const HeadArgs &a, int p)
{
    const int axis = a.axis[p];
    return axis >= 0 && axis < a.axes ? axis : 0;
}

// N elements that lie at a multiple of A elements.
template <class T, int N, int A = N>
struct alignas(sizeof(T) * A) Piece {
    T e[N];
};

// 1 / sqrt(v), a unit in the last place off; the instruction takes numbers below
// the smallest normal one for 0.
__device__ inline float inverse_root(float v)
{
    const bool small = v < 0x1p-100f;
    return __builtin_amdgcn_rsqf(small ? v * 0x1p64f : v) * (small ? 0x1p32f : 1.f);
}

// A vector's elements over the lanes of its group: U units each.  A unit is W
// elements of both halves of the pairs, or the pairs of W elements side by side
// (one pair where W is 1); units beyond the turning ones are W elements that
// the rotation copies.
template <class T, int W, bool APART, int U>
struct Layout {
    static constexpr int P = APART ? W : W > 1 ? W / 2 : 1;  // pairs of a unit
    static constexpr int E = 2 * P;                          // its elements (W where it does not turn)
    int pairs, turning, units, first, group;

    __device__ inline Layout(const HeadArgs &a, int lane)
        : pairs(a.rotated / 2), turning(pairs / P), units(turning + (a.dim - a.rotated) / W),
          first(lane & (a.group - 1)), group(a.group)
    {
    }
    __device__ inline int unit(int i) const { return first + i * group; }
    // Whether the lane's unit i turns: elements that are copied, two of which would
    // make a pair of it, leave each other alone (0 times an infinity is none).  With
    // the halves apart a copied element's partner is none and stays 0.
    __device__ inline bool turns(int i) const { return APART || unit(i) < turning; }
    // Whether element e of unit u exists.
    __device__ inline bool inside(int u, int e) const { return u < turning || (u < units && e < W); }
    __device__ inline int element(int u, int e) const
    {
        if (u >= turning)
            return 2 * pairs + (u - turning) * W + e;
        return APART ? u * W + e % W + e / W * pairs : u * E + e;
    }

    struct Raw {
        T e[U][E];
    };
    __device__ inline void load(const T *p, Raw &r) const
    {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = unit(i);
#pragma unroll
            for (int e = 0; e < E; ++e)
                r.e[i][e] = (T)0.f;
            if (u < turning) {
                if constexpr (APART) {
                    const Piece<T, W> x = *(const Piece<T, W> *)(p + u * W), y = *(const Piece<T, W> *)(p + pairs + u * W);
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        r.e[i][e] = x.e[e];
                        r.e[i][W + e] = y.e[e];
                    }
                } else {
                    const Piece<T, E, W> x = *(const Piece<T, E, W> *)(p + u * E);
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        r.e[i][e] = x.e[e];
                }
            } else if (u < units) {
                const Piece<T, W> x = *(const Piece<T, W> *)(p + 2 * pairs + (u - turning) * W);
#pragma unroll
                for (int e = 0; e < W; ++e)
                    r.e[i][e] = x.e[e];
            }
        }
    }
    __device__ inline void store(T *p, const Raw &r) const
    {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = unit(i);
            if (u < turning) {
                if constexpr (APART) {
                    Piece<T, W> x, y;
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        x.e[e] = r.e[i][e];
                        y.e[e] = r.e[i][W + e];
                    }
                    *(Piece<T, W> *)(p + u * W) = x;
                    *(Piece<T, W> *)(p + pairs + u * W) = y;
                } else {
                    Piece<T, E, W> x;
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        x.e[e] = r.e[i][e];
                    *(Piece<T, E, W> *)(p + u * E) = x;
                }
            } else if (u < units) {
                Piece<T, W> x;
#pragma unroll
                for (int e = 0; e < W; ++e)
                    x.e[e] = r.e[i][e];
                *(Piece<T, W> *)(p + 2 * pairs + (u - turning) * W) = x;
            }
        }
    }
    __device__ inline void widen(const Raw &r, float (&v)[U][E]) const
    {
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[i][e] = (float)r.e[i][e];
    }
    __device__ inline void round(const float (&v)[U][E], Raw &r) const
    {
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)
                r.e[i][e] = (T)v[i][e];
    }
    __device__ inline void weights(const void *w, float (&v)[U][E]) const
    {
        if (w) {
            Raw r;
            load((const T *)w, r);
            widen(r, v);
            return;
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[i][e] = 1.f;
    }
    // Sum over a vector's lanes, the same in all of them.
    __device__ inline float sum(float v) const
    {
        if (group > 1)
            v += moved<0xb1, 0xf>(v);  // quad_perm 1 0 3 2
        if (group > 2)
            v += moved<0x4e, 0xf>(v);  // quad_perm 2 3 0 1
        if (group > 4)
            v += moved<0x141, 0xf>(v);  // row_half_mirror
        if (group > 8)
            v += moved<0x140, 0xf>(v);  // row_mirror
        if (group > 16)
            v += __shfl_xor(v, 16);
        if (group > 32)
            v += __shfl_xor(v, 32);
        return v;
    }
    // t = x - mean (layer) or x becomes u = t / sqrt(mean(t^2) + eps); returns
    // the factor.
    __device__ inline float normalise(const HeadArgs &a, float (&v)[U][E]) const
    {
        const float scale = 1.f / a.dim;
        if (a.kind == MTPX_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    s += v[i][e];
            const float mean = sum(s) * scale;
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    v[i][e] = inside(unit(i), e) ? v[i][e] - mean : 0.f;
        }
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)
                q = fmaf(v[i][e], v[i][e], q);
        const float inv = inverse_root(fmaf(sum(q), scale, a.eps));
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[i][e] *= inv;
        return inv;
    }
    // Elements of a unit's pair j.
    static __device__ inline constexpr int one(int j) { return APART ? j : 2 * j; }
    static __device__ inline constexpr int two(int j) { return APART ? W + j : 2 * j + 1; }
};

// cos and sin of a row's pairs, each formed once for all of its heads: the
// angle is reduced to a fraction of a turn in 64 bits.
__device__ inline void fill_table(const HeadArgs &a, int64_t row, int lane, float2 *table)
{
    for (int p = lane; p < a.rotated / 2; p += a.lanes) {
        const double turns = position(a, row, pair_axis(a, p)) * (double)a.freq[p] * 0.15915494309189533577;
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        table[p] = make_float2(c, s);
    }
}

// A unit's cos and sin; the copied units turn by 0.
template <class L, int U, int P>
__device__ inline void read_table(const L &at, const float2 *table, float (&c)[U][P], float (&s)[U][P])
{
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const bool turns = at.unit(i) < at.turning;
            const float2 cs = turns ? table[at.unit(i) * P + j] : make_float2(1.f, 0.f);
            c[i][j] = cs.x;
            s[i][j] = cs.y;
        }
}

__device__ inline void wave_order()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The same for all lanes of a row: one wave's, or a workgroup's.
__device__ inline void row_order(const HeadArgs &a)
{
    if (a.lanes > kWave)
        __syncthreads();
    else
        wave_order();
}

// `lanes` lanes per row (several rows a wave where a row has little work, a
// whole workgroup where there are few rows), `group` of them per vector.  A lane
// keeps its unit's place in every vector, and so its cos, sin and weights, and
// reads a vector ahead of the one that it works on.
template <class T, int W, bool APART, int U, bool APPEND>
__global__ __launch_bounds__(kThreads) void head_forward_kernel(HeadArgs a)
{
    using L = Layout<T, W, APART, U>;
    __shared__ float2 tables[kThreads * L::P * U];
    const int lane = threadIdx.x & (a.lanes - 1), mine = threadIdx.x / a.lanes;
    const L at(a, lane);
    const int64_t row = (int64_t)blockIdx.x * (kThreads / a.lanes) + mine;
    bool there = row < a.rows;
    T *to_k = nullptr, *to_v = nullptr;
    if constexpr (APPEND) {
        const int i = last_true([&](int j) { return row_offset(a.offsets, j, a.rows) <= row; }, a.sequences + 1,
                                min(a.lanes, kWave));
        there = there && i >= 0 && i < a.sequences;
        if (there) {
            const mtpx_pages &c = a.cache;
            const int64_t t = (int64_t)a.lengths[i] - row_offset(a.offsets, i + 1, a.rows) + row;
            if (t >= 0 && t < (int64_t)c.table_width * c.page_rows) {
                const int p = c.table[i * c.table_row + (int)t / c.page_rows], slot = (int)t % c.page_rows;
                if (p >= 0 && p < c.pages) {
                    to_k = (T *)c.k.data + p * c.k_page + slot * c.k.row;
                    to_v = (T *)c.v.data + p * c.v_page + slot * c.v.row;
                }
            }
        }
    }
    const int first = lane / a.group, step = a.lanes / a.group, bits = a.maps - 1;
    // the first vectors come while the table is filled
    typename L::Raw early[2];
#pragma unroll
    for (int job = 0; job < 2; ++job)
        if (there && first < a.vectors[job])
            at.load((const T *)a.in[job].data + row * a.in[job].row + (first >> bits) * a.in[job].head + (first & bits) * a.in[job].map, early[job]);
    float2 *table = tables + mine * at.pairs;
    if (there)
        fill_table(a, row, lane, table);
    row_order(a);
    if (!there)
        return;
    float c[U][L::P], s[U][L::P];
    read_table<L, U, L::P>(at, table, c, s);

#pragma unroll
    for (int job = 0; job < 2; ++job) {
        const int n = a.vectors[job];
        if (first >= n || (APPEND && job == 1 && !to_k))
            continue;
        const mtpx_rows &from = a.in[job], &to = APPEND && job == 1 ? a.cache.k : a.out[job];
        const T *x = (const T *)from.data + row * from.row;
        T *y = APPEND && job == 1 ? to_k : (T *)to.data + row * to.row;
        float w[U][L::E];
        at.weights(a.weight[job], w);
        typename L::Raw next = early[job];
        for (int v = first; v < n; v += step) {
            float z[U][L::E];
            at.widen(next, z);
            const int ahead = v + step;
            if (ahead < n)
                at.load(x + (ahead >> bits) * from.head + (ahead & bits) * from.map, next);
            if (a.kind != MTPX_NORM_NONE)
                at.normalise(a, z);
#pragma unroll
            for (int i = 0; i < U; ++i) {
#pragma unroll
                for (int e = 0; e < L::E; ++e)
                    z[i][e] *= w[i][e];
                if (!at.turns(i))
                    continue;
#pragma unroll
                for (int j = 0; j < L::P; ++j) {
                    const float z1 = z[i][L::one(j)], z2 = z[i][L::two(j)];
                    z[i][L::one(j)] = z1 * c[i][j] - z2 * s[i][j];
                    z[i][L::two(j)] = z1 * s[i][j] + z2 * c[i][j];
                }
            }
            typename L::Raw r;
            at.round(z, r);
            at.store(y + (v >> bits) * to.head + (v & bits) * to.map, r);
        }
    }
    if constexpr (APPEND) {
        if (!to_v)
            return;
        const T *x = (const T *)a.v.data + row * a.v.row;
        for (int v = first; v < a.vectors[1]; v += step) {
            typename L::Raw r;
            at.load(x + (v >> bits) * a.v.head + (v & bits) * a.v.map, r);
            at.store(to_v + (v >> bits) * a.cache.v.head + (v & bits) * a.cache.v.map, r);
        }
    }
}

// With g = dz w:  dx = (g - [mean g] - u mean(g u)) / size,  dw = sum dz u, and
// a pair's share of the positions' gradient freq (dz2 z1 - dz1 z2), which the
// rotation leaves as it is.  u is formed again from x.  A row's lanes are a part of
// a wave or a workgroup; a workgroup takes rows part, part + groups, ... and keeps its share of
// the weights' gradients in registers until the end: a.parts partial rows.
template <class T, int W, bool APART, int U, bool MOVED>
__global__ __launch_bounds__(kThreads) void head_backward_kernel(HeadArgs a)
{
    using L = Layout<T, W, APART, U>;
    // the tables of the rows, and at the end the lanes' sums
    __shared__ float shared[kThreads * L::E * U];
    __shared__ float moved[MOVED ? kMaxAxes : 1][kThreads / kWave];  // the waves' sums
    const int lane = threadIdx.x & (a.lanes - 1), mine = threadIdx.x / a.lanes;
    const L at(a, lane);
    float2 *table = (float2 *)shared + mine * at.pairs;
    const int first = lane / a.group, step = a.lanes / a.group, bits = a.maps - 1;
    const float scale = 1.f / a.dim;
    float dw[2][U][L::E];
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < L::E; ++e)
            dw[0][i][e] = dw[1][i][e] = 0.f;

    const int together = kThreads / a.lanes;
    for (int64_t row = (int64_t)blockIdx.x * together + mine; row < a.rows; row += (int64_t)gridDim.x * together) {
        typename L::Raw early[2][2];
#pragma unroll
        for (int job = 0; job < 2; ++job)
            if (first < a.vectors[job]) {
                const mtpx_rows &x = a.in[job], &y = a.grad[job];
                at.load((const T *)x.data + row * x.row + (first >> bits) * x.head + (first & bits) * x.map, early[job][0]);
                at.load((const T *)y.data + row * y.row + (first >> bits) * y.head + (first & bits) * y.map, early[job][1]);
            }
        row_order(a);  // the last row's reads of the table
        fill_table(a, row, lane, table);
        row_order(a);
        float c[U][L::P], s[U][L::P], d[U][L::P];
        read_table<L, U, L::P>(at, table, c, s);
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < L::P; ++j)
                d[i][j] = 0.f;
#pragma unroll
        for (int job = 0; job < 2; ++job) {
            const int n = a.vectors[job];
            if (first >= n)
                continue;
            const mtpx_rows &fx = a.in[job], &fy = a.grad[job], &to = a.out[job];
            const T *x = (const T *)fx.data + row * fx.row, *dy = (const T *)fy.data + row * fy.row;
            T *dx = (T *)to.data + row * to.row;
            float w[U][L::E];
            at.weights(a.weight[job], w);
            auto read = [&](int v, typename L::Raw &rx, typename L::Raw &ry) {
                if (v < n) {
                    at.load(x + (v >> bits) * fx.head + (v & bits) * fx.map, rx);
                    at.load(dy + (v >> bits) * fy.head + (v & bits) * fy.map, ry);
                }
            };
            typename L::Raw rx = early[job][0], ry = early[job][1];
            for (int v = first; v < n; v += step) {
                float u[U][L::E], g[U][L::E];
                at.widen(rx, u);
                at.widen(ry, g);
                read(v + step, rx, ry);
                const float inv = at.normalise(a, u);
                float s0 = 0.f, s1 = 0.f;
#pragma unroll
                for (int i = 0; i < U; ++i) {
#pragma unroll
                    for (int j = 0; j < L::P; ++j) {
                        const int k = L::one(j), l = L::two(j);
                        const float d1 = g[i][k], d2 = g[i][l];
                        // (a choice of the partner, not a branch: a step of 4,001 rows of 10 and 5
                        // heads of 40 in 32 bits, 36 turning, takes 40.8 us, 41.4 us with one)
                        g[i][k] = d1 * c[i][j] + (at.turns(i) ? d2 : 0.f) * s[i][j];
                        g[i][l] = d2 * c[i][j] - (at.turns(i) ? d1 : 0.f) * s[i][j];
                        if constexpr (MOVED)
                            d[i][j] += g[i][l] * (u[i][k] * w[i][k]) - g[i][k] * (u[i][l] * w[i][l]);
                    }
#pragma unroll
                    for (int e = 0; e < L::E; ++e) {
                        dw[job][i][e] = fmaf(g[i][e], u[i][e], dw[job][i][e]);
                        g[i][e] *= w[i][e];
                        s1 = fmaf(g[i][e], u[i][e], s1);
                    }
                }
                if (a.kind == MTPX_NORM_LAYER) {
#pragma unroll
                    for (int i = 0; i < U; ++i)
#pragma unroll
                        for (int e = 0; e < L::E; ++e)
                            s0 += g[i][e];
                    s0 = at.sum(s0) * scale * inv;
                }
                s1 = at.sum(s1) * scale * inv;
#pragma unroll
                for (int i = 0; i < U; ++i)
#pragma unroll
                    for (int e = 0; e < L::E; ++e)
                        g[i][e] = fmaf(-u[i][e], s1, fmaf(g[i][e], inv, -s0));
                typename L::Raw r;
                at.round(g, r);
                at.store(dx + (v >> bits) * to.head + (v & bits) * to.map, r);
            }
        }
        if constexpr (MOVED) {
            float sums[kMaxAxes] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int j = 0; j < L::P; ++j)
                    if (at.unit(i) < at.turning) {
                        const int p = at.unit(i) * L::P + j, axis = pair_axis(a, p);
                        const float v = d[i][j] * a.freq[p];
#pragma unroll
                        for (int k = 0; k < kMaxAxes; ++k)
                            sums[k] += axis == k ? v : 0.f;
                    }
#pragma unroll
            for (int k = 0; k < kMaxAxes; ++k) {
                if (k >= a.axes)
                    break;
                float v = sums[k];
                for (int o = min(a.lanes, kWave) / 2; o > 0; o >>= 1)
                    v += __shfl_xor(v, o);
                if (a.lanes > kWave) {
                    if (lane % kWave == 0)
                        moved[k][lane / kWave] = v;
                    __syncthreads();
                    v = moved[k][0];
                    for (int w = 1; w < kThreads / kWave; ++w)
                        v += moved[k][w];
                }
                if (lane == 0) {
                    if (a.position_dtype == MTPX_F64)
                        ((double *)a.dpositions)[row * a.axes + k] = v;
                    else
                        ((float *)a.dpositions)[row * a.axes + k] = v;
                }
            }
        }
    }

    // the lanes of a workgroup that hold the same elements, in a fixed order: an
    // element a thread, of short vectors, which many lanes hold, a part of one's (one
    // row of vectors of 16: 13.6 us, 17.6 us an element a thread; 4,001 rows of 40:
    // 25.8 and 24.9 us)
    const int runs = a.dim <= 32 ? kThreads / a.dim : 1;
#pragma unroll
    for (int job = 0; job < 2; ++job) {
        if (!a.dweight[job])
            continue;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int x = 0; x < L::E; ++x)
                if (at.inside(at.unit(i), x))
                    shared[threadIdx.x / a.group * a.dim + at.element(at.unit(i), x)] = dw[job][i][x];
        __syncthreads();
        float *const part = a.part + ((int64_t)job * a.parts + blockIdx.x) * a.dim;
        if (runs == 1) {
            for (int e = threadIdx.x; e < a.dim; e += kThreads) {
                float v = 0.f;
                for (int k = 0; k < kThreads / a.group; ++k)
                    v += shared[k * a.dim + e];
                part[e] = v;
            }
            continue;
        }
        const int e = threadIdx.x % a.dim, run = threadIdx.x / a.dim;
        float v = 0.f;
        if (run < runs)
#pragma unroll 4
            for (int k = run; k < kThreads / a.group; k += runs)
                v += shared[k * a.dim + e];
        __syncthreads();
        shared[threadIdx.x] = v;
        __syncthreads();
        if (run == 0) {
#pragma unroll 4
            for (int k = 1; k < runs; ++k)
                v += shared[k * a.dim + e];
            part[e] = v;
        }
    }
}

// Sums the parts of the weights' gradients: 16 columns and 64 runs of parts a
// workgroup, the runs in a fixed order (64 columns and 16 runs, with a fourth of
// the workgroups and four times the reads one after the other: 6.4 us of 4,001
// rows, 4.6 us so).
template <class T>
__global__ __launch_bounds__(1024) void head_parts_kernel(HeadArgs a)
{
    constexpr int kColumns = 16, kRuns = 1024 / kColumns, kEach = kRuns / (kWave / kColumns);
    __shared__ float red[kRuns][kColumns];
    const int job = blockIdx.y, column = threadIdx.x % kColumns, run = threadIdx.x / kColumns;
    T *out = (T *)a.dweight[job];
    if (!out)
        return;
    const int c = blockIdx.x * kColumns + column;
    float v = 0.f;
    if (c < a.dim) {
#pragma unroll 8
        for (int p = run; p < a.parts; p += kRuns)
            v += a.part[((int64_t)job * a.parts + p) * a.dim + c];
    }
    red[run][column] = v;
    __syncthreads();
    if (threadIdx.x >= kWave)
        return;
    v = 0.f;
#pragma unroll
    for (int r = 0; r < kEach; ++r)
        v += red[run * kEach + r][column];
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    if (run == 0 && c < a.dim)
        out[c] = (T)v;
}

enum Pass { kForward, kAppend, kBackward };

template <int W, bool APART, int U>
hipError_t launch(const HeadArgs &a, Pass pass, hipStream_t s)
{
    const int rows = kThreads / a.lanes;
    const dim3 grid((unsigned)(pass == kBackward ? a.parts : (a.rows + rows - 1) / rows)), block(kThreads);
    const auto kernel = pass == kForward   ? head_forward_kernel<Type, W, APART, U, false>
                        : pass == kAppend  ? head_forward_kernel<Type, W, APART, U, true>
                        : a.dpositions     ? head_backward_kernel<Type, W, APART, U, true>
                                           : head_backward_kernel<Type, W, APART, U, false>;
    return launch_kernel(kernel, grid, block, 0, s, a);
}
template <int W, int U>
hipError_t by_pairs(const HeadArgs &a, Pass pass, hipStream_t s)
{
    return a.interleaved ? launch<W, false, U>(a, pass, s) : launch<W, true, U>(a, pass, s);
}
hipError_t by_width(const HeadArgs &a, Pass pass, hipStream_t s)
{
    // a vector in a group's lanes: one unit each, or up to four
    const int unit = a.interleaved ? (a.width > 1 ? a.width / 2 : 1) : a.width;
    const int units = a.rotated / 2 / unit + (a.dim - a.rotated) / a.width;
    if (units <= a.group) {
        switch (a.width) {
        case 8:
            if constexpr (sizeof(Type) == 2)
                return by_pairs<8, 1>(a, pass, s);
            return hipErrorInvalidValue;
        case 4: return by_pairs<4, 1>(a, pass, s);
        case 2: return by_pairs<2, 1>(a, pass, s);
        default: return by_pairs<1, 1>(a, pass, s);
        }
    }
    if (units > 4 * a.group)
        return hipErrorInvalidValue;
    return a.width == 2 ? by_pairs<2, 4>(a, pass, s) : a.width == 1 ? by_pairs<1, 4>(a, pass, s) : hipErrorInvalidValue;
}

}  // namespace

hipError_t MTPX_OPS_NAME(head_pass)(const HeadArgs &a, int pass, hipStream_t s)
{
    if (pass != kBackward)
        return by_width(a, (Pass)pass, s);
    if (a.rows > 0)
        if (hipError_t e = by_width(a, kBackward, s))
            return e;
    if (!a.dweight[0] && !a.dweight[1])
        return hipSuccess;
    // (without rows it writes zeros)
    return launch_kernel(head_parts_kernel<Type>, dim3((a.dim + 15) / 16, 2), dim3(1024), 0, s, a);
}

#if MTPX_OPS_TYPE == 0
hipError_t head_pass_bf16(const HeadArgs &, int, hipStream_t);
hipError_t head_pass_f16(const HeadArgs &, int, hipStream_t);

namespace {
hipError_t by_type(int dtype, const HeadArgs &a, int pass, hipStream_t s)
{
    return dtype == MTPX_F32    ? head_pass_f32(a, pass, s)
           : dtype == MTPX_BF16 ? head_pass_bf16(a, pass, s)
                                : head_pass_f16(a, pass, s);
}
}  // namespace
hipError_t launch_head_forward(int dtype, const HeadArgs &a, hipStream_t s) { return by_type(dtype, a, kForward, s); }
hipError_t launch_head_append(int dtype, const HeadArgs &a, hipStream_t s) { return by_type(dtype, a, kAppend, s); }
hipError_t launch_head_backward(int dtype, const HeadArgs &a, hipStream_t s) { return by_type(dtype, a, kBackward, s); }
#endif

}  // namespace mtpx
