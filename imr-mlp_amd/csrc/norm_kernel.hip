// The norms around a block with its gate and residual (mtpx_norm_block and
// its backward pass):
//
//   u = norm(y),  s = alpha x + beta act(g) (u w1),  n = norm(s) w2.
//
// Both kernels keep a row in registers between its sums, so every input is
// read once and every output written once; they are bound by those bytes.
#include "ops_device.hpp"

namespace mtpx {

namespace {

constexpr int kMaxBlock = 1024;

// A row's columns over NT threads, E of them each, in pieces of V elements
// that are read at once (V 1 where rows are not whole 16-byte pieces).
template <class T, int NT, int E, int V>
struct Row {
    static constexpr int kBlock = NT <= kWave ? 256 : NT;
    static constexpr int kPerBlock = kBlock / NT;                    // rows of a workgroup
    static constexpr int kPerWave = NT < kWave ? kWave / NT : 1;      // and of a wave
    static constexpr int kPieces = E / V;
    static __device__ inline int column(int i, int t) { return (i * NT + t) * V; }

    // A row as it lies in memory: read ahead, widened when it is needed.
    // Columns beyond width are 0.
    struct alignas(V * sizeof(T)) Piece {
        T e[V];
    };
    struct Raw {
        Piece p[kPieces];
    };
    static __device__ inline void fetch(const T *p, int width, int t, Raw &r)
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int c = column(i, t);
            r.p[i] = Piece{};
            if (c < width)
                r.p[i] = *reinterpret_cast<const Piece *>(p + c);
        }
    }
    static __device__ inline void widen(const Raw &r, float (&v)[E])
    {
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] = (float)r.p[e / V].e[e % V];
    }
    static __device__ inline void load(const T *p, int width, int t, float (&v)[E])
    {
        Raw r;
        fetch(p, width, t, r);
        widen(r, v);
    }
    static __device__ inline void store(T *p, int width, int t, const float (&v)[E])
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int c = column(i, t);
            if (c >= width)
                continue;
            Piece u;
#pragma unroll
            for (int j = 0; j < V; ++j)
                u.e[j] = (T)v[i * V + j];
            *reinterpret_cast<Piece *>(p + c) = u;
        }
    }
    static __device__ inline bool inside(int e, int t, int width)
    {
        return column(e / V, t) + e % V < width;
    }
    // Sum over the row's threads, in a fixed order.
    static __device__ inline float sum(float v, float *red)
    {
        if constexpr (NT < kWave) {
            v = row16_sum(v);
            return NT == 32 ? v + __shfl_xor(v, 16) : v;
        }
        v = wave_sum(v);
        if constexpr (NT > kWave) {
            constexpr int kWavesRow = NT / kWave;
            const int wave = threadIdx.x / kWave;
            __syncthreads();
            if (threadIdx.x % kWave == 0)
                red[wave] = v;
            __syncthreads();
            v = 0.f;
#pragma unroll
            for (int w = 0; w < kWavesRow; ++w)
                v += red[w];
        }
        return v;
    }
};

// 1 / (1 + e^-g) and tanh(g) from one exponential and one reciprocal (a unit
// in the last place each); tanh near 0, where 1 - e cancels, from its series,
// whose first term left out is 9e-9 of it at 1/4.
__device__ inline float act(int kind, float g)
{
    if (kind == MTPX_GATE_SIGMOID)
        return __builtin_amdgcn_rcpf(1.f + exp2_fast(-g * kLog2e));
    if (kind == MTPX_GATE_TANH) {
        const float e = exp2_fast(-2.f * kLog2e * fabsf(g));
        const float far = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), g);
        const float q = g * g;
        const float near = g + g * q * fmaf(q, fmaf(q, fmaf(q, 62.f / 2835, -17.f / 315), 2.f / 15), -1.f / 3);
        return fabsf(g) < 0.25f ? near : far;
    }
    return g;
}
// Derivative from the activation's value.
__device__ inline float act_slope(int kind, float a)
{
    return kind == MTPX_GATE_SIGMOID ? a * (1.f - a) : kind == MTPX_GATE_TANH ? 1.f - a * a : 1.f;
}

// Mean (0 for RMS) and 1 / sqrt(variance + eps) of a row; v is left centred.
template <class R, int E>
__device__ inline void normalise(float (&v)[E], int kind, int width, float eps, int t, float *red, float &mean,
                                 float &inv)
{
    mean = 0.f;
    if (kind == MTPX_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            s += v[e];
        mean = R::sum(s, red) / width;
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] = R::inside(e, t, width) ? v[e] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
        q = fmaf(v[e], v[e], q);
    inv = 1.f / sqrtf(R::sum(q, red) / width + eps);
}

// A group of NT threads takes rows part, part + groups, ...: the weights and a
// gate shared by all rows stay in registers, and a row's inputs are read while
// the row before is worked on.
template <class T, int NT, int E, int V>
__global__ __launch_bounds__((Row<T, NT, E, V>::kBlock)) void norm_forward_kernel(NormArgs a)
{
    using R = Row<T, NT, E, V>;
    __shared__ float red[kMaxBlock / kWave];
    const int t = threadIdx.x % NT;
    const int64_t part = (int64_t)blockIdx.x * R::kPerBlock + threadIdx.x / NT;
    const int64_t groups = (int64_t)gridDim.x * R::kPerBlock;
    const bool own_gate = a.gate && a.gate_row != 0;
    if (NT >= kWave && part >= a.rows)  // a row's threads leave together
        return;
    float post[E], pre[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        post[e] = pre[e] = 1.f;
    if (a.post)
        R::load((const T *)a.post, a.width, t, post);
    if (a.pre)
        R::load((const T *)a.pre, a.width, t, pre);
    if (a.gate && !own_gate) {
        float g[E];
        R::load((const T *)a.gate, a.width, t, g);
#pragma unroll
        for (int e = 0; e < E; ++e)
            post[e] *= act(a.act, g[e]);
    }
    typename R::Raw ry, rx, rg;
    auto ahead = [&](int64_t row) {
        if (row >= a.rows)
            return;
        R::fetch((const T *)a.y + row * a.y_row, a.width, t, ry);
        if (a.x)
            R::fetch((const T *)a.x + row * a.x_row, a.width, t, rx);
        if (own_gate)
            R::fetch((const T *)a.gate + row * a.gate_row, a.width, t, rg);
    };
    ahead(part);
    // (a wave's rows end together: one beyond the last is worked on unseen)
    for (int64_t row0 = part - part % R::kPerWave; row0 < a.rows; row0 += groups) {
        const int64_t row = row0 + part % R::kPerWave;
        const bool there = row < a.rows;
        float v[E], x[E], g[E];
        R::widen(ry, v);
        R::widen(rx, x);
        R::widen(rg, g);
        ahead(row + groups);
        float mean, inv;
        normalise<R>(v, a.kind, a.width, a.eps, t, red, mean, inv);
        if (a.stats && t == 0 && there) {
            a.stats[4 * row] = mean;
            a.stats[4 * row + 1] = inv;
        }
        const float b = a.block_scale * inv;
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] *= b * post[e];
        if (own_gate) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[e] *= act(a.act, g[e]);
        }
        if (a.x) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[e] = fmaf(a.residual_scale, x[e], v[e]);
        }
        R::store((T *)a.s + row * a.s_row, there ? a.width : 0, t, v);
        if (!a.n)
            continue;
        normalise<R>(v, a.kind, a.width, a.eps, t, red, mean, inv);
        if (a.stats && t == 0 && there) {
            a.stats[4 * row + 2] = mean;
            a.stats[4 * row + 3] = inv;
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] *= inv * pre[e];
        R::store((T *)a.n + row * a.n_row, there ? a.width : 0, t, v);
    }
}

// With v = (s - mean) r:  ds = ds_in + r (dv - [mean dv] - v mean(dv v)),
// dv = dn w2; the same again through the first norm.  s is formed again from
// x, y and the gate (the bytes of reading it back, without its rounding).
// A group of NT threads takes rows part, part + groups, ... and keeps its
// share of the weights' gradients in registers; a.parts workgroups leave one
// partial row of each.
template <class T, int NT, int E, int V>
__global__ __launch_bounds__((Row<T, NT, E, V>::kBlock), NT < 1024 ? 3 : 4) void norm_backward_kernel(NormArgs a)
{
    using R = Row<T, NT, E, V>;
    __shared__ float red[kMaxBlock / kWave];
    const int t = threadIdx.x % NT;
    // (a group without a row stays for the sums at the end)
    const int64_t part = (int64_t)blockIdx.x * R::kPerBlock + threadIdx.x / NT;
    const int64_t groups = (int64_t)gridDim.x * R::kPerBlock;
    const bool layer = a.kind == MTPX_NORM_LAYER;
    const float scale = 1.f / a.width;
    float dw1[E], dw2[E], dgs[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        dw1[e] = dw2[e] = dgs[e] = 0.f;
    const bool own_gate = a.gate && a.gate_row != 0;
    float g[E];
    if (a.gate && !own_gate) {
        R::load((const T *)a.gate, a.width, t, g);
#pragma unroll
        for (int e = 0; e < E; ++e)
            g[e] = act(a.act, g[e]);
    }
    // what a row starts with is read one row ahead
    typename R::Raw ry, rx, rdn, rds, rpost, rpre;
    if (a.post)
        R::fetch((const T *)a.post, a.width, t, rpost);
    if (a.pre)
        R::fetch((const T *)a.pre, a.width, t, rpre);
    f32x4 rst;
    auto ahead = [&](int64_t row) {
        if (row >= a.rows) {
            // zeros take part in the sums of a wave's other rows
            rst = f32x4{0, 0, 0, 0};
            ry = rx = rdn = rds = typename R::Raw{};
            return;
        }
        R::fetch((const T *)a.y + row * a.y_row, a.width, t, ry);
        if (a.x)
            R::fetch((const T *)a.x + row * a.x_row, a.width, t, rx);
        if (a.dn)
            R::fetch((const T *)a.dn + row * a.dn_row, a.width, t, rdn);
        if (a.ds)
            R::fetch((const T *)a.ds + row * a.ds_row, a.width, t, rds);
        rst = *reinterpret_cast<const f32x4 *>(a.stats + 4 * row);
    };
    ahead(part);
    for (int64_t row0 = part - part % R::kPerWave; row0 < a.rows; row0 += groups) {
        const int64_t row = row0 + part % R::kPerWave;
        const bool there = row < a.rows;
        const f32x4 st = rst;
        float u[E], v[E], w[E], ds[E];
        R::widen(ry, u);
        R::widen(rx, v);
        R::widen(rdn, ds);
        const typename R::Raw into = rds;
        if (own_gate)
            R::load((const T *)a.gate + row * a.gate_row, there ? a.width : 0, t, g);
        if (a.post)
            R::widen(rpost, w);
        ahead(row + groups);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            u[e] = R::inside(e, t, a.width) ? (u[e] - st[0]) * st[1] : 0.f;
            if (!a.gate)
                g[e] = 1.f;
            else if (own_gate)
                g[e] = act(a.act, g[e]);
            if (!a.post)
                w[e] = 1.f;
            const float z = a.block_scale * g[e] * u[e] * w[e];
            v[e] = a.x ? fmaf(a.residual_scale, v[e], z) : z;
        }
        if (a.dn) {
            float w2[E], s0 = 0.f, s1 = 0.f;
            if (a.pre)
                R::widen(rpre, w2);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[e] = R::inside(e, t, a.width) ? (v[e] - st[2]) * st[3] : 0.f;
                dw2[e] = fmaf(ds[e], v[e], dw2[e]);
                if (a.pre)
                    ds[e] *= w2[e];
                s0 += ds[e];
                s1 = fmaf(ds[e], v[e], s1);
            }
            s0 = layer ? R::sum(s0, red) * scale : 0.f;
            s1 = R::sum(s1, red) * scale;
#pragma unroll
            for (int e = 0; e < E; ++e)
                ds[e] = st[3] * (ds[e] - s0 - v[e] * s1);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                ds[e] = 0.f;
        }
        if (a.ds) {
            R::widen(into, v);
#pragma unroll
            for (int e = 0; e < E; ++e)
                ds[e] += v[e];
        }
        if (a.dx) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[e] = a.residual_scale * ds[e];
            R::store((T *)a.dx + row * a.dx_row, there ? a.width : 0, t, v);
        }
        // through the gate and the first norm
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = R::inside(e, t, a.width) ? a.block_scale * ds[e] : 0.f;
            v[e] = act_slope(a.act, g[e]) * u[e] * w[e] * d;
            dgs[e] += v[e];
            const float dz = g[e] * d;
            dw1[e] = fmaf(dz, u[e], dw1[e]);
            ds[e] = dz * w[e];
            s0 += ds[e];
            s1 = fmaf(ds[e], u[e], s1);
        }
        if (a.dgate && a.gate_row != 0)
            R::store((T *)a.dgate + row * a.dgate_row, there ? a.width : 0, t, v);
        if (a.dy) {
            s0 = layer ? R::sum(s0, red) * scale : 0.f;
            s1 = R::sum(s1, red) * scale;
#pragma unroll
            for (int e = 0; e < E; ++e)
                ds[e] = st[1] * (ds[e] - s0 - u[e] * s1);
            R::store((T *)a.dy + row * a.dy_row, there ? a.width : 0, t, ds);
        }
    }
    // The rows of a workgroup are summed through LDS, in their order.
    auto leave = [&](int which, const float (&d)[E]) {
        float *p = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * a.width;
        if constexpr (R::kPerBlock == 1) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (R::inside(e, t, a.width))
                    p[R::column(e / V, t) + e % V] = d[e];
        } else {
            __shared__ float sums[R::kPerBlock][NT * E];
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e)
                sums[threadIdx.x / NT][R::column(e / V, t) + e % V] = d[e];
            __syncthreads();
            for (int c = threadIdx.x; c < a.width; c += R::kBlock) {
                float s = 0.f;
#pragma unroll
                for (int r = 0; r < R::kPerBlock; ++r)
                    s += sums[r][c];
                p[c] = s;
            }
        }
    };
    if (a.dpost)
        leave(0, dw1);
    if (a.dpre)
        leave(1, dw2);
    if (a.dgate && a.gate_row == 0)
        leave(2, dgs);
}

// Sums the parts of the weights' gradients: 64 columns and 16 runs of parts
// a workgroup, the runs in a fixed order.
template <class T>
__global__ __launch_bounds__(kMaxBlock) void norm_parts_kernel(NormArgs a)
{
    constexpr int kRuns = kMaxBlock / kWave;
    __shared__ float red[kRuns][kWave];
    const int which = blockIdx.y, lane = threadIdx.x % kWave, run = threadIdx.x / kWave;
    T *out = (T *)(which == 0 ? a.dpost : which == 1 ? a.dpre : a.gate_row == 0 ? a.dgate : nullptr);
    if (!out)
        return;
    const int c = blockIdx.x * kWave + lane;
    float v = 0.f;
    if (c < a.width) {
#pragma unroll 8
        for (int p = run; p < a.parts; p += kRuns)
            v += a.part[((int64_t)which * a.parts + p) * a.width + c];
    }
    red[run][lane] = v;
    __syncthreads();
    if (run == 0 && c < a.width) {
        for (int r = 1; r < kRuns; ++r)
            v += red[r][lane];
        out[c] = (T)v;
    }
}

template <class T, int NT, int E, int V>
hipError_t run(const NormArgs &a, bool back, hipStream_t s)
{
    using R = Row<T, NT, E, V>;
    // the forward pass: what its registers let in at once, four waves per SIMD
    const int64_t need = (a.rows + R::kPerBlock - 1) / R::kPerBlock;
    const int64_t most = 256 * (16 * kWave / R::kBlock);
    const dim3 grid((unsigned)(back ? a.parts : need < most ? need : most)), block(R::kBlock);
    return launch_kernel(back ? norm_backward_kernel<T, NT, E, V> : norm_forward_kernel<T, NT, E, V>, grid, block, 0, s, a);
}

// The fewest threads that hold a row with 8 elements each (16 beyond 8,192
// columns), a power of two from 16 on or, of whole waves, 3/4 of one (forward
// and backward of 51,198 rows of 2,352 columns in 16 bits: 887 us with 512
// threads, 740 us with 384).  More elements leave the backward pass fewer waves
// per SIMD to hide its reads (160,000 rows of 1,024: 611 us with 16 elements a
// thread).
int row_threads(int width)
{
    int n = 16;
    while (n < kMaxBlock && width > 8 * n)
        n *= 2;
    return n > 2 * kWave && width <= 6 * n ? n / 4 * 3 : n;
}
template <class T, int V>
hipError_t by_width(const NormArgs &a, bool back, hipStream_t s)
{
    switch (row_threads(a.width)) {
    case 16: return run<T, 16, 8, V>(a, back, s);
    case 32: return run<T, 32, 8, V>(a, back, s);
    case 64: return run<T, 64, 8, V>(a, back, s);
    case 128: return run<T, 128, 8, V>(a, back, s);
    case 192: return run<T, 192, 8, V>(a, back, s);
    case 256: return run<T, 256, 8, V>(a, back, s);
    case 384: return run<T, 384, 8, V>(a, back, s);
    case 512: return run<T, 512, 8, V>(a, back, s);
    case 768: return run<T, 768, 8, V>(a, back, s);
    default: return a.width <= 8192 ? run<T, 1024, 8, V>(a, back, s) : run<T, 1024, 16, V>(a, back, s);
    }
}

template <class T>
hipError_t by_vec(const NormArgs &a, bool back, hipStream_t s)
{
    const hipError_t e = a.vec ? by_width<T, 16 / sizeof(T)>(a, back, s) : by_width<T, 1>(a, back, s);
    if (e != hipSuccess || !back || !(a.dpost || a.dpre || (a.dgate && a.gate_row == 0)))
        return e;
    return launch_kernel(norm_parts_kernel<T>, dim3((a.width + kWave - 1) / kWave, 3), dim3(kMaxBlock), 0, s, a);
}

hipError_t by_type(int dtype, const NormArgs &a, bool back, hipStream_t s)
{
    return dtype == MTPX_F32 ? by_vec<float>(a, back, s)
                             : dtype == MTPX_BF16 ? by_vec<__bf16>(a, back, s) : by_vec<_Float16>(a, back, s);
}

}  // namespace

// Workgroups of the backward pass: as many as the chip holds at once (three
// waves per SIMD by their registers, four of the largest workgroup), so that a weight gradient takes the
// fewest partial rows; rows of one wave and less share a workgroup.
int norm_backward_parts(int64_t rows, int width)
{
    const int n = row_threads(width);
    const int block = n <= kWave ? 256 : n, together = block / n;
    const int64_t need = (rows + together - 1) / together, most = 256 * std::max(12 * kWave / block, 1);
    return (int)(need < most ? need : most);
}
hipError_t launch_norm_forward(int dtype, const NormArgs &a, hipStream_t s)
{
    return a.rows == 0 ? hipSuccess : by_type(dtype, a, false, s);
}
// Without rows the parts kernel still writes the (zero) weight gradients.
hipError_t launch_norm_backward(int dtype, const NormArgs &a, hipStream_t s)
{
    if (a.rows > 0)
        return by_type(dtype, a, true, s);
    const dim3 grid((a.width + kWave - 1) / kWave, 3), block(kMaxBlock);
    return launch_kernel(dtype == MTPX_F32    ? norm_parts_kernel<float>
                         : dtype == MTPX_BF16 ? norm_parts_kernel<__bf16>
                                              : norm_parts_kernel<_Float16>,
                         grid, block, 0, s, a);
}

}  // namespace mtpx
