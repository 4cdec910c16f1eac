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
    static constexpr int kBlock = NT < 256 ? 256 : NT;
    static constexpr int kPerBlock = kBlock / NT;  // rows of a workgroup
    static constexpr int kPieces = E / V;
    static __device__ inline int column(int i, int t) { return (i * NT + t) * V; }

    // Columns beyond width are `beyond`.
    static __device__ inline void load(const T *p, int width, int t, float beyond, float (&v)[E])
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int c = column(i, t);
            if constexpr (V == 1) {
                v[i] = c < width ? (float)p[c] : beyond;
            } else {
                union {
                    u32x4 v;
                    T e[V];
                } u;
                if (c < width)
                    u.v = *reinterpret_cast<const u32x4 *>(p + c);
#pragma unroll
                for (int j = 0; j < V; ++j)
                    v[i * V + j] = c < width ? (float)u.e[j] : beyond;
            }
        }
    }
    static __device__ inline void store(T *p, int width, int t, const float (&v)[E])
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int c = column(i, t);
            if (c >= width)
                continue;
            if constexpr (V == 1) {
                p[c] = (T)v[i];
            } else {
                union {
                    u32x4 v;
                    T e[V];
                } u;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    u.e[j] = (T)v[i * V + j];
                *reinterpret_cast<u32x4 *>(p + c) = u.v;
            }
        }
    }
    static __device__ inline bool inside(int e, int t, int width)
    {
        return column(e / V, t) + e % V < width;
    }
    // Sum over the row's threads, in a fixed order.
    static __device__ inline float sum(float v, float *red)
    {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            v += __shfl_xor(v, o);
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

__device__ inline float act(int kind, float g)
{
    if (kind == MTPX_GATE_SIGMOID)
        return 1.f / (1.f + __expf(-g));
    if (kind == MTPX_GATE_TANH)
        return tanhf(g);
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

template <class T, int NT, int E, int V>
__global__ __launch_bounds__((Row<T, NT, E, V>::kBlock)) void norm_forward_kernel(NormArgs a)
{
    using R = Row<T, NT, E, V>;
    __shared__ float red[kMaxBlock / kWave];
    const int t = threadIdx.x % NT;
    const int64_t row = (int64_t)blockIdx.x * R::kPerBlock + threadIdx.x / NT;
    if (row >= a.rows)  // whole waves: a row's threads leave together
        return;
    float v[E], w[E], x[E];
    R::load((const T *)a.y + row * a.y_row, a.width, t, 0.f, v);
    if (a.x)
        R::load((const T *)a.x + row * a.x_row, a.width, t, 0.f, x);
    if (a.gate)
        R::load((const T *)a.gate + row * a.gate_row, a.width, t, 0.f, w);
    float mean, inv;
    normalise<R>(v, a.kind, a.width, a.eps, t, red, mean, inv);
    if (a.stats && t == 0) {
        a.stats[4 * row] = mean;
        a.stats[4 * row + 1] = inv;
    }
    const float b = a.block_scale * inv;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] *= a.gate ? b * act(a.act, w[e]) : b;
    }
    if (a.post) {
        R::load((const T *)a.post, a.width, t, 0.f, w);
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] *= w[e];
    }
    if (a.x) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] = fmaf(a.residual_scale, x[e], v[e]);
    }
    R::store((T *)a.s + row * a.s_row, a.width, t, v);
    if (!a.n)
        return;
    normalise<R>(v, a.kind, a.width, a.eps, t, red, mean, inv);
    if (a.stats && t == 0) {
        a.stats[4 * row + 2] = mean;
        a.stats[4 * row + 3] = inv;
    }
    if (a.pre)
        R::load((const T *)a.pre, a.width, t, 0.f, w);
#pragma unroll
    for (int e = 0; e < E; ++e)
        v[e] *= a.pre ? inv * w[e] : inv;
    R::store((T *)a.n + row * a.n_row, a.width, t, v);
}

// With v = (s - mean) r:  ds = ds_in + r (dv - [mean dv] - v mean(dv v)),
// dv = dn w2; the same again through the first norm.  s is formed again from
// x, y and the gate (the bytes of reading it back, without its rounding).
// A group of NT threads takes rows part, part + parts, ... and keeps its
// share of the weights' gradients in registers.
template <class T, int NT, int E, int V>
__global__ __launch_bounds__((Row<T, NT, E, V>::kBlock)) void norm_backward_kernel(NormArgs a)
{
    using R = Row<T, NT, E, V>;
    __shared__ float red[kMaxBlock / kWave];
    const int t = threadIdx.x % NT;
    const int part = blockIdx.x * R::kPerBlock + threadIdx.x / NT;
    if (part >= a.parts)
        return;
    const bool layer = a.kind == MTPX_NORM_LAYER;
    const float scale = 1.f / a.width;
    float dw1[E], dw2[E], dgs[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        dw1[e] = dw2[e] = dgs[e] = 0.f;
    for (int64_t row = part; row < a.rows; row += a.parts) {
        const f32x4 st = *reinterpret_cast<const f32x4 *>(a.stats + 4 * row);
        float u[E], v[E], g[E], w[E], ds[E];
        R::load((const T *)a.y + row * a.y_row, a.width, t, 0.f, u);
        if (a.x)
            R::load((const T *)a.x + row * a.x_row, a.width, t, 0.f, v);
        if (a.gate)
            R::load((const T *)a.gate + row * a.gate_row, a.width, t, 0.f, g);
        if (a.dn)
            R::load((const T *)a.dn + row * a.dn_row, a.width, t, 0.f, ds);
        if (a.post)
            R::load((const T *)a.post, a.width, t, 0.f, w);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            u[e] = R::inside(e, t, a.width) ? (u[e] - st[0]) * st[1] : 0.f;
            g[e] = a.gate ? act(a.act, g[e]) : 1.f;
            if (!a.post)
                w[e] = 1.f;
            const float z = a.block_scale * g[e] * u[e] * w[e];
            v[e] = a.x ? fmaf(a.residual_scale, v[e], z) : z;
        }
        if (a.dn) {
            float w2[E], s0 = 0.f, s1 = 0.f;
            if (a.pre)
                R::load((const T *)a.pre, a.width, t, 0.f, w2);
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
            R::load((const T *)a.ds + row * a.ds_row, a.width, t, 0.f, v);
#pragma unroll
            for (int e = 0; e < E; ++e)
                ds[e] += v[e];
        }
        if (a.dx) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[e] = a.residual_scale * ds[e];
            R::store((T *)a.dx + row * a.dx_row, a.width, t, v);
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
            R::store((T *)a.dgate + row * a.dgate_row, a.width, t, v);
        if (a.dy) {
            s0 = layer ? R::sum(s0, red) * scale : 0.f;
            s1 = R::sum(s1, red) * scale;
#pragma unroll
            for (int e = 0; e < E; ++e)
                ds[e] = st[1] * (ds[e] - s0 - u[e] * s1);
            R::store((T *)a.dy + row * a.dy_row, a.width, t, ds);
        }
    }
    auto leave = [&](int which, const float (&d)[E]) {
        float *p = a.part + ((int64_t)which * a.parts + part) * a.width;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (R::inside(e, t, a.width))
                p[R::column(e / V, t) + e % V] = d[e];
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
    if (c < a.width)
        for (int p = run; p < a.parts; p += kRuns)
            v += a.part[((int64_t)which * a.parts + p) * a.width + c];
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
    const int64_t groups = back ? a.parts : a.rows;
    const dim3 grid((unsigned)((groups + R::kPerBlock - 1) / R::kPerBlock)), block(R::kBlock);
    if (back)
        norm_backward_kernel<T, NT, E, V><<<grid, block, 0, s>>>(a);
    else
        norm_forward_kernel<T, NT, E, V><<<grid, block, 0, s>>>(a);
    return hipGetLastError();
}

// The fewest threads that hold a row with 8 or 16 elements each.
template <class T, int V>
hipError_t by_width(const NormArgs &a, bool back, hipStream_t s)
{
    if (a.width <= 512)
        return run<T, 64, 8, V>(a, back, s);
    if (a.width <= 1024)
        return run<T, 64, 16, V>(a, back, s);
    if (a.width <= 4096)
        return run<T, 256, 16, V>(a, back, s);
    return run<T, 1024, 16, V>(a, back, s);
}

template <class T>
hipError_t by_vec(const NormArgs &a, bool back, hipStream_t s)
{
    const hipError_t e = a.vec ? by_width<T, 16 / sizeof(T)>(a, back, s) : by_width<T, 1>(a, back, s);
    if (e != hipSuccess || !back || !(a.dpost || a.dpre || (a.dgate && a.gate_row == 0)))
        return e;
    norm_parts_kernel<T><<<dim3((a.width + kWave - 1) / kWave, 3), dim3(kMaxBlock), 0, s>>>(a);
    return hipGetLastError();
}

hipError_t by_type(int dtype, const NormArgs &a, bool back, hipStream_t s)
{
    return dtype == MTPX_F32 ? by_vec<float>(a, back, s)
                             : dtype == MTPX_BF16 ? by_vec<__bf16>(a, back, s) : by_vec<_Float16>(a, back, s);
}

}  // namespace

// Rows are spread over as many groups as fill the chip a few times over;
// each leaves one partial row per weight gradient.
int norm_backward_parts(int64_t rows, int width)
{
    const int most = width <= 1024 ? 4096 : width <= 4096 ? 1024 : 512;
    return (int)(rows < most ? rows : most);
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
    if (dtype == MTPX_F32)
        norm_parts_kernel<float><<<grid, block, 0, s>>>(a);
    else if (dtype == MTPX_BF16)
        norm_parts_kernel<__bf16><<<grid, block, 0, s>>>(a);
    else
        norm_parts_kernel<_Float16><<<grid, block, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace mtpx
