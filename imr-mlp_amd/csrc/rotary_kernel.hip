// Rotary positions with several axes (mtpx_rotary): every pair of a head
// turns by the position of its row on the pair's axis, and in the backward
// pass the gradient of the positions is summed over the row's heads.
#include "ops_device.hpp"

namespace mtpx {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kMaxPairs = 512, kMaxAxes = 8;

__device__ inline double position(const RotaryArgs &a, int64_t row, int axis)
{
    const int64_t i = row * a.position_row + axis * a.position_axis;
    switch (a.position_dtype) {
    case MTPX_F32: return ((const float *)a.positions)[i];
    case MTPX_F64: return ((const double *)a.positions)[i];
    case MTPX_I32: return ((const int *)a.positions)[i];
    default: return (double)((const int64_t *)a.positions)[i];
    }
}

// N elements that lie at a multiple of A elements.
template <class T, int N, int A = N>
struct alignas(sizeof(T) * A) Piece {
    T e[N];
};

// A group of `lanes` lanes (a wave, or a part of one where a row has little
// work) per row.  They first put cos and sin of the row's pairs into LDS (each
// once, for all heads: the angle is reduced to a fraction of a turn in 64
// bits), then walk the heads: lane l keeps unit l % units of every head, W
// elements of one or both halves of the pairs, and takes heads l / units,
// + lanes / units, ...  So a lane reads its cos and sin once, and in the
// backward pass sums the pairs' gradients over heads in registers.  The work
// is bound by the reads and writes of x and y (160,000 rows of 32 heads, 64
// wide, 16 bits: 233 us, 5.6 TB/s).
template <class T, int W, bool PAIRS_APART, bool GRAD>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a)
{
    __shared__ float2 tables[kWaves][kMaxPairs];
    const int wave = threadIdx.x >> 6, in_wave = threadIdx.x & 63;
    const int lanes = a.lanes, lane = in_wave % lanes, pairs = a.rotated / 2;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
    const bool there = row < a.rows;
    float2 *table = tables[wave] + in_wave / lanes * pairs;
    for (int p = lane; there && p < pairs; p += lanes) {
        int axis = a.axis[p];
        axis = axis >= 0 && axis < a.axes ? axis : 0;
        const double turns = position(a, row, axis) * (double)a.freq[p] * 0.15915494309189533577;
        const float f = (float)(2.0 * (turns - rint(turns)));
        float s, c;
        sincospif(f, &s, &c);
        table[p] = make_float2(c, a.inverse ? -s : s);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (!there)
        return;

    // units of a head: W pairs (both halves) or W elements of pairs side by
    // side, then W elements beyond the rotated ones
    // (a pair side by side in rows without any alignment: its two elements)
    constexpr int P = PAIRS_APART ? W : W > 1 ? W / 2 : 1;  // pairs of a unit
    constexpr int N = PAIRS_APART ? W : 2 * P;              // elements read at once
    const int turning = pairs / P, units = turning + (a.dim - a.rotated) / W;
    const int step = units < lanes ? lanes / units : 1;
    const T *x = (const T *)a.x.data + row * a.x.row;
    T *y = (T *)a.y.data + row * a.y.row;
    const T *fw = GRAD ? (const T *)a.forward.data + row * a.forward.row : nullptr;
    float sum[kMaxAxes] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};

    for (int u0 = 0; u0 < units; u0 += lanes) {
        const int here = min(units - u0, lanes);
        const int u = u0 + lane % here, h0 = lane / here;
        if (h0 >= step)
            continue;
        if (u >= turning) {
            const int64_t e = a.rotated + (int64_t)(u - turning) * W;
            for (int h = h0; h < a.heads; h += step)
                *(Piece<T, W> *)(y + h * a.y.head + e) = *(const Piece<T, W> *)(x + h * a.x.head + e);
            continue;
        }
        float c[P], s[P], d[P];
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const float2 cs = table[u * P + j];
            c[j] = cs.x;
            s[j] = cs.y;
            d[j] = 0.f;
        }
        for (int h = h0; h < a.heads; h += step) {
            const T *px = x + h * a.x.head + u * N;
            T *py = y + h * a.y.head + u * N;
            if constexpr (PAIRS_APART) {
                const Piece<T, W> x1 = *(const Piece<T, W> *)px, x2 = *(const Piece<T, W> *)(px + pairs);
                Piece<T, W> y1, y2, f1, f2;
                if constexpr (GRAD) {
                    f1 = *(const Piece<T, W> *)(fw + h * a.forward.head + u * W);
                    f2 = *(const Piece<T, W> *)(fw + h * a.forward.head + u * W + pairs);
                }
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float v1 = (float)x1.e[j] * c[j] - (float)x2.e[j] * s[j];
                    const float v2 = (float)x1.e[j] * s[j] + (float)x2.e[j] * c[j];
                    y1.e[j] = (T)v1;
                    y2.e[j] = (T)v2;
                    if constexpr (GRAD)
                        d[j] += v2 * (float)f1.e[j] - v1 * (float)f2.e[j];
                }
                *(Piece<T, W> *)py = y1;
                *(Piece<T, W> *)(py + pairs) = y2;
            } else {
                const Piece<T, N, W> xx = *(const Piece<T, N, W> *)px;
                Piece<T, N, W> yy, ff;
                if constexpr (GRAD)
                    ff = *(const Piece<T, N, W> *)(fw + h * a.forward.head + u * N);
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const float v1 = (float)xx.e[2 * j] * c[j] - (float)xx.e[2 * j + 1] * s[j];
                    const float v2 = (float)xx.e[2 * j] * s[j] + (float)xx.e[2 * j + 1] * c[j];
                    yy.e[2 * j] = (T)v1;
                    yy.e[2 * j + 1] = (T)v2;
                    if constexpr (GRAD)
                        d[j] += v2 * (float)ff.e[2 * j] - v1 * (float)ff.e[2 * j + 1];
                }
                *(Piece<T, N, W> *)py = yy;
            }
        }
        if constexpr (GRAD) {
#pragma unroll
            for (int j = 0; j < P; ++j) {
                int axis = a.axis[u * P + j];
                axis = axis >= 0 && axis < a.axes ? axis : 0;
                const float v = d[j] * a.freq[u * P + j];
#pragma unroll
                for (int k = 0; k < kMaxAxes; ++k)
                    sum[k] += axis == k ? v : 0.f;
            }
        }
    }
    if constexpr (GRAD) {
#pragma unroll
        for (int k = 0; k < kMaxAxes; ++k) {
            if (k >= a.axes)
                break;
            float v = sum[k];
            for (int o = lanes / 2; o > 0; o >>= 1)
                v += __shfl_xor(v, o);
            if (lane == 0) {
                const int64_t at = row * a.axes + k;
                if (a.position_dtype == MTPX_F64)
                    ((double *)a.dpositions)[at] = v;
                else
                    ((float *)a.dpositions)[at] = v;
            }
        }
    }
}

template <class T, int W>
hipError_t launch(const RotaryArgs &a, hipStream_t s)
{
    const int rows = kThreads / a.lanes;
    const dim3 grid((unsigned)((a.rows + rows - 1) / rows)), block(kThreads);
    const auto kernel = a.interleaved ? (a.dpositions ? rotary_kernel<T, W, false, true> : rotary_kernel<T, W, false, false>)
                                      : (a.dpositions ? rotary_kernel<T, W, true, true> : rotary_kernel<T, W, true, false>);
    return launch_kernel(kernel, grid, block, 0, s, a);
}

template <class T>
hipError_t by_width(const RotaryArgs &a, hipStream_t s)
{
    switch (a.width) {
    case 8:
        if constexpr (sizeof(T) == 2)
            return launch<T, 8>(a, s);
        return hipErrorInvalidValue;
    case 4: return launch<T, 4>(a, s);
    case 2: return launch<T, 2>(a, s);
    default: return launch<T, 1>(a, s);
    }
}

}  // namespace

hipError_t launch_rotary(int dtype, const RotaryArgs &a, hipStream_t s)
{
    if (a.rows == 0)
        return hipSuccess;
    return dtype == MTPX_F32 ? by_width<float>(a, s)
                             : dtype == MTPX_BF16 ? by_width<__bf16>(a, s) : by_width<_Float16>(a, s);
}

}  // namespace mtpx
