// Device helpers of the operators on device tensors: element types, matrix
// fragments, tiles in LDS.
//
// Fragments.  A fragment holds 8 contraction elements of one row (operand A)
// or column (operand B) per lane: lane l has row or column l % 16 and the
// elements 8 (l / 16) + j, j < 8, of a block of 32.  mma() multiplies a
// 16x32 by a 32x16 block: one v_mfma_f32_16x16x32 in 16-bit types, eight
// v_mfma_f32_16x16x4 in 32 bits, the j-th over element j of every lane.  The
// result's lane l holds rows 4 (l / 16) + r, r < 4, of column l % 16.
//
// The order of the 32 contraction elements is free as long as both operands
// agree.  Two results that lie below one another (32 rows) hold, in lane l,
// rows 16 t + 4 (l / 16) + r, t < 2: read as a fragment with j = 4 t + r they
// are operand B of a product that contracts over those rows, without moving
// between lanes.  column_frag() reads operand A in that same order.
#pragma once

#include "mtpx_internal.hpp"
#include "ops_internal.hpp"

namespace mtpx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <class T>
struct Elem;
template <>
struct Elem<float> {
    typedef f32x8 frag;
};
template <>
struct Elem<__bf16> {
    typedef bf16x8 frag;
};
template <>
struct Elem<_Float16> {
    typedef f16x8 frag;
};
template <class T>
using Frag = typename Elem<T>::frag;

__device__ inline f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mma(f16x8 a, f16x8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mma(f32x8 a, f32x8 b, f32x4 c)
{
#pragma unroll
    for (int j = 0; j < 8; ++j)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// Two results below one another as operand B, rounded to T once.
template <class T>
__device__ inline Frag<T> pack(f32x4 a, f32x4 b)
{
    const f32x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_convertvector(v, Frag<T>);
}

// 16 bytes (E elements) of a row, of which `valid` exist; the others are 0.
template <class T>
__device__ inline u32x4 load16(const T *p, int valid, int vec)
{
    constexpr int E = 16 / sizeof(T);
    u32x4 v = {0, 0, 0, 0};
    if (valid <= 0)
        return v;
    if (vec)
        return *reinterpret_cast<const u32x4 *>(p);
    union {
        u32x4 v;
        T e[E];
    } u;
    u.v = v;
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (j < valid)
            u.e[j] = p[j];
    return u.v;
}

// 8 elements of a row from column c on, columns beyond dim 0.
template <class T>
__device__ inline Frag<T> load_frag(const T *row, int c, int dim, bool live, int vec)
{
    constexpr int E = 16 / sizeof(T), N = 8 / E;
    union {
        u32x4 v[N];
        Frag<T> f;
    } u;
#pragma unroll
    for (int i = 0; i < N; ++i)
        u.v[i] = load16(row + c + i * E, live ? dim - c - i * E : 0, vec);
    return u.f;
}

// Stores 4 consecutive results at column c of a row, columns beyond dim left out.
template <class T>
__device__ inline void store4(T *row, int c, int dim, f32x4 v, int vec)
{
    typedef T t4 __attribute__((ext_vector_type(4)));
    if (c >= dim)
        return;
    if (vec) {
        *reinterpret_cast<t4 *>(row + c) = __builtin_convertvector(v, t4);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < dim)
            row[c + j] = (T)v[j];
}

// A tile of rows in LDS: [rows][2 D] elements, each row's 16-byte pieces
// permuted by piece ^ (row % 8), so that 8 rows' pieces of one column fall
// into different banks, in row reads as in transposed ones.
template <class T, int D>
struct Tile {
    static constexpr int E = 16 / sizeof(T);
    static constexpr int kPieces = 2 * D / E;
    static constexpr int kRowBytes = 32 * D / E;  // 2 D sizeof(T)

    static __device__ inline int at(int row, int piece)
    {
        return row * kRowBytes + ((piece ^ (row & 7)) << 4);
    }
    // Operand A: row r0 + l % 16, columns c0 + 8 (l / 16) + j.
    static __device__ inline Frag<T> row_frag(const char *tile, int r0, int c0, int lane)
    {
        constexpr int N = 8 / E;
        const int row = r0 + (lane & 15), piece = c0 / E + (lane >> 4) * N;
        union {
            u32x4 v[N];
            Frag<T> f;
        } u;
#pragma unroll
        for (int i = 0; i < N; ++i)
            u.v[i] = *reinterpret_cast<const u32x4 *>(tile + at(row, piece + i));
        return u.f;
    }
    // Operand A of the transposed tile: column c0 + l % 16, contraction over
    // rows r0 + 16 t + 4 (l / 16) + r at j = 4 t + r.
    static __device__ inline Frag<T> column_frag(const char *tile, int r0, int c0, int lane)
    {
        const int g = lane >> 4, i = lane & 15;
        if constexpr (sizeof(T) == 2) {
            // ds_read_b64_tr_b16: of 16 lanes that read 4 rows of 16 elements
            // (lane i: row i / 4, elements 4 (i % 4) ...), lane i gets column i
            union {
                s16x4 h[2];
                Frag<T> f;
            } u;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int row = r0 + 16 * t + 4 * g + (i >> 2);
                const char *p = tile + at(row, c0 / E + ((i & 3) >> 1)) + ((i & 1) << 3);
                u.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *)p);
            }
            return u.f;
        } else {
            Frag<T> f;
            const int c = c0 + i;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = r0 + 16 * (j >> 2) + 4 * g + (j & 3);
                f[j] = *reinterpret_cast<const T *>(tile + at(row, c / E) + (c % E) * sizeof(T));
            }
            return f;
        }
    }
};

// The way of a tile from global memory through registers into LDS, by a
// workgroup of NT threads: thread t moves piece t % kPieces of rows
// t / kPieces, + NT / kPieces, ...
template <class T, int D, int ROWS, int NT>
struct Stage {
    using TL = Tile<T, D>;
    static constexpr int kStep = NT / TL::kPieces;
    static constexpr int N = ROWS / kStep;
    static_assert(ROWS % kStep == 0, "rows of a tile");
    u32x4 r[N];

    // Rows first, first + 1, ... of head-shifted `base`; a row whose bit in
    // `live` is not set, and columns beyond dim of either map, are 0.
    __device__ inline void load(const T *base, const mtpx_rows &s, int dim, int64_t first,
                                unsigned long long live, int tid, int vec)
    {
        const int piece = tid % TL::kPieces, row = tid / TL::kPieces;
        const int col = piece * TL::E, map = col / D, c = col % D;
        const T *p = base + (first + row) * s.row + map * s.map + c;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool on = live >> (row + i * kStep) & 1;
            r[i] = load16(p + (int64_t)(i * kStep) * s.row, on ? dim - c : 0, vec);
        }
    }
    __device__ inline void store(char *tile, int tid) const
    {
        const int piece = tid % TL::kPieces, row = tid / TL::kPieces;
#pragma unroll
        for (int i = 0; i < N; ++i)
            *reinterpret_cast<u32x4 *>(tile + TL::at(row + i * kStep, piece)) = r[i];
    }
};

// Consecutive workgroups go to the 8 XCDs in turn; this order gives each XCD
// a contiguous run of work items, so that neighbours share its L2.
__device__ inline int xcd_order(int b, int n)
{
    const int per = n / 8, rest = n % 8, x = b % 8;
    return x * per + (x < rest ? x : rest) + b / 8;
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Maximum and sum over the four lanes that hold one column of a result.
__device__ inline float column_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float column_sum(float v)
{
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

}  // namespace mtpx
