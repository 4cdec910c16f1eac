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

#include <tuple>
#include <utility>

namespace mtpx {

// Launches a kernel and returns the launch's own error: the runtime's last
// error may be an earlier call's, and is its caller's to read.
template <class... P, size_t... I>
hipError_t launch_with(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t s, std::tuple<P...> values,
                       std::index_sequence<I...>)
{
    void *each[] = {&std::get<I>(values)...};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, each, lds, s);
}
template <class... P, class... A>
hipError_t launch_kernel(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t s, const A &...args)
{
    return launch_with(kernel, grid, block, lds, s, std::tuple<P...>(args...), std::index_sequence_for<P...>());
}

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

// Results below one another as operand B, rounded to T once.
template <class T>
using Half = T __attribute__((ext_vector_type(4)));
template <class T>
__device__ inline Half<T> round4(f32x4 a)
{
    return __builtin_convertvector(a, Half<T>);
}
template <class T>
__device__ inline Frag<T> join(Half<T> a, Half<T> b)
{
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <class T>
__device__ inline Frag<T> pack(f32x4 a, f32x4 b)
{
    return join<T>(round4<T>(a), round4<T>(b));
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
};

// A lane's byte offsets of its fragments in a tile.  The permutation touches
// only the low three bits of a piece's number, so the places of all pieces
// follow from a few, to which whole constants are added.
template <class T, int D>
struct Reader {
    using TL = Tile<T, D>;
    static constexpr int E = TL::E, RB = TL::kRowBytes;
    static constexpr bool kHalf = sizeof(T) == 2;
    int row[2];   // row_frag: the pieces whose bit 2 is clear, set (32 bits: first, second)
    int col[kHalf ? 4 : 8];

    __device__ inline void init(int lane)
    {
        const int g = lane >> 4, i = lane & 15;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            row[h] = TL::at(i, kHalf ? 4 * h + g : 2 * g + h);
        if constexpr (kHalf) {
#pragma unroll
            for (int h = 0; h < 4; ++h)
                col[h] = TL::at(4 * g + (i >> 2), 2 * h + ((i & 3) >> 1)) + ((i & 1) << 3);
        } else {
#pragma unroll
            for (int h = 0; h < 8; ++h)
                col[h] = TL::at(4 * g + (h & 3), (h & 4) + (i >> 2)) + (i & 3) * 4;
        }
    }
    // Operand A: row r0 + l % 16, columns c0 + 8 (l / 16) + j; r0 a multiple
    // of 8, c0 a constant multiple of 32.
    __device__ inline Frag<T> row_frag(const char *tile, int r0, int c0) const
    {
        union {
            u32x4 v[8 / E];
            Frag<T> f;
        } u;
        if constexpr (kHalf) {
            const int piece = c0 / E;
            u.v[0] = *reinterpret_cast<const u32x4 *>(tile + row[piece >> 2 & 1] +
                                                      (r0 * RB + (piece & ~7) * 16));
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                u.v[h] = *reinterpret_cast<const u32x4 *>(tile + row[h] + (r0 * RB + c0 / E * 16));
        }
        return u.f;
    }
    // Operand A of the transposed tile: column c0 + l % 16 (c0 a constant
    // multiple of 16), contraction over rows r0 + 16 t + 4 (l / 16) + r at
    // j = 4 t + r.
    __device__ inline Frag<T> column_frag(const char *tile, int r0, int c0) const
    {
        const int piece = c0 / E;
        if constexpr (kHalf) {
            // ds_read_b64_tr_b16: of 16 lanes that read 4 rows of 16 elements
            // (lane i: row i / 4, elements 4 (i % 4) ...), lane i gets column i
            union {
                s16x4 h[2];
                Frag<T> f;
            } u;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                u.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *)(tile + col[piece >> 1 & 3] +
                                                                ((r0 + 16 * t) * RB + (piece & ~7) * 16)));
            return u.f;
        } else {
            Frag<T> f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                f[j] = *reinterpret_cast<const T *>(tile + col[(piece & 4) + (j & 3)] +
                                                    ((r0 + 16 * (j >> 2)) * RB + (piece & ~7) * 16));
            return f;
        }
    }
};

// The way of a tile from global memory through registers into LDS, by one
// wave: lane l moves piece l % kPieces of rows l / kPieces, + 64 / kPieces, ...
template <class T, int D, int ROWS, int NT>
struct Stage {
    using TL = Tile<T, D>;
    static constexpr int kStep = NT / TL::kPieces;
    static constexpr int N = ROWS / kStep;
    static_assert(ROWS % kStep == 0, "rows of a tile");
    u32x4 r[N ? N : 1];

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

// 16 bytes of zeros that a load takes in the place of a row that is not there.
__device__ const u32x4 kZeroPiece = {0, 0, 0, 0};

// 16 bytes per lane from global memory straight into LDS, at byte `offset`
// (the same in every lane) + 16 lane of the workgroup's LDS.  They are there
// after wait_loads().
// (As assembly text, since the compiler would wait for such loads before any
// read of the LDS that it cannot tell from their target.  It has no output
// register, and what it writes is waited for in wait_loads().  A write of m0
// takes one wait state to reach it.)
__device__ inline void load_to_lds(const void *p, unsigned offset)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(offset) : "memory");
}
// (After the reads of what lay there: wait_reads() or a barrier.)
__device__ inline void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// Waits for them and all other loads.  (The instruction itself, not assembly
// text: the compiler then knows that its own loads have come too and does not
// wait for those again, and so for the loads into LDS, where they are used.)
__device__ inline void wait_loads()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    asm volatile("" ::: "memory");
}

// A tile's way from global memory straight into LDS, by a workgroup of W
// waves, without passing through registers.  A wave's instruction fills 1 KiB
// of the tile: kGroup rows; lane l fills the piece that lies at place
// l % kPieces of its row and so reads the one that the permutation puts there.
// The lane's address moves from tile to tile by whole strides.
template <class T, int D, int ROWS, int W>
struct Loader {
    using TL = Tile<T, D>;
    static constexpr int kGroup = 1024 / TL::kRowBytes;
    static constexpr int N = ROWS / (kGroup * W);
    static_assert(N * kGroup * W == ROWS, "rows of a tile");
    // the permutation is the same in all of a lane's rows, or changes
    static constexpr bool kSame = W * kGroup % 8 == 0;
    const T *at;  // the lane's row of the next tile
    int64_t row, map;
    int dim, vec, lane, wave;

    __device__ inline int column(int i) const
    {
        const int r = (kSame ? 0 : i * W * kGroup) + wave * kGroup + lane / TL::kPieces;
        return ((lane % TL::kPieces) ^ (r & 7)) * TL::E;
    }
    // From row 0 of the sequence (`base`, of the head) on.
    __device__ inline void init(const T *base, const mtpx_rows &s, int d, int v, int tid)
    {
        row = s.row;
        map = s.map;
        dim = d;
        vec = v;
        lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        at = base + (wave * kGroup + lane / TL::kPieces) * row;
        if constexpr (kSame)
            at += column(0) / D * map + column(0) % D;
    }
    __device__ inline void move(int64_t elements) { at += elements; }
    __device__ inline void next() { at += ROWS * row; }
    // The tile at `at` to byte `tile` of the workgroup's LDS (`smem` its
    // start); a row whose bit in `live` is not set (`all`: every bit is), and
    // columns beyond dim of either map, become 0.
    __device__ inline void load(char *smem, int tile, unsigned long long live, bool all) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int to = tile + (i * W + wave) * 1024;
            const T *p = at + i * (W * kGroup * row);
            if constexpr (!kSame)
                p += column(i) / D * map + column(i) % D;
            if (vec && all && dim == D) {
                load_to_lds(p, to);
                continue;
            }
            const int c = column(i) % D;
            const bool on = (live >> ((i * W + wave) * kGroup + lane / TL::kPieces) & 1) && c < dim;
            if (vec)
                load_to_lds(on ? (const void *)p : (const void *)&kZeroPiece, to);
            else
                *reinterpret_cast<u32x4 *>(smem + to + lane * 16) = load16(p, on ? dim - c : 0, 0);
        }
    }
};

// The tile and head of workgroup b.  Consecutive workgroups go to the 8 XCDs
// in turn, each with an L2 of its own: a head's tiles stay on one XCD where
// the heads go round evenly (then head by head), and on as few as there are
// heads to go round otherwise.  Tiles come with the most work first.
struct Work {
    int tile, head;
};
__device__ inline Work work_item(int b, int ntiles, int heads)
{
    if (heads % 8 != 0)
        return {b / heads, b % heads};
    const int y = b / 8;
    return {y % ntiles, y / ntiles * 8 + b % 8};
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The largest of three, without the quieting of NaNs that fmaxf comes with.
__device__ inline float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// The largest absolute value of three.
__device__ inline float max3_abs(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// The exponent e of 2^(e-1) <= v < 2^e; 0 of 0, infinities and NaN.
__device__ inline int exponent(float v) { return __builtin_amdgcn_frexp_expf(v); }

// Sum over 16 lanes or a wave, in a fixed order, in every lane: rotations or
// shifts within rows of 16 lanes, then from row to row, by data-parallel moves
// that need no LDS.
template <int CONTROL, int ROWS>
__device__ inline float moved(float v)
{
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CONTROL, ROWS, 0xf, false));
}
__device__ inline float row16_sum(float v)
{
    v += moved<0x128, 0xf>(v);  // row_ror:8
    v += moved<0x124, 0xf>(v);
    v += moved<0x122, 0xf>(v);
    return v + moved<0x121, 0xf>(v);
}
__device__ inline float wave_sum(float v)
{
    v += moved<0x111, 0xf>(v);  // row_shr:1
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);  // row_bcast:15
    v += moved<0x143, 0xc>(v);  // row_bcast:31
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Maximum over a wave of values that are not negative, in every lane.
__device__ inline float wave_max(float v)
{
    v = fmaxf(v, moved<0x111, 0xf>(v));
    v = fmaxf(v, moved<0x112, 0xf>(v));
    v = fmaxf(v, moved<0x114, 0xf>(v));
    v = fmaxf(v, moved<0x118, 0xf>(v));
    v = fmaxf(v, moved<0x142, 0xa>(v));
    v = fmaxf(v, moved<0x143, 0xc>(v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

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
