// Launch arguments of the operators on device tensors (include/mtpx.h),
// shared by the host file (ops_api.cpp) and the kernels.
#pragma once

#include "mtpx.h"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mtpx {

// A run of rows of one sequence of a ragged batch that one workgroup takes:
// queries or keys start .. start + tile rows - 1, with the sequence's place.
struct SeqTile {
    int64_t q0, k0;
    int nq, nk, start;
};

// Row counts of the tile tables a sequence handle keeps.
constexpr int kTileRows[2] = {64, 128};

struct TileTable {
    const SeqTile *q[2], *k[2];  // by kTileRows
    int nq[2], nk[2];
    int longest_q, longest_k;  // most rows and keys of a sequence
};

struct AttnArgs {
    TileTable tiles;
    int heads, kv_heads, dim, causal;
    int64_t total_q, total_k;
    float scale;
    mtpx_rows q, k, v, out, dout, dq, dk, dv;
    const unsigned char *mask;
    const float *lambda;
    void *out1;
    float *lse, *delta, *dlam_part, *dlambda;
    int vec;  // every row is a whole number of 16-byte pieces at a 16-byte address
    // the key pass's walk over the rows in so many parts, each with its sums in
    // kv_part [part][kv head][key][dv, dk: 4 dim] (one part: none)
    int kv_parts;
    float *kv_part;
};

constexpr int kMaxSplits = 128;  // of one sequence's cache

struct CacheArgs {
    int sequences, heads, kv_heads, dim, splits;
    int64_t capacity, k_sequence, v_sequence;
    float scale;
    mtpx_rows q, k, v, out;
    const int *lengths;
    const float *lambda;
    float *part;
    int vec;
};

struct RotaryArgs {
    int64_t rows;
    int heads, dim, rotated, interleaved, inverse, axes, position_dtype;
    mtpx_rows x, y, forward;
    const void *positions;
    int64_t position_row, position_axis;
    const float *freq;
    const int *axis;
    void *dpositions;
    int width;  // elements of one access
    int lanes;  // of a row: a power of two up to 64
};

struct NormArgs {
    int64_t rows;
    int width, kind, act;
    float residual_scale, block_scale, eps;
    const void *x, *y, *gate, *post, *pre;
    int64_t x_row, y_row, gate_row;
    void *s, *n;
    int64_t s_row, n_row;
    float *stats;
    const void *ds, *dn;
    int64_t ds_row, dn_row;
    void *dx, *dy, *dgate, *dpost, *dpre;
    int64_t dx_row, dy_row, dgate_row;
    float *part;  // [3][parts][width]: post, pre, shared gate
    int parts;
    int vec;
};

// Norms and rotation of heads: [0] is q, [1] is k; a vector is a head's map.
struct HeadArgs {
    int64_t rows;
    int vectors[2], maps;
    int dim, rotated, interleaved, kind, axes, position_dtype;
    float eps;
    mtpx_rows in[2], out[2];  // backward: out is the gradient of in
    const void *weight[2];
    const void *positions;
    int64_t position_row, position_axis;
    const float *freq;
    const int *axis;
    // append
    mtpx_rows v;
    mtpx_pages cache;
    const int *offsets, *lengths;
    int sequences;
    // backward
    mtpx_rows grad[2];
    void *dweight[2], *dpositions;
    float *part;  // [2][parts][dim]
    int parts;
    int width;  // elements of one access
    int group;  // lanes of a vector: a power of two up to 64
    int lanes;  // of a row: a power of two from group up to 256 (backward: not 128)
};

// n / d for n below 2^31: the upper half of 2 n magic, shifted.
struct Divisor {
    unsigned magic;
    int shift;
};

// A search by `lanes` places at a time (a power of two) for the first place below
// n at which something no longer holds that holds at all places before.  Every
// round leaves fewer places, by one lane too, which bisects them: of 4,096 places
// 64 lanes find one in two rounds, one lane in at most 13.
struct Search {
    int from = 0, to;  // it holds below `from`, and no longer from `to` on
    int lanes, shift, step = 0;

    __host__ __device__ inline Search(int n, int by) : to(n), lanes(by), shift(by > 1 ? 31 - __builtin_clz(by) : 1) {}
    // Whether places are left; where lane l looks: at no place if that is not below `to`.
    __host__ __device__ inline bool next()
    {
        step = (int)(((int64_t)to - from + (1 << shift) - 1) >> shift);
        return from < to;
    }
    __host__ __device__ inline int64_t place(int l) const { return from + (int64_t)(l + 1) * step - 1; }
    // The first `count` of the lanes' places hold.
    __host__ __device__ inline void narrow(int count)
    {
        const int64_t end = place(count);
        if (count < lanes && end < to)
            to = (int)end;
        from += count * step;
    }
};

// What the first t tiles of a sequence's columns cost, in steps of `step` keys:
// `start` and no less than its steps each.  Where the new rows are a small part,
// every tile as much as the last.  Else tile t sees `before` + (t + 1) columns /
// heads keys, rounded up; the sum's rounding may leave a step off and the keys'
// two more, so four are added.
__host__ __device__ inline int tile_costs(bool causal, int length, int rows, int shift, int heads, int columns, int step, int start, int t)
{
    if (!causal || rows <= length / 8)  // (without a division: one row of 997 takes 10.1 us, 10.8 us with it)
        return t * (start + (length + step - 1) / step);
    const int before = (shift < 0 ? 0 : shift < length ? shift : length) / step + 4;
    return t * (start + before) + (int)((int64_t)t * (t + 1) / 2 * columns / (heads * step));
}

// How the tiles of one width are given to workgroups.
struct RoleArgs {
    int groups;     // workgroups (0: none)
    int each_unit;  // one takes one tile; else they share all keys evenly, their
    float *part;    // partial results here: [groups][2][columns][2][4 + 2 D] (NULL: one group)
    // wide: the most tiles of a key head, as many of every sequence (`level`) or
    // by number; and of four times the columns (0: every tile in its turn)
    int tiles, level, quarters;
    int split;  // steps that writing and joining a partial result are worth
};

struct PagedArgs {
    int64_t rows;
    int sequences, heads, kv_heads, dim, causal;
    float scale;
    mtpx_rows q, out;
    mtpx_pages cache;
    const int *offsets, *lengths;
    const float *lambda;
    int vec;
    int alike;  // and keys and values have the same strides, within 32 bits a row
    int heads_each;       // of a group
    Divisor page, group;  // by page_rows and heads_each
    // sequences of up to so many columns (a row's head of the group that shares
    // a key head) have a narrow tile, the others wide ones
    int narrow_columns;
    RoleArgs narrow, wide;
};

// dtype is one of MTPX_F32, MTPX_BF16, MTPX_F16 (checked by the caller).
hipError_t launch_attn_forward(int dtype, const AttnArgs &a, hipStream_t s);
hipError_t launch_attn_backward(int dtype, const AttnArgs &a, hipStream_t s);
// Query tiles of the backward pass, each of which leaves one partial of dlambda per head.
int attn_backward_tiles(int dtype, int dim, int heads, const TileTable &t);
hipError_t launch_attn_cache(int dtype, const CacheArgs &a, hipStream_t s);
hipError_t launch_rotary(int dtype, const RotaryArgs &a, hipStream_t s);
hipError_t launch_norm_forward(int dtype, const NormArgs &a, hipStream_t s);
hipError_t launch_norm_backward(int dtype, const NormArgs &a, hipStream_t s);
int norm_backward_parts(int64_t rows, int width);
hipError_t launch_head_forward(int dtype, const HeadArgs &a, hipStream_t s);
hipError_t launch_head_append(int dtype, const HeadArgs &a, hipStream_t s);
hipError_t launch_head_backward(int dtype, const HeadArgs &a, hipStream_t s);
hipError_t launch_paged(int dtype, const PagedArgs &a, hipStream_t s);

}  // namespace mtpx
