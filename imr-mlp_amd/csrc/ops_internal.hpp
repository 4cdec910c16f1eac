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

}  // namespace mtpx
