// Checks that the C entry points of the operators on device tensors share
// (include/mtpx.h).
#pragma once

#include "context.hpp"

#include <cmath>
#include <string>

namespace mtpx {

// a launch's threads are counted in 32 bits: workgroups of 512, rows of 64 in
// workgroups of 256, the last one whole
constexpr int64_t kMaxGroups = UINT32_MAX / 512, kMaxRows = (UINT32_MAX - 255) / 64;

inline int invalid(mtpx_context *ctx, const std::string &msg) { return set_error(ctx, MTPX_E_INVALID, msg); }

inline size_t dtype_bytes(int dtype) { return dtype == MTPX_F32 ? 4 : 2; }
inline bool is_dtype(int d) { return d == MTPX_F32 || d == MTPX_BF16 || d == MTPX_F16; }
inline bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A tensor of rows: present, element-aligned, strides that count forward.
inline int check_rows(mtpx_context *ctx, const mtpx_rows &r, int dtype, const char *name)
{
    if (!r.data)
        return invalid(ctx, std::string("null ") + name);
    if (!aligned(r.data, dtype_bytes(dtype)))
        return invalid(ctx, std::string(name) + " is not aligned to its elements");
    if (r.row < 0 || r.head < 0 || r.map < 0)
        return invalid(ctx, std::string(name) + " has a negative stride");
    return MTPX_OK;
}
inline int check_flat(mtpx_context *ctx, const void *p, size_t align, const char *name)
{
    if (!p)
        return invalid(ctx, std::string("null ") + name);
    if (!aligned(p, align))
        return invalid(ctx, std::string(name) + " is not aligned to its elements");
    return MTPX_OK;
}

// The context's device while a call queues its work, then the caller's again:
// these calls run inside programs that keep a current device of their own.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device)
    {
        int d = -1;
        if (hipGetDevice(&d) == hipSuccess && d == device)
            return;
        before = d;
        (void)hipSetDevice(device);
    }
    ~OnDevice()
    {
        if (before >= 0)
            (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

inline bool whole_pieces(const mtpx_rows &r, size_t size)
{
    return aligned(r.data, 16) && r.row * size % 16 == 0 && r.head * size % 16 == 0 &&
           r.map * size % 16 == 0;
}

#define MTPX_TRY(expr)                                                                     \
    do {                                                                                   \
        if (int rc_ = (expr))                                                              \
            return rc_;                                                                    \
    } while (0)

inline int check_heads(mtpx_context *ctx, int dtype, int heads, int kv_heads, int dim, float scale)
{
    if (!is_dtype(dtype))
        return invalid(ctx, "dtype must be MTPX_F32, MTPX_BF16 or MTPX_F16");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0)
        return invalid(ctx, "heads must be a positive multiple of kv_heads");
    if (dim < 1)
        return invalid(ctx, "dim must be positive");
    if (dim > 128)
        return set_error(ctx, MTPX_E_CAPACITY, "dim beyond 128");
    if (!(scale > 0.f) || !std::isfinite(scale))
        return invalid(ctx, "scale must be positive and finite");
    return MTPX_OK;
}

inline int check_workspace(mtpx_context *ctx, const void *p, size_t have, size_t need)
{
    if (need == 0)
        return MTPX_OK;
    if (have < need || !p)
        return invalid(ctx, "the workspace holds " + std::to_string(p ? have : 0) + " bytes, " +
                                std::to_string(need) + " are needed");
    if (!aligned(p, 16))
        return invalid(ctx, "the workspace is not aligned to 16 bytes");
    return MTPX_OK;
}

}  // namespace mtpx
