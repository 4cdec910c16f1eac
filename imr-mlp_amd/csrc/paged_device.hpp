// Where the rows of a batch stand in a paged cache (mtpx_pages), for the
// kernels that write and read it.
#pragma once

#include "ops_device.hpp"

namespace mtpx {

// The largest i < n for which pred(i) holds, -1 if none: pred holds up to some
// i and not beyond.  `lanes` neighbouring lanes (a power of two up to a wave)
// search together, as many places at a time.
template <class P>
__device__ inline int last_true(const P &pred, int n, int lanes)
{
    const int l = threadIdx.x & (lanes - 1), base = (threadIdx.x & (kWave - 1)) & ~(lanes - 1);
    const unsigned long long all = ~0ull >> (kWave - lanes);
    Search s(n, lanes);
    while (s.next()) {
        const int64_t at = s.place(l);
        const unsigned long long holds = __ballot(at < s.to && pred((int)at)) >> base & all;
        s.narrow(holds == all ? lanes : __ffsll(~holds) - 1);
    }
    return s.from - 1;
}

// The first row of sequence i (of sequence n: the end of the last one).
__device__ inline int row_offset(const int *offsets, int i, int64_t rows)
{
    const int o = offsets[i];
    return o < 0 ? 0 : o > rows ? (int)rows : o;
}

}  // namespace mtpx
