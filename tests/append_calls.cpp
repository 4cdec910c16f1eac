// The plan of an append and the search of its rows for their sequences, without a GPU.
//
//   append_calls search         every number of lanes, many lengths and ends: how many
//                               were searched, and how many ended at another place or
//                               took more rounds than they may
//   append_calls lanes DTYPE DIM ROTATED INTERLEAVED HEADS
//                               lanes of a vector and of a row for rows from 1 up to
//                               the most, one line each
//   append_calls backward ROWS HEADS MAPS DIM ROTATED INTERLEAVED DTYPE
//                               lanes of a row and workgroups of the backward pass of
//                               head norms on a device of 256 compute units
//   append_calls weights        the code of an append with a weight for each norm, and
//                               whether its work was queued
#include "../imr-mlp_amd/csrc/paged_api.cpp"

#include <cstdio>
#include <cstdlib>
#include <cstring>

static mtpx::HeadArgs seen;
static bool queued = false;

extern "C" {
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevice(int *d)
{
    *d = 0;
    return hipSuccess;
}
hipError_t hipMalloc(void **, size_t) { return hipErrorOutOfMemory; }
hipError_t hipFree(void *) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
}

namespace mtpx {
hipError_t launch_head_forward(int, const HeadArgs &, hipStream_t) { return hipSuccess; }
hipError_t launch_head_append(int, const HeadArgs &a, hipStream_t)
{
    seen = a;
    queued = true;
    return hipSuccess;
}
hipError_t launch_head_backward(int, const HeadArgs &a, hipStream_t)
{
    seen = a;
    return hipSuccess;
}
hipError_t launch_paged(int, const PagedArgs &, hipStream_t) { return hipSuccess; }
}  // namespace mtpx

// What last_true does, the lanes one after the other; -2 after too many rounds.
static int searched(int n, int lanes, int holds, int most)
{
    mtpx::Search s(n, lanes);
    for (int rounds = 0; s.next(); ++rounds) {
        if (rounds == most)
            return -2;
        int count = 0;
        while (count < lanes && s.place(count) < s.to && s.place(count) < holds)
            ++count;
        s.narrow(count);
    }
    return s.from - 1;
}

static int search()
{
    long looked = 0, wrong = 0;
    for (int lanes = 1; lanes <= 64; lanes *= 2) {
        auto look = [&](int n, int holds) {
            // a round leaves a part of the places, rounded up
            int most = 1;
            for (int64_t left = n; left > 1; left = (left + std::max(lanes, 2) - 1) / std::max(lanes, 2))
                ++most;
            ++looked;
            wrong += searched(n, lanes, holds, most) != holds - 1;
        };
        for (int n = 0; n <= 300; ++n)
            for (int holds = 0; holds <= n; ++holds)
                look(n, holds);
        for (int n : {1023, 1024, 1025, 4095, 4096, 4097, 4160, 4161, 5001})
            for (int holds = 0; holds <= n; ++holds)
                look(n, holds);
        for (int n : {1 << 20, (1 << 24) + 1, INT32_MAX - 1, INT32_MAX})
            for (int holds : {0, 1, 2, n / 3, n / 2, n - 2, n - 1, n})
                look(n, holds);
    }
    std::printf("%ld %ld\n", looked, wrong);
    return 0;
}

alignas(16) static float room[4096];
static int numbers[16] = {0};
static mtpx_context ctx;

static mtpx_append_paged_request append(int dtype, int dim, int rotated, int kv_heads)
{
    mtpx_append_paged_request r{};
    r.dtype = dtype, r.dim = dim, r.rotated = rotated, r.kv_heads = kv_heads;
    r.rows = r.sequences = 1, r.axes = 1, r.kind = MTPX_NORM_NONE;
    const int64_t map = r.dim, head = 2 * map, row = head * r.kv_heads;
    r.k = r.v = mtpx_rows{room, row, head, map};
    r.positions = room, r.freq = room, r.axis = numbers, r.offsets = r.lengths = numbers;
    r.cache.k = r.cache.v = r.k;
    r.cache.k_page = r.cache.v_page = row * 16;
    r.cache.pages = 4, r.cache.page_rows = 16, r.cache.table = numbers, r.cache.table_row = 2, r.cache.table_width = 2;
    return r;
}

static int lanes(char **v)
{
    auto r = append(std::atoi(v[0]), std::atoi(v[1]), std::atoi(v[2]), std::atoi(v[4]));
    r.interleaved = std::atoi(v[3]);
    for (int bit = 1; bit <= 26; ++bit)
        for (int64_t rows : {(int64_t(1) << bit) - 4, (int64_t(1) << bit) - 1, int64_t(1) << bit, (int64_t(1) << bit) + 1}) {
            if (rows < 1)
                continue;
            r.rows = rows;
            if (const int code = mtpx_append_paged(&ctx, &r)) {
                std::printf("%lld refused %d\n", (long long)rows, code);
                continue;
            }
            std::printf("%lld %d %d\n", (long long)rows, seen.group, seen.lanes);
        }
    return 0;
}

static int backward(char **v)
{
    mtpx_head_norm_rotary_request r{};
    r.rows = std::atoll(v[0]), r.heads = std::atoi(v[1]), r.maps = std::atoi(v[2]), r.dim = std::atoi(v[3]);
    r.rotated = std::atoi(v[4]), r.interleaved = std::atoi(v[5]), r.dtype = std::atoi(v[6]);
    r.axes = 1, r.positions = r.freq = room, r.axis = numbers;
    const int64_t map = r.dim, head = r.maps * map;
    r.q = r.dq_out = r.dq = mtpx_rows{room, head * r.heads, head, map};
    r.workspace = room, r.workspace_bytes = size_t(1) << 40;
    ctx.num_cus = 256;
    if (const int code = mtpx_head_norm_rotary_backward(&ctx, &r))
        return code;
    std::printf("%d %d\n", seen.lanes, seen.parts);
    return 0;
}

static int weights()
{
    for (int kind : {MTPX_NORM_RMS, MTPX_NORM_LAYER, MTPX_NORM_NONE})
        for (int given = 0; given < 4; ++given) {
            auto r = append(MTPX_F32, 8, 8, 1);
            r.kind = kind, r.heads = 1, r.q = r.k, r.q_out = r.k;
            r.q_weight = given & 1 ? room : nullptr, r.k_weight = given & 2 ? room : nullptr;
            queued = false;
            const int code = mtpx_append_paged(&ctx, &r);
            std::printf("%d %d %d %d\n", kind, given, code, queued);
        }
    return 0;
}

int main(int argc, char **argv)
{
    if (argc > 1 && !std::strcmp(argv[1], "search"))
        return search();
    if (argc > 6 && !std::strcmp(argv[1], "lanes"))
        return lanes(argv + 2);
    if (argc > 8 && !std::strcmp(argv[1], "backward"))
        return backward(argv + 2);
    if (argc > 1 && !std::strcmp(argv[1], "weights"))
        return weights();
    return 2;
}
