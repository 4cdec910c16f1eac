// The C entry points of the operators on device tensors with the HIP runtime's
// calls and the kernel launches replaced by records of them.
//
//   ops_calls device   every entry point, for a context on device 0 called with
//                      device 1 current: prints its name, its code, the device
//                      its work was queued on (-1: none) and the one current
//                      afterwards
//   ops_calls sequences n rows megabytes
//                      a handle of n sequences of so many rows, with so much
//                      address space left to the process: prints its code
#include "../imr-mlp_amd/csrc/ops_api.cpp"

#include <cstdio>
#include <cstdlib>
#include <cstring>

#include <sys/resource.h>
#include <unistd.h>

static int current = 1, queued = -1;

extern "C" {
hipError_t hipSetDevice(int d)
{
    current = d;
    return hipSuccess;
}
hipError_t hipGetDevice(int *d)
{
    *d = current;
    return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t bytes)
{
    queued = current;
    *p = std::malloc(bytes);
    return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void *p)
{
    queued = current;
    std::free(p);
    return hipSuccess;
}
hipError_t hipMemcpyAsync(void *to, const void *from, size_t bytes, hipMemcpyKind, hipStream_t)
{
    std::memcpy(to, from, bytes);
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
}

namespace mtpx {
static hipError_t launched()
{
    queued = current;
    return hipSuccess;
}
hipError_t launch_attn_forward(int, const AttnArgs &, hipStream_t) { return launched(); }
hipError_t launch_attn_backward(int, const AttnArgs &, hipStream_t) { return launched(); }
int attn_backward_tiles(int, int, int, const TileTable &) { return 1; }
hipError_t launch_attn_cache(int, const CacheArgs &, hipStream_t) { return launched(); }
hipError_t launch_rotary(int, const RotaryArgs &, hipStream_t) { return launched(); }
hipError_t launch_norm_forward(int, const NormArgs &, hipStream_t) { return launched(); }
hipError_t launch_norm_backward(int, const NormArgs &, hipStream_t) { return launched(); }
int norm_backward_parts(int64_t, int) { return 1; }
}  // namespace mtpx

static void report(const char *name, int code)
{
    std::printf("%s %d %d %d\n", name, code, queued, current);
    current = 1;
    queued = -1;
}

static int devices()
{
    mtpx_context ctx;
    alignas(16) static float room[1 << 12];
    static int numbers[16] = {0};
    const mtpx_rows rows{room, 64, 16, 8};
    const int64_t offsets[] = {0, 4};
    mtpx_sequences *seqs = nullptr;
    report("sequences_create", mtpx_sequences_create(&ctx, 1, offsets, nullptr, &seqs));
    if (!seqs)
        return 1;

    mtpx_rotary_request r{};
    r.rows = 4, r.heads = 1, r.dim = 4, r.rotated = 2, r.axes = 1;
    r.x = rows, r.y = mtpx_rows{room + 1024, 64, 16, 8}, r.positions = room, r.freq = room, r.axis = numbers;
    report("rotary", mtpx_rotary(&ctx, &r));

    mtpx_diff_attention_request a{};
    a.sequences = seqs, a.heads = a.kv_heads = 1, a.dim = 8, a.scale = 1.f;
    for (mtpx_rows *t : {&a.q, &a.k, &a.v, &a.out, &a.dout, &a.dq, &a.dk, &a.dv})
        *t = rows;
    a.lambda = a.dlambda = a.lse = room, a.out1 = room, a.workspace = room, a.workspace_bytes = sizeof room;
    report("diff_attention", mtpx_diff_attention(&ctx, &a));
    report("diff_attention_backward", mtpx_diff_attention_backward(&ctx, &a));

    mtpx_diff_attention_cache_request c{};
    c.sequences = c.heads = c.kv_heads = 1, c.dim = 8, c.scale = 1.f;
    c.q = c.out = rows, c.lengths = numbers, c.lambda = room;
    report("diff_attention_cache", mtpx_diff_attention_cache(&ctx, &c));

    mtpx_norm_block_request n{};
    n.rows = 4, n.width = 8, n.y = room, n.s = room, n.stats = room, n.workspace = room, n.workspace_bytes = sizeof room;
    report("norm_block", mtpx_norm_block(&ctx, &n));
    report("norm_block_backward", mtpx_norm_block_backward(&ctx, &n));
    mtpx_sequences_destroy(seqs);
    report("sequences_destroy", 0);
    return 0;
}

static int sequences(int n, int64_t rows, size_t megabytes)
{
    mtpx_context ctx;
    std::vector<int64_t> offsets(n + 1);
    for (int i = 0; i <= n; ++i)
        offsets[i] = i * rows;
    long long pages = 0;
    if (std::FILE *f = std::fopen("/proc/self/statm", "r")) {
        if (std::fscanf(f, "%lld", &pages) != 1)
            return 1;
        std::fclose(f);
    }
    const rlim_t limit = (rlim_t)pages * sysconf(_SC_PAGESIZE) + ((rlim_t)megabytes << 20);
    const rlimit space{limit, limit};
    if (setrlimit(RLIMIT_AS, &space))
        return 1;
    mtpx_sequences *seqs = nullptr;
    std::printf("%d\n", mtpx_sequences_create(&ctx, n, offsets.data(), nullptr, &seqs));
    return 0;
}

int main(int argc, char **argv)
{
    if (argc > 4 && !std::strcmp(argv[1], "sequences"))
        return sequences(std::atoi(argv[2]), std::atoll(argv[3]), std::atoi(argv[4]));
    if (argc > 1 && !std::strcmp(argv[1], "device"))
        return devices();
    return 2;
}
