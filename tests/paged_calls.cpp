// The C entry points of the paged cache and of the norms of heads with the HIP
// runtime's calls and the kernel launches replaced by records of them.
//
//   paged_calls device   every entry point, for a context on device 0 called with
//                        device 1 current: prints its name, its code, the device
//                        its work was queued on (-1: none) and the one current
//                        afterwards
//   paged_calls refuse   one line per refused request: its name, its code, and
//                        whether anything was queued
//   paged_calls pages    page_rows, magic and shift of every page size up to 4100
//   paged_calls costs n  n sequences and tiles at random: how many tiles were looked
//                        at, and how many cost less than they take
//   paged_calls plan rows sequences max_rows heads kv_heads dim dtype page width
//                        how a call's work is split, and its workspace
#include "../imr-mlp_amd/csrc/paged_api.cpp"

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>

static int current = 1, queued = -1;
static mtpx::PagedArgs seen;

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
hipError_t hipMalloc(void **, size_t) { return hipErrorOutOfMemory; }
hipError_t hipFree(void *) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
}

namespace mtpx {
static hipError_t launched()
{
    queued = current;
    return hipSuccess;
}
hipError_t launch_head_forward(int, const HeadArgs &, hipStream_t) { return launched(); }
hipError_t launch_head_append(int, const HeadArgs &, hipStream_t) { return launched(); }
hipError_t launch_head_backward(int, const HeadArgs &, hipStream_t) { return launched(); }
hipError_t launch_paged(int, const PagedArgs &a, hipStream_t)
{
    seen = a;
    return launched();
}
}  // namespace mtpx

alignas(16) static float room[1 << 16];
static int numbers[16] = {0};
static const mtpx_rows rows{room, 64, 16, 8};

static mtpx_pages pages()
{
    mtpx_pages p{};
    p.k = p.v = rows;
    p.k_page = p.v_page = 1024;
    p.pages = 4;
    p.page_rows = 16;
    p.table = numbers;
    p.table_row = 2;
    p.table_width = 2;
    return p;
}
static mtpx_head_norm_rotary_request heads()
{
    mtpx_head_norm_rotary_request r{};
    r.rows = 4, r.heads = 2, r.kv_heads = 1, r.maps = 2, r.dim = 8, r.rotated = 8, r.axes = 1, r.eps = 1e-6f;
    r.q = r.k = r.dq_out = r.dk_out = rows;
    r.q_out = r.k_out = r.dq = r.dk = mtpx_rows{room + 4096, 64, 16, 8};
    r.q_weight = r.k_weight = r.dq_weight = r.dk_weight = r.dpositions = room;
    r.positions = room, r.freq = room, r.axis = numbers;
    r.workspace = room, r.workspace_bytes = sizeof room;
    return r;
}
static mtpx_append_paged_request append()
{
    mtpx_append_paged_request r{};
    r.rows = 4, r.sequences = 2, r.heads = 2, r.kv_heads = 1, r.dim = 8, r.rotated = 8, r.axes = 1;
    r.kind = MTPX_NORM_NONE;
    r.q = r.k = r.v = rows, r.q_out = mtpx_rows{room + 4096, 64, 16, 8};
    r.positions = room, r.freq = room, r.axis = numbers;
    r.cache = pages(), r.offsets = r.lengths = numbers;
    return r;
}
static mtpx_diff_attention_paged_request attend()
{
    mtpx_diff_attention_paged_request r{};
    r.rows = 4, r.sequences = 2, r.heads = 2, r.kv_heads = 1, r.dim = 8, r.scale = 1.f;
    r.q = r.out = rows, r.cache = pages(), r.offsets = r.lengths = numbers, r.lambda = room;
    r.workspace = room, r.workspace_bytes = sizeof room;
    return r;
}

static mtpx_context ctx;

static int devices()
{
    auto report = [](const char *name, int code) {
        std::printf("%s %d %d %d\n", name, code, queued, current);
        current = 1;
        queued = -1;
    };
    const auto h = heads();
    report("head_norm_rotary", mtpx_head_norm_rotary(&ctx, &h));
    report("head_norm_rotary_backward", mtpx_head_norm_rotary_backward(&ctx, &h));
    const auto a = append();
    report("append_paged", mtpx_append_paged(&ctx, &a));
    const auto d = attend();
    report("diff_attention_paged", mtpx_diff_attention_paged(&ctx, &d));
    return 0;
}

static void line(const char *name, int code)
{
    std::printf("%s %d %d\n", name, code, queued);
    queued = -1;
}
static void head(const char *name, const std::function<void(mtpx_head_norm_rotary_request &)> &change, bool back = false)
{
    auto r = heads();
    change(r);
    line(name, back ? mtpx_head_norm_rotary_backward(&ctx, &r) : mtpx_head_norm_rotary(&ctx, &r));
}
static void app(const char *name, const std::function<void(mtpx_append_paged_request &)> &change)
{
    auto r = append();
    change(r);
    line(name, mtpx_append_paged(&ctx, &r));
}
static void att(const char *name, const std::function<void(mtpx_diff_attention_paged_request &)> &change)
{
    auto r = attend();
    change(r);
    line(name, mtpx_diff_attention_paged(&ctx, &r));
}

static int refusals()
{
    using H = mtpx_head_norm_rotary_request &;
    void *odd = reinterpret_cast<char *>(room) + 2;
    head("head_dtype", [](H r) { r.dtype = MTPX_F64; });
    head("head_rows", [](H r) { r.rows = -1; });
    head("head_many_rows", [](H r) { r.rows = int64_t(1) << 27; });
    head("head_dim", [](H r) { r.dim = 0, r.rotated = 0; });
    head("head_wide", [](H r) { r.dim = 257; });
    head("head_rotated", [](H r) { r.rotated = 10; });
    head("head_odd_rotated", [](H r) { r.rotated = 3; });
    head("head_maps", [](H r) { r.maps = 3; });
    head("head_none", [](H r) { r.kind = MTPX_NORM_NONE; });
    head("head_eps", [](H r) { r.eps = -1.f; });
    head("head_axes", [](H r) { r.axes = 9; });
    head("head_positions", [](H r) { r.position_dtype = MTPX_F16; });
    head("head_null_q", [](H r) { r.q.data = nullptr; });
    head("head_null_out", [](H r) { r.k_out.data = nullptr; });
    head("head_stride", [](H r) { r.k.head = -1; });
    head("head_alignment", [=](H r) { r.q.data = odd; });
    head("head_weight_alignment", [=](H r) { r.k_weight = odd; });
    head("head_in_place", [](H r) { r.q_out = r.q, r.q_out.row = 65; });
    head("back_workspace", [](H r) { r.workspace_bytes = 64; }, true);
    head("back_null_workspace", [](H r) { r.workspace = nullptr; }, true);
    head("back_weight", [](H r) { r.q_weight = nullptr; }, true);
    head("back_integer", [](H r) { r.position_dtype = MTPX_I32; }, true);
    head("back_null_dq", [](H r) { r.dq.data = nullptr; }, true);
    head("back_null_gradient", [](H r) { r.dk_out.data = nullptr; }, true);
    using A = mtpx_append_paged_request &;
    app("append_kv", [](A r) { r.kv_heads = 0; });
    app("append_kind", [](A r) { r.kind = 3; });
    app("append_sequences", [](A r) { r.sequences = -1; });
    app("append_many_sequences", [](A r) { r.sequences = (1 << 24) + 1; });
    app("append_offsets", [](A r) { r.offsets = nullptr; });
    app("append_lengths", [=](A r) { r.lengths = static_cast<int *>(odd); });
    app("append_table", [](A r) { r.cache.table = nullptr; });
    app("append_page_rows", [](A r) { r.cache.page_rows = 0; });
    app("append_room", [](A r) { r.cache.page_rows = 1 << 20, r.cache.table_width = 1025; });
    app("append_pages", [](A r) { r.cache.pages = int64_t(1) << 31; });
    app("append_page_stride", [](A r) { r.cache.v_page = -1; });
    app("append_null_pages", [](A r) { r.cache.k.data = nullptr; });
    app("append_null_v", [](A r) { r.v.data = nullptr; });
    app("append_null_q_out", [](A r) { r.q_out.data = nullptr; });
    app("append_in_place", [](A r) { r.q_out = r.q, r.q_out.map = 9; });
    using D = mtpx_diff_attention_paged_request &;
    att("attend_heads", [](D r) { r.heads = 3, r.kv_heads = 2; });
    att("attend_dim", [](D r) { r.dim = 129; });
    att("attend_scale", [](D r) { r.scale = 0.f; });
    att("attend_max_rows", [](D r) { r.max_rows = -1; });
    att("attend_rows", [](D r) { r.rows = int64_t(1) << 26; });
    att("attend_launch", [](D r) { r.rows = 1 << 20, r.heads = 16, r.kv_heads = 16; });
    att("attend_page_rows", [](D r) { r.cache.page_rows = -1; });
    att("attend_room", [](D r) { r.cache.page_rows = 1 << 20, r.cache.table_width = 1025; });
    att("attend_null_q", [](D r) { r.q.data = nullptr; });
    att("attend_null_out", [](D r) { r.out.data = nullptr; });
    att("attend_lambda", [](D r) { r.lambda = nullptr; });
    att("attend_offsets", [](D r) { r.offsets = nullptr; });
    att("attend_workspace", [](D r) { r.cache.table_width = 1000, r.workspace_bytes = 1024; });
    return 0;
}

static int page_sizes()
{
    for (int n = 1; n <= 4100; ++n) {
        auto r = attend();
        r.cache.page_rows = n, r.cache.table_width = 0;
        if (mtpx_diff_attention_paged(&ctx, &r))
            return 1;
        std::printf("%d %u %d\n", n, seen.page.magic, seen.page.shift);
    }
    return 0;
}

static int costs(int n)
{
    unsigned long long state = 88172645463325252ull;
    auto random = [&](int most) {  // 1 to most, spread over its logarithm
        state ^= state << 13, state ^= state >> 7, state ^= state << 17;
        int bits = 1;
        while (bits < 30 && (1 << bits) < most)
            ++bits;
        const int top = 1 << (state >> 40) % (bits + 1), v = 1 + (int)((state >> 8) % (unsigned)top);
        return v < most ? v : most;
    };
    long looked = 0, wrong = 0;
    const int shapes[][2] = {{32, 64}, {32, 32}, {128, 64}, {64, 32}, {64, 64}};
    for (int i = 0; i < n; ++i) {
        const int *s = shapes[i % 5], heads = random(80), rows = random(100000 / heads + 1), given = random(200000) - 1;
        const int room = i % 3 ? given : random(200000), length = given < room ? given : room, shift = given - rows, start = 128 / s[1];
        const int columns = rows * heads, tiles = (columns + s[0] - 1) / s[0], first = random(tiles) - 1;
        for (int t = first; t < tiles && t < first + 50; ++t) {
            const int last = ((t + 1) * s[0] < columns ? (t + 1) * s[0] : columns) - 1;
            int keys = shift + last / heads + 1;
            keys = keys < 0 ? 0 : keys < length ? keys : length;
            for (bool causal : {false, true}) {
                const int steps = ((causal ? keys : length) + s[1] - 1) / s[1];
                auto cost = [&](int at) { return mtpx::tile_costs(causal, length, rows, shift, heads, s[0], s[1], start, at); };
                wrong += cost(t + 1) - cost(t) < start + steps;
                ++looked;
            }
        }
    }
    std::printf("%ld %ld\n", looked, wrong);
    return 0;
}

static int plan(char **v)
{
    mtpx_diff_attention_paged_request r{};
    r.rows = std::atoll(v[0]), r.sequences = std::atoi(v[1]), r.max_rows = std::atoi(v[2]), r.heads = std::atoi(v[3]);
    r.kv_heads = std::atoi(v[4]), r.dim = std::atoi(v[5]), r.dtype = std::atoi(v[6]);
    r.cache.page_rows = std::atoi(v[7]), r.cache.table_width = std::atoi(v[8]), r.scale = 1.f;
    const mtpx::PagedPlan p = mtpx::paged_plan(&ctx, r);
    size_t bytes = 0;
    const int code = mtpx_diff_attention_paged_workspace(&ctx, &r, &bytes);
    std::printf("%d %d %d %d %d %d %d %d %d %zu\n", code, p.narrow_columns, p.narrow.groups, p.narrow.each_unit, p.wide.groups,
                p.wide.each_unit, p.wide.tiles, p.wide.level, p.wide.quarters, bytes);
    return 0;
}

int main(int argc, char **argv)
{
    if (argc > 1 && !std::strcmp(argv[1], "device"))
        return devices();
    if (argc > 1 && !std::strcmp(argv[1], "refuse"))
        return refusals();
    if (argc > 1 && !std::strcmp(argv[1], "pages"))
        return page_sizes();
    if (argc > 2 && !std::strcmp(argv[1], "costs"))
        return costs(std::atoi(argv[2]));
    if (argc > 10 && !std::strcmp(argv[1], "plan"))
        return plan(argv + 2);
    return 2;
}
