// Differential attention (mtpx_diff_attention, _backward, _cache): two
// softmax maps over the same values,
//
//   out = (P_0 - lambda P_1) V,   P_m = softmax(scale Q_m K_m^T).
//
//   attn_forward_kernel   out, and lse and P_1 V for the backward pass
//   attn_dq_kernel        dq, and per row D_m = sum_j P_m dP (for the next)
//   attn_dkv_kernel       dk, dv; the group of query heads that share them
//                         is summed in registers; dlambda from its shares
//   attn_dkv_join         sums its parts where few keys leave the device idle
//   dlambda_kernel        dlambda where there are no keys
//   attn_cache_kernel     one row per sequence, keys split over workgroups
//   attn_cache_join       joins their partial results
//
// Compiled once per element type (MTPX_OPS_TYPE).
#include "ops_device.hpp"

namespace mtpx {

namespace {

#if MTPX_OPS_TYPE == 0
typedef float Type;
#define MTPX_OPS_NAME(f) f##_f32
#elif MTPX_OPS_TYPE == 1
typedef __bf16 Type;
#define MTPX_OPS_NAME(f) f##_bf16
#else
typedef _Float16 Type;
#define MTPX_OPS_NAME(f) f##_f16
#endif

constexpr int kThreads = 256, kWaves = kThreads / kWave;

// Which of the keys k0 .. k0 + 63 of a sequence of nk are there and not
// masked; the mask is read `step` keys ahead, so that no step waits for it.
struct SeenKeys {
    const unsigned char *mask;
    int nk, lane;
    unsigned char ahead = 0;

    __device__ inline SeenKeys(const unsigned char *m, int n, int l) : mask(m), nk(n), lane(l)
    {
        if (mask && lane < nk)
            ahead = mask[lane];
    }
    __device__ inline unsigned long long at(int k0, int step)
    {
        if (!mask) {
            const int there = nk - k0;
            return there >= 64 ? ~0ull : (1ull << there) - 1;
        }
        const int k = k0 + lane;
        const unsigned long long bits = __ballot(k < nk && ahead);
        if (k + step < nk)
            ahead = mask[k + step];
        return bits;
    }
};

// Whether no row up to `last` sees any of the 32 keys from k0 + 32 b on.
__device__ inline bool empty_block(unsigned long long seen, int b, int causal, int k0, int last)
{
    return (unsigned)(seen >> (32 * b)) == 0 || (causal && k0 + 32 * b > last);
}

// Rounds per-lane column results 16 t + 4 (l / 16) + r, of width 2 D, to the
// row that lane l % 16 stands for.
template <class T, int D>
__device__ inline void store_columns(T *row, int64_t map, int dim, int t, int lane, f32x4 v, int vec)
{
    const int m = t * 16 / D, c = t * 16 % D + 4 * (lane >> 4);
    store4(row + m * map, c, dim, v, vec);
}

// A row's exponentials are taken relative to a level (in powers of two) that
// is renewed, and the row's products rescaled, only when a score passes it by
// this much: exp2 then stays below 2^8, within every type's range, and most
// steps need no comparison between lanes.  kNoLevel, the level of a row that
// has seen no key, is passed by every finite score.
constexpr float kSlack = 8.f, kNoLevel = -3.0e38f;

// float16 has five bits of exponent: what is rounded to it for a product is
// scaled by powers of two first, so that gradients of the size of a mean loss
// (1e-4 and less) or of a scaled one keep their bits, and no product passes its
// largest number where inputs and results do not.  (P of the forward pass is
// relative to a row's largest as it is.)  A training step of 160,000 rows, 64
// wide, takes 2.07 ms, 1.97 ms without.
template <class T>
constexpr bool kNarrowRange = __is_same(T, _Float16);
constexpr int kMostLift = 80;  // exponent of the scale where there is nothing to scale yet

// Rows that see no more keys than this sum D from 32-bit products.
constexpr int kFewKeys = 64;

// Forward.  A workgroup takes kWaves * QT * 16 query rows of one head, each
// wave QT * 16 of them; the keys and values come in tiles of KB rows straight
// into LDS, the next tile while the present one is worked on (BUF 2).
// S^T = K Q^T leaves a query per lane column: its running maximum and sum are
// per lane, and exp(S^T) is operand B of O^T += V^T P^T as it stands.  The two
// maps keep their own maximum, sum and product, since their normalisers are
// known only at the end; each V fragment read from LDS serves both.  P is
// rounded to T for the product (its 32-bit sum is the normaliser), as V is in
// T already.  32,000 rows of 8 heads, 64 wide, in 16 bits: 5.9 ms, 1,070
// TFLOP/s of the matrix units (a loop of nothing else reaches 1,200 at two
// waves a SIMD), with the vector units issuing half of the time.
template <class T, int D, int W, int QT, int KB, int BUF, int OCC>
__global__ __launch_bounds__(W * kWave, OCC) void attn_forward_kernel(AttnArgs a, int table, int ntiles)
{
    using TL = Tile<T, D>;
    constexpr int kTile = KB * TL::kRowBytes;
    constexpr unsigned long long kFull = ~0ull >> (64 - KB);
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Work wk = work_item(blockIdx.x, ntiles, a.heads);
    const int head = wk.head, kv = head / (a.heads / a.kv_heads);
    const SeqTile sq = a.tiles.q[table][wk.tile];
    const int shift = sq.nk - sq.nq;
    const float lambda = a.lambda[head];
    const float c = a.scale * kLog2e;

    Reader<T, D> rd;
    rd.init(lane);
    const unsigned char *mask = a.mask ? a.mask + sq.k0 : nullptr;
    Loader<T, D, KB, W> lk, lv;
    lk.init((const T *)a.k.data + kv * a.k.head + sq.k0 * a.k.row, a.k, a.dim, a.vec, tid);
    lv.init((const T *)a.v.data + kv * a.v.head + sq.k0 * a.v.row, a.v, a.dim, a.vec, tid);

    const int w0 = sq.start + wave * QT * 16;  // first row of the wave
    Frag<T> qf[2][QT][D / 32];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int row = w0 + t * 16 + (lane & 15);
        const T *qp = (const T *)a.q.data + head * a.q.head + (sq.q0 + row) * a.q.row;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
                qf[m][t][kk] = load_frag(qp + m * a.q.map, kk * 32 + 8 * g, a.dim, row < sq.nq, a.vec);
    }
    f32x4 acc[2][QT][D / 8];
    float level[2][QT], sum[2][QT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            level[m][t] = kNoLevel;
            sum[m][t] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                acc[m][t][i] = f32x4{0, 0, 0, 0};
        }

    // keys that the last row of the workgroup sees
    int nk = sq.nk;
    if (a.causal)
        nk = min(nk, min(sq.start + W * QT * 16, sq.nq) + shift);
    unsigned long long bits = 0;
    SeenKeys seen(mask, nk, lane);
    if (nk > 0) {
        bits = seen.at(0, KB) & kFull;
        lk.load(smem, 0, bits, bits == kFull);
        lv.load(smem, kTile, bits, bits == kFull);
    }
    int buf = 0;
    for (int k0 = 0; k0 < nk; k0 += KB) {
        wait_loads();
        __syncthreads();
        const unsigned long long now = bits;
        const char *kt = smem + buf * 2 * kTile, *vt = kt + kTile;
        auto next = [&] {
            if (k0 + KB < nk) {
                buf = BUF - 1 - buf;
                bits = seen.at(k0 + KB, KB) & kFull;
                lk.next();
                lv.next();
                lk.load(smem, buf * 2 * kTile, bits, bits == kFull);
                lv.load(smem, buf * 2 * kTile + kTile, bits, bits == kFull);
            }
        };
        if constexpr (BUF == 2)
            next();
        const bool idle = now == 0 || w0 >= sq.nq || (a.causal && k0 > w0 + QT * 16 - 1 + shift);
        const bool partly = now != kFull || (a.causal && k0 + KB - 1 > w0 + shift);
        if (!idle) {
#pragma unroll 1
            for (int b = 0; b < KB / 32; ++b) {
                if (empty_block(now, b, a.causal, k0, w0 + QT * 16 - 1 + shift))
                    continue;
                f32x4 s[2][2][QT];
                {
                    // u, then map, then columns: one K fragment ahead
                    constexpr int kSteps = 2 * 2 * (D / 32);
                    Frag<T> kf = rd.row_frag(kt, b * 32, 0);
#pragma unroll
                    for (int x = 0; x < kSteps; ++x) {
                        const int u = x / (D / 16), m = x / (D / 32) % 2, kk = x % (D / 32);
                        Frag<T> ahead;
                        if (x + 1 < kSteps) {
                            const int y = x + 1, mc = y / (D / 32) % 2 * D + y % (D / 32) * 32;
                            ahead = rd.row_frag(kt, b * 32 + y / (D / 16) * 16, mc);
                        }
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int t = 0; t < QT; ++t)
                            s[m][u][t] = mma(kf, qf[m][t][kk], kk ? s[m][u][t] : f32x4{0, 0, 0, 0});
                        __builtin_amdgcn_sched_barrier(0);
                        kf = ahead;
                    }
                }
                if (partly) {
                    const unsigned mine = (unsigned)(now >> (32 * b + 4 * g));
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        const int last =
                            a.causal ? w0 + t * 16 + (lane & 15) + shift - k0 - 32 * b - 4 * g : 32;
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const bool on = (mine >> (16 * u + r) & 1) && 16 * u + r <= last;
                                s[0][u][t][r] = on ? s[0][u][t][r] : -INFINITY;
                                s[1][u][t][r] = on ? s[1][u][t][r] : -INFINITY;
                            }
                    }
                }
                float hi[2][QT];
                bool passed = false;
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        const f32x4 x = s[m][0][t], y = s[m][1][t];
                        hi[m][t] = max3(max3(x[0], x[1], x[2]), max3(x[3], y[0], y[1]), max3(y[2], y[3], y[3]));
                        passed |= fmaf(hi[m][t], c, -level[m][t]) > kSlack;
                    }
                if (__any(passed)) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int t = 0; t < QT; ++t) {
                            const float up = fmaxf(level[m][t], column_max(hi[m][t]) * c);
                            const float f = exp2_fast(level[m][t] - up);
                            level[m][t] = up;
                            sum[m][t] *= f;
#pragma unroll
                            for (int i = 0; i < D / 8; ++i)
                                acc[m][t][i] *= f;
                        }
                }
                Frag<T> pf[2][QT];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        float part[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float p = exp2_fast(fmaf(s[m][u][t][r], c, -level[m][t]));
                                s[m][u][t][r] = p;
                                part[u] = r ? part[u] + p : p;
                            }
                        sum[m][t] += part[0] + part[1];
                        pf[m][t] = pack<T>(s[m][0][t], s[m][1][t]);
                    }
                // one V fragment ahead of the products, so that none waits for LDS
                Frag<T> vf = rd.column_frag(vt, b * 32, 0);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    Frag<T> ahead;
                    if (i + 1 < D / 8)
                        ahead = rd.column_frag(vt, b * 32, (i + 1) * 16);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int t = 0; t < QT; ++t)
                            acc[m][t][i] = mma(vf, pf[m][t], acc[m][t][i]);
                    __builtin_amdgcn_sched_barrier(0);
                    vf = ahead;
                }
            }
        }
        if constexpr (BUF == 1) {
            __syncthreads();
            next();
        }
    }

#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int row = w0 + t * 16 + (lane & 15);
        float inv[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const float total = column_sum(sum[m][t]);
            inv[m] = total > 0.f || total != total ? 1.f / total : 0.f;
            if (a.lse && row < sq.nq && g == 0)
                a.lse[((int64_t)m * a.heads + head) * a.total_q + sq.q0 + row] =
                    total == 0.f ? -INFINITY : fmaf(level[m][t], kLn2, __logf(total));
        }
        if (row >= sq.nq)
            continue;
        T *op = (T *)a.out.data + head * a.out.head + (sq.q0 + row) * a.out.row;
        T *o1 = (T *)a.out1 + ((sq.q0 + row) * a.heads + head) * 2 * a.dim;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const f32x4 second = acc[1][t][i] * inv[1];
            store_columns<T, D>(op, a.out.map, a.dim, i, lane, acc[0][t][i] * inv[0] - lambda * second, a.vec);
            if (a.out1)
                store_columns<T, D>(o1, a.dim, a.dim, i, lane, second, a.vec);
        }
    }
}

// S^T (both maps) and dP^T = V dO^T of 32 keys: those of block b of the tiles.
template <class T, int D, int QT>
__device__ inline void score_block(const Reader<T, D> &rd, const char *kt, const char *vt, int b,
                                   const Frag<T> (&qf)[2][QT][D / 32], const Frag<T> (&df)[2][QT][D / 32],
                                   f32x4 (&s)[2][2][QT], f32x4 (&dp)[2][QT])
{
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r0 = b * 32 + u * 16;
#pragma unroll
        for (int t = 0; t < QT; ++t)
            s[0][u][t] = s[1][u][t] = dp[u][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) {
                const Frag<T> kf = rd.row_frag(kt, r0, m * D + kk * 32);
                const Frag<T> vf = rd.row_frag(vt, r0, m * D + kk * 32);
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    s[m][u][t] = mma(kf, qf[m][t][kk], s[m][u][t]);
                    dp[u][t] = mma(vf, df[m][t][kk], dp[u][t]);
                }
            }
    }
}

// Scores that a lane's row does not see become -inf.  seen: the bits of the
// lane's first key and those after it; last: the last of them that its row of
// group 0 sees.
template <int QT>
__device__ inline void hide(f32x4 (&s)[2][2][QT], unsigned seen, int last, bool causal)
{
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool on = (seen >> (16 * u + r) & 1) && (!causal || 16 * u + r <= last + 16 * t);
                s[0][u][t][r] = on ? s[0][u][t][r] : -INFINITY;
                s[1][u][t][r] = on ? s[1][u][t][r] : -INFINITY;
            }
}

// Gradient of the queries.  Work split, tiles and fragments as in the forward
// pass: S^T and dP^T = V dO^T come out with a query per lane column, so
// dS_m^T = P_m (dP - D_m) is operand B of dQ_m^T += K_m^T dS_m^T, rounded to T
// for it.  The rows' D_m = dO . O_m are formed here from out and out1 (O_0 =
// out + lambda O_1).  The roundings of 16-bit out and out1 reach q's gradient
// through them (in bfloat16 it is then off by 0.0027 of its size, where the
// roundings of dS and of the result leave 0.0023; keeping what out and out1
// leave off, a byte each, made a training step of 1,000 structures 23% longer).
// The sum of P_m (dP - D_m) over a row is what they took from D_m: with it added,
// D_m for the key pass and for dlambda = -sum D_1 comes from 32-bit values.
//
// Where rows see few keys, dS is small beside D and those roundings are as
// large as dS itself (bfloat16 rows of two to four keys: 0.0038 of q's gradient
// where one rounding of dS and of the result leave 0.0032).  A workgroup whose
// rows see few keys (kFewKeys, or the first rows of causal sequences)
// therefore walks them once more first and sums D from 32-bit products
// (18 us of a training step of 1,000 bfloat16 sequences of about 50 rows, which
// takes 677 us).  D from 32-bit out and out1 is as good as that sum.
//
// float16: dS is scaled row by row (both maps alike).  The scale, 2^lift, sits
// in the exponent of P and is lowered, and the row's products with it, when a
// scaled dS passes 2^15; it is set so that the largest then lies below 2^8.
template <class T, int D, int QT, int KB, int BUF, int OCC>
__global__ __launch_bounds__(kThreads, OCC) void attn_dq_kernel(AttnArgs a, int table, int ntiles)
{
    using TL = Tile<T, D>;
    constexpr int kTile = KB * TL::kRowBytes;
    constexpr unsigned long long kFull = ~0ull >> (64 - KB);
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Work wk = work_item(blockIdx.x, ntiles, a.heads);
    const int head = wk.head, kv = head / (a.heads / a.kv_heads);
    const SeqTile sq = a.tiles.q[table][wk.tile];
    const int shift = sq.nk - sq.nq;
    const float c = a.scale * kLog2e, lambda = a.lambda[head];

    Loader<T, D, KB, kWaves> lk, lv;
    lk.init((const T *)a.k.data + kv * a.k.head + sq.k0 * a.k.row, a.k, a.dim, a.vec, tid);
    lv.init((const T *)a.v.data + kv * a.v.head + sq.k0 * a.v.row, a.v, a.dim, a.vec, tid);
    const unsigned char *mask = a.mask ? a.mask + sq.k0 : nullptr;
    Reader<T, D> rd;
    rd.init(lane);

    // keys that the last row of the workgroup sees (a single one gives its
    // row's scores no gradient)
    constexpr int kRows = kWaves * QT * 16;
    int nk = sq.nk > 1 ? sq.nk : 0;
    if (a.causal)
        nk = min(nk, min(sq.start + kRows, sq.nq) + shift);
    const bool twice = sizeof(T) == 2 && nk > 0 && nk <= (a.causal ? max(kRows, kFewKeys) : kFewKeys);

    const int w0 = sq.start + wave * QT * 16;
    constexpr bool kScaled = kNarrowRange<T>;
    Frag<T> qf[2][QT][D / 32], df[2][QT][D / 32];
    float base[2][QT], delta[2][QT];
    int lift[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int row = w0 + t * 16 + (lane & 15);
        const bool live = row < sq.nq;
        const T *qp = (const T *)a.q.data + head * a.q.head + (sq.q0 + row) * a.q.row;
        const T *dp = (const T *)a.dout.data + head * a.dout.head + (sq.q0 + row) * a.dout.row;
        const T *op = (const T *)a.out.data + head * a.out.head + (sq.q0 + row) * a.out.row;
        const T *o1 = (const T *)a.out1 + ((sq.q0 + row) * a.heads + head) * 2 * a.dim;
        float dot = 0.f, dot1 = 0.f, most = 0.f;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) {
                const int col = kk * 32 + 8 * g;
                qf[m][t][kk] = load_frag(qp + m * a.q.map, col, a.dim, live, a.vec);
                df[m][t][kk] = load_frag(dp + m * a.dout.map, col, a.dim, live, a.vec);
                const Frag<T> of = load_frag(op + m * a.out.map, col, a.dim, live, a.vec);
                const Frag<T> o1f = load_frag(o1 + m * a.dim, col, a.dim, live, a.vec);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    dot = fmaf((float)df[m][t][kk][j], (float)of[j], dot);
                    dot1 = fmaf((float)df[m][t][kk][j], (float)o1f[j], dot1);
                    if constexpr (kScaled)
                        most = fmaxf(most, fabsf((float)df[m][t][kk][j]));
                }
            }
        delta[1][t] = column_sum(dot1);
        delta[0][t] = fmaf(lambda, delta[1][t], column_sum(dot));
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int64_t at = ((int64_t)m * a.heads + head) * a.total_q + sq.q0 + row;
            const float lse = live ? a.lse[at] : -INFINITY;
            // a row without a key: exp2(s c - inf) is 0
            base[m][t] = lse == -INFINITY ? INFINITY : lse * kLog2e;
        }
        if constexpr (kScaled) {
            // for the key pass's scale
            most = column_max(most);
            if (live && g == 0)
                a.delta[((int64_t)2 * a.heads + head) * a.total_q + sq.q0 + row] = most;
        }
    }

    unsigned long long bits = 0;
    SeenKeys seen(mask, nk, lane);
    auto load = [&](int k0, int to) {
        bits = seen.at(k0, KB) & kFull;
        lk.load(smem, to * 2 * kTile, bits, bits == kFull);
        lv.load(smem, to * 2 * kTile + kTile, bits, bits == kFull);
    };
    auto idle = [&](int k0) { return bits == 0 || w0 >= sq.nq || (a.causal && k0 > w0 + QT * 16 - 1 + shift); };
    auto last = [&](int k) { return w0 + (lane & 15) + shift - k - 4 * g; };
    if (nk > 0)
        load(0, 0);
    if (twice) {
        float summed[2][QT];
#pragma unroll
        for (int t = 0; t < QT; ++t)
            summed[0][t] = summed[1][t] = 0.f;
        for (int k0 = 0;;) {
            wait_loads();
            __syncthreads();
#pragma unroll 1
            for (int b = 0; b < KB / 32 && !idle(k0); ++b) {
                if (empty_block(bits, b, a.causal, k0, w0 + QT * 16 - 1 + shift))
                    continue;
                f32x4 s[2][2][QT], dp[2][QT];
                score_block<T, D, QT>(rd, smem, smem + kTile, b, qf, df, s, dp);
                hide<QT>(s, (unsigned)(bits >> (32 * b + 4 * g)), last(k0 + 32 * b), a.causal);
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int t = 0; t < QT; ++t)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                summed[m][t] = fmaf(exp2_fast(fmaf(s[m][u][t][r], c, -base[m][t])), dp[u][t][r],
                                                    summed[m][t]);
            }
            if (k0 + KB >= nk) {
                if (k0 > 0) {  // back to the first tile; the only one stays
                    __syncthreads();
                    lk.move(-(int64_t)k0 * a.k.row);
                    lv.move(-(int64_t)k0 * a.v.row);
                    seen = SeenKeys(mask, nk, lane);
                    load(0, 0);
                }
                break;
            }
            __syncthreads();
            k0 += KB;
            lk.next();
            lv.next();
            load(k0, 0);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int t = 0; t < QT; ++t)
                delta[m][t] = column_sum(summed[m][t]);
    }
    constexpr bool kRounded = sizeof(T) == 2;
    float missing[2][QT];  // sums of the lane's P (dP - D)
    f32x4 acc[2][QT][D / 16];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        lift[t] = kScaled ? kMostLift : 0;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            missing[m][t] = 0.f;
            base[m][t] -= lift[t];
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                acc[m][t][i] = f32x4{0, 0, 0, 0};
        }
    }
    int buf = 0;
    for (int k0 = 0; k0 < nk; k0 += KB) {
        wait_loads();
        __syncthreads();
        const unsigned long long now = bits;
        const bool rest = idle(k0);
        const char *kt = smem + buf * 2 * kTile, *vt = kt + kTile;
        auto next = [&] {
            if (k0 + KB < nk) {
                buf = BUF - 1 - buf;
                lk.next();
                lv.next();
                load(k0 + KB, buf);
            }
        };
        if constexpr (BUF == 2)
            next();
        const bool partly = now != kFull || (a.causal && k0 + KB - 1 > w0 + shift);
#pragma unroll 1
        for (int b = 0; b < KB / 32 && !rest; ++b) {
            if (empty_block(now, b, a.causal, k0, w0 + QT * 16 - 1 + shift))
                continue;
            f32x4 s[2][2][QT], dp[2][QT];
            score_block<T, D, QT>(rd, kt, vt, b, qf, df, s, dp);
            if (partly)
                hide<QT>(s, (unsigned)(now >> (32 * b + 4 * g)), last(k0 + 32 * b), a.causal);
            Frag<T> sf[2][QT];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int t = 0; t < QT; ++t) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float p = exp2_fast(fmaf(s[m][u][t][r], c, -base[m][t]));
                            s[m][u][t][r] = p * (dp[u][t][r] - delta[m][t]);
                            if (!kScaled && (kRounded || m == 1))
                                missing[m][t] += s[m][u][t][r];
                        }
                    if constexpr (!kScaled)
                        sf[m][t] = pack<T>(s[m][0][t], s[m][1][t]);
                }
            if constexpr (kScaled) {
                float hi[QT];
                bool passed = false;
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    hi[t] = 0.f;
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const f32x4 x = s[m][u][t];
                            hi[t] = max3_abs(max3_abs(hi[t], x[0], x[1]), x[2], x[3]);
                        }
                    passed |= hi[t] > 32768.f;
                }
                if (__any(passed)) {
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        const int down = min(0, 8 - exponent(column_max(hi[t])));
                        const float f = ldexpf(1.f, down);
                        lift[t] += down;
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            base[m][t] -= down;
                            missing[m][t] *= f;
                            s[m][0][t] *= f;
                            s[m][1][t] *= f;
#pragma unroll
                            for (int i = 0; i < D / 16; ++i)
                                acc[m][t][i] *= f;
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < QT; ++t) {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                missing[m][t] += s[m][u][t][r];
                        sf[m][t] = pack<T>(s[m][0][t], s[m][1][t]);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const Frag<T> kf = rd.column_frag(kt, b * 32, m * D + i * 16);
#pragma unroll
                    for (int t = 0; t < QT; ++t)
                        acc[m][t][i] = mma(kf, sf[m][t], acc[m][t][i]);
                }
        }
        if constexpr (BUF == 1) {
            __syncthreads();
            next();
        }
    }

    float dlam = 0.f;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int row = w0 + t * 16 + (lane & 15);
#pragma unroll
        for (int m = 0; m < 2; ++m)
            if (kRounded || m == 1)
                delta[m][t] += column_sum(ldexpf(missing[m][t], -lift[t]));
        if (row >= sq.nq)
            continue;
        if (g == 0) {
            dlam += delta[1][t];
#pragma unroll
            for (int m = 0; m < 2; ++m)
                a.delta[((int64_t)m * a.heads + head) * a.total_q + sq.q0 + row] = delta[m][t];
        }
        T *qp = (T *)a.dq.data + head * a.dq.head + (sq.q0 + row) * a.dq.row;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                store4(qp + m * a.dq.map, i * 16 + 4 * g, a.dim,
                       acc[m][t][i] * ldexpf(m ? -lambda * a.scale : a.scale, -lift[t]), a.vec);
    }
    // this workgroup's share of dlambda
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        dlam += __shfl_xor(dlam, o);
    __syncthreads();
    float *red = reinterpret_cast<float *>(smem);
    if (lane == 0)
        red[wave] = dlam;
    __syncthreads();
    if (tid == 0) {
        float total = 0.f;
        for (int w = 0; w < kWaves; ++w)
            total += red[w];
        a.dlam_part[(int64_t)head * ntiles + wk.tile] = -total;
    }
}

// dlambda of one head from the query tiles' shares, by one workgroup.
template <int THREADS>
__device__ inline void sum_shares(const float *part, int n, float *dlambda, float *red, int tid)
{
    float v = 0.f;
    for (int i = tid; i < n; i += THREADS)
        v += part[i];
    v = wave_sum(v);
    __syncthreads();
    if (tid % kWave == 0)
        red[tid / kWave] = v;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < THREADS / kWave; ++w)
            v += red[w];
        *dlambda = v;
    }
}

#if MTPX_OPS_TYPE == 0
// The same where no key pass runs (the workgroups of its last tile do it
// otherwise).
__global__ __launch_bounds__(kThreads) void dlambda_kernel(const float *part, float *dlambda, int n)
{
    __shared__ float red[kWaves];
    sum_shares<kThreads>(part + (int64_t)blockIdx.x * n, n, dlambda + blockIdx.x, red, threadIdx.x);
}
#endif

// Gradient of the keys and values.  A workgroup takes W * KT * 8 keys of one
// key head; the rows' q, dO and statistics come in tiles of QB rows through
// LDS.  S and dP come out with a key per lane column: P = P_0 - lambda P_1 and
// dS_m are operand B of dV^T += dO^T P and dK_m^T += Q_m^T dS_m, rounded to T
// for them: k's and v's gradients in bfloat16 are off by 0.0023 of their size,
// 0.0017 of which is the rounding of the results.
//
// Two waves share KT * 16 keys.  Of a tile's rows, each forms the scores of
// half; the first then hands its dS to the second, which sums dK, and gets P
// for the other rows, as it sums dV.  One wave alone would hold both sums and
// could afford half as many keys, at twice the reads of the tiles from LDS
// (8,192 causal rows of 16 heads, 64 wide: 1.75 ms; 1.54 to 1.59 ms so).  The query
// heads that share the key head follow one another, so their sum stays in
// registers.  What bounds it now are the waits at its two barriers a tile.
//
// float16: P is scaled by 2^rise, with which P_0 - lambda P_1 stays below 2^15,
// and dS tile by tile by what its elements may be at most: |dO| of the tile's
// rows times the sum of |V| of the pair's keys bounds dP, the statistics D.  The
// scale follows the tiles down, and up where it would lose six bits.
template <class T, int D, int W, int KT, int QB, int BUF, int OCC>
__global__ __launch_bounds__(W * kWave, OCC) void attn_dkv_kernel(AttnArgs a, int table, int ntiles, int shares)
{
    using TL = Tile<T, D>;
    constexpr int kTile = QB * TL::kRowBytes;
    extern __shared__ __align__(16) char smem[];
    float *stats = reinterpret_cast<float *>(smem + BUF * 2 * kTile);  // [BUF][4][QB]
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pair = wave >> 1, half = wave & 1;
    // what one wave of a pair hands to the other: [3][U][KT][lane]
    constexpr int U = QB / 32;
    Half<T> *given = reinterpret_cast<Half<T> *>(stats + BUF * 4 * QB) + pair * (3 * U * KT * kWave) + lane;
    const Work wk = work_item(blockIdx.x, ntiles * a.kv_parts, a.kv_heads);
    const int kv = wk.head, group = a.heads / a.kv_heads;
    const int tile_id = wk.tile / a.kv_parts, part = wk.tile % a.kv_parts;
    const SeqTile sq = a.tiles.k[table][tile_id];
    const int shift = sq.nk - sq.nq;
    const float c = a.scale * kLog2e;
    Reader<T, D> rd;
    rd.init(lane);

    const int w0 = sq.start + pair * KT * 16;  // first key of the pair
    Frag<T> kf[2][KT][D / 32], vf[2][KT][D / 32];
    bool live[KT];
    bool any = false;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const int key = w0 + t * 16 + (lane & 15);
        live[t] = key < sq.nk && (!a.mask || a.mask[sq.k0 + key]);
        any |= live[t];
        const T *kp = (const T *)a.k.data + kv * a.k.head + (sq.k0 + key) * a.k.row;
        const T *vp = (const T *)a.v.data + kv * a.v.head + (sq.k0 + key) * a.v.row;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) {
                kf[m][t][kk] = load_frag(kp + m * a.k.map, kk * 32 + 8 * g, a.dim, live[t], a.vec);
                vf[m][t][kk] = load_frag(vp + m * a.v.map, kk * 32 + 8 * g, a.dim, live[t], a.vec);
            }
    }
    const bool busy = __any(any);
    constexpr bool kScaled = kNarrowRange<T>;
    int rise = 0, lift = 0;
    float value_sum = 0.f;  // largest of the pair's keys
    if constexpr (kScaled) {
        float most = 0.f;
        for (int h = 0; h < group; ++h)
            most = fmaxf(most, fabsf(a.lambda[kv * group + h]));
        rise = 15 - exponent(1.f + most);
        lift = kMostLift;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            float v = 0.f;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        v += fabsf((float)vf[m][t][kk][j]);
            value_sum = fmaxf(value_sum, column_sum(v));
        }
        value_sum = wave_max(value_sum);
    }
    // dV of the first wave, dK_0 and dK_1 side by side of the second
    f32x4 acc[KT][D / 8];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
            acc[t][i] = f32x4{0, 0, 0, 0};

    // rows before the first that sees a key of this workgroup are left out
    const int first = a.causal ? max(0, sq.start - shift) / QB * QB : 0;
    const int per = sq.nq > first ? (sq.nq - first + QB - 1) / QB : 0;
    // of the walk over the rows of all its heads, this workgroup's part
    const int step0 = (int)((int64_t)per * group * part / a.kv_parts);
    const int steps = (int)((int64_t)per * group * (part + 1) / a.kv_parts) - step0;
    const int head0 = kv * group + (steps ? step0 / per : 0), skip = (steps ? step0 % per : 0) * QB;
    Loader<T, D, QB, W> lq, ld;
    lq.init((const T *)a.q.data + sq.q0 * a.q.row, a.q, a.dim, a.vec, tid);
    ld.init((const T *)a.dout.data + sq.q0 * a.dout.row, a.dout, a.dim, a.vec, tid);
    lq.move(head0 * a.q.head + (first + skip) * a.q.row);
    ld.move(head0 * a.dout.head + (first + skip) * a.dout.row);
    // The tiles go round the rows once per query head.
    int to_head = head0, to_q0 = first + skip, head = to_head, q0 = to_q0;
    auto onward = [&](int &h, int &q) {
        q += QB;
        if (q >= sq.nq) {
            q = first;
            ++h;
            return true;
        }
        return false;
    };
    // A step's tiles go into buffer `to`; its statistics and lambda come into
    // registers, and the statistics from there into LDS once no wave reads the
    // buffer any more.
    float st_reg = 0.f, lambda = 0.f, lambda_to = 0.f, most = 0.f, most_to = 0.f;
    auto fetch = [&](int to) {
        const int there = sq.nq - to_q0;
        const unsigned long long bits = there >= 64 ? ~0ull : (1ull << there) - 1;
        if (tid < 4 * QB) {
            const int which = tid / QB, row = to_q0 + tid % QB;
            const float *src = which < 2 ? a.lse : a.delta;
            st_reg = which < 2 ? -INFINITY : 0.f;
            if (row < sq.nq)
                st_reg = src[((int64_t)(which & 1) * a.heads + to_head) * a.total_q + sq.q0 + row];
        }
        lambda_to = a.lambda[to_head];
        if constexpr (kScaled) {
            const int row = to_q0 + lane % QB;
            most_to = row < sq.nq ? a.delta[((int64_t)2 * a.heads + to_head) * a.total_q + sq.q0 + row] : 0.f;
        }
        lq.load(smem, to * 2 * kTile, bits, there >= QB);
        ld.load(smem, to * 2 * kTile + kTile, bits, there >= QB);
        lq.next();
        ld.next();
        if (onward(to_head, to_q0)) {
            lq.move(a.q.head - (int64_t)per * QB * a.q.row);
            ld.move(a.dout.head - (int64_t)per * QB * a.dout.row);
        }
    };
    auto keep = [&](int to) {
        if (tid < 4 * QB)
            stats[to * 4 * QB + tid] =
                tid >= 2 * QB ? st_reg : st_reg == -INFINITY ? INFINITY : st_reg * kLog2e - rise;
        lambda = lambda_to;
        most = most_to;
    };
    static_assert(4 * QB <= W * kWave, "a thread per statistic");
    if (steps > 0) {
        fetch(0);
        keep(0);
    }
    int buf = 0;
    for (int step = 0; step < steps; ++step) {
        wait_loads();
        __syncthreads();
        const char *qt = smem + buf * 2 * kTile, *dt = qt + kTile;
        const float *stat = stats + buf * 4 * QB;
        if constexpr (BUF == 2) {
            buf ^= 1;
            if (step + 1 < steps)
                fetch(buf);
        }
        const bool idle = !busy || (a.causal && q0 + QB - 1 + shift < w0);
        const bool partly = a.causal && q0 + shift < w0 + KT * 16 - 1;
        // a tile of 64 rows: 32 for each wave of the pair; of 32: 16 each
        Half<T> ph[U][KT], sh[2][U][KT];
        float scale = 1.f;
        if constexpr (kScaled) {
            if (!idle) {
                const float d = fmaxf(fabsf(stat[2 * QB + lane % QB]), fabsf(stat[3 * QB + lane % QB]));
                const float bound = wave_max(fmaf(most, value_sum, d)) * fmaxf(1.f, fabsf(lambda));
                const int want = min(15 - exponent(bound) - rise, kMostLift);
                if (bound > 0.f && (want < lift || want > lift + 6)) {
                    if (half) {
                        const float f = ldexpf(1.f, want - lift);
#pragma unroll
                        for (int t = 0; t < KT; ++t)
#pragma unroll
                            for (int i = 0; i < D / 8; ++i)
                                acc[t][i] *= f;
                    }
                    lift = want;
                }
                scale = ldexpf(1.f, lift);
            }
        }
        if (!idle) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r0 = (half * U + u) * 16;
                f32x4 s[2][KT], dp[KT];
#pragma unroll
                for (int t = 0; t < KT; ++t)
                    s[0][t] = s[1][t] = dp[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int kk = 0; kk < D / 32; ++kk) {
                        const Frag<T> qf = rd.row_frag(qt, r0, m * D + kk * 32);
                        const Frag<T> df = rd.row_frag(dt, r0, m * D + kk * 32);
#pragma unroll
                        for (int t = 0; t < KT; ++t) {
                            s[m][t] = mma(qf, kf[m][t][kk], s[m][t]);
                            dp[t] = mma(df, vf[m][t][kk], dp[t]);
                        }
                    }
                const f32x4 l0 = *reinterpret_cast<const f32x4 *>(stat + r0 + 4 * g);
                const f32x4 l1 = *reinterpret_cast<const f32x4 *>(stat + QB + r0 + 4 * g);
                f32x4 d0 = *reinterpret_cast<const f32x4 *>(stat + 2 * QB + r0 + 4 * g);
                f32x4 d1 = *reinterpret_cast<const f32x4 *>(stat + 3 * QB + r0 + 4 * g);
                if constexpr (kScaled) {
                    d0 *= scale;
                    d1 *= scale;
                }
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    // the first row of these that sees the lane's key
                    const int from = partly ? w0 + t * 16 + (lane & 15) - shift - q0 - r0 - 4 * g : -1;
                    f32x4 both;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float p0 = exp2_fast(fmaf(s[0][t][r], c, -l0[r]));
                        float p1 = exp2_fast(fmaf(s[1][t][r], c, -l1[r]));
                        if (partly && r < from)
                            p0 = p1 = 0.f;
                        p1 *= -lambda;
                        both[r] = p0 + p1;
                        s[0][t][r] = p0 * (kScaled ? fmaf(dp[t][r], scale, -d0[r]) : dp[t][r] - d0[r]);
                        s[1][t][r] = p1 * (kScaled ? fmaf(dp[t][r], scale, -d1[r]) : dp[t][r] - d1[r]);
                    }
                    ph[u][t] = round4<T>(both);
                    sh[0][u][t] = round4<T>(s[0][t]);
                    sh[1][u][t] = round4<T>(s[1][t]);
                    if (half) {
                        given[(u * KT + t) * kWave] = ph[u][t];
                    } else {
                        given[((U + u) * KT + t) * kWave] = sh[0][u][t];
                        given[((2 * U + u) * KT + t) * kWave] = sh[1][u][t];
                    }
                }
            }
        }
        __syncthreads();
        if (!idle) {
            // operand B of the wave's products: P twice, or dS_0 and dS_1
            auto mine = [&](int m, int u, int t) { return half ? sh[m][u][t] : ph[u][t]; };
            auto other = [&](int m, int u, int t) {
                return given[((half ? (1 + m) * U : 0) + u) * KT * kWave + t * kWave];
            };
            const char *tile = half ? qt : dt;
            constexpr int kSteps = U * (D / 8);
            Frag<T> xf = rd.column_frag(tile, 0, 0), bf[2][KT];
#pragma unroll
            for (int x = 0; x < kSteps; ++x) {
                const int b = x / (D / 8), i = x % (D / 8);
                if (i == 0) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int t = 0; t < KT; ++t) {
                            if constexpr (U == 1) {
                                const Half<T> o = other(m, 0, t), w = mine(m, 0, t);
                                bf[m][t] = half ? join<T>(o, w) : join<T>(w, o);
                            } else {
                                bf[m][t] = b == half ? join<T>(mine(m, 0, t), mine(m, 1, t))
                                                     : join<T>(other(m, 0, t), other(m, 1, t));
                            }
                        }
                }
                Frag<T> ahead;
                if (x + 1 < kSteps)
                    ahead = rd.column_frag(tile, (x + 1) / (D / 8) * 32, (x + 1) % (D / 8) * 16);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < KT; ++t)
                    acc[t][i] = mma(xf, bf[i / (D / 16)][t], acc[t][i]);
                __builtin_amdgcn_sched_barrier(0);
                xf = ahead;
            }
        }
        if constexpr (BUF == 1)
            __syncthreads();
        if (step + 1 < steps) {
            if constexpr (BUF == 1)
                fetch(0);
            keep(buf);
        }
        onward(head, q0);
    }

    // the last tile has the least work: it sums its heads' shares of dlambda
    if (tile_id == ntiles - 1 && part == a.kv_parts - 1)
        for (int h = kv * group; h < (kv + 1) * group; ++h)
            sum_shares<W * kWave>(a.dlam_part + (int64_t)h * shares, shares, a.dlambda + h,
                                  reinterpret_cast<float *>(smem), tid);

    const mtpx_rows &to = half ? a.dk : a.dv;
    const float factor = half ? ldexpf(a.scale, -lift - rise) : ldexpf(1.f, -rise);
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const int key = w0 + t * 16 + (lane & 15);
        if (key >= sq.nk)
            continue;
        T *p = (T *)to.data + kv * to.head + (sq.k0 + key) * to.row;
        float *sums = a.kv_part + ((((int64_t)part * a.kv_heads + kv) * a.total_k + sq.k0 + key) * 2 + half) * 2 * a.dim;
        // a masked key's gradients are 0, whatever its column holds, and a
        // single key's score has none
        const f32x4 none = {0, 0, 0, 0};
        const bool some = live[t] && !(half && sq.nk == 1);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
            if (a.kv_parts == 1)
                store_columns<T, D>(p, to.map, a.dim, i, lane, some ? acc[t][i] * factor : none, a.vec);
            else
                store_columns<float, D>(sums, a.dim, a.dim, i, lane, some ? acc[t][i] * factor : none,
                                        a.dim % 4 == 0);
    }
}

// Sums the parts of the key pass, in their order, and rounds them once.
template <class T>
__global__ __launch_bounds__(kThreads) void attn_dkv_join(AttnArgs a)
{
    const int width = 4 * a.dim;
    const int64_t each = (int64_t)a.kv_heads * a.total_k * width;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= each)
        return;
    float v = 0.f;
#pragma unroll 4
    for (int p = 0; p < a.kv_parts; ++p)
        v += a.kv_part[p * each + i];
    const int e = (int)(i % width), m = e / a.dim % 2, c = e % a.dim;
    const int64_t key = i / width % a.total_k, kv = i / width / a.total_k;
    const mtpx_rows &to = e >= 2 * a.dim ? a.dk : a.dv;
    ((T *)to.data)[kv * to.head + key * to.row + m * to.map + c] = (T)v;
}

// One query row per sequence.  A workgroup takes one key head of one sequence
// and one of `splits` runs of its keys, for up to 16 of the query heads that
// share the key head (the columns of S^T; fewer leave columns empty, which
// costs nothing, as the reads of the cache bound the kernel).  Its waves take
// steps of 32 keys in turn, each with its own maxima and sums: no wave waits
// for another until the end.  A wave reads K as operand A straight from
// memory; V goes through LDS of its own to be read by columns.  The waves'
// results are joined through LDS.  With one split they are the result; the
// workgroups' are joined by attn_cache_join otherwise, from
// [sequence][head][map][split][2 + 2 D] floats (maximum, sum, product).  The
// reads of the cache bound it (64 caches of 4,096 to 8,192 rows of 4 heads, 64
// wide, in 16 bits: 160 us, 4.8 TB/s).
template <class T, int D, int W, int OCC>
__global__ __launch_bounds__(W * kWave, OCC) void attn_cache_kernel(CacheArgs a)
{
    using TL = Tile<T, D>;
    constexpr int kTile = 32 * TL::kRowBytes;
    constexpr int kPart = 2 + 2 * D;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = a.heads / a.kv_heads, blocks = (group + 15) / 16;
    const int split = blockIdx.x, kv = blockIdx.y / blocks, seq = blockIdx.z;
    const int head0 = kv * group + blockIdx.y % blocks * 16;
    const int count = min(16, (kv + 1) * group - head0);
    const float c = a.scale * kLog2e;
    char *tile = smem + wave * kTile;
    Reader<T, D> rd;
    rd.init(lane);

    int64_t len = a.lengths[seq];
    len = len < 0 ? 0 : len > a.capacity ? a.capacity : len;
    // whole steps, split as evenly as they go
    const int64_t nsteps = (len + 31) / 32;
    const int64_t s0 = nsteps * split / a.splits, s1 = nsteps * (split + 1) / a.splits;

    const T *kp = (const T *)a.k.data + seq * a.k_sequence + kv * a.k.head;
    const T *vp = (const T *)a.v.data + seq * a.v_sequence + kv * a.v.head;

    const int col = lane & 15;
    const T *qp = (const T *)a.q.data + seq * a.q.row + (head0 + col) * a.q.head;
    Frag<T> qf[2][D / 32];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)
            qf[m][kk] = load_frag(qp + m * a.q.map, kk * 32 + 8 * g, a.dim, col < count, a.vec);

    f32x4 acc[2][D / 8];
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
        acc[0][i] = acc[1][i] = f32x4{0, 0, 0, 0};

    // Rows of 256 bytes a map and more leave no registers to read a step ahead:
    // there the values go straight into LDS, and other waves hide the wait.
    constexpr bool kAhead = D * sizeof(T) < 256;
    Stage<T, D, kAhead ? 32 : 0, kWave> sv;
    Frag<T> kf[2][2][D / 32];
    auto fetch = [&](int64_t step) {
        const int64_t k0 = step * 32;
        const int there = (int)min((int64_t)32, len - k0);
        const unsigned long long bits = (1ull << there) - 1;
        if constexpr (kAhead)
            sv.load(vp, a.v, a.dim, k0, bits, lane, a.vec);
        else {
            Loader<T, D, 32, 1> lv;
            lv.init(vp, a.v, a.dim, a.vec, lane);
            lv.move(k0 * a.v.row);
            lv.load(smem, wave * kTile, bits, there == 32);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = 16 * u + (lane & 15);
            const T *p = kp + (k0 + r) * a.k.row;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int kk = 0; kk < D / 32; ++kk)
                    kf[u][m][kk] = load_frag(p + m * a.k.map, kk * 32 + 8 * g, a.dim, r < there, a.vec);
        }
    };
    if (kAhead && s0 + wave < s1)
        fetch(s0 + wave);
    for (int64_t step = s0 + wave; step < s1; step += W) {
        const int there = (int)min((int64_t)32, len - step * 32);
        if constexpr (!kAhead) {
            wait_reads();
            fetch(step);
        }
        f32x4 s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                s[m][u] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int kk = 0; kk < D / 32; ++kk)
                    s[m][u] = mma(kf[u][m][kk], qf[m][kk], s[m][u]);
            }
        if constexpr (kAhead) {
            // the wave's own reads of the last step's values are done before
            // these writes: both go through the LDS in program order
            sv.store(tile, lane);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (step + W < s1)
                fetch(step + W);
        } else {
            wait_loads();
        }
        if (there < 32) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * u + 4 * g + r >= there)
                        s[0][u][r] = s[1][u][r] = -INFINITY;
        }
        Frag<T> pf[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float hi = s[m][0][0];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    hi = fmaxf(hi, s[m][u][r]);
            hi = fmaxf(top[m], column_max(hi));
            if (__any(hi > top[m])) {
                const float f = top[m] == -INFINITY ? 0.f : exp2_fast((top[m] - hi) * c);
                top[m] = hi;
                sum[m] *= f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    acc[m][i] *= f;
            }
            const float base = hi == -INFINITY ? 0.f : hi * c;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = exp2_fast(fmaf(s[m][u][r], c, -base));
                    s[m][u][r] = p;
                    sum[m] += p;
                }
            pf[m] = pack<T>(s[m][0], s[m][1]);
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const Frag<T> vf = rd.column_frag(tile, 0, i * 16);
            acc[0][i] = mma(vf, pf[0], acc[0][i]);
            acc[1][i] = mma(vf, pf[1], acc[1][i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // Join the waves, one map at a time: column-major products in LDS, and the
    // first map's result beside them while the second's are joined.
    float *red = reinterpret_cast<float *>(smem);  // [W][16][kPart], [16][2 D]
    float *first = red + W * 16 * kPart;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float total = column_sum(sum[m]);
        __syncthreads();
        float *mine = red + (wave * 16 + col) * kPart;
        if (g == 0) {
            mine[0] = top[m];
            mine[1] = total;
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                mine[2 + i * 16 + 4 * g + r] = acc[m][i][r];
        __syncthreads();
        for (int e = tid; e < count * 2 * D; e += W * kWave) {
            const int h = e / (2 * D), x = e % (2 * D);
            float hi = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w)
                hi = fmaxf(hi, red[(w * 16 + h) * kPart]);
            float v = 0.f, l = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float *o = red + (w * 16 + h) * kPart;
                const float f = o[0] == -INFINITY ? 0.f : exp2_fast((o[0] - hi) * c);
                v = fmaf(f, o[2 + x], v);
                l = fmaf(f, o[1], l);
            }
            if (a.splits > 1) {
                float *p = a.part + ((((int64_t)seq * a.heads + head0 + h) * 2 + m) * a.splits + split) * kPart;
                if (x == 0) {
                    p[0] = hi;
                    p[1] = l;
                }
                p[2 + x] = v;
                continue;
            }
            v = l == 0.f ? 0.f : v / l;
            if (m == 0) {
                first[e] = v;
            } else if (x % D < a.dim) {
                ((T *)a.out.data)[seq * a.out.row + (head0 + h) * a.out.head + x / D * a.out.map + x % D] =
                    (T)(first[e] - a.lambda[head0 + h] * v);
            }
        }
    }
}

// Joins the splits of one sequence and head: a thread per map and column,
// the splits' weights in LDS.
template <class T, int D>
__global__ __launch_bounds__(4 * D) void attn_cache_join(CacheArgs a)
{
    constexpr int kPart = 2 + 2 * D;
    __shared__ float weight[2][kMaxSplits], joined[2 * D];
    const int tid = threadIdx.x, m = tid / (2 * D), x = tid % (2 * D), head = blockIdx.x, seq = blockIdx.y;
    const float c = a.scale * kLog2e;
    const float *p = a.part + (((int64_t)seq * a.heads + head) * 2 + m) * a.splits * kPart;
    // maxima, then weights, of this map's splits (a map has 2 D >= 64 threads)
    for (int i = x; i < a.splits; i += 2 * D)
        weight[m][i] = p[i * kPart];
    __syncthreads();
    float hi = -INFINITY;
    for (int i = 0; i < a.splits; ++i)
        hi = fmaxf(hi, weight[m][i]);
    __syncthreads();
    for (int i = x; i < a.splits; i += 2 * D)
        weight[m][i] = weight[m][i] == -INFINITY ? 0.f : exp2_fast((weight[m][i] - hi) * c);
    __syncthreads();
    float total = 0.f, v = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.splits; ++i) {
        total = fmaf(weight[m][i], p[i * kPart + 1], total);
        v = fmaf(weight[m][i], p[i * kPart + 2 + x], v);
    }
    v = total == 0.f ? 0.f : v / total;
    if (m == 1)
        joined[x] = v;
    __syncthreads();
    if (m == 0 && x % D < a.dim)
        ((T *)a.out.data)[seq * a.out.row + head * a.out.head + x / D * a.out.map + x % D] =
            (T)(v - a.lambda[head] * joined[x]);
}

// Tile shapes by head width: rows of a wave (16 QT), rows of a tile in LDS.
template <class T, int D>
struct Shape {
    static constexpr int kRows = 2 * D * (int)sizeof(T) <= 256 ? 64 : 32;
    // 16-row groups of a wave: two share the reads from LDS that bound 16-bit
    // products; 32-bit products take so long that more waves serve them better
    static constexpr int kWide = D <= 64 && sizeof(T) == 2 ? 2 : 1;
    // 64 keys: two pairs of waves that share 32 keys where a wave's registers
    // hold those (and two workgroups' LDS a CU), four pairs that share 16 else
    static constexpr int kKeyWide = D <= 64 && sizeof(T) == 2 ? 2 : 1;
    static constexpr int kKeyWaves = 8 / kKeyWide;
    static constexpr size_t kLds = 2 * (size_t)kRows * 2 * D * sizeof(T);
    // two buffers of both tiles within the 64 KiB that loads into LDS address
    static constexpr int kBuffers = kLds <= 32768 ? 2 : 1;
    // waves per SIMD that the registers of one let in
    static constexpr int kOccupancy = kLds > 32768 ? 1 : D == 32 && sizeof(T) == 2 ? 3 : 2;
    // narrow 32-bit heads: three and four, to which one buffer leaves the LDS
    // (200 structures of 84 atoms: forward 103 us with two buffers and two
    // waves, 92 us so; key pass 164 us with 64 rows twice, 128 us with 32 once)
    static constexpr bool kMore = D == 32 && sizeof(T) == 4;
    static constexpr int kQueryBuffers = kMore ? 1 : kBuffers, kQueryOccupancy = kMore ? 3 : kOccupancy;
    static constexpr int kKeyRows = kMore ? 32 : kRows, kKeyBuffers = kMore ? 1 : kBuffers;
    static constexpr int kKeyOccupancy = kMore ? 4 : kOccupancy > 2 ? 3 : 2;
    static constexpr size_t kKeyLds = kKeyBuffers * (4 * (size_t)kKeyRows * D * sizeof(T) + 4 * kKeyRows * sizeof(float)) +
                                      kKeyWaves / 2 * 3 * (kKeyRows / 32) * kKeyWide * kWave * 4 * sizeof(T);
};

// Tables of 64 and 128 rows.
constexpr int kNarrow = 0, kBroad = 1;

// 32 rows a wave halve the reads from LDS per product and are right for work
// that fills the device (32,000 rows of 8 heads, 64 wide: 5.9 ms, 6.9 ms with
// 16 rows a wave); where tiles of 128 rows are fewer than two workgroups a CU,
// tiles of 64 spread the work further (997 rows of 8 heads: 41 us and 31 us a call).
// Sequences of few keys have as few rows where they attend to themselves.
template <int D>
int query_table(const TileTable &t, int heads)
{
    if (t.longest_k <= kFewKeys)
        return kNarrow;
    return Shape<Type, D>::kWide == 2 && (int64_t)t.nq[kBroad] * heads >= 512 ? kBroad : kNarrow;
}

template <int D, int QT>
hipError_t forward_rows(const AttnArgs &a, int table, hipStream_t s)
{
    using S = Shape<Type, D>;
    const int n = a.tiles.nq[table];
    return launch_kernel(attn_forward_kernel<Type, D, 4, QT, S::kRows, S::kQueryBuffers, S::kQueryOccupancy>,
                         dim3((unsigned)((int64_t)n * a.heads)), dim3(kThreads), S::kQueryBuffers * S::kLds, s, a, table, n);
}
template <int D>
hipError_t forward(const AttnArgs &a, hipStream_t s)
{
    if (query_table<D>(a.tiles, a.heads) == kBroad)
        return forward_rows<D, Shape<Type, D>::kWide>(a, kBroad, s);
    return forward_rows<D, 1>(a, kNarrow, s);
}

template <int D, int QT>
hipError_t dq_rows(const AttnArgs &a, int table, hipStream_t s)
{
    using S = Shape<Type, D>;
    const int n = a.tiles.nq[table];
    return launch_kernel(attn_dq_kernel<Type, D, QT, S::kRows, S::kQueryBuffers, S::kQueryOccupancy>,
                         dim3((unsigned)((int64_t)n * a.heads)), dim3(kThreads), S::kQueryBuffers * S::kLds, s, a, table, n);
}
template <int D>
hipError_t backward(const AttnArgs &a, hipStream_t s)
{
    using S = Shape<Type, D>;
    if (a.tiles.nq[kNarrow] > 0) {
        const bool broad = query_table<D>(a.tiles, a.heads) == kBroad;
        if (hipError_t e = broad ? dq_rows<D, S::kWide>(a, kBroad, s) : dq_rows<D, 1>(a, kNarrow, s))
            return e;
    }
    const int nk = a.tiles.nk[kNarrow];
    if (nk == 0)
        return hipSuccess;
    const hipError_t e = launch_kernel(
        attn_dkv_kernel<Type, D, S::kKeyWaves, S::kKeyWide, S::kKeyRows, S::kKeyBuffers, S::kKeyOccupancy>,
        dim3((unsigned)((int64_t)nk * a.kv_heads * a.kv_parts)), dim3(S::kKeyWaves * kWave), S::kKeyLds, s, a, kNarrow,
        nk, a.tiles.nq[query_table<D>(a.tiles, a.heads)]);
    if (e != hipSuccess || a.kv_parts == 1)
        return e;
    const int64_t n = a.kv_heads * a.total_k * 4 * a.dim;
    return launch_kernel(attn_dkv_join<Type>, dim3((unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
}

template <int D, int W>
hipError_t cache_waves(const CacheArgs &a, hipStream_t s)
{
    const int group = a.heads / a.kv_heads;
    constexpr size_t tiles = (size_t)W * 32 * 2 * D * sizeof(Type);
    static_assert(tiles <= 65536, "what loads into LDS address");
    constexpr size_t join = ((size_t)W * 16 * (2 + 2 * D) + 16 * 2 * D) * sizeof(float);
    constexpr int occ = D * sizeof(Type) < 256 ? 2 : 1;
    return launch_kernel(attn_cache_kernel<Type, D, W, occ>, dim3(a.splits, a.kv_heads * ((group + 15) / 16), a.sequences),
                         dim3(W * kWave), tiles > join ? tiles : join, s, a);
}
// Eight waves where one workgroup takes a whole cache, four where splits
// share it, fewer where their tiles would not fit.
template <int D>
hipError_t cache(const CacheArgs &a, hipStream_t s)
{
    constexpr int most = 1024 / (D * (int)sizeof(Type));
    if (a.splits == 1)
        return cache_waves<D, most < 8 ? most : 8>(a, s);
    const hipError_t e = cache_waves<D, most < 4 ? most : 4>(a, s);
    if (e != hipSuccess)
        return e;
    return launch_kernel(attn_cache_join<Type, D>, dim3(a.heads, a.sequences), dim3(4 * D), 0, s, a);
}

}  // namespace

hipError_t MTPX_OPS_NAME(attn_forward)(const AttnArgs &a, hipStream_t s)
{
    return a.dim <= 32 ? forward<32>(a, s) : a.dim <= 64 ? forward<64>(a, s) : forward<128>(a, s);
}
hipError_t MTPX_OPS_NAME(attn_backward)(const AttnArgs &a, hipStream_t s)
{
    return a.dim <= 32 ? backward<32>(a, s) : a.dim <= 64 ? backward<64>(a, s) : backward<128>(a, s);
}
hipError_t MTPX_OPS_NAME(attn_cache)(const CacheArgs &a, hipStream_t s)
{
    return a.dim <= 32 ? cache<32>(a, s) : a.dim <= 64 ? cache<64>(a, s) : cache<128>(a, s);
}
int MTPX_OPS_NAME(attn_tiles)(int dim, int heads, const TileTable &t)
{
    return t.nq[dim <= 32 ? query_table<32>(t, heads)
                          : dim <= 64 ? query_table<64>(t, heads) : query_table<128>(t, heads)];
}

#if MTPX_OPS_TYPE == 0
hipError_t attn_forward_bf16(const AttnArgs &, hipStream_t);
hipError_t attn_forward_f16(const AttnArgs &, hipStream_t);
hipError_t attn_backward_bf16(const AttnArgs &, hipStream_t);
hipError_t attn_backward_f16(const AttnArgs &, hipStream_t);
hipError_t attn_cache_bf16(const CacheArgs &, hipStream_t);
hipError_t attn_cache_f16(const CacheArgs &, hipStream_t);
int attn_tiles_bf16(int, int, const TileTable &);
int attn_tiles_f16(int, int, const TileTable &);

int attn_backward_tiles(int dtype, int dim, int heads, const TileTable &t)
{
    return dtype == MTPX_F32    ? attn_tiles_f32(dim, heads, t)
           : dtype == MTPX_BF16 ? attn_tiles_bf16(dim, heads, t)
                                : attn_tiles_f16(dim, heads, t);
}
hipError_t launch_attn_forward(int dtype, const AttnArgs &a, hipStream_t s)
{
    return dtype == MTPX_F32 ? attn_forward_f32(a, s)
                             : dtype == MTPX_BF16 ? attn_forward_bf16(a, s) : attn_forward_f16(a, s);
}
hipError_t launch_attn_backward(int dtype, const AttnArgs &a, hipStream_t s)
{
    const hipError_t e = dtype == MTPX_F32 ? attn_backward_f32(a, s)
                         : dtype == MTPX_BF16 ? attn_backward_bf16(a, s) : attn_backward_f16(a, s);
    if (e != hipSuccess || a.tiles.nk[kNarrow] > 0)
        return e;
    return launch_kernel(dlambda_kernel, dim3(a.heads), dim3(kThreads), 0, s, a.dlam_part, a.dlambda,
                         attn_backward_tiles(dtype, a.dim, a.heads, a.tiles));
}
hipError_t launch_attn_cache(int dtype, const CacheArgs &a, hipStream_t s)
{
    return dtype == MTPX_F32 ? attn_cache_f32(a, s)
                             : dtype == MTPX_BF16 ? attn_cache_bf16(a, s) : attn_cache_f16(a, s);
}
#endif

}  // namespace mtpx
