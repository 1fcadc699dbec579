// Group normalisation with its activation, channels last.
//
//   y[i][r][c] = act((x[i][r][c] - mean) / sqrt(var + eps) * gamma[c] + beta[c])
//
// with the mean and the biased variance of image i over all rows and the
// `width` channels of c's group.  Memory-bound: 16 bytes per lane per access
// where the layout allows them (V elements, else one).
//
// Statistics.  Every thread keeps V fixed channels and walks rows; it forms
// the mean and the sum of squared differences of a few rows held in registers
// in two passes, and joins such pieces pairwise (n, mean, M2), so that no
// difference of large sums is taken however far the mean is from zero.  The
// pieces of a workgroup are joined per group through LDS the same way: the
// weighted mean first (as differences from one of the means), then
// M2 + n (mean_i - mean)^2.  All of it in a fixed order: the same input gives
// the same output.
//
// Two forms, by the size of an image.
//   slab   a workgroup holds the rows of some whole groups of an image in
//          registers (128 KB at most): one launch, x read once.
//   rows   three launches: every workgroup reduces a run of rows, a small
//          kernel joins the runs, and a last pass reads x again.
//
// What it reaches: 3 x 230400 x 256 bf16 with SiLU 185 us (rows form: 65 us of
// statistics at 5.4 TB/s, 4 to join, 116 for the last pass at 6.1 TB/s, read and
// write; one read and one write at a large copy's rate would be 142), with rows
// of 264 elements 218, of 257 (one element a lane) 293; 480 x 512 fp16 7.5 us
// (slab form, the latency of one launch); 3 x 3600 x 320 fp32 17 us (three
// launches of 4 to 7).  Tried and taken back: image by image, so that the
// last pass reads from the last-level cache (no faster, more launches); joining
// in the last pass (15.6 us for the last case, 21 images 59 against 51).
#include "sv2_internal.h"
#include "activation.h"
#include "vec_io.h"

#include <algorithm>
#include <type_traits>

namespace sv2
{
namespace
{

using namespace vec;

struct NormArgs
{
    const void* x;
    void* y;
    long long x_image, x_row, y_image, y_row; // strides in elements
    const float* gamma;
    const float* beta;
    int rows, channels, groups, width;
    int unit;                 // channels of a thread's V that surely share a group: gcd(width, V)
    float eps;
    int slab_groups, slabs, blocks; // slab form
    int chunk_rows, chunks;   // rows form
    float2* part;             // rows form: (mean, M2) [image][group][chunk], then (mean, rstd) [image][group]
    float2* stat;
};

constexpr int kSlabThreads = 1024;
constexpr int kRowThreads = 256;
constexpr int kMaxChannels = 8192;

template <typename T>
constexpr int elem_bytes()
{
    return std::is_same_v<T, F32> ? 4 : 2;
}

typedef __attribute__((ext_vector_type(4))) unsigned u4;

// Outputs go past the caches: written through the last-level cache they leave
// dirty lines there, whose eviction costs the statistics of the next call half
// of their rate (3 x 230400 x 256 bf16: statistics 85 against 58 us, the whole
// 213 against 193).
__device__ inline void put16(void* to, u4 v)
{
    __builtin_nontemporal_store(v, static_cast<u4*>(to));
}

// V elements of one row piece, as loaded.
template <typename T, int V>
struct Piece;
template <typename T>
struct Piece<T, 1>
{
    float v;
    __device__ void load(const void* base, long long i)
    {
        if constexpr (std::is_same_v<T, F32>)
            v = static_cast<const float*>(base)[i];
        else if constexpr (std::is_same_v<T, F16>)
            v = static_cast<float>(static_cast<const _Float16*>(base)[i]);
        else
            v = __builtin_bit_cast(float, static_cast<uint32_t>(static_cast<const uint16_t*>(base)[i]) << 16);
    }
    __device__ void get(float x[1]) const { x[0] = v; }
    __device__ static void store(void* base, long long i, const float x[1])
    {
        if constexpr (std::is_same_v<T, F32>)
            static_cast<float*>(base)[i] = x[0];
        else if constexpr (std::is_same_v<T, F16>)
            static_cast<_Float16*>(base)[i] = static_cast<_Float16>(x[0]);
        else
            static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(to_bf16_bits(x[0]));
    }
};
template <typename T>
struct Piece<T, 8>
{
    Raw8<T> r;
    __device__ void load(const void* base, long long i) { ld_raw8<T>(base, i, r); }
    __device__ void get(float x[8]) const { raw8_float(r, x); }
    __device__ static void store(void* base, long long i, const float x[8])
    {
        if constexpr (std::is_same_v<T, BF16>)
        {
            // v_cvt_pk_bf16_f32 (nearest even)
            typedef __attribute__((ext_vector_type(8))) __bf16 b8;
            b8 v;
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[e] = static_cast<__bf16>(x[e]);
            put16(static_cast<uint16_t*>(base) + i, __builtin_bit_cast(u4, v));
        }
        else
        {
            f16x8 v;
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[e] = static_cast<_Float16>(x[e]);
            put16(static_cast<uint16_t*>(base) + i, __builtin_bit_cast(u4, v));
        }
    }
};
template <>
struct Piece<F32, 4>
{
    float4 r;
    __device__ void load(const void* base, long long i) { r = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i); }
    __device__ void get(float x[4]) const
    {
        x[0] = r.x; x[1] = r.y; x[2] = r.z; x[3] = r.w;
    }
    __device__ static void store(void* base, long long i, const float x[4])
    {
        typedef __attribute__((ext_vector_type(4))) float f4;
        put16(static_cast<float*>(base) + i, __builtin_bit_cast(u4, f4{x[0], x[1], x[2], x[3]}));
    }
};

// Elements of a 16-byte access.
template <typename T>
constexpr int wide()
{
    return 16 / elem_bytes<T>();
}

// Over the `team` lanes (a power of two) that share lane / team.
__device__ inline float team_sum(float v, int team)
{
    for (int d = team >> 1; d > 0; d >>= 1)
        v += __shfl_xor(v, d, 64);
    return v;
}

// Joins `entries` pieces (count n(e), mean, M2) whose counts add up to `total`
// by a team of lanes, `lane` being the caller's place in it; every lane
// receives the result.
template <typename N, typename E>
__device__ inline void join(int entries, float total, int team, int lane, N n, E entry, float* out_mean, float* out_m2)
{
    const float ref = entry(0).x;
    float d = 0.f;
    for (int e = lane; e < entries; e += team)
        d += n(e) * (entry(e).x - ref);
    const float mu = ref + team_sum(d, team) / total;
    float s = 0.f;
    for (int e = lane; e < entries; e += team)
    {
        const float2 p = entry(e);
        const float off = p.x - mu;
        s += p.y + n(e) * off * off;
    }
    *out_mean = mu;
    *out_m2 = team_sum(s, team);
}

// Lanes per group, so that a workgroup's threads take its groups at once
// where they can.
__device__ inline int team_of(int threads, int groups)
{
    int team = 64;
    while (team > 1 && threads / team < groups)
        team >>= 1;
    return team;
}

// Joins the V channels' pieces (each over n rows) by spans of `unit` channels,
// which lie in one group, and writes one piece a span.
template <int V>
__device__ inline void put_pieces(float2* to, float mean[V], float m2[V], float n, int unit)
{
#pragma unroll
    for (int span = 1; span < V; span *= 2)
        if (span < unit)
#pragma unroll
            for (int e = 0; e < V; e += 2 * span)
            {
                const float d = mean[e + span] - mean[e];
                mean[e] += 0.5f * d;
                m2[e] += m2[e + span] + d * d * (0.5f * n * static_cast<float>(span));
            }
    int k = 0;
#pragma unroll
    for (int e = 0; e < V; e++)
        if ((e & (unit - 1)) == 0)
            to[k++] = make_float2(mean[e], m2[e]);
}

// How `rows` rows fall to row lanes: lane r takes rows r, r + lanes, ...
struct Share
{
    int each, more; // lanes 0 .. more - 1 take one row more
    __device__ Share(int rows, int lanes) : each(rows / lanes), more(rows - each * lanes) {}
    __device__ int of(int r) const { return each + (r < more ? 1 : 0); }
};

// e / d for 0 <= e < 2^21 (threads, channels, pieces in LDS) and inv = 1 / d: the half keeps the
// quotient's rounding errors, 2^-22 of it, from reaching a whole number.
__device__ inline int quick_div(int e, float inv)
{
    return static_cast<int>((static_cast<float>(e) + 0.5f) * inv);
}

// gamma and beta of V channels, then with the group's mean and
// 1 / sqrt(var + eps) folded into the scale.
template <int V>
struct Affine
{
    float mean[V], a[V], b[V];
    __device__ void load(const float* gamma, const float* beta, int c0)
    {
#pragma unroll
        for (int e = 0; e < V; e++)
        {
            a[e] = gamma ? gamma[c0 + e] : 1.f;
            b[e] = beta ? beta[c0 + e] : 0.f;
        }
    }
    template <typename G>
    __device__ void scale(G stat)
    {
#pragma unroll
        for (int e = 0; e < V; e++)
        {
            const float2 s = stat(e);
            mean[e] = s.x;
            a[e] *= s.y;
        }
    }
    template <int ACT, bool EXACT>
    __device__ void apply(float x[V]) const
    {
#pragma unroll
        for (int e = 0; e < V; e++)
            x[e] = activate<ACT, EXACT>(__builtin_fmaf(x[e] - mean[e], a[e], b[e]));
    }
};

// Slab form: workgroup (image, slab of slab_groups groups), at most KEEP rows
// of V channels per thread.
template <typename T, int V, int KEEP, int ACT>
__global__ __launch_bounds__(kSlabThreads) void norm_slab_kernel(NormArgs p)
{
    extern __shared__ __attribute__((aligned(16))) float smem[];
    // XCD x (workgroup id mod 8) takes a contiguous run: slabs that share a
    // 128-byte line share an L2
    const int id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (id >= p.blocks)
        return;
    const int image = id / p.slabs;
    const int g0 = (id - image * p.slabs) * p.slab_groups;
    const int ng = min(p.slab_groups, p.groups - g0);
    const int c_base = g0 * p.width;
    const int sc = ng * p.width;     // channels of this slab, a multiple of V
    const int nc = sc / V;
    const int lanes = blockDim.x / nc;
    const int r0 = quick_div(threadIdx.x, 1.f / static_cast<float>(nc));
    const int c = (threadIdx.x - r0 * nc) * V;
    const bool active = r0 < lanes;
    const Share share(p.rows, lanes);
    const int mine = active ? share.of(r0) : 0;
    const long long xi = image * p.x_image + c_base + c;

    Piece<T, V> keep[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; k++)
        if (k < mine)
            keep[k].load(p.x, xi + static_cast<long long>(r0 + k * lanes) * p.x_row);
    Affine<V> f;
    if (active)
        f.load(p.gamma, p.beta, c_base + c);
    float mean[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; e++)
        mean[e] = m2[e] = 0.f;
#pragma unroll
    for (int k = 0; k < KEEP; k++)
        if (k < mine)
        {
            float x[V];
            keep[k].get(x);
#pragma unroll
            for (int e = 0; e < V; e++)
                mean[e] += x[e];
        }
    const float inv = 1.f / static_cast<float>(max(mine, 1));
#pragma unroll
    for (int e = 0; e < V; e++)
        mean[e] *= inv;
#pragma unroll
    for (int k = 0; k < KEEP; k++)
        if (k < mine)
        {
            float x[V];
            keep[k].get(x);
#pragma unroll
            for (int e = 0; e < V; e++)
                m2[e] += (x[e] - mean[e]) * (x[e] - mean[e]);
        }
    // pieces [row lane][span of unit channels], then (mean, rstd) per group
    const int unit = p.unit;
    const int spans = sc / unit;
    float2* s_piece = reinterpret_cast<float2*>(smem);
    float2* s_stat = s_piece + lanes * spans;
    if (active)
        put_pieces<V>(s_piece + r0 * spans + c / unit, mean, m2, static_cast<float>(mine), unit);
    __syncthreads();
    const int used = min(lanes, p.rows); // row lanes that hold a row
    const float total = static_cast<float>(p.rows) * static_cast<float>(p.width);
    const int team = team_of(blockDim.x, ng);
    const int per = p.width / unit;
    const float inv_per = 1.f / static_cast<float>(per);
    for (int g = threadIdx.x / team; g < ng; g += blockDim.x / team)
    {
        float mu, s;
        join(used * per, total, team, threadIdx.x & (team - 1),
             [&](int e) { return static_cast<float>(share.of(quick_div(e, inv_per)) * unit); },
             [&](int e) { const int r = quick_div(e, inv_per); return s_piece[r * (spans - per) + g * per + e]; }, &mu, &s);
        if ((threadIdx.x & (team - 1)) == 0)
            s_stat[g] = make_float2(mu, 1.f / sqrtf(s / total + p.eps));
    }
    __syncthreads();
    if (!active)
        return;
    const float inv_width = 1.f / static_cast<float>(p.width);
    if (unit == V)
    {
        const float2 one = s_stat[quick_div(c, inv_width)];
        f.scale([&](int) { return one; });
    }
    else
        f.scale([&](int e) { return s_stat[quick_div(c + e, inv_width)]; });
    const long long yi = image * p.y_image + c_base + c;
#pragma unroll
    for (int k = 0; k < KEEP; k++)
        if (k < mine)
        {
            float x[V];
            keep[k].get(x);
            f.template apply<ACT, std::is_same_v<T, F32>>(x);
            Piece<T, V>::store(p.y, yi + static_cast<long long>(r0 + k * lanes) * p.y_row, x);
        }
}

// Channels are taken by the 256 threads of a workgroup V at a time; where they
// are more than 256 V, in rounds.
struct Columns
{
    int nc, lanes, rounds;
};
template <int V>
__host__ __device__ inline Columns columns(int channels)
{
    Columns k;
    k.nc = channels / V;
    k.lanes = k.nc >= kRowThreads ? 1 : kRowThreads / k.nc;
    k.rounds = (k.nc + kRowThreads - 1) / kRowThreads;
    return k;
}

// Rows form, first launch: workgroup (image, run of chunk_rows rows).
template <typename T, int V>
__global__ __launch_bounds__(kRowThreads, 4) void norm_stats_kernel(NormArgs p)
{
    extern __shared__ __attribute__((aligned(16))) float smem[];
    constexpr int kHeld = V == 1 ? 16 : 8; // rows in registers at a time
    const int image = blockIdx.x / p.chunks;
    const int chunk = blockIdx.x - image * p.chunks;
    const int first = chunk * p.chunk_rows;
    const int rows = min(p.chunk_rows, p.rows - first);
    const Columns k = columns<V>(p.channels);
    const Share share(rows, k.lanes);
    const int spans = p.channels / p.unit;
    float2* s_piece = reinterpret_cast<float2*>(smem); // [row lane][span of unit channels]
    for (int round = 0; round < k.rounds; round++)
    {
        // (quick_div here costs the large case 4 us of 188: its loop comes out differently)
        const int r0 = k.rounds > 1 ? 0 : threadIdx.x / k.nc;
        const int col = k.rounds > 1 ? round * kRowThreads + threadIdx.x : threadIdx.x - r0 * k.nc;
        if (r0 >= k.lanes || col >= k.nc)
            continue;
        const int mine = share.of(r0);
        long long at = image * p.x_image + static_cast<long long>(first + r0) * p.x_row + col * V;
        const long long step = k.lanes * p.x_row;
        float mean[V], m2[V];
#pragma unroll
        for (int e = 0; e < V; e++)
            mean[e] = m2[e] = 0.f;
        // the next rows are on their way while these are summed
        Piece<T, V> ahead[kHeld];
        if (kHeld <= mine)
#pragma unroll
            for (int i = 0; i < kHeld; i++)
                ahead[i].load(p.x, at + i * step);
        int done = 0;
        for (; done + kHeld <= mine; done += kHeld)
        {
            Piece<T, V> h[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; i++)
                h[i] = ahead[i];
            at += kHeld * step;
            if (done + 2 * kHeld <= mine)
#pragma unroll
                for (int i = 0; i < kHeld; i++)
                    ahead[i].load(p.x, at + i * step);
            // sums of differences from the mean so far (the first row at the
            // start): of kHeld rows the subtraction below takes at most
            // (kHeld - 1) / kHeld of s2 away, 7/8 or 15/16, the reference being
            // one of the values or the mean of as many
            float ref[V], s1[V], s2[V];
            if (done == 0)
                h[0].get(mean);
#pragma unroll
            for (int e = 0; e < V; e++)
            {
                ref[e] = mean[e];
                s1[e] = s2[e] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < kHeld; i++)
            {
                float x[V];
                h[i].get(x);
#pragma unroll
                for (int e = 0; e < V; e++)
                {
                    const float d = x[e] - ref[e];
                    s1[e] += d;
                    s2[e] = __builtin_fmaf(d, d, s2[e]);
                }
            }
            const float inv = 1.f / static_cast<float>(done + kHeld);
#pragma unroll
            for (int e = 0; e < V; e++)
            {
                const float d = s1[e] * inv;
                mean[e] += d;
                m2[e] += __builtin_fmaf(-d, s1[e], s2[e]);
            }
        }
        for (; done < mine; done++)
        {
            Piece<T, V> h;
            h.load(p.x, at);
            at += step;
            float x[V];
            h.get(x);
            const float share = 1.f / static_cast<float>(done + 1);
#pragma unroll
            for (int e = 0; e < V; e++)
            {
                const float d = x[e] - mean[e];
                mean[e] += d * share;
                m2[e] += d * (x[e] - mean[e]);
            }
        }
        put_pieces<V>(s_piece + r0 * spans + col * V / p.unit, mean, m2, static_cast<float>(mine), p.unit);
    }
    __syncthreads();
    const int used = min(k.lanes, rows);
    const float total = static_cast<float>(rows) * static_cast<float>(p.width);
    const int team = team_of(kRowThreads, p.groups);
    const int per = p.width / p.unit;
    const float inv_per = 1.f / static_cast<float>(per);
    for (int g = threadIdx.x / team; g < p.groups; g += kRowThreads / team)
    {
        float mu, s;
        join(used * per, total, team, threadIdx.x & (team - 1),
             [&](int e) { return static_cast<float>(share.of(quick_div(e, inv_per)) * p.unit); },
             [&](int e) { const int r = quick_div(e, inv_per); return s_piece[r * (spans - per) + g * per + e]; }, &mu, &s);
        if ((threadIdx.x & (team - 1)) == 0)
            p.part[(static_cast<long long>(image) * p.groups + g) * p.chunks + chunk] = make_float2(mu, s);
    }
}

// Rows form, second launch: a workgroup per (image, group), the pieces in
// registers.
constexpr int kJoinThreads = 256;
constexpr int kJoinHeld = 8;
constexpr int kMaxChunks = kJoinThreads * kJoinHeld;

__device__ inline float block_sum(float v, float* scratch)
{
    v = team_sum(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 64; w++)
        s += scratch[w];
    return s;
}

__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(NormArgs p)
{
    __shared__ float scratch[kJoinThreads / 64];
    const float2* part = p.part + static_cast<long long>(blockIdx.x) * p.chunks;
    const float w = static_cast<float>(p.width);
    const float total = static_cast<float>(p.rows) * w;
    const float ref = part[0].x;
    float2 v[kJoinHeld];
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < kJoinHeld; i++)
    {
        const int e = threadIdx.x + kJoinThreads * i;
        v[i] = e < p.chunks ? part[e] : make_float2(ref, 0.f);
    }
#pragma unroll
    for (int i = 0; i < kJoinHeld; i++)
    {
        const int e = threadIdx.x + kJoinThreads * i;
        d += w * static_cast<float>(min(p.chunk_rows, p.rows - min(e, p.chunks - 1) * p.chunk_rows)) * (v[i].x - ref);
    }
    const float mu = ref + block_sum(d, scratch) / total;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kJoinHeld; i++)
    {
        const int e = threadIdx.x + kJoinThreads * i;
        const float off = v[i].x - mu;
        if (e < p.chunks)
            s += v[i].y + w * static_cast<float>(min(p.chunk_rows, p.rows - e * p.chunk_rows)) * off * off;
    }
    s = block_sum(s, scratch);
    if (threadIdx.x == 0)
        p.stat[blockIdx.x] = make_float2(mu, 1.f / sqrtf(s / total + p.eps));
}

// Rows form, third launch.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kRowThreads) void norm_apply_kernel(NormArgs p)
{
    constexpr int kHeld = 4;
    // backwards: what the statistics read last may still be in the last-level
    // cache
    const int block = gridDim.x - 1 - blockIdx.x;
    const int image = block / p.chunks;
    const int first = (block - image * p.chunks) * p.chunk_rows;
    const int rows = min(p.chunk_rows, p.rows - first);
    const Columns k = columns<V>(p.channels);
    const float2* stat = p.stat + static_cast<long long>(image) * p.groups;
    const float inv_width = 1.f / static_cast<float>(p.width);
    for (int round = 0; round < k.rounds; round++)
    {
        const int r0 = k.rounds > 1 ? 0 : quick_div(threadIdx.x, 1.f / static_cast<float>(k.nc));
        const int col = k.rounds > 1 ? round * kRowThreads + threadIdx.x : threadIdx.x - r0 * k.nc;
        if (r0 >= k.lanes || col >= k.nc)
            continue;
        const int mine = Share(rows, k.lanes).of(r0);
        long long xi = image * p.x_image + static_cast<long long>(first + r0) * p.x_row + col * V;
        long long yi = image * p.y_image + static_cast<long long>(first + r0) * p.y_row + col * V;
        const long long xs = k.lanes * p.x_row;
        const long long ys = k.lanes * p.y_row;
        // the next rows are on their way while these are normalised, the first
        // while the factors are
        Piece<T, V> ahead[kHeld];
        if (kHeld <= mine)
#pragma unroll
            for (int i = 0; i < kHeld; i++)
                ahead[i].load(p.x, xi + i * xs);
        Affine<V> f;
        f.load(p.gamma, p.beta, col * V);
        if (p.unit == V)
        {
            const float2 one = stat[quick_div(col * V, inv_width)];
            f.scale([&](int) { return one; });
        }
        else
            f.scale([&](int e) { return stat[quick_div(col * V + e, inv_width)]; });
        auto finish = [&](const Piece<T, V>& h, long long to) {
            float x[V];
            h.get(x);
            f.template apply<ACT, std::is_same_v<T, F32>>(x);
            Piece<T, V>::store(p.y, to, x);
        };
        int done = 0;
        for (; done + kHeld <= mine; done += kHeld)
        {
            Piece<T, V> h[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; i++)
                h[i] = ahead[i];
            xi += kHeld * xs;
            if (done + 2 * kHeld <= mine)
#pragma unroll
                for (int i = 0; i < kHeld; i++)
                    ahead[i].load(p.x, xi + i * xs);
#pragma unroll
            for (int i = 0; i < kHeld; i++)
                finish(h[i], yi + i * ys);
            yi += kHeld * ys;
        }
        for (; done < mine; done++)
        {
            Piece<T, V> h;
            h.load(p.x, xi);
            finish(h, yi);
            xi += xs;
            yi += ys;
        }
    }
}

// The rows form's runs: enough workgroups for 256 CUs, at least 32 KB each.
void plan_rows(NormArgs* p, int images, int bytes)
{
    const long long row_bytes = static_cast<long long>(p->channels) * bytes;
    // kMaxChunks runs in all, so no image has more
    const long long want = (static_cast<long long>(images) * p->rows + kMaxChunks - 1) / kMaxChunks;
    const long long least = std::max(1LL, 32768 / row_bytes);
    p->chunk_rows = static_cast<int>(std::min<long long>(p->rows, std::max(want, least)));
    p->chunks = (p->rows + p->chunk_rows - 1) / p->chunk_rows;
}

// Bytes of (mean, M2) of every run and (mean, rstd) of every group.
long long rows_workspace(const NormArgs& p, int images)
{
    return static_cast<long long>(images) * p.groups * (p.chunks + 1) * static_cast<long long>(sizeof(float2));
}

// Pieces a thread of the slab form holds: 128 KB a workgroup.  Past that the
// rows form is the faster one, though it reads twice: one image of 32 groups of
// 16 in fp16 takes 10.0 / 14.4 / 20.3 us at 960 / 1920 / 3600 rows (61 / 123 /
// 230 KB a workgroup) against 15.7 / 15.8 / 16.0.
constexpr int keep_of(int v)
{
    return v == 1 ? 32 : 8;
}

// The slab form's shape for pieces of V elements, or threads = 0 where an
// image does not fit: whole groups whose channels are a multiple of V, 64
// bytes of a row at least (a quarter of the groups otherwise share a line).
struct Slab
{
    int groups, threads, lds;
};
Slab plan_slab(const NormArgs& p, int v, int bytes)
{
    const int keep = keep_of(v);
    int g = 1;
    while (g < p.groups && (g * p.width % v != 0 || g * p.width * bytes < 64))
        g++;
    const int sc = g * p.width;
    const int nc = sc / v;
    if (sc % v != 0 || nc > kSlabThreads)
        return Slab{0, 0, 0};
    // the fewest threads that hold the rows in half of the registers, or all
    // of them
    for (int threads : {256, 512, 1024})
    {
        const int lanes = threads / nc;
        if (lanes > 0 && p.rows <= lanes * (threads < 1024 ? keep / 2 : keep))
            // the last slab may be narrower and have more row lanes
            return Slab{g, threads, 2 * threads * v * 4 + g * 8};
    }
    return Slab{0, 0, 0};
}

template <typename T, int V, int ACT>
int run_norm(NormArgs p, int images, bool slab, const Slab& s, hipStream_t stream)
{
    if (slab)
    {
        constexpr int kKeep = keep_of(V);
        p.slab_groups = s.groups;
        p.slabs = (p.groups + s.groups - 1) / s.groups;
        const long long grid = static_cast<long long>(images) * p.slabs;
        if (!grid_fits(grid + 7, s.threads))
            return set_error(SV2_EUNSUPPORTED, "sv2_group_norm: too many images");
        p.blocks = static_cast<int>(grid);
        const void* fn = reinterpret_cast<const void*>(&norm_slab_kernel<T, V, kKeep, ACT>);
        const int rc = set_dynamic_lds(fn, s.lds, "norm_slab: dynamic LDS attribute");
        if (rc != SV2_OK)
            return rc;
        hipLaunchKernelGGL((norm_slab_kernel<T, V, kKeep, ACT>), dim3((static_cast<unsigned>(grid) + 7) / 8 * 8),
                           dim3(s.threads), s.lds, stream, p);
    }
    else
    {
        const long long grid = static_cast<long long>(images) * p.chunks;
        const long long joins = static_cast<long long>(images) * p.groups;
        if (!grid_fits(grid, kRowThreads) || !grid_fits(joins, kJoinThreads))
            return set_error(SV2_EUNSUPPORTED, "sv2_group_norm: too many images");
        const int lds = 2 * columns<V>(p.channels).lanes * p.channels * 4;
        const void* fn = reinterpret_cast<const void*>(&norm_stats_kernel<T, V>);
        const int rc = set_dynamic_lds(fn, lds, "norm_stats: dynamic LDS attribute");
        if (rc != SV2_OK)
            return rc;
        hipLaunchKernelGGL((norm_stats_kernel<T, V>), dim3(static_cast<unsigned>(grid)), dim3(kRowThreads), lds, stream, p);
        hipLaunchKernelGGL(norm_join_kernel, dim3(static_cast<unsigned>(joins)), dim3(kJoinThreads), 0, stream,
                           p);
        hipLaunchKernelGGL((norm_apply_kernel<T, V, ACT>), dim3(static_cast<unsigned>(grid)), dim3(kRowThreads), 0, stream, p);
    }
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? SV2_OK : hip_error(err, "sv2_group_norm launch");
}

template <typename T, int V>
int run_act(const NormArgs& p, int images, int activation, bool slab, const Slab& s, hipStream_t stream)
{
    switch (activation)
    {
    case SV2_ACT_SILU: return run_norm<T, V, SV2_ACT_SILU>(p, images, slab, s, stream);
    case SV2_ACT_GELU: return run_norm<T, V, SV2_ACT_GELU>(p, images, slab, s, stream);
    case SV2_ACT_GELU_TANH: return run_norm<T, V, SV2_ACT_GELU_TANH>(p, images, slab, s, stream);
    default: return run_norm<T, V, SV2_ACT_NONE>(p, images, slab, s, stream);
    }
}

int check_sizes(int dtype, int images, int rows, int channels, int groups, const char* what)
{
    if ((dtype != SV2_F32 && dtype != SV2_F16 && dtype != SV2_BF16) || images < 0 || rows < 0 || channels <= 0 ||
        groups <= 0 || channels % groups != 0)
        return set_error(SV2_EINVAL, std::string(what) + ": bad type or sizes (channels must be a multiple of groups)");
    if (channels > kMaxChannels)
        return set_error(SV2_EUNSUPPORTED, std::string(what) + ": more than 8192 channels");
    return SV2_OK;
}

} // namespace
} // namespace sv2

extern "C" int64_t sv2_group_norm_workspace(int dtype, int images, int rows, int channels, int groups)
try
{
    using namespace sv2;
    const int rc = check_sizes(dtype, images, rows, channels, groups, "sv2_group_norm_workspace");
    if (rc != SV2_OK)
        return rc;
    if (images == 0 || rows == 0)
        return 0;
    NormArgs p{};
    p.rows = rows;
    p.channels = channels;
    p.groups = groups;
    p.width = channels / groups;
    const int bytes = dtype == SV2_F32 ? 4 : 2;
    // where even single elements fit the slab form, every layout does
    if (plan_slab(p, 1, bytes).threads > 0 && plan_slab(p, 16 / bytes, bytes).threads > 0)
        return 0;
    plan_rows(&p, images, bytes);
    return rows_workspace(p, images);
}
catch (...)
{
    return sv2::caught_exception("sv2_group_norm_workspace");
}

extern "C" int sv2_group_norm(const void* x, int64_t x_image_stride, int64_t x_row_stride, void* y,
                              int64_t y_image_stride, int64_t y_row_stride, int dtype, int images, int rows,
                              int channels, int groups, float eps, const float* gamma, const float* beta,
                              int activation, void* workspace, size_t workspace_bytes, void* stream)
try
{
    using namespace sv2;
    const int rc = check_sizes(dtype, images, rows, channels, groups, "sv2_group_norm");
    if (rc != SV2_OK)
        return rc;
    if (activation < SV2_ACT_NONE || activation > SV2_ACT_GELU_TANH || !(eps >= 0.f))
        return set_error(SV2_EINVAL, "sv2_group_norm: unknown activation or negative eps");
    if (images == 0 || rows == 0)
        return SV2_OK;
    const int bytes = dtype == SV2_F32 ? 4 : 2;
    if (!x || !y)
        return set_error(SV2_EINVAL, "sv2_group_norm: null pointer");
    if (misaligned(x, bytes) || misaligned(y, bytes) || misaligned(gamma, 4) || misaligned(beta, 4) ||
        misaligned(workspace, 8))
        return set_error(SV2_EINVAL, "sv2_group_norm: a pointer is not aligned to its elements");
    if (x_row_stride < channels || y_row_stride < channels ||
        (images > 1 && (x_image_stride < 0 || y_image_stride < channels)))
        return set_error(SV2_EINVAL, "sv2_group_norm: a stride below the channel count");
    if (x == y && ((rows > 1 && x_row_stride != y_row_stride) || (images > 1 && x_image_stride != y_image_stride)))
        return set_error(SV2_EINVAL, "sv2_group_norm: y is x with other strides");
    NormArgs p{};
    p.x = x;
    p.y = y;
    p.x_image = x_image_stride;
    p.x_row = x_row_stride;
    p.y_image = y_image_stride;
    p.y_row = y_row_stride;
    p.gamma = gamma;
    p.beta = beta;
    p.rows = rows;
    p.channels = channels;
    p.groups = groups;
    p.width = channels / groups;
    p.eps = eps;
    const int v = 16 / bytes;
    const bool one_image = images == 1; // its image strides are not read
    const bool wide = channels % v == 0 && x_row_stride % v == 0 && y_row_stride % v == 0 && !misaligned(x, 16) &&
                      !misaligned(y, 16) && (one_image || (x_image_stride % v == 0 && y_image_stride % v == 0));
    p.unit = 1;
    while (wide && p.unit < v && p.width % (2 * p.unit) == 0)
        p.unit *= 2;
    const Slab s = plan_slab(p, wide ? v : 1, bytes);
    const bool slab = s.threads > 0;
    if (!slab)
    {
        plan_rows(&p, images, bytes);
        if (!workspace || workspace_bytes < static_cast<size_t>(rows_workspace(p, images)))
            return set_error(SV2_EINVAL, "sv2_group_norm: workspace missing or too small");
        p.part = static_cast<float2*>(workspace);
        p.stat = p.part + static_cast<long long>(images) * groups * p.chunks;
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == SV2_F32)
        return wide ? run_act<vec::F32, 4>(p, images, activation, slab, s, st)
                    : run_act<vec::F32, 1>(p, images, activation, slab, s, st);
    if (dtype == SV2_F16)
        return wide ? run_act<vec::F16, 8>(p, images, activation, slab, s, st)
                    : run_act<vec::F16, 1>(p, images, activation, slab, s, st);
    return wide ? run_act<vec::BF16, 8>(p, images, activation, slab, s, st)
                : run_act<vec::BF16, 1>(p, images, activation, slab, s, st);
}
catch (...)
{
    return sv2::caught_exception("sv2_group_norm");
}
