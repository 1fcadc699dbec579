// Attention of a chunk of tokens over a cache, with a sliding window and first
// tokens that stay visible.
//
// Query i of a sequence with nq queries and nk cached keys stands at position
// p = nk - nq + i and sees key j where
//   j < nk,  j <= p + right,  j < sinks or j >= p - left.
//   o_i = sum_j w_ij v_j,  w_ij = exp(scale q_i k_j) / sum over the visible j
//
// One pass over the keys with a running maximum and sum (fp32), on
// v_mfma_f32_32x32x16 in both products:
//   S^T = K Q^T   32 keys x 32 queries: a lane holds 16 scores of one query, so
//                 the softmax is in-lane but for one exchange of half-waves;
//   O^T += V^T P^T  P^T leaves the scores' registers as the operand as it is:
//                 the order of the keys in the product's sum is free, and the
//                 values come from LDS by transposing reads in that order.
// P is rounded to the inputs' type (the matrix instruction takes no mixed
// types); the sum of the weights is of the unrounded ones.
//
// A query row here is a (position, head) pair: the heads that share a key head
// are packed into one tile of rows, position-major, so that a tile covers few
// positions (little of its window is masked) and its keys are read once for
// all of them.
//
// Tiles of keys outside every row's window are not visited.  A tile in which
// some row sees some key only is masked per element; there, values that are
// not finite are kept out of the product (0 * Inf would poison the rows that
// do not see them) and enter through products of indicators instead.
#include "sv2_internal.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace sv2
{
namespace
{

typedef __attribute__((ext_vector_type(8))) _Float16 h8;
typedef __attribute__((ext_vector_type(8))) __bf16 b8;
typedef __attribute__((ext_vector_type(16))) float f16v;
typedef __attribute__((ext_vector_type(4))) unsigned u4;
typedef __attribute__((ext_vector_type(2))) unsigned u2;

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct HalfIO
{
    static constexpr unsigned kExpMask = 0x7c007c00u; // exponent bits of a pair
    static constexpr unsigned kExpOne = 0x04000400u;  // the exponent's lowest bit
    static constexpr unsigned kOne = 0x3c00u;
    static __device__ f16v mfma(u4 a, u4 b, f16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    // nearest even
    static __device__ unsigned pack(float lo, float hi)
    {
        typedef __attribute__((ext_vector_type(2))) _Float16 h2;
        return __builtin_bit_cast(unsigned, h2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
    }
};
struct BfloatIO
{
    static constexpr unsigned kExpMask = 0x7f807f80u;
    static constexpr unsigned kExpOne = 0x00800080u;
    static constexpr unsigned kOne = 0x3f80u;
    static __device__ f16v mfma(u4 a, u4 b, f16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ unsigned pack(float lo, float hi)
    {
        typedef __attribute__((ext_vector_type(2))) __bf16 b2;
        return __builtin_bit_cast(unsigned, b2{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
    }
};

struct SlideParams
{
    const char* q;
    const char* k;
    const char* v;
    char* out;
    // strides in bytes
    long long q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h, o_b, o_t, o_h;
    const int32_t* q_lens;
    const int32_t* kv_lens;
    float* lse;
    float* part;    // splits > 1: sums [split][batch][heads][q_len][head_dim]
    float2* part_ml; // maxima (scaled, base 2) and sums of weights [split][batch][heads][q_len]
    float scale2;   // scale * log2(e)
    int batch, q_len, kv_len, heads, kv_heads, group;
    int left, right, sinks;
    int row_tiles, splits, blocks;
};

constexpr int kKeys = 64;      // keys of a tile
constexpr int kWaves = 4;
constexpr int kRows = 32 * kWaves; // query rows of a workgroup

__device__ inline int clamp_len(const int32_t* lens, int b, int most)
{
    return lens ? min(max(lens[b], 0), most) : most;
}

// 16 bytes per lane from global memory (uniform base + 32-bit lane offset)
// straight into LDS at lds + 16 * lane (lds wave-uniform, in M0; one wait
// state between the write of M0 and its use).  The compiler does not count
// these loads; the loop waits for them itself.
__device__ inline void dma16(const char* base, unsigned voff, unsigned lds)
{
    const unsigned long long b = reinterpret_cast<unsigned long long>(base);
    const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(b));
    const unsigned hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(b >> 32));
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(voff), "s"(static_cast<unsigned long long>(hi) << 32 | lo)
                 : "memory", "m0");
}

template <int N>
__device__ inline void wait_vm()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A workgroup barrier that waits for this wave's LDS reads, but not for the
// fetches in flight.
__device__ inline void bar()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The values of lanes l % 32 and l % 32 + 32, in the same order in both: from
// two copies of v one register ends up with the lower half-wave's values in
// every lane, the other with the upper's (with the wait states a VALU write
// needs before a permlane read).
__device__ inline void with_partner(float v, float* a, float* b)
{
    float x = v;
    float y = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x), "+v"(y));
    *a = x;
    *b = y;
}
__device__ inline float partner_max(float v)
{
    float a, b;
    with_partner(v, &a, &b);
    return fmaxf(a, b);
}
__device__ inline float partner_sum(float v)
{
    float a, b;
    with_partner(v, &a, &b);
    return a + b;
}

// Four keys of one dim: within each 16-lane group such a read hands lane i
// element i % 4 of the 8-byte pieces addressed by group lanes i / 4 + 4 j,
// j = 0..3; when group lane k addresses key row r0 + k / 4 at dims
// d0 + 4 (k % 4), lane i receives keys r0 .. r0 + 3 of dim d0 + i.
__device__ inline u2 keys4(const char* at)
{
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at)));
}

// The keys a tile of rows at positions p0 .. p1 visits: tiles of the first
// tokens, then those of the window.
struct KeyTiles
{
    int sink, start, count;
    __device__ int at(int i) const { return i < sink ? i : start + i - sink; }
};
__device__ inline KeyTiles key_tiles(const SlideParams& p, int nk, int p0, int p1)
{
    const int hi = min(nk, p1 + p.right + 1); // one past the last visible key
    KeyTiles t{0, 0, 0};
    if (hi <= 0)
        return t;
    const int lo = max(0, p0 - p.left);
    t.sink = (min(p.sinks, hi) + kKeys - 1) / kKeys;
    t.start = max(lo / kKeys, t.sink);
    t.count = t.sink + max(0, (hi + kKeys - 1) / kKeys - t.start);
    return t;
}

// LDS of one tile: keys, then values, rows of D elements.  16-byte chunk c of
// row r sits in slot c ^ key_swz(r) (the 16 rows that an operand read takes
// fall on different bank groups) or c ^ value_swz(r) (the four rows of a
// transposing read do).
template <int D>
__device__ inline unsigned key_swz(unsigned r)
{
    return D == 128 ? r & 15 : r & 7;
}
template <int D>
__device__ inline unsigned value_swz(unsigned r)
{
    return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
}

template <typename IO, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void slide_tile_kernel(SlideParams p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int kRowBytes = 2 * D;
    constexpr int kChunks = kRowBytes / 16;
    constexpr int kTileBytes = kKeys * kRowBytes;
    constexpr int kBuf = 2 * kTileBytes;
    constexpr int kSteps = D / 16;
    constexpr int kBlocks = D / 32;
    constexpr int kRowsPerDma = 64 / kChunks;
    constexpr int kDma = kKeys / kRowsPerDma / kWaves; // of each of K and V per wave

    // XCD x (workgroup id mod 8) takes a contiguous run of blocks: tiles of one
    // key head share an L2
    const int per = gridDim.x >> 3;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= p.blocks)
        return;
    const int tile = id % p.row_tiles;
    int rest = id / p.row_tiles;
    const int split = rest % p.splits;
    rest /= p.splits;
    const int kvh = rest % p.kv_heads;
    const int b = rest / p.kv_heads;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5;
    const int nq = __builtin_amdgcn_readfirstlane(clamp_len(p.q_lens, b, p.q_len));
    const int nk = __builtin_amdgcn_readfirstlane(clamp_len(p.kv_lens, b, p.kv_len));
    const int rows = nq * p.group;
    const int first = tile * kRows;
    if (first >= rows)
        return;
    const int off = nk - nq;
    const int p0 = off + first / p.group;
    const int p1 = off + (min(first + kRows, rows) - 1) / p.group;
    const KeyTiles kt = key_tiles(p, nk, p0, p1);
    const int share = (kt.count + p.splits - 1) / p.splits;
    const int t0 = min(split * share, kt.count);
    const int t1 = min(t0 + share, kt.count);

    const int row = first + wave * 32 + (lane & 31);
    const bool live = row < rows;
    const int rowc = min(row, rows - 1);
    const int qi = rowc / p.group;
    const int head = kvh * p.group + (rowc - qi * p.group);
    const int pos = off + qi;
    const int hi_key = min(pos + p.right, nk - 1);
    const int lo_key = pos - p.left;

    u4 q[kSteps];
    {
        const char* qr = p.q + b * p.q_b + qi * p.q_t + head * p.q_h + 16 * half;
#pragma unroll
        for (int s = 0; s < kSteps; s++)
            q[s] = *reinterpret_cast<const u4*>(qr + 32 * s);
    }

    const char* kb = p.k + b * p.k_b + kvh * p.k_h;
    const char* vb = p.v + b * p.v_b + kvh * p.v_h;
    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<size_t>(smem));
    const unsigned k_step = static_cast<unsigned>(p.k_t);
    const unsigned v_step = static_cast<unsigned>(p.v_t);
    auto fetch = [&](int t, int buf) {
        const int k0 = t * kKeys;
        const int last = nk - 1 - k0; // rows past the end repeat the last one
        const char* kp = kb + k0 * p.k_t;
        const char* vp = vb + k0 * p.v_t;
        const unsigned d = lds0 + buf * kBuf;
#pragma unroll
        for (int i = 0; i < kDma; i++)
        {
            const int r0 = (wave * kDma + i) * kRowsPerDma;
            const unsigned r = r0 + lane / kChunks;
            const unsigned c = lane % kChunks;
            const unsigned rr = min(static_cast<int>(r), last);
            dma16(kp, rr * k_step + ((c ^ key_swz<D>(r)) << 4), d + r0 * kRowBytes);
            dma16(vp, rr * v_step + ((c ^ value_swz<D>(r)) << 4), d + kTileBytes + r0 * kRowBytes);
        }
    };

    f16v o[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; i++)
#pragma unroll
        for (int e = 0; e < 16; e++)
            o[i][e] = 0.f;
    float m = kNegInf; // largest score so far, times scale2
    float l = 0.f;     // this half-wave's part of the sum of weights

    // operand reads
    const unsigned krow = lane & 31;
    unsigned koff[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; s++)
        koff[s] = krow * kRowBytes + (((2 * s + half) ^ key_swz<D>(krow)) << 4);
    // transposing reads: rows 4 half + (lane % 16) / 4 of a group of 8 keys,
    // dims 32 blk + 16 (lane / 16 % 2) + 4 (lane % 4)
    const unsigned vrow = 4 * half + ((lane & 15) >> 2);
    unsigned voff[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; i++)
    {
        const unsigned c = 4 * i + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        voff[i] = kTileBytes + vrow * kRowBytes + ((c ^ value_swz<D>(vrow)) << 4) + 8 * (lane & 1);
    }

    if (t0 < t1)
    {
        fetch(kt.at(t0), 0);
    }
    for (int t = t0; t < t1; t++)
    {
        const int buf = (t - t0) & 1;
        wait_vm<0>();
        bar(); // the tile is whole, and the other buffer's readers are done
        if (t + 1 < t1)
            fetch(kt.at(t + 1), buf ^ 1);
        const int k0 = kt.at(t) * kKeys;
        const char* st = smem + buf * kBuf;
        f16v s[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
        {
#pragma unroll
            for (int e = 0; e < 16; e++)
                s[i][e] = 0.f;
#pragma unroll
            for (int c = 0; c < kSteps; c++)
                s[i] = IO::mfma(*reinterpret_cast<const u4*>(st + i * 32 * kRowBytes + koff[c]), q[c], s[i]);
        }
        const bool masked = !(k0 + kKeys <= nk && k0 + kKeys - 1 <= p0 + p.right &&
                              (k0 + kKeys <= p.sinks || k0 >= p1 - p.left));
        auto key_of = [&](int i, int e) { return k0 + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3); };
        auto sees = [&](int j) { return j <= hi_key && (j < p.sinks || j >= lo_key); };
        if (masked)
        {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    s[i][e] = sees(key_of(i, e)) ? s[i][e] : kNegInf;
        }
        float top = kNegInf;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                top = fmaxf(top, s[i][e]);
        top = partner_max(top) * p.scale2;
        // the sums are rescaled only when some row's maximum rose
        if (__builtin_amdgcn_ballot_w64(top > m) != 0)
        {
            const float next = fmaxf(top, m);
            const float alpha = next == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    o[i][e] *= alpha;
        }
        const float base = m == kNegInf ? 0.f : m;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
            {
                s[i][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e], p.scale2, -base));
                l += s[i][e];
            }
        u4 w[4];
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                w[c][e] = IO::pack(s[c >> 1][8 * (c & 1) + 2 * e], s[c >> 1][8 * (c & 1) + 2 * e + 1]);
#pragma unroll
        for (int i = 0; i < kBlocks; i++)
        {
            u4 a[4];
#pragma unroll
            for (int c = 0; c < 4; c++)
            {
                const u2 lo = keys4(st + voff[i] + 16 * c * kRowBytes);
                const u2 hi = keys4(st + voff[i] + (16 * c + 8) * kRowBytes);
                a[c] = u4{lo.x, lo.y, hi.x, hi.y};
            }
            if (masked)
            {
                unsigned bad = 0;
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        bad |= (a[c][e] & IO::kExpMask) + IO::kExpOne;
                if (__builtin_amdgcn_ballot_w64((bad & 0x80008000u) != 0) != 0)
                {
                    // the sums of visible values that are +Inf, -Inf or NaN,
                    // by counting them
                    u4 vis[4];
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                        {
                            const int at = 8 * (c & 1) + 2 * e;
                            vis[c][e] = (sees(key_of(c >> 1, at)) ? IO::kOne : 0u) |
                                        (sees(key_of(c >> 1, at + 1)) ? IO::kOne << 16 : 0u);
                        }
                    const unsigned inf = IO::kExpMask & 0xffffu;
#pragma unroll
                    for (int kind = 0; kind < 3; kind++)
                    {
                        f16v n;
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            n[e] = 0.f;
#pragma unroll
                        for (int c = 0; c < 4; c++)
                        {
                            u4 is;
#pragma unroll
                            for (int e = 0; e < 4; e++)
                            {
                                auto flag = [&](unsigned x) {
                                    const bool hit = kind == 0   ? x == inf
                                                     : kind == 1 ? x == (inf | 0x8000u)
                                                                 : (x & 0x7fffu) > inf;
                                    return hit ? IO::kOne : 0u;
                                };
                                is[e] = flag(a[c][e] & 0xffffu) | flag(a[c][e] >> 16) << 16;
                            }
                            n = IO::mfma(is, vis[c], n);
                        }
                        const float add = kind == 0 ? -kNegInf : kind == 1 ? kNegInf : __builtin_nanf("");
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            o[i][e] = n[e] > 0.f ? o[i][e] + add : o[i][e];
                    }
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                        {
                            unsigned x = a[c][e];
                            x = (x & inf) == inf ? x & 0xffff0000u : x;
                            x = (x >> 16 & inf) == inf ? x & 0xffffu : x;
                            a[c][e] = x;
                        }
                }
            }
#pragma unroll
            for (int c = 0; c < 4; c++)
                o[i] = IO::mfma(a[c], w[c], o[i]);
        }
    }

    l = partner_sum(l);
    if (!live)
        return;
    const long long at = (static_cast<long long>(b) * p.heads + head) * p.q_len + qi;
    if (p.splits > 1)
    {
        const long long to = static_cast<long long>(split) * p.batch * p.heads * p.q_len + at;
        float* dst = p.part + to * D + 4 * half;
#pragma unroll
        for (int i = 0; i < kBlocks; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                *reinterpret_cast<float4*>(dst + 32 * i + 8 * e) =
                    make_float4(o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]);
        if (half == 0)
            p.part_ml[to] = make_float2(m, l);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    char* dst = p.out + b * p.o_b + qi * p.o_t + head * p.o_h + 8 * half;
#pragma unroll
    for (int i = 0; i < kBlocks; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            *reinterpret_cast<u2*>(dst + 64 * i + 16 * e) =
                u2{IO::pack(o[i][4 * e] * inv, o[i][4 * e + 1] * inv), IO::pack(o[i][4 * e + 2] * inv, o[i][4 * e + 3] * inv)};
    if (p.lse && half == 0)
        p.lse[at] = l == 0.f ? kNegInf : m * kLn2 + logf(l);
}

// Joins the splits of one query row: one wave per row.
template <typename IO, int D>
__global__ __launch_bounds__(256) void slide_join_kernel(SlideParams p)
{
    const int lane = threadIdx.x & 63;
    const long long rows = static_cast<long long>(p.batch) * p.heads * p.q_len;
    const long long at = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (at >= rows)
        return;
    const int qi = static_cast<int>(at % p.q_len);
    const long long bh = at / p.q_len;
    const int head = static_cast<int>(bh % p.heads);
    const int b = static_cast<int>(bh / p.heads);
    if (qi >= clamp_len(p.q_lens, b, p.q_len))
        return;
    float m = kNegInf;
    for (int s = 0; s < p.splits; s++)
        m = fmaxf(m, p.part_ml[s * rows + at].x);
    const float base = m == kNegInf ? 0.f : m;
    float l = 0.f;
    constexpr int kPer = D / 64;
    float o[kPer];
#pragma unroll
    for (int e = 0; e < kPer; e++)
        o[e] = 0.f;
    for (int s = 0; s < p.splits; s++)
    {
        const float2 ml = p.part_ml[s * rows + at];
        if (ml.y == 0.f)
            continue; // no visible key in this split
        const float a = __builtin_amdgcn_exp2f(ml.x - base);
        l += a * ml.y;
        const float* src = p.part + (s * rows + at) * D + kPer * lane;
#pragma unroll
        for (int e = 0; e < kPer; e++)
            o[e] += a * src[e];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    char* dst = p.out + b * p.o_b + qi * p.o_t + head * p.o_h + 2 * kPer * lane;
    if constexpr (kPer == 2)
        *reinterpret_cast<unsigned*>(dst) = IO::pack(o[0] * inv, o[1] * inv);
    else
        *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(IO::pack(o[0] * inv, 0.f));
    if (p.lse && lane == 0)
        p.lse[at] = l == 0.f ? kNegInf : m * kLn2 + logf(l);
}

// Splits of the keys where the row tiles alone leave CUs without work: two
// workgroups a CU at most, two tiles of keys each at least.
int plan_splits(const SlideParams& p, long long tiles)
{
    const long long positions = std::min<long long>(p.q_len, (kRows + p.group - 1) / p.group + 1);
    const long long span = std::min<long long>(p.kv_len, static_cast<long long>(p.sinks) + p.left + p.right + positions + kKeys);
    const long long keys = (span + kKeys - 1) / kKeys;
    const long long want = 512 / std::max(1LL, tiles);
    return static_cast<int>(std::max(1LL, std::min(want, keys / 2)));
}

long long part_rows(const SlideParams& p)
{
    return static_cast<long long>(p.splits) * p.batch * p.heads * p.q_len;
}

int make_params(const sv2_sliding_attn_args* a, const char* what, SlideParams* out)
{
    auto bad = [&](const char* why) { return set_error(SV2_EINVAL, std::string(what) + ": " + why); };
    if (!a)
        return bad("null arguments");
    if (a->batch < 0 || a->q_len < 0 || a->kv_len < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads != 0)
        return bad("negative sizes, or heads not a multiple of kv_heads");
    if (a->left < 0 || a->right < 0 || a->sinks < 0)
        return bad("left, right and sinks must not be negative");
    if (!(a->scale > 0.f) || !std::isfinite(a->scale))
        return bad("scale must be positive and finite");
    if (a->dtype != SV2_F16 && a->dtype != SV2_BF16)
        return set_error(a->dtype == SV2_F32 ? SV2_EUNSUPPORTED : SV2_EINVAL, std::string(what) + ": dtype must be SV2_F16 or SV2_BF16");
    if (a->head_dim != 64 && a->head_dim != 128)
        return set_error(SV2_EUNSUPPORTED, std::string(what) + ": head_dim must be 64 or 128");
    constexpr int kMost = 1 << 30;
    if (a->q_len > kMost / a->heads || a->kv_len > kMost)
        return set_error(SV2_EUNSUPPORTED, std::string(what) + ": more than 2^30 query rows or keys");
    SlideParams p{};
    p.batch = a->batch;
    p.q_len = a->q_len;
    p.kv_len = a->kv_len;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    // a reach past 2^30 sees the same keys
    p.left = std::min(a->left, kMost);
    p.right = std::min(a->right, kMost - 1);
    p.sinks = std::min(a->sinks, kMost);
    p.scale2 = a->scale * kLog2e;
    const long long rows = static_cast<long long>(p.q_len) * p.group;
    p.row_tiles = static_cast<int>((rows + kRows - 1) / kRows);
    const long long tiles = static_cast<long long>(p.row_tiles) * p.kv_heads * p.batch;
    p.splits = plan_splits(p, tiles);
    if (tiles * p.splits > INT_MAX - 8)
        return set_error(SV2_EUNSUPPORTED, std::string(what) + ": too many tiles");
    p.blocks = static_cast<int>(tiles * p.splits);
    *out = p;
    return SV2_OK;
}

long long workspace_of(const SlideParams& p, int head_dim)
{
    return p.splits > 1 ? part_rows(p) * (head_dim + 2) * 4 : 0;
}

template <typename IO, int D>
int run_slide(const SlideParams& p, hipStream_t stream)
{
    constexpr int kLds = 2 * 2 * kKeys * 2 * D;
    const int rc = set_dynamic_lds(reinterpret_cast<const void*>(&slide_tile_kernel<IO, D>), kLds, "slide_tile: dynamic LDS attribute");
    if (rc != SV2_OK)
        return rc;
    const unsigned grid = (static_cast<unsigned>(p.blocks) + 7) / 8 * 8;
    hipLaunchKernelGGL((slide_tile_kernel<IO, D>), dim3(grid), dim3(64 * kWaves), kLds, stream, p);
    if (p.splits > 1)
    {
        const long long rows = static_cast<long long>(p.batch) * p.heads * p.q_len;
        hipLaunchKernelGGL((slide_join_kernel<IO, D>), dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, stream, p);
    }
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? SV2_OK : hip_error(err, "sv2_sliding_attention launch");
}

} // namespace
} // namespace sv2

extern "C" int64_t sv2_sliding_attention_workspace(const sv2_sliding_attn_args* args)
try
{
    sv2::SlideParams p;
    const int rc = sv2::make_params(args, "sv2_sliding_attention_workspace", &p);
    return rc != SV2_OK ? rc : sv2::workspace_of(p, args->head_dim);
}
catch (...)
{
    return sv2::caught_exception("sv2_sliding_attention_workspace");
}

extern "C" int sv2_sliding_attention(const sv2_sliding_attn_args* args, void* stream)
try
{
    using namespace sv2;
    SlideParams p;
    const int rc = make_params(args, "sv2_sliding_attention", &p);
    if (rc != SV2_OK)
        return rc;
    if (p.batch == 0 || p.q_len == 0)
        return SV2_OK;
    const sv2_sliding_attn_args& a = *args;
    if (!a.q || !a.out || (p.kv_len > 0 && (!a.k || !a.v)))
        return set_error(SV2_EINVAL, "sv2_sliding_attention: null pointer");
    if (misaligned(a.q, 16) || misaligned(a.k, 16) || misaligned(a.v, 16) || misaligned(a.out, 16) ||
        misaligned(a.q_lens, 4) || misaligned(a.kv_lens, 4) || misaligned(a.lse, 4))
        return set_error(SV2_EINVAL, "sv2_sliding_attention: q, k, v and out must be 16-byte aligned, the rest 4-byte");
    const int64_t strides[12] = {a.q_batch_stride, a.q_token_stride, a.q_head_stride, a.k_batch_stride, a.k_token_stride,
                                 a.k_head_stride, a.v_batch_stride, a.v_token_stride, a.v_head_stride,
                                 a.out_batch_stride, a.out_token_stride, a.out_head_stride};
    for (int64_t s : strides)
        if (s < 0 || s % 8 != 0 || s > INT64_MAX / 4)
            return set_error(SV2_EINVAL, "sv2_sliding_attention: strides must be non-negative multiples of 8 elements");
    // a tile's rows are addressed by 32-bit offsets from its first
    constexpr int64_t kMostStride = INT32_MAX / (2 * kKeys) - 256;
    if (a.k_token_stride > kMostStride || a.v_token_stride > kMostStride)
        return set_error(SV2_EUNSUPPORTED, "sv2_sliding_attention: token stride of k or v above 2^24 elements");
    const long long need = workspace_of(p, a.head_dim);
    if (need > 0 && (!a.workspace || a.workspace_bytes < static_cast<size_t>(need) || misaligned(a.workspace, 16)))
        return set_error(SV2_EINVAL, "sv2_sliding_attention: workspace missing, too small or not 16-byte aligned");
    p.q = static_cast<const char*>(a.q);
    p.k = static_cast<const char*>(a.k);
    p.v = static_cast<const char*>(a.v);
    p.out = static_cast<char*>(a.out);
    long long* const to[12] = {&p.q_b, &p.q_t, &p.q_h, &p.k_b, &p.k_t, &p.k_h, &p.v_b, &p.v_t, &p.v_h, &p.o_b, &p.o_t, &p.o_h};
    for (int i = 0; i < 12; i++)
        *to[i] = 2 * strides[i];
    p.q_lens = a.q_lens;
    p.kv_lens = a.kv_lens;
    p.lse = a.lse;
    p.part = static_cast<float*>(a.workspace);
    if (need > 0)
        p.part_ml = reinterpret_cast<float2*>(p.part + part_rows(p) * a.head_dim);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.dtype == SV2_F16)
        return a.head_dim == 128 ? run_slide<HalfIO, 128>(p, st) : run_slide<HalfIO, 64>(p, st);
    return a.head_dim == 128 ? run_slide<BfloatIO, 128>(p, st) : run_slide<BfloatIO, 64>(p, st);
}
catch (...)
{
    return sv2::caught_exception("sv2_sliding_attention");
}
