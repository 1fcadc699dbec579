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
// types), which adds as much to the output's error as its own rounding does;
// the sum of the weights is of the unrounded ones.  Where the cache's bytes
// are the bound (the few form) P goes in as two such numbers, the second the
// first one's rounding error: its products cost nothing there.  In the tile
// form they cost 274 us for 215 at the prompt below, 39.5 for 33.5 at 480 new
// tokens and 27.7 for 22.5 at head size 64, for an error against float64 of 1.0
// times the output's own rounding in place of 1.35: the caller's choice there,
// one term unless it asks for two.
//
// A query row here is a (position, head) pair: the heads that share a key head
// are packed into one tile of rows, position-major, so that a tile covers few
// positions (little of its window is masked) and its keys are read once for
// all of them.
//
// Tiles of keys outside every row's window are not visited.  A tile in which
// some row sees some key only is masked per element; there, values that are
// not finite are kept out of the product (0 * Inf would poison the rows that
// do not see them).  A value that is not finite is the sum of the rows that see
// it, whatever its weight: where the tiles held one (or the sums show one), a
// second walk over the tiles counts them by products of indicators (with one such
// key the prompt below takes 268 us for 214).
//
// Forms, by the rows (heads of a key head x positions):
//   few   up to 32 rows (single tokens): a stream of the cache, one row tile a
//         wave, the keys split over waves and workgroups.  Bound by the cache's
//         bytes: sixteen tokens over 16 ragged caches, 227 MB of bf16 keys and
//         values, 52 us (4.4 TB/s, two sets in turn; a large copy reaches 4.9),
//         4.6 more to join the splits.
//   tile  more rows: 128 of them a workgroup.  A tile of 64 keys is 32 matrix
//         instructions a wave (1024 cycles) and about 220 vector ones beside
//         its LDS reads; the two waves of a SIMD overlap them in part only
//         (matrix unit 37% busy, vector unit 42%; 35% of a wave's time waiting
//         to issue).  8250 tokens, window 2048, 20 heads
//         of 128, bf16: 214 us, 0.72 PFLOP/s; 480 new tokens over 2400 of a
//         cache 34 us, of which 27 this kernel.
//         Tried and slower for that prompt: both products and the softmax of
//         three successive tiles interleaved in one stream (235 us beside 208;
//         64 rows a wave 392), eight waves in two groups a phase apart (257), wave
//         priorities (208 either way), the first rows last (215).
//   join  where the keys were split: sums of a row in one team of lanes each.
#include "sv2_internal.h"

#include <algorithm>
#include <climits>
#include <cmath>

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
    static __device__ float to_float(unsigned bits)
    {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
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
    static __device__ float to_float(unsigned bits) { return __builtin_bit_cast(float, bits << 16); }
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
    float2* part_ml; // maxima (unscaled) and sums of weights [split][batch][heads][q_len]
    float scale, scale2; // scale2 = scale * log2(e)
    int batch, q_len, kv_len, heads, kv_heads, group;
    int left, right, sinks;
    int few, row_tiles, splits, blocks;
    int terms; // of a weight in the tile form
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

// sum * a, a >= 0 finite; a sum that is not finite stays as it is (a weight
// too small for fp32 would make a NaN of an infinity).
__device__ inline float rescaled(float sum, float a)
{
    const float x = sum * a;
    return x == x ? x : sum;
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

// The keys that rows at positions p0 .. p1 visit, in tiles of KEYS: those of
// the first tokens, then those of the window.
template <int KEYS>
struct KeyTiles
{
    int sink, start, count;
    __device__ KeyTiles(const SlideParams& p, int nk, int p0, int p1) : sink(0), start(0), count(0)
    {
        const int hi = min(nk, p1 + p.right + 1); // one past the last visible key
        if (hi <= 0)
            return;
        sink = (min(p.sinks, hi) + KEYS - 1) / KEYS;
        start = max(max(0, p0 - p.left) / KEYS, sink);
        count = sink + max(0, (hi + KEYS - 1) / KEYS - start);
    }
    // first key of tile i
    __device__ int key(int i) const { return (i < sink ? i : start + i - sink) * KEYS; }
};

// LDS tiles of keys and values: rows of D elements, 16-byte chunk c of row r
// in slot c ^ key_swz(r) (the 16 rows that an operand read takes fall on
// different bank groups) or c ^ value_swz(r) (the four rows of a transposing
// read do).
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

// Largest rise of a row's maximum, in powers of two, that its weights absorb:
// up to 2^8, far inside both types.
constexpr float kRise = 8.f;

// Scores (times scale2) up to here are brought down to the maximum by one
// fused product: its rounding of the maximum moves a row's weights by 2^-16 of
// themselves at most.  Larger ones (whose rounding would take the weights out
// of their type's range in the end) by a difference first.
constexpr float kFar = 256.f;

// 32 query rows in one wave: lane % 32 is the row (its two half-waves hold
// different keys of the scores and different dims of the sums).
template <typename IO, int D>
struct Rows
{
    static constexpr int kRowBytes = 2 * D;
    static constexpr int kSteps = D / 16;
    static constexpr int kBlocks = D / 32;
    static constexpr unsigned kInf = IO::kExpMask & 0xffffu;

    u4 q[kSteps];
    f16v o[kBlocks]; // sums, dims 32 i + 8 (e / 4) + 4 half + e % 4
    float m;         // the largest score in use, unscaled
    bool far;        // some row's largest score is past kFar (wave-uniform)
    bool found;      // a masked tile held a value that is not finite (wave-uniform)
    float l;         // this half-wave's part of the sum of weights
    int half, qi, head, hi_key, lo_key, sinks;
    float scale2;
    unsigned koff[kSteps], voff[kBlocks];

    // row `row` (a packed one, clamped by the caller) of key head kvh, the
    // sequence's first query at position `off`
    __device__ void init(const SlideParams& p, int b, int kvh, int row, int off, int nk, int lane)
    {
        half = lane >> 5;
        qi = row / p.group;
        head = kvh * p.group + (row - qi * p.group);
        hi_key = min(off + qi + p.right, nk - 1);
        lo_key = off + qi - p.left;
        sinks = p.sinks;
        scale2 = p.scale2;
        const char* qr = p.q + b * p.q_b + qi * p.q_t + head * p.q_h + 16 * half;
#pragma unroll
        for (int c = 0; c < kSteps; c++)
            q[c] = *reinterpret_cast<const u4*>(qr + 32 * c);
#pragma unroll
        for (int i = 0; i < kBlocks; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                o[i][e] = 0.f;
        m = kNegInf;
        far = false;
        found = false;
        l = 0.f;
        const unsigned krow = lane & 31;
#pragma unroll
        for (int c = 0; c < kSteps; c++)
            koff[c] = krow * kRowBytes + (((2 * c + half) ^ key_swz<D>(krow)) << 4);
        // transposing reads: rows 4 half + (lane % 16) / 4 of a group of 8 keys,
        // dims 32 i + 16 (lane / 16 % 2) + 4 (lane % 4)
        const unsigned vrow = 4 * half + ((lane & 15) >> 2);
#pragma unroll
        for (int i = 0; i < kBlocks; i++)
        {
            const unsigned c = 4 * i + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            voff[i] = vrow * kRowBytes + ((c ^ value_swz<D>(vrow)) << 4) + 8 * (lane & 1);
        }
    }
    // key of score e of key block i of a tile from key k0 on
    __device__ int key_of(int k0, int i, int e) const { return k0 + 4 * half + 32 * i + 8 * (e >> 2) + (e & 3); }
    __device__ bool sees(int j) const { return (j <= hi_key) & ((j < sinks) | (j >= lo_key)); }

    template <int NB>
    __device__ void scores(f16v (&s)[NB], const char* keys) const
    {
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                s[i][e] = 0.f;
        // the blocks in turn (a product that waits for the one before it costs
        // the matrix unit its latency), operands read kAhead products ahead: the
        // compiler, left to itself, reads each where it is used
        constexpr int kAhead = 3;
        constexpr int kAll = NB * kSteps;
        u4 a[kAhead + 1];
        auto read = [&](int j) {
            a[j % (kAhead + 1)] = *reinterpret_cast<const u4*>(keys + (j % NB) * 32 * kRowBytes + koff[j / NB]);
        };
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            read(j);
#pragma unroll
        for (int j = 0; j < kAll; j++)
        {
            if (j + kAhead < kAll)
                read(j + kAhead);
            s[j % NB] = IO::mfma(a[j % (kAhead + 1)], q[j / NB], s[j % NB]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    template <int NB>
    __device__ void mask(f16v (&s)[NB], int k0) const
    {
        if (k0 >= sinks)
        {
            // lo_key <= j <= hi_key in one comparison (hi_key < lo_key: nothing)
            const bool any = hi_key >= lo_key;
            const unsigned range = any ? static_cast<unsigned>(hi_key) - static_cast<unsigned>(lo_key) : 0u;
            const unsigned d = any ? static_cast<unsigned>(key_of(k0, 0, 0)) - static_cast<unsigned>(lo_key) : 1u << 30;
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    s[i][e] = d + (32u * i + 8u * (e >> 2) + (e & 3)) <= range ? s[i][e] : kNegInf;
            return;
        }
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                s[i][e] = sees(key_of(k0, i, e)) ? s[i][e] : kNegInf;
    }
    // scores to weights exp2((s - m) scale2), rounded for the product.  m is the
    // largest score but for a rise of up to kRise that the weights absorb; the
    // sums are rescaled when some row's maximum rises further (of 32 rows one
    // finds a larger score in nearly every tile: rescaling for each costs a
    // quarter of the vector work)
    template <int NB>
    __device__ void weights(f16v (&s)[NB], u4 (&w)[2 * NB])
    {
        float top = kNegInf;
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                top = fmaxf(top, s[i][e]);
        top = partner_max(top);
        if (__builtin_amdgcn_ballot_w64((top - m) * scale2 > kRise) != 0)
        {
            const float next = fmaxf(top, m);
            const float alpha = next == kNegInf ? 1.f : __builtin_amdgcn_exp2f((m - next) * scale2);
            m = next;
            far = __builtin_amdgcn_ballot_w64(m != kNegInf && fabsf(m * scale2) > kFar) != 0;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    o[i][e] *= alpha;
        }
        float base = m == kNegInf ? 0.f : m;
        if (__builtin_expect(far, 0))
        {
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    s[i][e] -= base;
            base = 0.f;
        }
        base *= scale2;
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
            {
                s[i][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e], scale2, -base));
                l += s[i][e];
            }
#pragma unroll
        for (int c = 0; c < 2 * NB; c++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                w[c][e] = IO::pack(s[c >> 1][8 * (c & 1) + 2 * e], s[c >> 1][8 * (c & 1) + 2 * e + 1]);
    }
    // what the rounded weights lack: their second terms
    template <int NB>
    static __device__ void rounding_of(const f16v (&s)[NB], const u4 (&w)[2 * NB], u4 (&rest)[2 * NB])
    {
#pragma unroll
        for (int c = 0; c < 2 * NB; c++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                rest[c][e] = IO::pack(s[c >> 1][8 * (c & 1) + 2 * e] - IO::to_float(w[c][e] & 0xffffu),
                                      s[c >> 1][8 * (c & 1) + 2 * e + 1] - IO::to_float(w[c][e] >> 16));
    }
    // values of keys 16 c .. 16 c + 15 of a tile, dims 32 i on
    __device__ u4 values(const char* vals, int i, int c) const
    {
        const u2 lo = keys4(vals + voff[i] + 16 * c * kRowBytes);
        const u2 hi = keys4(vals + voff[i] + (16 * c + 8) * kRowBytes);
        return u4{lo.x, lo.y, hi.x, hi.y};
    }
    // the operands of 16 keys from 16 c on
    __device__ void read_values(u4 (&a)[kBlocks], const char* vals, int c) const
    {
#pragma unroll
        for (int i = 0; i < kBlocks; i++)
            a[i] = values(vals, i, c);
    }
    // Whether an operand holds a value that is not finite: bit 15 or 31 set.
    static __device__ unsigned bad_bits(u4 a)
    {
        unsigned bad = 0;
#pragma unroll
        for (int e = 0; e < 4; e++)
            bad |= (a[e] & IO::kExpMask) + IO::kExpOne;
        return bad & 0x80008000u;
    }
    // sums += weights values (`first`: the operands of the first 16 keys;
    // `rest`: what the weights lack, if given); in a masked tile values that are
    // not finite stay out of the product
    template <int NB>
    __device__ void add(const u4 (&w)[2 * NB], u4 (&first)[kBlocks], const char* vals, bool masked,
                        const u4* rest = nullptr)
    {
        u4 next[kBlocks];
#pragma unroll
        for (int c = 0; c < 2 * NB; c++)
        {
            u4(&a)[kBlocks] = c & 1 ? next : first;
            if (c + 1 < 2 * NB)
                read_values(c & 1 ? first : next, vals, c + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (masked)
            {
                unsigned bad = 0;
#pragma unroll
                for (int i = 0; i < kBlocks; i++)
                    bad |= bad_bits(a[i]);
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad != 0) != 0, 0))
                {
                    found = true;
#pragma unroll
                    for (int i = 0; i < kBlocks; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                        {
                            const unsigned x = a[i][e];
                            a[i][e] = ((x & kInf) == kInf ? 0u : x & 0xffffu) |
                                      ((x >> 16 & kInf) == kInf ? 0u : x & 0xffff0000u);
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
                o[i] = IO::mfma(a[i], w[c], o[i]);
            if (rest)
#pragma unroll
                for (int i = 0; i < kBlocks; i++)
                    o[i] = IO::mfma(a[i], rest[c], o[i]);
        }
    }
    // Whether some value was not finite (wave-uniform): a masked tile held one,
    // or a sum is not, in a row whose weights are.
    __device__ bool odd() const
    {
        float t[4] = {0.f, 0.f, 0.f, 0.f}; // 0 or NaN
#pragma unroll
        for (int i = 0; i < kBlocks; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                t[e & 3] = __builtin_fmaf(o[i][e], 0.f, t[e & 3]);
        const float any = (t[0] + t[1]) + (t[2] + t[3]);
        return found || __builtin_amdgcn_ballot_w64(any != any && l == l) != 0;
    }
    // The values of a tile from key k0 on that are +Inf, -Inf or NaN, counted
    // per row that sees them by products of indicators: they are the sums of
    // those rows, whatever the weights (`given`, a bit a sum: one was there
    // before).  A product with the weights makes a NaN of an infinity where a
    // weight, or the second term of one, is 0 in 16 bits.
    template <int NB>
    __device__ void count(unsigned (&given)[kBlocks], const char* vals, int k0)
    {
        for (int c = 0; c < 2 * NB; c++)
        {
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
            {
                const u4 a = values(vals, i, c);
                if (__builtin_amdgcn_ballot_w64(bad_bits(a) != 0) != 0)
                    count_odd(a, key_of(k0, c >> 1, 8 * (c & 1)), o[i], given[i]);
            }
        }
    }
    // of one operand: 16 keys, this lane's from `first` on
    __device__ void count_odd(u4 a, int first, f16v& sum, unsigned& given) const
    {
#pragma nounroll
        for (int kind = 0; kind < 3; kind++)
        {
            const unsigned want = kind == 0 ? kInf : kInf | 0x8000u;
            auto flag = [&](unsigned x) {
                const unsigned hit = kind < 2 ? x == want : (x & 0x7fffu) > kInf;
                return hit ? IO::kOne : 0u;
            };
            u4 is, vis;
#pragma unroll
            for (int e = 0; e < 4; e++)
            {
                const int j = first + 8 * (e >> 1) + 2 * (e & 1);
                is[e] = flag(a[e] & 0xffffu) | flag(a[e] >> 16) << 16;
                vis[e] = (sees(j) ? IO::kOne : 0u) | (sees(j + 1) ? IO::kOne << 16 : 0u);
            }
            f16v n;
#pragma unroll
            for (int e = 0; e < 16; e++)
                n[e] = 0.f;
            n = IO::mfma(is, vis, n);
            const float extra = kind == 0 ? -kNegInf : kind == 1 ? kNegInf : __builtin_nanf("");
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (n[e] > 0.f)
                {
                    sum[e] = given >> e & 1 ? sum[e] + extra : extra;
                    given |= 1u << e;
                }
        }
    }
};

// Whether rows at positions p0 .. p1 do not all see all of n keys from k0 on.
__device__ inline bool is_masked(const SlideParams& p, int nk, int p0, int p1, int k0, int n)
{
    return !(k0 + n <= nk && k0 + n - 1 <= p0 + p.right && (k0 + n <= p.sinks || k0 >= p1 - p.left));
}

// What a workgroup works on: XCD x (workgroup id mod 8) takes a contiguous run
// of blocks, so that tiles of one key head share an L2.
struct Place
{
    int tile, split, kvh, b, nq, nk, rows, off;
    bool none;
    __device__ explicit Place(const SlideParams& p, int tile_rows)
    {
        const int id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
        none = id >= p.blocks;
        tile = id % p.row_tiles;
        int rest = id / p.row_tiles;
        split = rest % p.splits;
        rest /= p.splits;
        kvh = rest % p.kv_heads;
        b = none ? 0 : rest / p.kv_heads;
        nq = __builtin_amdgcn_readfirstlane(clamp_len(p.q_lens, b, p.q_len));
        nk = __builtin_amdgcn_readfirstlane(clamp_len(p.kv_lens, b, p.kv_len));
        rows = nq * p.group;
        off = nk - nq;
        none = none || tile * tile_rows >= rows;
    }
};

// Tile form: 128 rows by four waves of 32, tiles of 64 keys in two LDS
// buffers, the next one on its way while one is worked on; one barrier a tile.
// GROUPS = 2, for launches that give a CU one workgroup at most: a second
// group of four waves takes every other tile for the same rows, and its sums
// are joined to the first's in LDS.
// TERMS: 16-bit numbers that a weight goes into the product as.
template <typename IO, int D, int GROUPS, int TERMS>
__global__ __launch_bounds__(64 * kWaves * GROUPS, 2) void slide_tile_kernel(SlideParams p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int kRowBytes = 2 * D;
    constexpr int kChunks = kRowBytes / 16;
    constexpr int kTileBytes = kKeys * kRowBytes;
    constexpr int kBuf = 2 * kTileBytes;
    constexpr int kBlocks = D / 32;
    constexpr int kRowsPerDma = 64 / kChunks;
    constexpr int kDma = kKeys / kRowsPerDma / kWaves; // of each of K and V per wave

    const Place at(p, kRows);
    if (at.none)
        return;
    const int first = at.tile * kRows;
    const int p0 = at.off + first / p.group;
    const int p1 = at.off + (min(first + kRows, at.rows) - 1) / p.group;
    const KeyTiles<kKeys> kt(p, at.nk, p0, p1);
    const int share = (kt.count + p.splits - 1) / p.splits;
    const int t0 = min(at.split * share, kt.count);
    const int nt = min(share, kt.count - t0);
    const int steps = (nt + GROUPS - 1) / GROUPS; // of every group; its last may be empty

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kWaves;
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / kWaves;
    const int row = first + wave * 32 + (lane & 31);
    Rows<IO, D> r;
    r.init(p, at.b, at.kvh, min(row, at.rows - 1), at.off, at.nk, lane);

    const char* kb = p.k + at.b * p.k_b + at.kvh * p.k_h;
    const char* vb = p.v + at.b * p.v_b + at.kvh * p.v_h;
    char* const mine = smem + group * 2 * kBuf;
    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<size_t>(mine));
    const unsigned k_step = static_cast<unsigned>(p.k_t);
    const unsigned v_step = static_cast<unsigned>(p.v_t);
    auto fetch = [&](int i) {
        const int t = GROUPS * i + group;
        if (t >= nt)
            return;
        const int k0 = kt.key(t0 + t);
        const int last = at.nk - 1 - k0; // rows past the end repeat the last one
        const char* kp = kb + k0 * p.k_t;
        const char* vp = vb + k0 * p.v_t;
        const unsigned d = lds0 + (i & 1) * kBuf;
#pragma unroll
        for (int j = 0; j < kDma; j++)
        {
            const int r0 = (wave * kDma + j) * kRowsPerDma;
            const unsigned r = r0 + lane / kChunks;
            const unsigned c = lane % kChunks;
            const unsigned rr = min(static_cast<int>(r), last);
            dma16(kp, rr * k_step + ((c ^ key_swz<D>(r)) << 4), d + r0 * kRowBytes);
            dma16(vp, rr * v_step + ((c ^ value_swz<D>(r)) << 4), d + kTileBytes + r0 * kRowBytes);
        }
    };
    fetch(0);
    for (int i = 0; i < steps; i++)
    {
        wait_vm<0>();
        bar(); // the tile is whole, and the other buffer's readers are done
        fetch(i + 1);
        const int t = GROUPS * i + group;
        if (GROUPS > 1 && t >= nt)
            continue;
        const int k0 = kt.key(t0 + t);
        const char* st = mine + (i & 1) * kBuf;
        const bool masked = is_masked(p, at.nk, p0, p1, k0, kKeys);
        f16v s[2];
        u4 w[4];
        r.template scores<2>(s, st);
        if (masked)
            r.template mask<2>(s, k0);
        u4 v0[Rows<IO, D>::kBlocks];
        r.read_values(v0, st + kTileBytes, 0);
        r.template weights<2>(s, w);
        if constexpr (TERMS == 2)
        {
            u4 rest[4];
            r.template rounding_of<2>(s, w, rest);
            r.template add<2>(w, v0, st + kTileBytes, masked, rest);
        }
        else
            r.template add<2>(w, v0, st + kTileBytes, masked);
    }
    bool again;
    {
        // where some wave met a value that is not finite, all go over the tiles
        // again for these (the votes go through the buffers: their readers are
        // done after the first barrier)
        const bool odd = r.odd();
        int* const votes = reinterpret_cast<int*>(smem);
        bar();
        if (lane == 0)
            votes[kWaves * group + wave] = odd;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int i = 0; i < kWaves * GROUPS; i++)
            all |= votes[i];
        again = __builtin_amdgcn_readfirstlane(all) != 0;
        if (__builtin_expect(again, 0))
        {
            unsigned given[kBlocks] = {};
            bar(); // the votes are read
            fetch(0);
            for (int i = 0; i < steps; i++)
            {
                wait_vm<0>();
                bar();
                fetch(i + 1);
                const int t = GROUPS * i + group;
                if (GROUPS == 1 || t < nt)
                    r.template count<2>(given, mine + (i & 1) * kBuf + kTileBytes, kt.key(t0 + t));
            }
        }
    }
    if constexpr (GROUPS > 1)
    {
        // the second group's registers, to the lanes that hold the same rows
        bar();
        float4* give = reinterpret_cast<float4*>(smem) + wave * 4 * kBlocks * 64 + lane;
        float2* give_ml = reinterpret_cast<float2*>(smem + kWaves * 4 * kBlocks * 64 * 16) + wave * 64 + lane;
        static_assert(kWaves * (4 * kBlocks * 64 * 16 + 64 * 8) <= GROUPS * 2 * kBuf, "the sums fit the buffers");
        if (group == 1)
        {
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    give[(4 * i + e) * 64] = make_float4(r.o[i][4 * e], r.o[i][4 * e + 1], r.o[i][4 * e + 2], r.o[i][4 * e + 3]);
            *give_ml = make_float2(r.m, r.l);
        }
        __syncthreads();
        if (group == 1)
            return;
        const float2 ml = *give_ml;
        const float m = fmaxf(r.m, ml.x);
        const float base = m == kNegInf ? 0.f : m;
        // of a group that saw no score of a row: 0
        const float ca = __builtin_amdgcn_exp2f((r.m - base) * p.scale2);
        const float cb = __builtin_amdgcn_exp2f((ml.x - base) * p.scale2);
        r.m = m;
        r.l = r.l * ca + ml.y * cb;
        auto join = [&](auto scaled) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                {
                    const float4 v = give[(4 * i + e) * 64];
                    r.o[i][4 * e] = scaled(r.o[i][4 * e], ca) + scaled(v.x, cb);
                    r.o[i][4 * e + 1] = scaled(r.o[i][4 * e + 1], ca) + scaled(v.y, cb);
                    r.o[i][4 * e + 2] = scaled(r.o[i][4 * e + 2], ca) + scaled(v.z, cb);
                    r.o[i][4 * e + 3] = scaled(r.o[i][4 * e + 3], ca) + scaled(v.w, cb);
                }
        };
        if (again)
            join([](float x, float c) { return rescaled(x, c); });
        else
            join([](float x, float c) { return x * c; });
    }

    const float l = partner_sum(r.l);
    if (row >= at.rows)
        return;
    const long long to = (static_cast<long long>(at.b) * p.heads + r.head) * p.q_len + r.qi;
    if (p.splits > 1)
    {
        const long long part = static_cast<long long>(at.split) * p.batch * p.heads * p.q_len + to;
        float* dst = p.part + part * D + 4 * r.half;
#pragma unroll
        for (int i = 0; i < kBlocks; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                *reinterpret_cast<float4*>(dst + 32 * i + 8 * e) =
                    make_float4(r.o[i][4 * e], r.o[i][4 * e + 1], r.o[i][4 * e + 2], r.o[i][4 * e + 3]);
        if (r.half == 0)
            p.part_ml[part] = make_float2(r.m, l);
        return;
    }
    const float inv = 1.f / l;
    char* dst = p.out + at.b * p.o_b + r.qi * p.o_t + r.head * p.o_h + 8 * r.half;
#pragma unroll
    for (int i = 0; i < kBlocks; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
        {
            const u2 v = {IO::pack(r.o[i][4 * e] * inv, r.o[i][4 * e + 1] * inv),
                          IO::pack(r.o[i][4 * e + 2] * inv, r.o[i][4 * e + 3] * inv)};
            *reinterpret_cast<u2*>(dst + 64 * i + 16 * e) = l == 0.f ? u2{0u, 0u} : v; // no key: 0
        }
    if (p.lse && r.half == 0)
        p.lse[to] = l == 0.f ? kNegInf : r.m * p.scale + logf(l);
}

// Few form, for at most 32 rows of a key head (single tokens): a stream of the
// cache.  The two waves of a workgroup take tiles of 32 keys in turn, each
// through LDS slots of its own with the next tiles on their way, so no barrier
// stands in the stream; their sums are joined in LDS at the end.
constexpr int kFewWaves = 2;
template <int D>
struct FewShape
{
    static constexpr int kTileBytes = 32 * 2 * D;
    static constexpr int kSlots = D == 128 ? 2 : 4;
    static constexpr int kWaveBytes = kSlots * 2 * kTileBytes; // 32 KB
    static constexpr int kLds = kFewWaves * kWaveBytes;
    static_assert(32 * (D + 4) * 4 + 256 <= kWaveBytes, "a wave's sums fit its slots");
};

template <typename IO, int D>
__global__ __launch_bounds__(64 * kFewWaves) void slide_few_kernel(SlideParams p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    using S = FewShape<D>;
    constexpr int kRowBytes = 2 * D;
    constexpr int kChunks = kRowBytes / 16;
    constexpr int kBlocks = D / 32;
    constexpr int kRowsPerDma = 64 / kChunks;
    constexpr int kDma = 32 / kRowsPerDma; // of each of K and V per tile

    const Place at(p, 32);
    if (at.none)
        return;
    const int p0 = at.off;
    const int p1 = at.off + at.nq - 1;
    const KeyTiles<32> kt(p, at.nk, p0, p1);
    const int share = (kt.count + p.splits - 1) / p.splits;
    const int t0 = min(at.split * share, kt.count);
    const int nt = min(share, kt.count - t0);

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int mine = wave < nt ? (nt - 1 - wave) / kFewWaves + 1 : 0; // tiles wave, wave + kFewWaves, ...

    const char* kb = p.k + at.b * p.k_b + at.kvh * p.k_h;
    const char* vb = p.v + at.b * p.v_b + at.kvh * p.v_h;
    char* const ring = smem + wave * S::kWaveBytes;
    const unsigned lds = static_cast<unsigned>(reinterpret_cast<size_t>(ring));
    const unsigned k_step = static_cast<unsigned>(p.k_t);
    const unsigned v_step = static_cast<unsigned>(p.v_t);
    auto fetch = [&](int i) {
        const int k0 = kt.key(t0 + wave + i * kFewWaves);
        const int last = at.nk - 1 - k0; // rows past the end repeat the last one
        const char* kp = kb + k0 * p.k_t;
        const char* vp = vb + k0 * p.v_t;
        const unsigned d = lds + (i % S::kSlots) * 2 * S::kTileBytes;
#pragma unroll
        for (int j = 0; j < kDma; j++)
        {
            const unsigned r = j * kRowsPerDma + lane / kChunks;
            const unsigned c = lane % kChunks;
            const unsigned rr = min(static_cast<int>(r), last);
            dma16(kp, rr * k_step + ((c ^ key_swz<D>(r)) << 4), d + j * 1024);
            dma16(vp, rr * v_step + ((c ^ value_swz<D>(r)) << 4), d + S::kTileBytes + j * 1024);
        }
    };
    for (int i = 0; i < min(mine, S::kSlots - 1); i++)
        fetch(i);
    const int row = min(lane & 31, at.rows - 1);
    Rows<IO, D> r;
    r.init(p, at.b, at.kvh, row, at.off, at.nk, lane);
    for (int i = 0; i < mine; i++)
    {
        if (i + S::kSlots - 1 < mine)
        {
            // the slot worked on before is free once its reads are done
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            fetch(i + S::kSlots - 1);
            wait_vm<(S::kSlots - 1) * 2 * kDma>();
        }
        else
            wait_vm<0>();
        const int k0 = kt.key(t0 + wave + i * kFewWaves);
        const char* st = ring + (i % S::kSlots) * 2 * S::kTileBytes;
        const bool masked = is_masked(p, at.nk, p0, p1, k0, 32);
        f16v s[1];
        u4 w[2];
        r.template scores<1>(s, st);
        if (masked)
            r.template mask<1>(s, k0);
        u4 v0[Rows<IO, D>::kBlocks];
        r.read_values(v0, st + S::kTileBytes, 0);
        r.template weights<1>(s, w);
        u4 rest[2];
        r.template rounding_of<1>(s, w, rest);
        r.template add<1>(w, v0, st + S::kTileBytes, masked, rest);
    }
    if (__builtin_expect(r.odd(), 0)) // again, for the values that are not finite
    {
        unsigned given[kBlocks] = {};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the slots are free
        for (int i = 0; i < mine; i++)
        {
            fetch(i);
            wait_vm<0>();
            r.template count<1>(given, ring + (i % S::kSlots) * 2 * S::kTileBytes + S::kTileBytes,
                                kt.key(t0 + wave + i * kFewWaves));
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }

    // the waves' sums, relative to the largest maximum of a row
    constexpr int kPitch = D + 4; // floats: rows start in different banks
    float2* ml = reinterpret_cast<float2*>(ring + 32 * kPitch * 4);
    float* sums = reinterpret_cast<float*>(ring);
    const float l = partner_sum(r.l);
    if ((lane & 31) < at.rows)
    {
#pragma unroll
        for (int i = 0; i < kBlocks; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                *reinterpret_cast<float4*>(sums + (lane & 31) * kPitch + 32 * i + 8 * e + 4 * r.half) =
                    make_float4(r.o[i][4 * e], r.o[i][4 * e + 1], r.o[i][4 * e + 2], r.o[i][4 * e + 3]);
        if (r.half == 0)
            ml[lane & 31] = make_float2(r.m, l);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < at.rows * (D / 4); x += 64 * kFewWaves)
    {
        const int rr = x / (D / 4);
        const int d = 4 * (x % (D / 4));
        float2 part[kFewWaves];
        float m = kNegInf;
#pragma unroll
        for (int w = 0; w < kFewWaves; w++)
        {
            part[w] = reinterpret_cast<const float2*>(smem + w * S::kWaveBytes + 32 * kPitch * 4)[rr];
            m = fmaxf(m, part[w].x);
        }
        const float base = m == kNegInf ? 0.f : m;
        float total = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kFewWaves; w++)
        {
            // of a wave that saw no score: 0
            const float a = __builtin_amdgcn_exp2f((part[w].x - base) * p.scale2);
            const float4 u = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * S::kWaveBytes) + rr * kPitch + d);
            total += a * part[w].y;
            v.x += rescaled(u.x, a);
            v.y += rescaled(u.y, a);
            v.z += rescaled(u.z, a);
            v.w += rescaled(u.w, a);
        }
        const int qi = rr / p.group;
        const int head = at.kvh * p.group + (rr - qi * p.group);
        const long long to = (static_cast<long long>(at.b) * p.heads + head) * p.q_len + qi;
        if (p.splits > 1)
        {
            const long long to_part = static_cast<long long>(at.split) * p.batch * p.heads * p.q_len + to;
            *reinterpret_cast<float4*>(p.part + to_part * D + d) = v;
            if (d == 0)
                p.part_ml[to_part] = make_float2(m, total);
            continue;
        }
        const float inv = 1.f / total;
        *reinterpret_cast<u2*>(p.out + at.b * p.o_b + qi * p.o_t + head * p.o_h + 2 * d) =
            total == 0.f ? u2{0u, 0u} : u2{IO::pack(v.x * inv, v.y * inv), IO::pack(v.z * inv, v.w * inv)};
        if (p.lse && d == 0)
            p.lse[to] = total == 0.f ? kNegInf : m * p.scale + logf(total);
    }
}

// Joins the splits of query rows: teams of 32 lanes (D / 32 dims each), `per`
// teams to a row, each with a share of its splits; all of a team's loads are
// under way before the first is used.
constexpr int kTeams = 8;
template <typename IO, int D>
__global__ __launch_bounds__(32 * kTeams) void slide_join_kernel(SlideParams p, int per)
{
    constexpr int kE = D / 32;
    typedef __attribute__((ext_vector_type(kE))) float fe;
    __shared__ float2 s_ml[kTeams];
    __shared__ fe s_sum[kTeams][32];
    const int lane = threadIdx.x & 31;
    const int team = threadIdx.x >> 5;
    const long long rows = static_cast<long long>(p.batch) * p.heads * p.q_len;
    const long long at = static_cast<long long>(blockIdx.x) * (kTeams / per) + team / per;
    const long long atc = at < rows ? at : rows - 1;
    const int mine = team % per;
    float m = kNegInf;
    float l = 0.f;
    fe o = {};
    // one part more; of one that saw no score the factor is 0
    auto take = [&](float2 ml, fe v) {
        const float next = fmaxf(m, ml.x);
        const float base = next == kNegInf ? 0.f : next;
        const float a = __builtin_amdgcn_exp2f((m - base) * p.scale2);
        const float c = __builtin_amdgcn_exp2f((ml.x - base) * p.scale2);
        m = next;
        l = l * a + c * ml.y;
#pragma unroll
        for (int e = 0; e < kE; e++)
            o[e] = rescaled(o[e], a) + rescaled(v[e], c);
    };
    for (int s0 = mine; s0 < p.splits; s0 += 4 * per)
    {
        float2 ml[4];
        fe v[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            const int s = min(s0 + i * per, p.splits - 1);
            ml[i] = p.part_ml[s * rows + atc];
            v[i] = *reinterpret_cast<const fe*>(p.part + (s * rows + atc) * D + kE * lane);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (s0 + i * per < p.splits)
                take(ml[i], v[i]);
    }
    s_sum[team][lane] = o;
    if (lane == 0)
        s_ml[team] = make_float2(m, l);
    __syncthreads();
    if (mine != 0 || at >= rows)
        return;
    const int qi = static_cast<int>(at % p.q_len);
    const long long bh = at / p.q_len;
    const int head = static_cast<int>(bh % p.heads);
    const int b = static_cast<int>(bh / p.heads);
    if (qi >= clamp_len(p.q_lens, b, p.q_len))
        return;
    for (int t = 1; t < per; t++)
        take(s_ml[team + t], s_sum[team + t][lane]);
    if (l == 0.f)
        o = fe{}; // no key
    const float inv = l == 0.f ? 0.f : 1.f / l;
    char* dst = p.out + b * p.o_b + qi * p.o_t + head * p.o_h + 2 * kE * lane;
    if constexpr (kE == 4)
        *reinterpret_cast<u2*>(dst) = u2{IO::pack(o[0] * inv, o[1] * inv), IO::pack(o[2] * inv, o[3] * inv)};
    else
        *reinterpret_cast<unsigned*>(dst) = IO::pack(o[0] * inv, o[1] * inv);
    if (p.lse && lane == 0)
        p.lse[at] = l == 0.f ? kNegInf : m * p.scale + logf(l);
}

// The form, and splits of the keys where the rows alone leave CUs without
// work: up to one workgroup a CU in the tile form (which then has two groups of
// waves) with two tiles of keys each at least, up to two in the few form (two
// fit) with a tile for each wave.
void plan_tiles(SlideParams* p)
{
    const long long rows = static_cast<long long>(p->q_len) * p->group;
    const long long heads = static_cast<long long>(p->kv_heads) * p->batch;
    p->few = rows <= 32;
    const int tile_rows = p->few ? 32 : kRows;
    const int tile_keys = p->few ? 32 * kFewWaves : kKeys;
    p->row_tiles = static_cast<int>((rows + tile_rows - 1) / tile_rows);
    const long long positions = std::min<long long>(p->q_len, (tile_rows + p->group - 1) / p->group + 1);
    const long long span = std::min<long long>(p->kv_len, static_cast<long long>(p->sinks) + p->left + p->right + positions + kKeys);
    const long long keys = (span + tile_keys - 1) / tile_keys;
    const long long want = (p->few ? 512 : 256) / std::max(1LL, p->row_tiles * heads);
    p->splits = static_cast<int>(std::max(1LL, std::min(want, p->few ? keys : keys / 2)));
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
    if (!(a->scale > 0.f) || !std::isfinite(a->scale * kLog2e))
        return bad("scale must be positive and finite");
    if (a->dtype != SV2_F16 && a->dtype != SV2_BF16)
        return set_error(a->dtype == SV2_F32 ? SV2_EUNSUPPORTED : SV2_EINVAL, std::string(what) + ": dtype must be SV2_F16 or SV2_BF16");
    if (a->head_dim != 64 && a->head_dim != 128)
        return set_error(SV2_EUNSUPPORTED, std::string(what) + ": head_dim must be 64 or 128");
    if (a->weight_terms < 0 || a->weight_terms > 2)
        return bad("weight_terms must be 0, 1 or 2");
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
    p.scale = a->scale;
    p.scale2 = a->scale * kLog2e;
    p.terms = std::max(1, a->weight_terms);
    plan_tiles(&p);
    const long long tiles = static_cast<long long>(p.row_tiles) * p.kv_heads * p.batch;
    if (!grid_fits(tiles * p.splits + 7, p.few ? 64 * kFewWaves : 64 * kWaves))
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
    const int groups = p.blocks <= 256 ? 2 : 1; // one workgroup a CU: twice the waves
    const int lds = p.few ? FewShape<D>::kLds : groups * 2 * 2 * kKeys * 2 * D;
    const int threads = 64 * (p.few ? kFewWaves : kWaves * groups);
    auto kernel = p.few          ? &slide_few_kernel<IO, D>
                  : p.terms == 2 ? (groups == 2 ? &slide_tile_kernel<IO, D, 2, 2> : &slide_tile_kernel<IO, D, 1, 2>)
                  : groups == 2  ? &slide_tile_kernel<IO, D, 2, 1>
                                 : &slide_tile_kernel<IO, D, 1, 1>;
    const int rc = set_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, "sv2_sliding_attention: dynamic LDS attribute");
    if (rc != SV2_OK)
        return rc;
    const unsigned grid = (static_cast<unsigned>(p.blocks) + 7) / 8 * 8;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), lds, stream, p);
    if (p.splits > 1)
    {
        const long long rows = static_cast<long long>(p.batch) * p.heads * p.q_len;
        const int per = p.splits > 8 ? 8 : p.splits > 4 ? 2 : 1;
        const long long grid = (rows + kTeams / per - 1) / (kTeams / per);
        if (grid > INT_MAX)
            return set_error(SV2_EUNSUPPORTED, "sv2_sliding_attention: too many rows");
        hipLaunchKernelGGL((slide_join_kernel<IO, D>), dim3(static_cast<unsigned>(grid)), dim3(32 * kTeams), 0, stream, p, per);
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
    // of a dimension of one element the stride says nothing
    const int64_t extents[12] = {a.batch, a.q_len, a.heads, a.batch, a.kv_len, a.kv_heads, a.batch, a.kv_len, a.kv_heads,
                                 a.batch, a.q_len, a.heads};
    int64_t strides[12] = {a.q_batch_stride, a.q_token_stride, a.q_head_stride, a.k_batch_stride, a.k_token_stride,
                           a.k_head_stride, a.v_batch_stride, a.v_token_stride, a.v_head_stride,
                           a.out_batch_stride, a.out_token_stride, a.out_head_stride};
    for (int i = 0; i < 12; i++)
    {
        if (extents[i] <= 1)
            strides[i] = 0;
        const int64_t s = strides[i];
        if (s < 0 || s % 8 != 0 || s > INT64_MAX / 4)
            return set_error(SV2_EINVAL, "sv2_sliding_attention: strides must be non-negative multiples of 8 elements");
        if (i >= 9 && s == 0 && extents[i] > 1)
            return set_error(SV2_EINVAL, "sv2_sliding_attention: a stride of out is 0");
    }
    // a tile's rows are addressed by 32-bit offsets from its first
    constexpr int64_t kMostStride = 1 << 24;
    static_assert((kKeys - 1) * 2 * kMostStride + 256 <= INT32_MAX, "offsets fit 32 bits");
    if (strides[4] > kMostStride || strides[7] > kMostStride)
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
