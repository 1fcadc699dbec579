// Matrix product with bias, activation and residual in its epilogue:
//
//   y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n]
//
// fp16 or bf16 operands, fp32 sums, one rounding at the end.  Any sizes, row
// strides and element alignment.  The product is computed transposed (w as the
// first operand of v_mfma_f32_16x16x32), so a lane holds four consecutive
// columns of one output row.
//
// Two forms, by the number of rows.
//   few   up to 64 rows (32 without alignment), and some blocks of 64 where these
//         leave tiles few: a stream of w.  A workgroup of four waves takes 16 CT
//         columns and splits K among its waves in blocks of 64 (interleaved:
//         together they read 512 consecutive bytes of a row).  Each wave
//         fetches whole 128-byte lines of w and x straight into a ring of LDS
//         slots of its own, so no barrier stands in the stream; the four
//         partial sums meet in LDS at the end.  One launch, no workspace.
//   any   operands that the tile kernel of the inner products does not take,
//         from 33 rows or 4097 columns on: tiles through registers.
//   tile  aligned operands of more rows: gemm.hip's persistent tiles.
//
// What they reach (MI355X): few, 1 x 2560 -> 15360 fp16 14 us (5.7 TB/s of w,
// which the last-level cache holds in part), 58 x 5120 -> 2560 bf16 11 to 12 us (bound
// by x: a workgroup brings 590 KB of it into LDS beside 160 of w);
// any, 1999 x 1001 -> 777 with GELU and residual 20 to 23 us (16 steps, each a
// barrier and LDS round trip for 416 workgroups of 4 waves), 16000 x 2561 ->
// 2561 430 us (0.49 PFLOP/s); tile, 21658 x 2560 -> 6912 bf16 with bias and tanh
// GELU 600 to 650 us by the card (1.18 to 1.28 PFLOP/s; torch's product of these
// sizes alone 631 to 654).
#include "sv2_internal.h"
#include "activation.h"
#include "vec_io.h"

#include <algorithm>
#include <cmath>

namespace sv2
{
namespace
{

typedef __attribute__((ext_vector_type(8))) _Float16 h8;
typedef __attribute__((ext_vector_type(8))) __bf16 b8;
typedef __attribute__((ext_vector_type(4))) float f4;
typedef __attribute__((ext_vector_type(4))) unsigned u4;
typedef __attribute__((ext_vector_type(2))) unsigned u2;
typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned u4u; // 16 bytes at any element

struct HalfIO
{
    static __device__ f4 mfma(u4 a, u4 b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    static __device__ float to_float(uint16_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
    static __device__ uint16_t from_float(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
};
struct BfloatIO
{
    static __device__ f4 mfma(u4 a, u4 b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ float to_float(uint16_t v) { return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16); }
    static __device__ uint16_t from_float(float v) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }
};

struct LinearParams
{
    const uint16_t* x;
    const uint16_t* w;
    uint16_t* y;
    const uint16_t* r;
    const float* bias;
    long long ldx, ldw, ldy, ldr;
    int m, n, k;
    int act;
    int tiles_m, tiles_n;
    int vec4; // rows of y and the residual hold whole aligned groups of 4
};

constexpr int kBK = 64; // K of a step: whole 128-byte lines of every row

// 8 elements of a row from column k on, zeros past `k_end`: past the end, the
// row's last 8 moved down.
__device__ inline u4 load8(const uint16_t* row, int k, int k_end)
{
    if (k_end >= 8)
    {
        const int at = min(k, k_end - 8);
        const u4 v = *reinterpret_cast<const u4u*>(row + at);
        const int gone = k - at;
        const unsigned __int128 bits = __builtin_bit_cast(unsigned __int128, v);
        return gone < 8 ? __builtin_bit_cast(u4, bits >> (16 * gone)) : u4{0u, 0u, 0u, 0u};
    }
    u4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (k + e < k_end)
            v[e >> 1] |= static_cast<unsigned>(row[k + e]) << (16 * (e & 1));
    return v;
}

// Four columns of one output row.
template <typename IO, typename A>
__device__ inline void finish4(const LinearParams& p, int m, int n, f4 v, A act)
{
    if (m >= p.m || n >= p.n)
        return;
    const int left = p.n - n;
    if (p.bias)
#pragma unroll
        for (int e = 0; e < 4; e++)
            v[e] += p.bias[min(n + e, p.n - 1)];
#pragma unroll
    for (int e = 0; e < 4; e++)
        v[e] = act(v[e]);
    uint16_t* y = p.y + m * p.ldy + n;
    const uint16_t* r = p.r ? p.r + m * p.ldr + n : nullptr;
    if (p.vec4)
    {
        if (r)
        {
            const u2 old = *reinterpret_cast<const u2*>(r);
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[e] += IO::to_float(static_cast<uint16_t>(old[e >> 1] >> (16 * (e & 1))));
        }
        *reinterpret_cast<u2*>(y) = u2{IO::from_float(v[0]) | static_cast<unsigned>(IO::from_float(v[1])) << 16,
                                       IO::from_float(v[2]) | static_cast<unsigned>(IO::from_float(v[3])) << 16};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < left)
            y[e] = IO::from_float(r ? v[e] + IO::to_float(r[e]) : v[e]);
}

// The activation by a uniform branch, for epilogues that are a small part of
// their kernel.
__device__ inline float activate_by(int act, float v)
{
    switch (act)
    {
    case SV2_ACT_SILU: return activate<SV2_ACT_SILU, false>(v);
    case SV2_ACT_GELU: return activate<SV2_ACT_GELU, false>(v);
    case SV2_ACT_GELU_TANH: return activate<SV2_ACT_GELU_TANH, false>(v);
    default: return v;
    }
}

// 16 bytes per lane from global memory (uniform base + 32-bit lane offset)
// straight into LDS at lds + 16 * lane (lds wave-uniform, in M0; one wait
// state between the write of M0 and its use).  The compiler does not count
// these loads; the loop waits for them itself.
__device__ inline void dma16(const void* base, unsigned voff, unsigned lds)
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
    static_assert(N >= 0 && N < 64, "vmcnt holds 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

constexpr int kFewWaves = 4;
constexpr int kFewRows = 64;
constexpr int kFewMost = 1 << 20; // rows the few form is weighed for (its grid holds 65535 blocks of rows)

// The few form's LDS: a ring of slots of 16 CT rows of w and 16 MT rows of x,
// 128 bytes each, per wave; 16-byte chunk c of row r sits in slot c ^ (r & 7),
// so the 16 rows an operand read takes at one chunk fall on different banks.
// Two workgroups a CU where three blocks ahead fit, else one.
template <int MT, int CT>
struct FewShape
{
    static constexpr int kSlot = (MT + CT) * 2048;
    static constexpr int kPer = 2 * (MT + CT); // fetches of a block
    static constexpr int kBudget = (80 * 1024 / (kFewWaves * kSlot) >= 4 ? 80 : 160) * 1024;
    static constexpr int kFit = kBudget / (kFewWaves * kSlot);
    static constexpr int kSlots = kFit > 6 ? 6 : kFit;
    static constexpr int kLds = kFewWaves * kSlots * kSlot;
    static_assert(kSlots >= 2 && MT * CT * 1024 <= kSlots * kSlot, "a wave's sums fit its ring");
};

// `WHOLE`: operands in 16-byte pieces (pointers 16-byte aligned, strides of w
// and x multiples of 8); else every piece is loaded through registers.
template <typename IO, int MT, int CT, bool WHOLE>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few_kernel(LinearParams p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    using S = FewShape<MT, CT>;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15;
    const int lq = lane >> 4;
    const int n0 = blockIdx.x * 16 * CT;
    const int m0 = blockIdx.y * kFewRows; // more rows: in blocks of kFewRows
    p.x += m0 * p.ldx;
    p.y += m0 * p.ldy;
    if (p.r)
        p.r += m0 * p.ldr;
    p.m = min(p.m - m0, kFewRows);
    f4 acc[CT][MT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int m = 0; m < MT; m++)
            acc[c][m] = f4{0.f, 0.f, 0.f, 0.f};
    char* ring = smem + wave * S::kSlots * S::kSlot;
    // rows past the end repeat the last one; their sums are not stored
    int done = 0; // k that the stream has taken
    if constexpr (WHOLE)
    {
        const int blocks = p.k / 64;
        done = blocks * 64;
        const int mine = wave < blocks ? (blocks - 1 - wave) / kFewWaves + 1 : 0;
        const char* wb = reinterpret_cast<const char*>(p.w + n0 * p.ldw) + 128 * wave;
        const char* xb = reinterpret_cast<const char*>(p.x) + 128 * wave;
        const int fr = lane >> 3;
        const unsigned chunk = ((lane & 7) ^ fr) << 4;
        unsigned wo[2 * CT], xo[2 * MT];
#pragma unroll
        for (int i = 0; i < 2 * CT; i++)
            wo[i] = static_cast<unsigned>(min(8 * i + fr, p.n - 1 - n0) * p.ldw * 2) + chunk;
#pragma unroll
        for (int i = 0; i < 2 * MT; i++)
            xo[i] = static_cast<unsigned>(min(8 * i + fr, p.m - 1) * p.ldx * 2) + chunk;
        const unsigned lds = static_cast<unsigned>(reinterpret_cast<size_t>(ring));
        int slot = 0;
        auto fetch = [&]() {
            const unsigned d = lds + slot * S::kSlot;
#pragma unroll
            for (int i = 0; i < 2 * CT; i++)
                dma16(wb, wo[i], d + 1024 * i);
#pragma unroll
            for (int i = 0; i < 2 * MT; i++)
                dma16(xb, xo[i], d + CT * 2048 + 1024 * i);
            wb += 128 * kFewWaves;
            xb += 128 * kFewWaves;
            slot = slot + 1 == S::kSlots ? 0 : slot + 1;
        };
        unsigned at[2];
#pragma unroll
        for (int s = 0; s < 2; s++)
            at[s] = lr * 128 + (((4 * s + lq) ^ (lr & 7)) << 4);
        const char* st = ring;
        auto multiply = [&]() {
#pragma unroll
            for (int s = 0; s < 2; s++)
            {
                u4 a[CT], b[MT];
#pragma unroll
                for (int c = 0; c < CT; c++)
                    a[c] = *reinterpret_cast<const u4*>(st + at[s] + 2048 * c);
#pragma unroll
                for (int m = 0; m < MT; m++)
                    b[m] = *reinterpret_cast<const u4*>(st + at[s] + 2048 * (CT + m));
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int m = 0; m < MT; m++)
                        acc[c][m] = IO::mfma(a[c], b[m], acc[c][m]);
            }
            st = st + S::kSlot == ring + S::kSlots * S::kSlot ? ring : st + S::kSlot;
        };
        for (int i = 0; i < min(mine, S::kSlots - 1); i++)
            fetch();
        int i = 0;
        for (; i + S::kSlots - 1 < mine; i++)
        {
            // the slot multiplied before is free once its reads are done
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            fetch();
            wait_vm<(S::kSlots - 1) * S::kPer>();
            multiply();
        }
        wait_vm<0>();
        for (; i < mine; i++)
            multiply();
    }
    // what the stream left: the last k of all (WHOLE), or everything
    const uint16_t* wr[CT];
    const uint16_t* xr[MT];
#pragma unroll
    for (int c = 0; c < CT; c++)
        wr[c] = p.w + min(n0 + 16 * c + lr, p.n - 1) * p.ldw;
#pragma unroll
    for (int m = 0; m < MT; m++)
        xr[m] = p.x + min(16 * m + lr, p.m - 1) * p.ldx;
    auto pieces = [&](auto load, int k) {
        u4 a[CT], b[MT];
#pragma unroll
        for (int c = 0; c < CT; c++)
            a[c] = load(wr[c], k);
#pragma unroll
        for (int m = 0; m < MT; m++)
            b[m] = load(xr[m], k);
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int m = 0; m < MT; m++)
                acc[c][m] = IO::mfma(a[c], b[m], acc[c][m]);
    };
    int k0 = done + 32 * wave;
#pragma unroll 4
    for (; k0 + 32 <= p.k; k0 += 32 * kFewWaves)
        pieces([](const uint16_t* row, int k) -> u4 { return *reinterpret_cast<const u4u*>(row + k); }, k0 + 8 * lq);
    if (k0 < p.k)
        pieces([&](const uint16_t* row, int k) { return load8(row, k, p.k); }, k0 + 8 * lq);
    // the waves' sums, added in wave order
    f4* sums = reinterpret_cast<f4*>(ring);
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int m = 0; m < MT; m++)
            sums[(c * MT + m) * 64 + lane] = acc[c][m];
    __syncthreads();
    for (int t = wave; t < CT * MT; t += kFewWaves)
    {
        f4 v = reinterpret_cast<const f4*>(smem)[t * 64 + lane];
#pragma unroll
        for (int w = 1; w < kFewWaves; w++)
            v += reinterpret_cast<const f4*>(smem + w * S::kSlots * S::kSlot)[t * 64 + lane];
        const int c = t / MT;
        finish4<IO>(p, 16 * (t - c * MT) + lr, n0 + 16 * c + 4 * lq, v, [&](float x) { return activate_by(p.act, x); });
    }
}

// Any form: TILE x TILE outputs by 4 waves, K in steps of 64 through registers
// (kHeld steps ahead) into two LDS buffers.  16-byte loads at any
// element alignment; only the last step looks at K's end.
template <int TILE>
struct AnyShape
{
    static constexpr int kPitch = kBK * 2 + 16; // bytes of an LDS row: 16 rows of one chunk start in different banks
    static constexpr int kOperand = TILE * kPitch;
    static constexpr int kLds = 2 * 2 * kOperand;
    static constexpr int kPieces = TILE * 8 / 256; // 16-byte pieces of an operand per thread and step
    static constexpr int kHeld = 2; // steps in registers (more: no faster, 1999 x 1001 -> 777 18.0 us, with five 19.8)
};

template <typename IO, int ACT, int TILE>
__global__ __launch_bounds__(256, TILE == 128 ? 2 : 3) void linear_any_kernel(LinearParams p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    using S = AnyShape<TILE>;
    constexpr int kPieces = S::kPieces;
    constexpr int kPart = TILE / 2; // of a wave, each way
    constexpr int kT = kPart / 16;
    // XCD x (workgroup id mod 8) takes a contiguous run of tiles, which share
    // rows of x in its L2
    const int id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int tm = id / p.tiles_n;
    const int tn = id - tm * p.tiles_n;
    if (tm >= p.tiles_m)
        return;
    const int m0 = tm * TILE;
    const int n0 = tn * TILE;
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int lr = lane & 15;
    const int lq = lane >> 4;
    const int wn = kPart * (wave & 1);
    const int wm = kPart * (wave >> 1);

    // this thread's pieces: rows threadIdx / 8 + 32 i, chunk threadIdx % 8
    const int cr = threadIdx.x >> 3;
    const int cc = threadIdx.x & 7;
    const uint16_t* xr[kPieces];
    const uint16_t* wr[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; i++)
    {
        // rows past the end repeat the last one; their sums are not stored
        xr[i] = p.x + min(m0 + cr + 32 * i, p.m - 1) * p.ldx;
        wr[i] = p.w + min(n0 + cr + 32 * i, p.n - 1) * p.ldw;
    }
    // whole steps; what K leaves follows them.  Loads stand in no branch: behind
    // one, the wait for a step's loads would be one for all loads under way
    const int steps = p.k / kBK;
    struct Held
    {
        u4 x[kPieces], w[kPieces];
    };
    auto load = [&](Held& h, int s) {
        const int k = min(s, steps - 1) * kBK + 8 * cc; // past the end: the last one again
#pragma unroll
        for (int i = 0; i < kPieces; i++)
        {
            h.x[i] = *reinterpret_cast<const u4u*>(xr[i] + k);
            h.w[i] = *reinterpret_cast<const u4u*>(wr[i] + k);
        }
    };
    auto put = [&](const Held& h, int s) {
        char* to = smem + (s & 1) * 2 * S::kOperand + cr * S::kPitch + 16 * cc;
#pragma unroll
        for (int i = 0; i < kPieces; i++)
        {
            *reinterpret_cast<u4*>(to + 32 * i * S::kPitch) = h.w[i];
            *reinterpret_cast<u4*>(to + S::kOperand + 32 * i * S::kPitch) = h.x[i];
        }
    };
    f4 acc[kT][kT];
#pragma unroll
    for (int t = 0; t < kT; t++)
#pragma unroll
        for (int u = 0; u < kT; u++)
            acc[t][u] = f4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int s) {
        const char* from = smem + (s & 1) * 2 * S::kOperand + lr * S::kPitch + 16 * lq;
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
        {
            u4 a[kT], b[kT];
#pragma unroll
            for (int t = 0; t < kT; t++)
            {
                a[t] = *reinterpret_cast<const u4*>(from + (wn + 16 * t) * S::kPitch + 64 * ks);
                b[t] = *reinterpret_cast<const u4*>(from + S::kOperand + (wm + 16 * t) * S::kPitch + 64 * ks);
            }
#pragma unroll
            for (int t = 0; t < kT; t++)
#pragma unroll
                for (int u = 0; u < kT; u++)
                    acc[t][u] = IO::mfma(a[t], b[u], acc[t][u]);
        }
    };
    const bool rest = p.k % kBK != 0;
    Held last;
    if (rest)
#pragma unroll
        for (int i = 0; i < kPieces; i++)
        {
            last.x[i] = load8(xr[i], steps * kBK + 8 * cc, p.k);
            last.w[i] = load8(wr[i], steps * kBK + 8 * cc, p.k);
        }
    if (steps > 0)
    {
        // step s: the next one's registers go to LDS and are loaded again, for
        // the step kHeld further
        Held held[S::kHeld];
#pragma unroll
        for (int i = 0; i < S::kHeld; i++)
            load(held[i], i);
        put(held[0], 0);
        load(held[0], S::kHeld);
        __syncthreads();
        for (int s0 = 0; s0 < steps; s0 += S::kHeld)
        {
#pragma unroll
            for (int u = 0; u < S::kHeld; u++)
            {
                const int s = s0 + u;
                if (s >= steps)
                    break;
                Held& h = held[(u + 1) % S::kHeld];
                put(h, s + 1);
                load(h, s + 1 + S::kHeld);
                multiply(s);
                __syncthreads();
            }
        }
    }
    if (rest)
    {
        put(last, 0);
        __syncthreads();
        multiply(0);
    }
#pragma unroll
    for (int t = 0; t < kT; t++)
#pragma unroll
        for (int u = 0; u < kT; u++)
            finish4<IO>(p, m0 + wm + 16 * u + lr, n0 + wn + 16 * t + 4 * lq, acc[t][u],
                        [](float v) { return activate<ACT, false>(v); });
}

template <typename IO, int ACT, int TILE>
int run_any(LinearParams p, hipStream_t stream)
{
    p.tiles_m = static_cast<int>((p.m + TILE - 1LL) / TILE);
    p.tiles_n = static_cast<int>((p.n + TILE - 1LL) / TILE);
    const long long total = static_cast<long long>(p.tiles_m) * p.tiles_n;
    if (!grid_fits(total + 7, 256))
        return set_error(SV2_EUNSUPPORTED, "sv2_linear: too many tiles");
    constexpr int kLds = AnyShape<TILE>::kLds;
    const int rc = set_dynamic_lds(reinterpret_cast<const void*>(&linear_any_kernel<IO, ACT, TILE>), kLds,
                                   "linear_any: dynamic LDS attribute");
    if (rc != SV2_OK)
        return rc;
    hipLaunchKernelGGL((linear_any_kernel<IO, ACT, TILE>), dim3((static_cast<unsigned>(total) + 7) / 8 * 8), dim3(256),
                       kLds, stream, p);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? SV2_OK : hip_error(err, "sv2_linear launch");
}

// The any form's tile: the large one where it gives two thirds of the CUs one
// and its rows are not mostly empty: 2561 -> 2561 at 1200 rows (210 of them) 52
// us in it and 72 in the small one, at 2000 (336) 81 and 109, 1001 -> 777 at
// 3000 (168) 24.5 and 23.8, at 1999 (112) 24 and 17
int any_tile(const LinearParams& p)
{
    const long long tiles = ((p.m + 127LL) / 128) * ((p.n + 127LL) / 128);
    return p.m > 64 && tiles >= 176 ? 128 : 64;
}

template <typename IO, int ACT>
int run_linear(const LinearParams& p, hipStream_t stream)
{
    return any_tile(p) == 128 ? run_any<IO, ACT, 128>(p, stream) : run_any<IO, ACT, 64>(p, stream);
}

template <typename IO, int MT, int CT, bool WHOLE>
int run_few(const LinearParams& p, hipStream_t stream)
{
    constexpr int kLds = FewShape<MT, CT>::kLds;
    if (!grid_fits((p.n + 16LL * CT - 1) / (16 * CT), 64 * kFewWaves))
        return set_error(SV2_EUNSUPPORTED, "sv2_linear: too many columns");
    const int rc = set_dynamic_lds(reinterpret_cast<const void*>(&linear_few_kernel<IO, MT, CT, WHOLE>), kLds,
                                   "linear_few: dynamic LDS attribute");
    if (rc != SV2_OK)
        return rc;
    const dim3 grid(static_cast<unsigned>((p.n + 16LL * CT - 1) / (16 * CT)), static_cast<unsigned>((p.m + kFewRows - 1) / kFewRows));
    hipLaunchKernelGGL((linear_few_kernel<IO, MT, CT, WHOLE>), grid, dim3(64 * kFewWaves), kLds, stream, p);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? SV2_OK : hip_error(err, "sv2_linear launch");
}

// Microseconds of the few form (MI355X): rounds of one workgroup a CU, each a
// stream of w and x through LDS (2560 -> 2560 takes 6.5 / 11 / 16 us at 64 /
// 128 / 256 rows: 160 / 320 / 640 workgroups, 5.5 us a round), and not faster
// than w comes from HBM and an x past an XCD's 4 MB of L2 comes once for every
// 16 CT columns (4538 x 5312 -> 96: 290 MB and 43 us in 16s, 97 MB in 64s).
double few_us(const LinearParams& p, int ct)
{
    const double groups = static_cast<double>((p.n + 16LL * ct - 1) / (16 * ct)) * ((p.m + kFewRows - 1) / kFewRows);
    const double round = ct == 4 ? 2.0 + 0.0041 * p.k : 1.4 + 0.0017 * p.k;
    const double x_bytes = 2.0 * p.m * p.k;
    const double x_us = x_bytes > (4 << 20) ? 1e-6 * x_bytes * ((p.n + 16LL * ct - 1) / (16 * ct)) / 7.0 : 0.0;
    return 1.5 + std::max({std::ceil(groups / 256) * round, 2e-6 * p.n * p.k / 5.0, x_us});
}
// Columns of a workgroup, in 16s: wide ones read x once for 64 columns and have
// fewer workgroups (only worth it with x of more than 32 rows in whole pieces).
int few_columns(const LinearParams& p, bool whole)
{
    return whole && p.m > 32 && few_us(p, 4) < few_us(p, 1) ? 4 : 1;
}

template <typename IO, bool WHOLE>
int run_few_rows(const LinearParams& p, hipStream_t stream)
{
    if (p.m <= 16)
        return run_few<IO, 1, 1, WHOLE>(p, stream);
    if (!WHOLE || p.m <= 32)
        return run_few<IO, 2, 1, WHOLE>(p, stream);
    return few_columns(p, true) == 4 ? run_few<IO, 4, 4, true>(p, stream) : run_few<IO, 4, 1, true>(p, stream);
}

template <typename IO>
int run_act(const LinearParams& p, int activation, hipStream_t stream)
{
    switch (activation)
    {
    case SV2_ACT_SILU: return run_linear<IO, SV2_ACT_SILU>(p, stream);
    case SV2_ACT_GELU: return run_linear<IO, SV2_ACT_GELU>(p, stream);
    case SV2_ACT_GELU_TANH: return run_linear<IO, SV2_ACT_GELU_TANH>(p, stream);
    default: return run_linear<IO, SV2_ACT_NONE>(p, stream);
    }
}

int check_linear(const sv2_linear_args* a)
{
    auto bad = [&](const char* why) { return set_error(SV2_EINVAL, std::string("sv2_linear: ") + why); };
    if (!a)
        return bad("null arguments");
    if (a->rows < 0 || a->in <= 0 || a->out < 0)
        return bad("negative rows or out, or in below 1");
    if (a->dtype != SV2_F16 && a->dtype != SV2_BF16)
        return set_error(a->dtype == SV2_F32 ? SV2_EUNSUPPORTED : SV2_EINVAL, "sv2_linear: dtype must be SV2_F16 or SV2_BF16");
    if (a->activation < SV2_ACT_NONE || a->activation > SV2_ACT_GELU_TANH)
        return bad("unknown activation");
    if (a->x_stride < a->in || a->w_stride < a->in || a->y_stride < a->out || (a->residual && a->residual_stride < a->out))
        return bad("a row stride below the row's length");
    if (a->rows > 1 && a->residual && a->residual == a->y && a->residual_stride != a->y_stride)
        return bad("the residual is y with another stride");
    return SV2_OK;
}

// A call of sv2_linear: its parameters and the kernel that takes it.
struct LinearCall
{
    LinearParams p;
    LinearOperands o;
    bool whole; // x and w in pieces of 16 bytes, the rows a workgroup fetches within 32-bit offsets
    int kernel; // SV2_LINEAR_*
};

int make_call(const sv2_linear_args& a, LinearCall* c)
{
    if (!a.x || !a.w || !a.y)
        return set_error(SV2_EINVAL, "sv2_linear: null pointer");
    if (misaligned(a.x, 2) || misaligned(a.w, 2) || misaligned(a.y, 2) || misaligned(a.residual, 2) || misaligned(a.bias, 4))
        return set_error(SV2_EINVAL, "sv2_linear: a pointer is not aligned to its elements");
    LinearParams p{};
    p.x = static_cast<const uint16_t*>(a.x);
    p.w = static_cast<const uint16_t*>(a.w);
    p.y = static_cast<uint16_t*>(a.y);
    p.r = static_cast<const uint16_t*>(a.residual);
    p.bias = a.bias;
    p.ldx = a.x_stride;
    p.ldw = a.w_stride;
    p.ldy = a.y_stride;
    p.ldr = a.residual ? a.residual_stride : 0;
    p.m = a.rows;
    p.n = a.out;
    p.k = a.in;
    p.vec4 = p.n % 4 == 0 && p.ldy % 4 == 0 && p.ldr % 4 == 0 && !misaligned(p.y, 8) && !misaligned(p.r, 8);
    p.act = a.activation;
    c->p = p;
    c->o = LinearOperands{p.x, p.w, p.y, p.r, p.bias, p.ldx, p.ldw, p.ldy, p.ldr, p.m, p.n, p.k, p.act, a.dtype == SV2_BF16};
    c->whole = p.ldx % 8 == 0 && p.ldw % 8 == 0 && !misaligned(p.x, 16) && !misaligned(p.w, 16) &&
               std::max(p.ldx, p.ldw) < (1LL << 31) / (2 * kFewRows);
    const bool tiles = linear_tiles_fit(c->o);
    // a few blocks of 64 rows stream faster than they fill tiles (2560 -> 2560
    // up to 384 rows, 640 -> 640 and 512 rows)
    // rows that are not in whole pieces: the few form loads each where it is
    // used, the tiles a step ahead (16 x 5001 -> 2001 26 us and 36, 24 x 1001 ->
    // 777 8.4 and 11, but 60 x 5001 -> 2001 60 and 35, 16 x 2561 -> 15001, in
    // rounds of workgroups, 65 and 26)
    const bool few = c->whole ? p.m <= kFewRows : p.m <= 32 && p.n <= 16 * 256;
    if (few || (c->whole && tiles && p.m <= kFewMost && few_us(p, few_columns(p, true)) < linear_tiles_us(c->o)))
        c->kernel = SV2_LINEAR_FEW;
    else
        c->kernel = tiles ? SV2_LINEAR_TILES : SV2_LINEAR_ANY;
    return SV2_OK;
}

} // namespace
} // namespace sv2

extern "C" int sv2_linear(const sv2_linear_args* args, void* stream)
try
{
    using namespace sv2;
    const int rc = check_linear(args);
    if (rc != SV2_OK)
        return rc;
    const sv2_linear_args& a = *args;
    if (a.rows == 0 || a.out == 0)
        return SV2_OK;
    LinearCall c;
    const int bad = make_call(a, &c);
    if (bad != SV2_OK)
        return bad;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool half = a.dtype == SV2_F16;
    switch (c.kernel)
    {
    case SV2_LINEAR_FEW:
        if (half)
            return c.whole ? run_few_rows<HalfIO, true>(c.p, st) : run_few_rows<HalfIO, false>(c.p, st);
        return c.whole ? run_few_rows<BfloatIO, true>(c.p, st) : run_few_rows<BfloatIO, false>(c.p, st);
    case SV2_LINEAR_TILES: return linear_tiles(st, c.o);
    default: return half ? run_act<HalfIO>(c.p, a.activation, st) : run_act<BfloatIO>(c.p, a.activation, st);
    }
}
catch (...)
{
    return sv2::caught_exception("sv2_linear");
}

extern "C" int sv2_linear_plan(const sv2_linear_args* args, sv2_linear_form* plan)
try
{
    using namespace sv2;
    const int rc = check_linear(args);
    if (rc != SV2_OK)
        return rc;
    if (!plan || args->rows == 0 || args->out == 0)
        return set_error(SV2_EINVAL, "sv2_linear_plan: null plan or no outputs");
    LinearCall c;
    const int bad = make_call(*args, &c);
    if (bad != SV2_OK)
        return bad;
    *plan = sv2_linear_form{c.kernel, 0, 0, -1};
    switch (c.kernel)
    {
    case SV2_LINEAR_FEW: plan->tile = 16 * few_columns(c.p, c.whole); break;
    case SV2_LINEAR_TILES: linear_tiles_plan(c.o, &plan->first_rows, &plan->form); break;
    default: plan->tile = any_tile(c.p); break;
    }
    return SV2_OK;
}
catch (...)
{
    return sv2::caught_exception("sv2_linear_plan");
}
