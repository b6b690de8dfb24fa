// 4-bit weights with group scales: quantisation, packing, and the products of
// a few activation rows with them (decode), dense and grouped by expert.
//
// Weight (k, n) of group g of G is q[g][k][n] * scale[g][k / gs][n] with q an
// integer in [-7, 7] and gs = 32, 64 or 128 consecutive k sharing a scale:
//   out[m, n] = sum_b scale[b, n] * sum_{k in block b} q[k, n] x[m, k]
//
// The weights need no arithmetic to reach the tensor cores: an 8-bit float
// (e4m3) whose exponent field is zero is m * 2^-9 for its mantissa m = 0..7,
// so a sign and three magnitude bits ARE the e4m3 code of q * 2^-9.  Eight
// packed weights become two operand registers by one mask, one rotation and
// another mask.  The activations take part as e5m2 terms: with rho = the
// power of two that brings the row's largest finite magnitude into
// [2^15, 2^16), x * rho = t_0 + t_1 + ... where t_j is what is left after
// t_0 .. t_{j-1}, truncated to e5m2's three significant bits (down to 2^-16).
// Three terms hold a bf16 value unless its last bits lie below that.  A float32
// value takes three such windows, each 2^9 larger than the one before, with sums
// of their own.  Elements that are 2^24 (float32: 2^26, 2^23 in few rows) below
// their row's largest may end below the last window: what is left of them is
// multiplied in float32 and added at the end, so every bit of x takes part.  A
// row's terms sit side by side in MMA columns whose sums are added (few rows: a
// tile is 16 columns at least), or follow one another into the window's column.
// Every product is exact, sums are float32 (tcgen05, accumulators in TMEM), and
// the scales multiply them in float32: no rounded weight ever exists.
//
// What has to be moved is the weight stream, K*N/2 bytes plus the scales.
// 4096 x 14336, groups of 128, one bf16 row: 10.9 us, 2.8 TB/s of that stream,
// from a cold L2 as from a warm one (about 2 us to the first product, 4 of
// products, 1.5 of sums between CTAs, the rest the launch).  64 rows of 14336 x
// 4096, groups of 64: 22.5 us (18.1 for 4096 x 14336, groups of 128), where
// unpacking, taking the sums back from tensor memory and the latency from one
// unit to the next bound it.  Forms that could not keep up (4096 x 14336, one
// row): warp MMAs (mma.sync m16n8k16 occupies its sub-core's tensor pipe for 32
// cycles: 16.6 us, 47.6 for 64 rows), and bf16 operands for tcgen05 (7 logic
// operations and 4 subtractions per 8 weights, the logic pipe the bound: 17.3 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <new>
#include <type_traits>

#include "common.cuh"
#include "runtime.h"

namespace aem {

// Packed 4-bit weight (device): [G][NC][NP] blocks of `block` bytes, NC =
// ceil(N / 128) channel blocks and NP = ceil(K / 128).  A block holds 128
// channels x 128 k and their scales, so one bulk copy brings both:
//   [4][128][16 B]   weights: 32-k quarter, channel.  A word holds 8
//                    consecutive k.  Byte j < 4: magnitude of weight j in bits
//                    0-2, its sign in bit 7; magnitude of weight 4 + j in bits
//                    4-6, its sign in bit 3 of byte (j + 1) % 4
//   [128 / gs][128]  scales in the caller's type
// Padding is zero.
struct Q4Weight {
    int device = 0;
    int64_t G = 0, K = 0, N = 0, NC = 0, NP = 0;
    int gs = 0, block = 0;
    bool scale_bf16 = false;
    uint8_t* data = nullptr;
};

namespace {

constexpr int kThreads = 256;  // pack

// ------------------------------------------------------------------ quantise
// One block per (128 float32 or 256 bf16 columns, scale group): GS / 8 warps
// hold 8 rows of the group each in registers, 16 bytes a lane, so w is read
// once; the column maxima meet in shared memory.  scale = max(amax / 7, 1e-12),
// rounded to the scale's type before q = clip(rint(w / scale), -7, 7) is taken
// with it (IEEE float32 division, ties to even).  |w / scale| is at most
// 7 (1 + 2^-8), so nothing is left to clip, and w * (1 / scale) is within 2^-20
// of it, so the division itself is only made where the product lies that near a
// half.  Adding 1.5 * 2^23 rounds to a whole number, ties to even, and leaves it
// in the low byte (the conversion instructions run at a quarter of the rate).
// 14336 x 4096, groups of 128: float32 51.4 us = 5.7 TB/s, memory bound (with a
// division per element 103); bf16 46.5, the wait for the maxima between loads
// and stores the bound.
constexpr float kRint = 12582912.0f;
// Maximum that keeps a NaN: its group's scale has to be one.
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
template <typename WT, typename ST, int GS, bool VEC>
__global__ void __launch_bounds__(4 * GS, 256 / GS)
    quantize_q4_kernel(const WT* __restrict__ w, int64_t K, int64_t N, int64_t KB,
                       int8_t* __restrict__ q, ST* __restrict__ scale) {
    // CL columns a lane: 16 bytes, kept as loaded
    constexpr int R = 8, W = GS / R, CL = VEC && sizeof(WT) == 2 ? 8 : 4, COLS = 32 * CL;
    __shared__ __align__(16) float amax[W][COLS], scales[COLS], inverses[COLS];
    const int lane = threadIdx.x & 31, wi = threadIdx.x >> 5;
    const int64_t g = blockIdx.x / KB, b = blockIdx.x % KB;
    const int64_t c0 = static_cast<int64_t>(blockIdx.y) * COLS, n0 = c0 + lane * CL, k0 = b * GS + wi;
    const int rows = static_cast<int>(min(static_cast<int64_t>(R), (K - k0 + W - 1) / W));  // k0 + i * W < K
    const int64_t at = (g * K + k0) * N + n0, step = W * N;
    const bool on = n0 < N;
    uint32_t v[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0;
        if (i >= rows || !on) continue;
        const WT* p = w + at + i * step;
        if constexpr (VEC) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            v[i][0] = u.x, v[i][1] = u.y, v[i][2] = u.z, v[i][3] = u.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < N) v[i][j] = __float_as_uint(static_cast<float>(p[j]));
        }
    }
    auto value = [&](int i, int j) {
        if constexpr (CL == 8) return __uint_as_float(j & 1 ? v[i][j / 2] & 0xffff0000u : v[i][j / 2] << 16);
        return __uint_as_float(v[i][j]);
    };
    float m[CL] = {};
    if constexpr (CL == 8) {  // two magnitudes at a time, as they are
        __nv_bfloat162 top[4] = {};
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                top[j] = __hmax2_nan(top[j], __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v[i][j])));
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = j & 1 ? __high2float(top[j / 2]) : __low2float(top[j / 2]);
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < CL; ++j) m[j] = max_nan(m[j], fabsf(value(i, j)));
    }
#pragma unroll
    for (int j = 0; j < CL; j += 4)
        *reinterpret_cast<float4*>(&amax[wi][lane * CL + j]) = make_float4(m[j], m[j + 1], m[j + 2], m[j + 3]);
    __syncthreads();
    for (int c = threadIdx.x; c < COLS; c += 4 * GS) {  // one thread per column
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) a = max_nan(a, amax[i][c]);
        float sc = max_nan(__fdiv_rn(a, 7.0f), 1e-12f);
        if constexpr (sizeof(ST) == 2) sc = __bfloat162float(__float2bfloat16_rn(sc));
        scales[c] = sc;
        inverses[c] = __frcp_rn(sc);
        if (c0 + c < N) scale[(g * KB + b) * N + c0 + c] = static_cast<ST>(sc);
    }
    __syncthreads();
    float inv[CL];
#pragma unroll
    for (int j = 0; j < CL; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(&inverses[lane * CL + j]);
        inv[j] = f.x, inv[j + 1] = f.y, inv[j + 2] = f.z, inv[j + 3] = f.w;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i >= rows || !on) continue;
        uint32_t c[CL];
        float off = 0.0f;  // the largest distance from a whole number
#pragma unroll
        for (int j = 0; j < CL; j += 2) {
            float r0, r1, e0, e1;
            asm("{\n.reg .b64 v, s, k, r, e;\nmov.b64 v, {%4, %5};\nmov.b64 s, {%6, %7};\nmov.b64 k, {%8, %8};\n"
                "fma.rn.f32x2 r, v, s, k;\nsub.rn.f32x2 e, k, r;\nfma.rn.f32x2 e, v, s, e;\n"
                "mov.b64 {%0, %1}, r;\nmov.b64 {%2, %3}, e;\n}"
                : "=f"(r0), "=f"(r1), "=f"(e0), "=f"(e1)
                : "f"(value(i, j)), "f"(value(i, j + 1)), "f"(inv[j]), "f"(inv[j + 1]), "f"(kRint));
            c[j] = __float_as_uint(r0), c[j + 1] = __float_as_uint(r1);
            off = fmaxf(off, fmaxf(fabsf(e0), fabsf(e1)));
        }
        if (off > 0.5f - 0x1p-18f)
#pragma unroll
            for (int j = 0; j < CL; ++j)
                c[j] = __float_as_uint(__fdiv_rn(value(i, j), scales[lane * CL + j]) + kRint);
        int8_t* p = q + at + i * step;
        if constexpr (VEC) {
            uint32_t o[CL / 4];
#pragma unroll
            for (int j = 0; j < CL; j += 4)
                o[j / 4] = __byte_perm(__byte_perm(c[j], c[j + 1], 0x0040), __byte_perm(c[j + 2], c[j + 3], 0x0040), 0x5410);
            if constexpr (CL == 8)
                *reinterpret_cast<uint2*>(p) = make_uint2(o[0], o[1]);
            else
                *reinterpret_cast<uint32_t*>(p) = o[0];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < N) p[j] = static_cast<int8_t>(c[j] & 0xff);
        }
    }
}

// ------------------------------------------------------------------ pack
// Once per weight: a thread gathers the 32 k of one channel, lanes lie along
// the channels.
__global__ void __launch_bounds__(kThreads)
    pack_q4_kernel(const int8_t* __restrict__ q, int64_t K, int64_t N, int64_t NC, int64_t NP,
                   int64_t pieces, int block, uint8_t* __restrict__ out, int* err) {
    bool bad = false;
    for (int64_t p = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; p < pieces;
         p += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t blk = p >> 9, kp = blk % NP, nc = blk / NP % NC, g = blk / NP / NC;
        const int64_t n = nc * 128 + (p & 127), k0 = kp * 128 + (p >> 7 & 3) * 32;
        uint32_t word[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            word[j] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t k = k0 + 8 * j + e;
                int v = k < K && n < N ? q[(g * K + k) * N + n] : 0;
                if (v < -7 || v > 7) {
                    bad = true;
                    v = v < 0 ? -7 : 7;
                }
                const uint32_t mag = static_cast<uint32_t>(v < 0 ? -v : v), neg = v < 0 ? 1u : 0u;
                word[j] |= e < 4 ? mag << (8 * e) | neg << (8 * e + 7)
                                 : mag << (8 * (e - 4) + 4) | neg << ((8 * (e - 4) + 11) & 31);
            }
        }
        *reinterpret_cast<uint4*>(out + blk * block + (p & 511) * 16) =
            make_uint4(word[0], word[1], word[2], word[3]);
    }
    if (bad) atomicOr(err, ERR_Q4_VALUE);
}

// s: [G][KB][N]; per block, `per` rows of 128 scales behind the weights.
template <typename ST>
__global__ void __launch_bounds__(kThreads)
    pack_q4_scale_kernel(const ST* __restrict__ s, int64_t KB, int64_t N, int64_t NC, int64_t NP,
                         int64_t total, int per, int block, uint8_t* __restrict__ out) {
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t row = i >> 7, blk = row / per, kp = blk % NP, nc = blk / NP % NC, g = blk / NP / NC;
        const int j = static_cast<int>(row % per);
        const int64_t n = nc * 128 + (i & 127), b = kp * per + j;
        reinterpret_cast<ST*>(out + blk * block + 8192)[j * 128 + (i & 127)] =
            n < N && b < KB ? s[(g * KB + b) * N + n] : ST(0.0f);
    }
}

// ------------------------------------------------------------------ product
using namespace aem::dev;

struct Q4Args {
    const uint8_t* w;
    const void* x;              // the caller's rows (ldx elements apart), for kernels that make the terms
    const uint32_t* tops;       // [M], from the terms kernel
    const uint8_t* cuts;        // [M][NP], from the terms kernel, for rows with bit 31 of tops
    void* out;
    const int32_t* group_rows;  // nullptr: one group of M rows, weight group `group`
    int64_t ldx, ldo, M, N, K;
    int64_t group;
    int* err;
    int NC, NP, G, block, S, rows;  // S: CTAs (one cluster) that split K; rows: rows of a row tile
    bool scale_bf16, out_bf16, relu, vec, ovec;  // vec, ovec: x, out can be moved in vectors of 4
};

// A row's activations as e5m2 terms, three to a window.  Window w holds
// x * rho * 2^(9 w) from 2^16 down to 2^-16, so a float32 row's three reach
// 2^-49 of its largest magnitude.
template <typename XT>
constexpr int kWin = sizeof(XT) == 4 ? 3 : 1;
template <typename XT>
constexpr int kTerms = 3 * kWin<XT>;
// Side by side a float32 row has eight, two in the last window: 16 columns hold
// two rows, and blocks of one row stay 1 KB apart.
template <typename XT>
constexpr int kSide = sizeof(XT) == 4 ? 8 : 3;
// An element whose exponent is further below the largest's may have bits that no
// term holds; they are added apart (cut_sum).
constexpr uint32_t span_of(int terms) { return terms == 9 ? 26 : terms == 8 ? 23 : 24; }

// Four elements of a row from k on, zero past K, as they lie in memory.
template <typename XT>
struct Four {
    uint32_t w[sizeof(XT)];
    // Running minimum of the magnitudes, zeros last; low_of() gives the form that
    // may_be_cut() reads.  bf16 in pairs: a magnitude less one, its sign set, orders
    // as a signed number, and zero becomes the largest.
    static constexpr uint32_t kNoLow = sizeof(XT) == 4 ? ~0u : 0x7fff7fffu;
    __device__ __forceinline__ void any_low(uint32_t& m) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(XT)); ++i)
            m = sizeof(XT) == 4 ? min(m, 2 * w[i] - 1) : __vmins2(m, (w[i] | 0x80008000u) - 0x00010001u);
    }
    __device__ static __forceinline__ uint32_t low_of(uint32_t m) {
        m ^= sizeof(XT) == 4 ? 0u : 0x80008000u;
        return sizeof(XT) == 4 ? m : min(m << 16, m & 0xffff0000u) << 1 | 0x1ffffu;
    }
    // VEC: rows of 4-element vectors, K a multiple of 4
    template <bool VEC>
    __device__ __forceinline__ void load(const XT* row, int64_t k, int64_t K) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(XT)); ++i) w[i] = 0;
        if constexpr (VEC && sizeof(XT) == 4) {
            if (k < K) {
                const uint4 u = *reinterpret_cast<const uint4*>(row + k);
                w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
            }
        } else if constexpr (VEC) {
            if (k < K) {
                const uint2 u = *reinterpret_cast<const uint2*>(row + k);
                w[0] = u.x, w[1] = u.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (k + i < K) {
                    if constexpr (sizeof(XT) == 4)
                        w[i] = __float_as_uint(row[k + i]);
                    else
                        w[i / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(row[k + i])) << (16 * (i & 1));
                }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(XT) == 4) return __uint_as_float(w[i]);
        return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
    // Running maximum of the magnitudes, non-finite ones included, in any form
    // that special() and bits() read.
    __device__ __forceinline__ void any_top(uint32_t& m) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(XT)); ++i)
            m = sizeof(XT) == 4 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
    }
    __device__ static __forceinline__ uint32_t bits(uint32_t m) {
        return sizeof(XT) == 4 ? m : max(m << 16, m & 0xffff0000u);
    }
    __device__ static __forceinline__ bool special(uint32_t m) { return bits(m) >= 0x7f800000u; }
    // Bits of the largest finite magnitude (they order as the magnitudes do).
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = __float_as_uint(get(i)) & 0x7fffffffu;
            if (u < 0x7f800000u) m = max(m, u);
        }
        return m;
    }
};
// rho = 2^up for a row whose top magnitude has these bits; 2^9 / rho.
__device__ __forceinline__ int rho_exponent(uint32_t top) { return 142 - static_cast<int>(top >> 23); }
// Whether the exponent of the smallest magnitude `low` is more than `span` below
// the largest's.
__device__ __forceinline__ bool may_be_cut(uint32_t low, uint32_t top, uint32_t span) {
    return low < (top >> 23 > span ? ((top >> 23) - span << 24) - 1 : 0);
}
__device__ __forceinline__ float unscale_of(uint32_t top) {
    const int e = 9 - rho_exponent(top);  // -133 .. 121
    return __uint_as_float(e >= -126 ? static_cast<uint32_t>(127 + e) << 23 : 1u << (149 + e));
}

// The terms of four elements, one byte each; t[3 w + j] is term j of window w.
// e5m2 is the upper byte of an fp16, so truncating an fp16 by a mask truncates
// the term.  What a window's terms leave of a value goes to the next, 2^9
// larger: three terms take nine significant bits of it or all down to 2^-16, so
// less than 2^7 is left, and all 24 bits are taken unless they end below the
// last window.  Every difference is exact.  An infinity or NaN is all in the
// first term.  REST: also what all terms leave of x * rho * 2^(9 (kWin - 1)).
template <bool REST, typename XT, int TERMS>
__device__ __forceinline__ void terms4(const Four<XT>& x, int up, uint32_t (&t)[TERMS], float (&r)[4]) {
    constexpr int WIN = kWin<XT>;
    // two factors: rho itself may be beyond float32
    const float f1 = __uint_as_float(static_cast<uint32_t>(127 + up / 2) << 23);
    const float f2 = __uint_as_float(static_cast<uint32_t>(127 + up - up / 2) << 23);
    uint32_t special = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = x.get(i);
        r[i] = v * f1 * f2;
        if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) {
            r[i] = 0.0f;
            special |= (v != v ? 0x7fu : v > 0.0f ? 0x7cu : 0xfcu) << (8 * i);
        }
    }
#pragma unroll
    for (int s = 0; s < WIN; ++s) {
        const bool on = REST || s + 1 < WIN;
        uint32_t h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(h[i]) : "f"(r[2 * i + 1]), "f"(r[2 * i]));
            if (on) {
                const __half2 hh = *reinterpret_cast<const __half2*>(&h[i]);
                r[2 * i] -= __low2float(hh);
                r[2 * i + 1] -= __high2float(hh);
            }
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            if (3 * s + j >= TERMS) continue;
            t[3 * s + j] = __byte_perm(h[0], h[1], 0x7531);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t m = h[i] & 0xff00ff00u;
                const __half2 left = __hsub2(*reinterpret_cast<const __half2*>(&h[i]), *reinterpret_cast<const __half2*>(&m));
                h[i] = *reinterpret_cast<const uint32_t*>(&left);
            }
        }
        if (on)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const __half2 left = *reinterpret_cast<const __half2*>(&h[i]);
                r[2 * i] = (r[2 * i] + __low2float(left)) * (s + 1 < WIN ? 512.0f : 1.0f);
                r[2 * i + 1] = (r[2 * i + 1] + __high2float(left)) * (s + 1 < WIN ? 512.0f : 1.0f);
            }
    }
    t[0] |= special;
}

// What TERMS terms leave of four elements of a row whose largest magnitude has
// the bits `top`.
template <int TERMS, typename XT>
__device__ __forceinline__ void cut4(const Four<XT>& x, uint32_t top, float (&r)[4]) {
    const int up = rho_exponent(top);
    uint32_t t[TERMS];
    terms4<true>(x, up, t, r);
    // (what is left has bits of x, and the first product fewer places: exact)
    const float f1 = __uint_as_float(static_cast<uint32_t>(127 - up / 2) << 23);
    const float f2 = __uint_as_float(static_cast<uint32_t>(127 - up + up / 2) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = __float_as_uint(x.get(i)) & 0x7fffffffu;
        // far below the last window, where x * rho may not be a float32 any more
        const bool all = (u >> 23) + 60 < top >> 23;
        r[i] = all ? x.get(i) : r[i] * (kWin<XT> == 3 ? 0x1p-18f : 1.0f) * f1 * f2;
    }
}

// Activations as the products read them: bytes [3][M][kWin][KP] (KP = K rounded
// up to 128, zero padded), tops [M], the bits of a row's largest finite magnitude,
// bit 31 where elements of the row may be cut, and cuts [M][KP / 128] for such a
// row: not zero where those of a block may be.  gridDim.y blocks share a row:
// each reads all of it for the largest magnitude and turns its slots (4 k a
// thread) into terms.  32 rows of 14336: done 2.4 us after the first block's
// start; one block of 1024 threads a row took 4.3 and kept whole SMs from the
// product's CTAs.
template <typename XT, bool VEC>
__global__ void __launch_bounds__(512)
    q4_terms_kernel(const XT* __restrict__ x, int64_t ldx, int64_t K, int64_t KP,
                    uint8_t* __restrict__ out, uint32_t* __restrict__ row_tops, uint8_t* __restrict__ cuts) {
    constexpr int TERMS = kTerms<XT>, WIN = kWin<XT>, HELD = 8;  // slots that stay in registers
    const int nt = blockDim.x, P = gridDim.y, y = blockIdx.y;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ uint32_t tops[16], lows[16];
    const XT* row = x + blockIdx.x * ldx;
    Four<XT> v[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) v[i].template load<VEC>(row, (i * nt + threadIdx.x) * 4ll, K);
    uint32_t top = 0, low = Four<XT>::kNoLow;
#pragma unroll
    for (int i = 0; i < HELD; ++i) v[i].any_top(top);
#pragma unroll
    for (int i = 0; i < HELD; ++i) v[i].any_low(low);
    if (Four<XT>::special(top)) {
        top = 0;
#pragma unroll
        for (int i = 0; i < HELD; ++i) top = max(top, v[i].top());
    } else {
        top = Four<XT>::bits(top);
    }
    for (int64_t k = (HELD * nt + threadIdx.x) * 4ll; k < K; k += nt * 4) {
        Four<XT> u;
        u.template load<VEC>(row, k, K);
        top = max(top, u.top());
        u.any_low(low);
    }
    low = __reduce_min_sync(~0u, Four<XT>::low_of(low));
    top = __reduce_max_sync(~0u, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top, lows[threadIdx.x >> 5] = low;
    __syncthreads();
    top = __reduce_max_sync(~0u, tops[threadIdx.x & (nt / 32 - 1)]);
    const int up = rho_exponent(top);
    const bool cut = may_be_cut(__reduce_min_sync(~0u, lows[threadIdx.x & (nt / 32 - 1)]), top, span_of(TERMS));
    if (threadIdx.x == 0 && y == 0) row_tops[blockIdx.x] = top | (cut ? 1u << 31 : 0u);
    auto put = [&](int64_t k, const Four<XT>& u) {
        uint32_t t[TERMS];
        float rest[4];
        terms4<false>(u, up, t, rest);
        if (cut) {  // a warp has a block
            uint32_t m = Four<XT>::kNoLow;
            u.any_low(m);
            const bool any = __any_sync(~0u, may_be_cut(Four<XT>::low_of(m), top, span_of(TERMS)));
            if ((threadIdx.x & 31) == 0) cuts[blockIdx.x * (KP >> 7) + (k >> 7)] = any;
        }
#pragma unroll
        for (int j = 0; j < TERMS; ++j)
            *reinterpret_cast<uint32_t*>(
                out + ((j % 3 * static_cast<int64_t>(gridDim.x) + blockIdx.x) * WIN + j / 3) * KP + k) = t[j];
    };
    int next = y;  // this block's next slot
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (i != next) continue;
        next += P;
        const int64_t k = (i * nt + threadIdx.x) * 4ll;
        if (k < KP) put(k, v[i]);
    }
    for (int64_t k = (static_cast<int64_t>(next) * nt + threadIdx.x) * 4; k < KP; k += P * nt * 4ll) {
        Four<XT> u;
        u.template load<VEC>(row, k, K);
        put(k, u);
    }
}

// Row tile `slot` of the groups' row tiles: its group, first row and rows.
// Every warp searches alike.  Offsets are clamped to [0, M].
__device__ __forceinline__ bool find_rows(const Q4Args& a, int slot, int64_t* g, int64_t* m0, int* rows) {
    if (!a.group_rows) {
        *g = a.group;
        *m0 = static_cast<int64_t>(slot) * a.rows;
        *rows = static_cast<int>(min(static_cast<int64_t>(a.rows), a.M - *m0));
        return *rows > 0;
    }
    const int lane = threadIdx.x & 31, M = static_cast<int>(a.M);
    int lo[8], hi[8];  // all offsets on their way at once
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo[i] = hi[i] = 0;
        if (i * 32 + lane < a.G) {
            lo[i] = a.group_rows[i * 32 + lane];
            hi[i] = a.group_rows[i * 32 + lane + 1];
        }
    }
    int before = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i * 32 >= a.G) break;
        lo[i] = min(max(lo[i], 0), M);
        hi[i] = min(max(hi[i], 0), M);
        const int n = hi[i] > lo[i] ? (hi[i] - lo[i] + a.rows - 1) / a.rows : 0;
        int s = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, s, o);
            if (lane >= o) s += v;
        }
        const int first = before + s - n;
        const unsigned hit = __ballot_sync(~0u, slot >= first && slot < first + n);
        if (hit) {
            const int l = __ffs(hit) - 1;
            const int m = lo[i] + (slot - first) * a.rows;
            *g = i * 32 + l;
            *m0 = __shfl_sync(~0u, m, l);
            *rows = __shfl_sync(~0u, min(a.rows, hi[i] - m), l);
            return true;
        }
        before += __shfl_sync(~0u, s, 31);
    }
    return false;
}

__device__ __forceinline__ void st_cluster(const float4* p, uint32_t rank, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mapa_u32(p, rank)), "f"(v.x),
                 "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}

__device__ __forceinline__ void store_out(const Q4Args& a, int64_t m, int64_t n, float4 v) {
    if (a.relu) {
        v.x = v.x < 0.0f ? 0.0f : v.x, v.y = v.y < 0.0f ? 0.0f : v.y;
        v.z = v.z < 0.0f ? 0.0f : v.z, v.w = v.w < 0.0f ? 0.0f : v.w;
    }
    const int64_t at = m * a.ldo + n;
    if (a.ovec && n + 3 < a.N) {
        if (a.out_bf16) {
            __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = *reinterpret_cast<uint2*>(h);
        } else {
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = v;
        }
        return;
    }
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (n + j >= a.N) return;
        if (a.out_bf16)
            static_cast<__nv_bfloat16*>(a.out)[at + j] = __float2bfloat16_rn(e[j]);
        else
            static_cast<float*>(a.out)[at + j] = e[j];
    }
}

// a0 += s * v0, a1 += s * v1
__device__ __forceinline__ void fma2(float& a0, float& a1, float s, uint32_t v0, uint32_t v1) {
    asm("{\n.reg .b64 a, s, v;\nmov.b64 a, {%0, %1};\nmov.b64 s, {%2, %2};\nmov.b64 v, {%3, %4};\n"
        "fma.rn.f32x2 a, s, v, a;\nmov.b64 {%0, %1}, a;\n}"
        : "+f"(a0), "+f"(a1)
        : "f"(s), "r"(v0), "r"(v1));
}

// What TERMS terms leave of a row, times the weights: the sums of four channels a
// lane over blocks p, p + step, ... of the CTA's np (at w; x their elements, k of
// them at most), in float32.  cuts, if given, says which blocks may have anything.
template <int TERMS, typename XT>
__device__ __forceinline__ float4 cut_sum(const XT* x, int64_t k, const uint8_t* cuts, const uint8_t* w, int p, int step,
                                          int np, int block, bool scale_bf16, uint32_t top) {
    const int lane = threadIdx.x & 31, gs = 128 * 128 * (scale_bf16 ? 2 : 4) / (block - 8192);
    float sum[4] = {};
    for (; p < np; p += 32 * step) {
        unsigned on = 0;  // bit i: block p + i * step may have something
        if (cuts) {
            on = __ballot_sync(~0u, p + lane * step < np && cuts[p + lane * step]);
        } else {
#pragma unroll 4
            for (int i = 0; i < 32 && p + i * step < np; ++i) {
                Four<XT> v;
                uint32_t low = Four<XT>::kNoLow;
                v.template load<false>(x, (p + i * step) * 128 + lane * 4, k);
                v.any_low(low);
                on |= __any_sync(~0u, may_be_cut(Four<XT>::low_of(low), top, span_of(TERMS))) ? 1u << i : 0u;
            }
        }
        for (; on; on &= on - 1) {
            const int at = p + (__ffs(on) - 1) * step;
            const uint8_t* blk = w + static_cast<int64_t>(at) * block;
            Four<XT> v;
            float r[4];
            v.template load<false>(x, at * 128 + lane * 4, k);
            cut4<TERMS>(v, top, r);
            const unsigned any = __ballot_sync(~0u, r[0] != 0.0f || r[1] != 0.0f || r[2] != 0.0f || r[3] != 0.0f);
            for (int i = 0; i < 4; ++i) {  // 32 k, eight lanes
                if (!(any >> 8 * i & 0xff)) continue;
                uint4 q[4];
                float s[4], part[4] = {};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int ch = lane * 4 + j, sc = i * 32 / gs * 128 + ch;
                    q[j] = *reinterpret_cast<const uint4*>(blk + i * 2048 + ch * 16);
                    s[j] = scale_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(blk + 8192)[sc])
                                      : reinterpret_cast<const float*>(blk + 8192)[sc];
                }
                for (int b = 0; b < 32; b += 4) {
                    if (!(any >> (8 * i + b / 4) & 1)) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float re = __shfl_sync(~0u, r[e], i * 8 + b / 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t lo = b & 8 ? q[j].y : q[j].x, hi = b & 8 ? q[j].w : q[j].z;
                            const uint32_t word = b & 16 ? hi : lo, mag = word >> (8 * e + (b & 4)) & 7;
                            const uint32_t neg = word >> (8 * e + (b & 4 ? 11 : 7) & 31) & 1;
                            part[j] = fmaf(s[j] * (neg ? -static_cast<float>(mag) : static_cast<float>(mag)), re, part[j]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += part[j];
            }
        }
    }
    return make_float4(sum[0], sum[1], sum[2], sum[3]);
}

// The end of a CTA, once the warpgroups' sums `fin` [2][ROWS][128] are in shared
// memory: rank ks sends its rows' sums to the ranks that write them, which add
// them in rank order in `recv` [S][share].  CUT: `cut` [ways of a row][128] holds
// what to add to a row, in `ways` parts.
struct Q4Sums {
    const float* fin;
    float *recv, *cut;
    const uint32_t* row_top;
    const uint8_t *cuts, *src;
    int64_t m0;
    int stride, rows, tile, ks, p0, np;
};
constexpr int kQ4Warps = 12, kQ4Threads = 32 * kQ4Warps;
template <int ROWS, bool CUT>
__device__ __forceinline__ void send_sums(const Q4Args& a, const Q4Sums& z, int ways) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int share = (z.rows + a.S - 1) / a.S;  // rows that a rank writes
    const int64_t n = z.tile * 128ll + lane * 4;  // a warp has a row, a lane four channels of it
    const float4* fin4 = reinterpret_cast<const float4*>(z.fin) + lane;
    float4* recv4 = reinterpret_cast<float4*>(z.recv) + lane;
    for (int c = w, to = 0, r = c; c < z.rows; c += kQ4Warps, r += kQ4Warps) {
        while (r >= share) r -= share, ++to;  // row c is row r of rank `to`
        const float4 u = fin4[c * 32], v = fin4[(ROWS + c) * 32];
        const float f = unscale_of(z.row_top[c] & 0x7fffffffu);
        float4 o = make_float4((u.x + v.x) * f, (u.y + v.y) * f, (u.z + v.z) * f, (u.w + v.w) * f);
        if constexpr (CUT)
            for (int i = 0; i < ways; ++i) {
                const float4 t = reinterpret_cast<const float4*>(z.cut)[(c * ways + i) * 32 + lane];
                o.x += t.x, o.y += t.y, o.z += t.z, o.w += t.w;
            }
        float4* p = recv4 + (z.ks * share + r) * 32;
        if (a.S > 1 && to != z.ks)
            st_cluster(p, to, o);
        else if (a.S > 1)
            *p = o;
        else
            store_out(a, z.m0 + c, n, o);
    }
    if (a.S == 1) return;
    cluster_sync();
    for (int r = w; r < share && z.ks * share + r < z.rows; r += kQ4Warps) {
        float4 v = recv4[r * 32];
        for (int s = 1; s < a.S; ++s) {
            const float4 u = recv4[(s * share + r) * 32];
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        store_out(a, z.m0 + z.ks * share + r, n, v);
    }
}
// The same where the terms may not hold all of a row, first the sums of what they
// leave: a warp has a row, or few rows' blocks go to several.  This is rare (8
// rows or more of 4096 x 14336 with one such element: 3 us more; rows of them, 30
// each).  A call that nothing outlives leaves the kernel's registers alone:
// as part of the loop above it cost every CTA 1 us.
template <typename XT, int ROWS, int TERMS>
__device__ __noinline__ void send_sums_and_cuts(const Q4Args& a, Q4Sums z) {
    const int lane = threadIdx.x & 31, ways = z.rows < kQ4Warps ? kQ4Warps / z.rows : 1;
    for (int i = threadIdx.x >> 5; i < z.rows * ways; i += kQ4Warps) {
        const int c = i / ways;
        const uint32_t top = z.row_top[c] & 0x7fffffffu;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (!z.cuts || z.row_top[c] != top)
            sum = cut_sum<TERMS>(static_cast<const XT*>(a.x) + (z.m0 + c) * a.ldx + z.p0 * 128ll, a.K - z.p0 * 128ll,
                                 z.cuts ? z.cuts + c * static_cast<int64_t>(z.stride) : nullptr, z.src, i - c * ways,
                                 ways, z.np, a.block, a.scale_bf16, top);
        reinterpret_cast<float4*>(z.cut)[i * 32 + lane] = sum;
    }
    __syncthreads();
    send_sums<ROWS, true>(a, z, ways);
}

// Shape of the product kernel: COLS MMA columns, scale groups of GS k, a row's
// TN * TK terms in TN columns, TK after one another (TK == 1: all side by side,
// window after window; else a column a window).  A block of the packed
// weight is 128 channels x 128 k; a unit is what a warpgroup hands to the
// tensor core at once: a block, with one accumulator per scale group side by
// side, or a half or quarter where a block's accumulators would not fit.  Two
// CTAs share an SM, so that one's set-up and end lie under the other's products,
// or a CTA has one to itself (ALONE) with room for two units in tensor memory
// and twice the registers: 32 rows, 4096 x 14336: 17.6 us shared, 15.7 alone; 64
// rows 25.0 as two shared tiles, 18.1 as one alone.  Few rows share: alone, one
// row takes 0.4 us more and four 5 more, where the stream is the bound and more
// CTAs ask for it.  With TK == 1 (few rows) the CTA makes the terms of its part
// of K itself and keeps them in shared memory; otherwise a terms kernel has made
// them and they come in a ring of their own.
template <int COLS, int GS, int ROWS, int TN, int TK, bool ALONE>
struct Q4Cfg {
    static constexpr bool XIN = TK == 1;
    static constexpr int CTAS = ALONE ? 1 : 2;         // on an SM
    static constexpr int TW = 256 / CTAS;              // TMEM columns of a warpgroup
    static constexpr int FULL = GS == 128 ? 1 : 128 / GS;  // scale groups of a block
    static constexpr bool QUEUE = ALONE;               // a unit's MMAs queue behind the last one's
    static constexpr int UB = QUEUE ? 2 : 1;           // units that tensor memory has to hold
    static constexpr int UK = UB * (32 + FULL * COLS) <= TW ? 128   // k of a unit
                              : UB * (16 + (64 / GS ? 64 / GS : 1) * COLS) <= TW ? 64 : 32;
    static constexpr int SUB = UK / GS;                // accumulators per unit
    static constexpr int UA = UK / 4;                  // columns of a unit's weights
    static constexpr int ND = UA + 2 * SUB * COLS <= TW ? 2 : 1;  // buffers of accumulators,
    static constexpr int NA = QUEUE || (ND == 1 && !XIN) ? 2 : 1;  // of weights
    static constexpr bool LATE = ND == 1 && NA == 1;   // weights unpacked after the sums are taken
    static constexpr int NB = QUEUE ? 2 : 1;           // units under way: their barriers
    static constexpr int XB = TK * COLS * 128;         // activation bytes of a block
    // XIN: bytes between the blocks' terms.  A tile of at most 8 columns takes
    // 1 KB; the MMA's other 8 columns, never read back, are then the next
    // block's bytes
    static constexpr int XSTEP = ROWS * TN <= 8 ? 1024 : XB;
    static constexpr int MAXP = XSTEP == 1024 ? 32 : 24;  // XIN: blocks whose terms are kept
    static constexpr int XRES = XIN ? MAXP * XSTEP : 0;
    static constexpr int WB = 8192 + (FULL * 512 + 1023) / 1024 * 1024;  // a block of weights and scales
    // the cluster's sums: S shares of ceil(rows / S) rows, for any S up to 8
    static constexpr int shares() {
        int most = 0;
        for (int rows = 1; rows <= ROWS; ++rows)
            for (int s = 1; s <= 8; ++s) most = s * ((rows + s - 1) / s) > most ? s * ((rows + s - 1) / s) : most;
        return most;
    }
    static constexpr int RECV = shares() * 128 * 4;
    // Even rings: a stage always comes back to the warpgroup that saw its
    // previous phase, so no parity wait can mistake a phase for the one two
    // back.  Activations stay in theirs until the MMAs are done, weights only
    // until they are read.
    static constexpr int NX = XIN ? 0 : 4;
    static constexpr int MOST = CTAS == 2 ? 113 * 1024 : 226 * 1024;
    static constexpr int FIT = (MOST - 2048 - XRES - RECV - NX * XB) / WB / 2 * 2;
    static constexpr int NW = FIT > 8 ? 8 : FIT;
    static constexpr int USED = 1024 + NW * WB + NX * XB + XRES + RECV + (2 * (NW + NX) + 9) * 8 + 12 + ROWS * 4;
    // so many CTAs on an SM and no more: no CTA ever waits for tensor memory
    static constexpr int LEAST = CTAS == 2 ? 78 * 1024 : 116 * 1024;
    static constexpr int SMEM = USED > LEAST ? USED : LEAST;
    static_assert(NA * UA + ND * SUB * COLS <= TW && NW >= 4 && SMEM <= MOST, "budgets");
    static_assert(ROWS * TN <= COLS && SUB >= 1, "a scale group inside a unit");
    static_assert(NW * WB >= ROWS * 1024, "the warpgroups' sums fit the ring");
    static_assert(XRES + NX * XB >= (ROWS < 12 ? 12 : ROWS) * 512, "what is added to them fits the activations'");
};
constexpr int kSMs = 148;

// A CTA computes 128 channels of one row tile over its part of K:
//   warps 0-7   two warpgroups, thread = channel = TMEM lane, that take the
//               weight's blocks in turn.  Per unit: the channel's 4-bit
//               weights come from the shared-memory ring and go to tensor
//               memory as e4m3 codes (8 columns per 32 k) once the MMAs of
//               the unit before are done; then that unit's accumulators come
//               back, a row's terms are added and scale * sum is added to the
//               row's float32 register.
//   warps 8-9   one per warpgroup, issue its MMAs (M = 128 channels, N =
//               columns, K = 32); one commit per unit.
//   warp 10     copies the weights with their scales, one bulk copy per block.
//   warp 11     copies the activations' terms, one TMA box per block
//               (128-byte swizzle), where the CTA does not make them itself.
// Two accumulator buffers let the sums be taken back under the next unit's
// MMAs.  Where only one fits, a second buffer of weights lets the next unit be
// unpacked under them, and it is handed over once the sums are taken.  The
// CTAs with an SM to themselves have two of both: a unit's MMAs queue up behind
// those of the one before.
// The S CTAs of a cluster take parts of K: each sends its sums to the rank
// that writes those outputs, which adds them in rank order.
// Every wait is bounded; a timeout sets the error word and ends all roles.
template <typename XT, int COLS, int GS, int ROWS, int TN, int TK, bool ALONE>
__global__ void __launch_bounds__(kQ4Threads, ALONE ? 1 : 2)
    q4_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ Q4Args a) {
    using C = Q4Cfg<COLS, GS, ROWS, TN, TK, ALONE>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* xres = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    uint8_t* xring = xres + C::XRES;
    uint8_t* ring = xring + C::NX * C::XB;
    float* recv = reinterpret_cast<float*>(ring + C::NW * C::WB);  // [S][share of ROWS * 128]
    uint64_t* w_full = reinterpret_cast<uint64_t*>(recv + C::RECV / 4);
    uint64_t* w_empty = w_full + C::NW;
    uint64_t* x_full = w_empty + C::NW;
    uint64_t* x_empty = x_full + C::NX;
    uint64_t* a_full = x_empty + C::NX;   // [2][2]: a unit's weights are in tensor memory
    uint64_t* done = a_full + 4;          // [2][2]: its MMAs have finished
    uint64_t* x_made = done + 4;          // XIN: the terms are in shared memory
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(x_made + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* any_cut = abort_flag + 1;  // the terms may not hold all of a row
    uint32_t* row_top = tmem_slot + 3;    // [ROWS]: the rows' tops

    constexpr int NX = C::XIN ? 1 : C::NX;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int tile = static_cast<int>(blockIdx.x) / a.S, ks = static_cast<int>(blockIdx.x) % a.S;
    int64_t g, m0;
    int rows;
    if (!find_rows(a, blockIdx.y, &g, &m0, &rows)) {  // the whole cluster alike
        if (!C::XIN) asm volatile("griddepcontrol.wait;" ::: "memory");  // this grid ends after the terms kernel
        return;
    }
    const int p0 = a.NP * ks / a.S, np = a.NP * (ks + 1) / a.S - p0;

    // XIN: a warp takes 128 k of a row, a lane four of them.  These loads go out
    // ahead of the weights, behind which they would wait for microseconds.
    constexpr int HELD = C::XIN ? (ROWS * C::MAXP + 7) / 8 : 1;
    Four<XT> xv[HELD];
    if (C::XIN && w < 8) {
        const XT* x = static_cast<const XT*>(a.x) + m0 * a.ldx + static_cast<int64_t>(p0) * 128 + lane * 4;
        const int64_t left = a.K - static_cast<int64_t>(p0) * 128 - lane * 4;
        auto load = [&](auto vec) {
            int r = 0, p = w;
#pragma unroll
            for (int h = 0; h < HELD; ++h, p += 8) {
                while (p >= np) p -= np, ++r;
                if (r >= rows) break;
                xv[h].template load<decltype(vec)::value>(x + r * a.ldx, p * 128, left);
            }
        };
        if (a.vec)
            load(std::true_type{});
        else
            load(std::false_type{});
    }
    const uint8_t* src = a.w + ((g * a.NC + tile) * a.NP + p0) * static_cast<int64_t>(a.block);
    auto copy_weights = [&](int p) {
        uint64_t* full = &w_full[p % C::NW];
        mbar_arrive_expect_tx(full, a.block);
        bulk_load(ring + p % C::NW * C::WB, src + static_cast<int64_t>(p) * a.block, a.block, full);
    };
    if (w == 9) {
        tmem_alloc(tmem_slot, 2 * C::TW);
        tmem_relinquish();
    } else if (w == 10 && lane == 0) {
        // the first weights are on their way before the rest of the set-up
        for (int i = 0; i < C::NW; ++i) {
            mbar_init(&w_full[i], 1);
            mbar_init(&w_empty[i], 4);  // the four warps of the block's warpgroup
        }
        for (int i = 0; i < C::NX; ++i) {
            mbar_init(&x_full[i], 1);
            mbar_init(&x_empty[i], 4);
        }
        for (int j = 0; j < 4; ++j) {
            mbar_init(&a_full[j], 4);
            mbar_init(&done[j], 1);
        }
        mbar_init(x_made, 8);
        *abort_flag = *any_cut = 0;
        fence_barrier_init();
        for (int p = 0; p < min(np, C::NW); ++p) copy_weights(p);
    } else if (w == 11) {
        if (C::XIN && lane < ROWS) row_top[lane] = 0;
        if (!C::XIN && lane == 0) tma_prefetch_desc(&xmap);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // the ranks' shared memory may be written from here on (waited for below)
    if (a.S > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    const int wg = w < 8 ? w >> 2 : w & 1;  // the warpgroup a channel or MMA warp belongs to
    const uint32_t td = tmem + static_cast<uint32_t>(wg * C::TW);  // accumulators, then the unit's weights
    const uint32_t ta = td + C::ND * C::SUB * COLS;
    a_full += 2 * wg;
    done += 2 * wg;
    auto wait = [&](uint64_t* bar, int phase) {  // whole warps
        if (__all_sync(~0u, mbar_try_wait(bar, phase & 1))) return true;
        return __all_sync(~0u, mbar_wait_bounded(bar, phase & 1, abort_flag, a.err, ERR_GEMM_TIMEOUT)) != 0;
    };

    float acc[ROWS] = {};
    const int ch = threadIdx.x & 127;
    if (w < 8) {
        if constexpr (C::XIN) {
            // terms of rows x [128 p0, 128 (p0 + np)), relative to the largest
            // magnitude in that part of the row
            int r = 0, p = w;
#pragma unroll
            for (int h = 0; h < HELD; ++h, p += 8) {
                while (p >= np) p -= np, ++r;
                if (r >= rows) break;
                const uint32_t top = __reduce_max_sync(~0u, xv[h].top());
                if (lane == 0) atomicMax(&row_top[r], top);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            bool cut = false;
            r = 0, p = w;
#pragma unroll
            for (int h = 0; h < HELD; ++h, p += 8) {
                while (p >= np) p -= np, ++r;
                if (r >= rows) break;
                uint32_t t[TN];
                const uint32_t top = row_top[r];
                uint32_t low = Four<XT>::kNoLow;
                xv[h].any_low(low);
                cut |= may_be_cut(Four<XT>::low_of(low), top, span_of(TN));
                float rest[4];
                terms4<false>(xv[h], rho_exponent(top), t, rest);
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const int col = r * TN + j;  // a 128-byte row of the swizzled tile
                    *reinterpret_cast<uint32_t*>(xres + p * C::XSTEP + col * 128 +
                                                 (((lane >> 2) ^ (col & 7)) << 4) + (lane & 3) * 4) = t[j];
                }
            }
            fence_proxy_async_smem();
            if (cut) *any_cut = 1;
            __syncwarp();
            if (lane == 0) mbar_arrive(x_made);
        }
        const uint32_t quarter = static_cast<uint32_t>(32 * (w & 3)) << 16;
        // columns taken back at once, PER of an accumulator
        constexpr int TC = C::SUB * COLS, CH = COLS % 48 == 0 ? 48 : TC == 16 ? 16 : 32, PER = COLS < CH ? COLS : CH;
        constexpr int WIN = kWin<XT>, SIDE = C::XIN ? 3 : 1;  // terms of a window side by side
        auto take = [&](int u, const float (&s)[C::SUB]) {  // unit u's sums, scaled
#pragma unroll
            for (int c0 = 0; c0 < TC; c0 += CH) {
                uint32_t r[CH];
                const uint32_t at = td + quarter + u % C::ND * TC + c0;
                if constexpr (CH == 16) {
                    tc_ld_32x32b_x16(at, r);
                } else if constexpr (CH == 32 && PER == 32 && ROWS * TN <= 24) {
                    tc_ld_32x32b_x16(at, *reinterpret_cast<uint32_t(*)[16]>(r));
                    tc_ld_32x32b_x8(at + 16, *reinterpret_cast<uint32_t(*)[8]>(r + 16));
                } else if constexpr (CH == 32) {
                    tc_ld_32x32b_x32(at, r);
                } else {
                    tc_ld_32x32b_x32(at, *reinterpret_cast<uint32_t(*)[32]>(r));
                    tc_ld_32x32b_x16(at + 32, *reinterpret_cast<uint32_t(*)[16]>(r + 32));
                }
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < CH / PER * (PER / TN); ++i) {  // PER columns hold PER / TN whole rows
                    const int c = i / (PER / TN) * PER + i % (PER / TN) * TN, row = (c0 + c) % COLS / TN;
                    if (row >= ROWS) continue;
                    if constexpr (TN == 1) {  // two rows an instruction
                        if (i % 2 == 0) fma2(acc[row], acc[row + 1], s[(c0 + c) / COLS], r[c], r[c + 1]);
                        continue;
                    }
                    float v = 0.0f;
#pragma unroll
                    for (int win = WIN - 1; win >= 0; --win) {
                        float a = __uint_as_float(r[c + win * SIDE]);
#pragma unroll
                        for (int t = 1; t < SIDE && win * SIDE + t < TN; ++t) a += __uint_as_float(r[c + win * SIDE + t]);
                        v = win == WIN - 1 ? a : fmaf(v, 0x1p-9f, a);
                    }
                    acc[row] = fmaf(s[(c0 + c) / COLS], v, acc[row]);
                }
            }
            tc_fence_before();
        };
        float s_prev[C::SUB];
        int u = 0;  // units of this warpgroup so far
        bool ok = true;
        for (int p = wg; ok && p < np; p += 2) {
            const uint8_t* st = ring + p % C::NW * C::WB;
            if (!(ok = wait(&w_full[p % C::NW], p / C::NW))) break;
            float s[C::FULL];
#pragma unroll
            for (int j = 0; j < C::FULL; ++j)
                s[j] = a.scale_bf16
                           ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(st + 8192)[j * 128 + ch])
                           : reinterpret_cast<const float*>(st + 8192)[j * 128 + ch];
#pragma unroll
            for (int j = 0; j < 128 / C::UK; ++j) {
                uint4 q[C::UK / 32];
#pragma unroll
                for (int i = 0; i < C::UK / 32; ++i)
                    q[i] = *reinterpret_cast<const uint4*>(st + (j * (C::UK / 32) + i) * 2048 + ch * 16);
                uint32_t v[C::UA];
                auto unpack = [&]() {
#pragma unroll
                    for (int i = 0; i < C::UK / 32; ++i) {
                        const uint32_t word[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[8 * i + 2 * e] = word[e] & 0x87878787u;
                            v[8 * i + 2 * e + 1] = __funnelshift_r(word[e], word[e], 4) & 0x87878787u;
                        }
                    }
                    if (j == 128 / C::UK - 1) {  // the block has been read
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&w_empty[p % C::NW]);
                    }
                };
                auto put = [&]() {
                    const uint32_t to = ta + quarter + u % C::NA * C::UA;
                    if constexpr (C::UA == 32)
                        tc_st_32x32b_x32(to, v);
                    else if constexpr (C::UA == 16)
                        tc_st_32x32b_x16(to, v);
                    else
                        tc_st_32x32b_x8(to, v);
                };
                auto hand_over = [&]() {
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&a_full[u % C::NB]);
                };
                // With two buffers of weights, unit u - 2's is free: its MMAs
                // were waited for a unit ago.
                if (!C::LATE) unpack();
                if (C::NA == 2) put();
                if (C::QUEUE) hand_over();
                if (u) {
                    // the unit before is done: its weights' columns, its
                    // accumulators and (at a block's start) its activations are free
                    if (!(ok = wait(&done[(u - 1) % C::NB], (u - 1) / C::NB))) break;
                    tc_fence_after();
                    if (!C::XIN && j == 0 && lane == 0) mbar_arrive(&x_empty[(p - 2) % NX]);
                    if (C::ND == 1 || C::QUEUE) take(u - 1, s_prev);
                }
                if (C::LATE) unpack();
                if (C::NA == 1) put();
                if (!C::QUEUE) hand_over();
                if (C::ND == 2 && !C::QUEUE && u) take(u - 1, s_prev);
#pragma unroll
                for (int i = 0; i < C::SUB; ++i) s_prev[i] = s[j * C::SUB + i];
                ++u;
            }
        }
        if (ok && u && wait(&done[(u - 1) % C::NB], (u - 1) / C::NB)) {
            tc_fence_after();
            take(u - 1, s_prev);
        }
    } else if (w < 10) {
        const uint32_t idesc = idesc_e4m3_e5m2_f32(128, static_cast<uint32_t>((rows * TN + 15) & ~15));
        int u = 0;
        bool ok = !C::XIN || wait(x_made, 0);
        for (int p = wg; ok && p < np; p += 2) {
            if (!C::XIN && !(ok = wait(&x_full[p % NX], p / NX))) break;
            const uint64_t bd = smem_desc_sw128(smem_u32(C::XIN ? xres + p * C::XSTEP : xring + p % NX * C::XB));
#pragma unroll
            for (int j = 0; j < 128 / C::UK; ++j) {
                if (!(ok = wait(&a_full[u % C::NB], u / C::NB))) break;
                tc_fence_after();
                const uint32_t d = td + static_cast<uint32_t>(u % C::ND * C::SUB * COLS);
#pragma unroll
                for (int m = 0; m < C::UK / 32; ++m)
#pragma unroll
                    for (int t = 0; t < TK; ++t)
                        tc_mma_f8_ts_elect(d + 32 * m / GS * COLS, ta + u % C::NA * C::UA + 8 * m,
                                           bd + t * (COLS * 8) + 2 * (j * (C::UK / 32) + m), idesc,
                                           32 * m % GS || t ? 1u : 0u);
                tc_commit_elect(&done[u % C::NB]);
                ++u;
            }
        }
    } else if (w == 10 || !C::XIN) {
        const bool weights = w == 10;
        if (!weights) {  // the terms and the tops are the terms kernel's
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (int r = lane; r < rows; r += 32) {
                row_top[r] = a.tops[m0 + r];
                if (row_top[r] >> 31) *any_cut = 1;
            }
        }
        const int ns = weights ? C::NW : C::NX;
        uint64_t *full = weights ? w_full : x_full, *empty = weights ? w_empty : x_empty;
        int p = lane != 0 ? np : weights ? min(np, C::NW) : 0;
        for (int at = 0, phase = weights ? 0 : 1; p < np; ++p) {
            if (!mbar_wait_bounded(&empty[at], phase, abort_flag, a.err, ERR_GEMM_TIMEOUT)) break;
            if (weights) {
                copy_weights(p);
            } else {
                mbar_arrive_expect_tx(&full[at], C::XB);
                tma_load_3d(xring + at * C::XB, &xmap, &full[at], (p0 + p) * 128, static_cast<int>(m0 * TN), 0);
            }
            if (++at == ns) at = 0, phase ^= 1;
        }
        if (lane == 0 && *abort_flag)  // a failed call leaves no copy in flight behind (bounded as well)
            for (int i = max(0, p - ns); i < p; ++i)
                for (int t = 0; t < 1 << 14 && !mbar_try_wait(&full[i % ns], i / ns & 1); ++t) {
                }
    }

    // every MMA has been waited for by the channel warps (or the call failed):
    // give the tensor memory back before any wait on another CTA
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (w == 9) tmem_dealloc(tmem, 2 * C::TW);
    // (This end runs once per CTA, from a cold instruction cache: the sums leave
    // the registers in one short unrolled piece and the rest is a loop.)
    float* fin = reinterpret_cast<float*>(ring);  // [2][ROWS][128]: the warpgroups' sums
    if (w < 8)
#pragma unroll
        for (int c = 0; c < ROWS; ++c) fin[(wg * ROWS + c) * 128 + ch] = acc[c];
    __syncthreads();
    if (a.S > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const Q4Sums z{fin, recv, reinterpret_cast<float*>(xres), row_top, C::XIN ? nullptr : a.cuts + m0 * a.NP + p0, src, m0, a.NP,
                   rows, tile, ks, p0, np};
    if (*any_cut)
        send_sums_and_cuts<XT, ROWS, TN * TK>(a, z);
    else
        send_sums<ROWS, false>(a, z, 0);
}

template <typename XT, int COLS, int GS, int ROWS, int TN, int TK, bool ALONE>
aem_status launch_q4(const CUtensorMap& xmap, const Q4Args& a, dim3 grid, cudaStream_t s) {
    using C = Q4Cfg<COLS, GS, ROWS, TN, TK, ALONE>;
    auto kern = q4_kernel<XT, COLS, GS, ROWS, TN, TK, ALONE>;
    static std::atomic<uint64_t> ready{0};  // bit per device: the shared memory opt-in is done
    const uint64_t bit = 1ull << (current_device() & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        AEM_TRY_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kQ4Threads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    int n = 0;
    if (!C::XIN) {  // starts under the terms kernel
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (a.S > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = a.S;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    AEM_TRY_CUDA(cudaLaunchKernelEx(&cfg, kern, xmap, a));
    count_launches(1);
    return AEM_OK;
}

// CTAs (at most 8, one cluster) that split K.  In blocks of a CTA that shares
// its SM, a CTA's set-up and end take about 14; one with the SM to itself does
// its blocks in 0.64 of the time and starts 1.5 sooner.  16 rows, 4096 x 4096:
// 4 CTAs (128 in all) 9.8 us, 8 CTAs 10.8; 14336 x 4096: 4 CTAs 19.1, 8 CTAs
// 17.2.  The wide tiles (`alone`) have an SM each and a wave costs 20 of their
// blocks: 32 rows, 14336 x 4096: 2, 3, 4, 5 CTAs 23.9, 18.8, 16.6, 25.2 us.
// Wide clusters leave slots of a GPC empty, more of them while blocks of the
// terms kernel hold some: 32 clusters of 8 took 19.4 us where 7 took 14.6
// (14336 x 4096, 4 float32 rows), so not all slots are counted on.
int split_k(int64_t ctas, int64_t blocks, int64_t most_blocks, bool terms, bool alone) {
    int best = 8;
    int64_t least = INT64_MAX;
    for (int S = 1; S <= 8; ++S) {
        const int64_t each = (blocks + S - 1) / S, n = ctas * S;
        if (each > most_blocks || (S > 1 && each < 2)) continue;
        const int64_t slots = alone ? (S == 3 ? 132 : S <= 4 ? 148 : S == 7 ? 104 : 120)
                                    : (S <= 4 ? 296 : terms ? 240 : 264);
        const int64_t waves = (n + slots - 1) / slots;
        const int64_t cost = alone ? waves * (2000 + 100 * each)
                             : n <= 148 ? 1400 + 64 * each : waves * (1550 + 100 * each);
        if (cost < least) {
            least = cost;
            best = S;
        }
    }
    return best;
}

template <typename XT, int COLS, int ROWS, int TN, int TK, bool ALONE = false>
aem_status launch_tile(const uint8_t* terms, Q4Args a, int gs, int64_t slots, cudaStream_t s) {
    CUtensorMap xmap{};
    constexpr bool XIN = TK == 1;
    const int64_t KP = a.NP * 128ll;
    if (!XIN)
        AEM_TRY(make_tmap_3d_u8(&xmap, terms, KP, a.M * TN, TK, KP, a.M * TN * KP, COLS, TK));
    a.S = split_k(a.NC * slots, a.NP, XIN ? Q4Cfg<COLS, 128, ROWS, TN, TK, ALONE>::MAXP : INT64_MAX, !XIN, ALONE);
    const dim3 grid(static_cast<unsigned>(a.NC * a.S), static_cast<unsigned>(slots));
    if (gs == 128) return launch_q4<XT, COLS, 128, ROWS, TN, TK, ALONE>(xmap, a, grid, s);
    if (gs == 64) return launch_q4<XT, COLS, 64, ROWS, TN, TK, ALONE>(xmap, a, grid, s);
    return launch_q4<XT, COLS, 32, ROWS, TN, TK, ALONE>(xmap, a, grid, s);
}

// Rows of a tile: as many as the call (grouped: an average group) has; few
// rows put their terms side by side in the 16 columns of the narrowest MMA.
// A CTA that makes its own terms spares the terms kernel and its wait, but
// every CTA of a row then does that work.  With the kernel, bf16 rows of 4096 x
// 14336 take 2.3 us more (one), the same (three) or 1.5 less (four), of 4096 x
// 4096 1.8 more (one) or 1.0 more (four).  A tile of 32 rows where 16 would do:
// 17.9 us instead of 15.0 (6 rows).  One of 64 takes 18.1 us where two of 32 take
// 25 (4096 x 14336), but 9.7 where those take 8.5 with K split three ways or more
// inside one wave (2048 x 1408).  A float32 row has three columns: 5 rows fill 16,
// 10 fill 32, 16 fill 48 and 32 fill 96.  Eight in a tile of eight, of which
// three quarters are read back: 16.7 us, in one of ten 17.3 (groups of 32), but
// groups of 6 rows on average have 9 or 10 often enough: 43.7 and 41.0 (64 of 2048
// x 1408).  Groups of 32 take three windows' sums back four times a block: 32
// float32 rows 29.6 us, of 128 19.1.
struct Q4Plan {
    bool few;
    int rows;
};
Q4Plan q4_plan(const Q4Weight* w, bool f32, int64_t M, bool grouped) {
    const int64_t groups = grouped ? std::min<int64_t>(w->G, M) : 1;
    const int64_t want = (M + groups - 1) / groups;
    const bool small = w->NC * groups * ((want + 31) / 32) * 3 <= kSMs;
    Q4Plan p;
    p.few = want <= (f32 ? 2 : 4) && w->NP <= 8 * 24;
    if (f32)
        p.rows = p.few ? (want <= 1 ? 1 : 2)
                 : want <= 5 ? 5 : want <= 8 && !grouped ? 8 : want <= 10 ? 10 : want <= 16 ? 16 : 32;
    else
        p.rows = p.few ? (want <= 2 ? 2 : 4) : want <= 16 ? 16 : want <= 32 || small ? 32 : 64;
    return p;
}
size_t q4_workspace(const Q4Weight* w, bool f32, int64_t M, bool grouped) {
    if (q4_plan(w, f32, M, grouped).few) return 0;
    return static_cast<size_t>(M) * ((f32 ? kTerms<float> : kTerms<__nv_bfloat16>) * w->NP * 128 + sizeof(uint32_t) + w->NP);
}

// x: the caller's rows.
template <typename XT>
aem_status q4_product(const Q4Weight* w, const char* what, Q4Args a, const XT* x, void* workspace,
                      size_t workspace_bytes, cudaStream_t s) {
    constexpr bool F32 = sizeof(XT) == 4;
    AEM_REQUIRE(current_device() == w->device, "%s: the weights are on device %d, the current one is %d",
                what, w->device, current_device());
    a.w = w->data;
    a.block = w->block;
    a.scale_bf16 = w->scale_bf16;
    a.N = w->N;
    a.K = w->K;
    a.NC = static_cast<int>(w->NC);
    a.NP = static_cast<int>(w->NP);
    a.x = x;
    a.err = device_error_word(w->device);
    if (!a.err) {
        set_error("%s: no device error word", what);
        return AEM_ENOMEM;
    }
    a.vec = reinterpret_cast<uintptr_t>(x) % (4 * sizeof(XT)) == 0 && a.ldx % 4 == 0 && a.K % 4 == 0;
    a.ovec = reinterpret_cast<uintptr_t>(a.out) % (a.out_bf16 ? 8 : 16) == 0 && a.ldo % 4 == 0;
    AEM_REQUIRE(a.M * kTerms<XT> < (1ll << 31), "%s: M=%lld out of range", what, (long long)a.M);
    const Q4Plan plan = q4_plan(w, F32, a.M, a.group_rows != nullptr);
    const size_t need = q4_workspace(w, F32, a.M, a.group_rows != nullptr);
    AEM_REQUIRE(!workspace || (workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                "%s: workspace of %zu bytes (%zu needed, 16-byte aligned)", what, workspace_bytes, need);
    a.rows = plan.rows;
    // row tiles at most: n groups with rows have up to n + (M - n) / rows
    const int64_t n = std::min<int64_t>(a.G, a.M);
    const int64_t slots = a.group_rows ? n + (a.M - n) / a.rows : (a.M + a.rows - 1) / a.rows;
    AEM_REQUIRE(slots <= 65535, "%s: M=%lld rows are too many for one call", what, (long long)a.M);
    if (plan.few)
        return a.rows == (F32 ? 1 : 2) ? launch_tile<XT, 16, F32 ? 1 : 2, kSide<XT>, 1>(nullptr, a, w->gs, slots, s)
                                       : launch_tile<XT, 16, F32 ? 2 : 4, kSide<XT>, 1>(nullptr, a, w->gs, slots, s);
    void* own = nullptr;
    if (!workspace) {
        AEM_TRY_CUDA(cudaMallocAsync(&own, need, s));
        workspace = own;
    }
    auto* terms = static_cast<uint8_t*>(workspace);
    auto* tops = reinterpret_cast<uint32_t*>(terms + static_cast<size_t>(a.M) * kTerms<XT> * w->NP * 128);
    auto* cuts = reinterpret_cast<uint8_t*>(tops + a.M);
    a.tops = tops;
    a.cuts = cuts;
    // at most 8 slots in registers up to K = 16384, and about two blocks an SM
    const int threads = w->K <= 4096 ? 128 : w->K <= 8192 ? 256 : 512;
    const int64_t slots_x = (w->NP * 32 + threads - 1) / threads;
    const dim3 blocks(static_cast<unsigned>(a.M),
                      static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(slots_x, 296 / a.M))));
    auto make_terms = a.vec ? q4_terms_kernel<XT, true> : q4_terms_kernel<XT, false>;
    make_terms<<<blocks, threads, 0, s>>>(x, a.ldx, w->K, w->NP * 128, terms, tops, cuts);
    count_launches(1);
    const cudaError_t e = cudaGetLastError();
    aem_status st;
    if (e != cudaSuccess) {
        set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
        st = AEM_ECUDA;
    } else if constexpr (F32) {
        st = a.rows == 5    ? launch_tile<XT, 16, 5, 3, 3>(terms, a, w->gs, slots, s)
             : a.rows == 8  ? launch_tile<XT, 32, 8, 3, 3>(terms, a, w->gs, slots, s)
             : a.rows == 10 ? launch_tile<XT, 32, 10, 3, 3>(terms, a, w->gs, slots, s)
             : a.rows == 16 ? launch_tile<XT, 48, 16, 3, 3, true>(terms, a, w->gs, slots, s)
                            : launch_tile<XT, 96, 32, 3, 3, true>(terms, a, w->gs, slots, s);
    } else {
        // 16 rows: an SM for each CTA while there are SMs (8 rows, 14336 x 4096:
        // 14.5 us, sharing 16.7), but not for many groups' tiles (64 tokens, 64
        // experts of 2048 x 1408: 39.2 us, sharing 29.4)
        st = a.rows == 64           ? launch_tile<XT, 64, 64, 1, 3, true>(terms, a, w->gs, slots, s)
             : a.rows == 32         ? launch_tile<XT, 32, 32, 1, 3, true>(terms, a, w->gs, slots, s)
             : a.NC * slots <= kSMs ? launch_tile<XT, 16, 16, 1, 3, true>(terms, a, w->gs, slots, s)
                                    : launch_tile<XT, 16, 16, 1, 3>(terms, a, w->gs, slots, s);
    }
    if (own) cudaFreeAsync(own, s);
    return st;
}

aem_status q4_any(const Q4Weight* w, const char* what, const Q4Args& a, const void* x, aem_dtype xd,
                  void* workspace, size_t bytes, cudaStream_t s) {
    if (xd == AEM_F32) return q4_product(w, what, a, static_cast<const float*>(x), workspace, bytes, s);
    return q4_product(w, what, a, static_cast<const __nv_bfloat16*>(x), workspace, bytes, s);
}

bool is_dtype(aem_dtype t) { return t == AEM_F32 || t == AEM_BF16; }
bool is_group(int gs) { return gs == 32 || gs == 64 || gs == 128; }

template <typename WT, typename ST>
void launch_quantize(const void* w, int64_t G, int64_t K, int64_t N, int gs, int8_t* q, void* scale,
                     cudaStream_t s) {
    const int64_t KB = (K + gs - 1) / gs;
    constexpr int CL = 16 / sizeof(WT);  // columns of a lane where rows can be read in vectors
    const bool vec = N % CL == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(q) % CL == 0;
    const int64_t cols = 32 * (vec ? CL : 4);
    const dim3 grid(static_cast<unsigned>(G * KB), static_cast<unsigned>((N + cols - 1) / cols));
    auto* wt = static_cast<const WT*>(w);
    auto* st = static_cast<ST*>(scale);
    auto go = [&](auto size) {
        constexpr int GS = decltype(size)::value;
        if (vec)
            quantize_q4_kernel<WT, ST, GS, true><<<grid, 4 * GS, 0, s>>>(wt, K, N, KB, q, st);
        else
            quantize_q4_kernel<WT, ST, GS, false><<<grid, 4 * GS, 0, s>>>(wt, K, N, KB, q, st);
    };
    if (gs == 32)
        go(std::integral_constant<int, 32>{});
    else if (gs == 64)
        go(std::integral_constant<int, 64>{});
    else
        go(std::integral_constant<int, 128>{});
}

void free_q4(Q4Weight* w) {
    cudaFree(w->data);
    delete w;
}

aem_status check_q4_shape(const char* what, int64_t G, int64_t K, int64_t N, int gs, aem_dtype sd) {
    AEM_REQUIRE(G >= 1 && K >= 1 && N >= 1, "%s: G=%lld K=%lld N=%lld must be >= 1", what,
                (long long)G, (long long)K, (long long)N);
    AEM_REQUIRE(K < (1ll << 30) && N < (1ll << 30) && G < (1ll << 31) && G * N < (1ll << 40),
                "%s: dimensions out of range", what);
    AEM_REQUIRE(is_group(gs), "%s: group_size=%d is not 32, 64 or 128", what, gs);
    AEM_REQUIRE(is_dtype(sd), "%s: bad scale dtype", what);
    return AEM_OK;
}

// Packs from device memory.  checked: waits, and a value out of range is an
// error of this call alone, through a flag behind the weight's blocks; else it
// is reported in the device's error word.
aem_status pack_q4(const int8_t* q, const void* scale, aem_dtype scale_dtype, int64_t G, int64_t K,
                   int64_t N, int group_size, cudaStream_t s, bool checked, aem_q4weight_t* out) {
    AEM_REQUIRE(out != nullptr, "aem_q4weight_pack: out is NULL");
    *out = nullptr;
    AEM_TRY(check_q4_shape("aem_q4weight_pack", G, K, N, group_size, scale_dtype));
    AEM_REQUIRE(q && scale, "aem_q4weight_pack: NULL buffer");
    int* err = device_error_word(current_device());
    auto* w = new (std::nothrow) Q4Weight();
    if (!err || !w) {
        delete w;
        set_error("aem_q4weight_pack: out of memory");
        return AEM_ENOMEM;
    }
    w->device = current_device();
    w->G = G;
    w->K = K;
    w->N = N;
    w->NC = (N + 127) / 128;
    w->NP = (K + 127) / 128;
    w->gs = group_size;
    w->scale_bf16 = scale_dtype == AEM_BF16;
    const int per = 128 / group_size;
    w->block = 8192 + per * 128 * (w->scale_bf16 ? 2 : 4);
    const int64_t blocks = G * w->NC * w->NP, KB = (K + group_size - 1) / group_size;
    const size_t bytes = static_cast<size_t>(blocks) * w->block;
    if (cudaMalloc(&w->data, bytes + sizeof(int)) != cudaSuccess) {
        cudaGetLastError();
        free_q4(w);
        set_error("aem_q4weight_pack: device allocation failed");
        return AEM_ENOMEM;
    }
    int* flag = reinterpret_cast<int*>(w->data + bytes);
    if (checked) {
        cudaMemsetAsync(flag, 0, sizeof(int), s);
        err = flag;
    }
    const unsigned g1 = static_cast<unsigned>(std::min<int64_t>(blocks * 2, 148 * 64));
    pack_q4_kernel<<<g1, kThreads, 0, s>>>(q, K, N, w->NC, w->NP, blocks * 512, w->block, w->data, err);
    const int64_t scales = blocks * per * 128;
    const unsigned g2 = static_cast<unsigned>(std::min<int64_t>((scales + 255) / 256, 148 * 64));
    if (w->scale_bf16)
        pack_q4_scale_kernel<__nv_bfloat16><<<g2, kThreads, 0, s>>>(
            static_cast<const __nv_bfloat16*>(scale), KB, N, w->NC, w->NP, scales, per, w->block, w->data);
    else
        pack_q4_scale_kernel<float><<<g2, kThreads, 0, s>>>(
            static_cast<const float*>(scale), KB, N, w->NC, w->NP, scales, per, w->block, w->data);
    cudaError_t e = cudaGetLastError();
    int bad = 0;
    if (checked && e == cudaSuccess) e = cudaMemcpyAsync(&bad, flag, sizeof(int), cudaMemcpyDeviceToHost, s);
    if (checked && e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess || bad) {
        free_q4(w);
        if (e == cudaSuccess) {
            set_error("aem_q4weight_pack: a 4-bit weight is outside [-7, 7]");
            return AEM_EINVAL;
        }
        set_error("aem_q4weight_pack: %s", cudaGetErrorString(e));
        return AEM_ECUDA;
    }
    count_launches(2);
    *out = reinterpret_cast<aem_q4weight_t>(w);
    return AEM_OK;
}

}  // namespace

}  // namespace aem

using aem::set_error;

extern "C" {

aem_status aem_quantize_q4(const void* w, aem_dtype w_dtype, int64_t G, int64_t K, int64_t N,
                           int group_size, int8_t* q, void* scale, aem_dtype scale_dtype,
                           void* stream) {
    AEM_TRY(aem::check_q4_shape("aem_quantize_q4", G, K, N, group_size, scale_dtype));
    AEM_REQUIRE(aem::is_dtype(w_dtype), "aem_quantize_q4: bad weight dtype");
    AEM_REQUIRE(w && q && scale, "aem_quantize_q4: NULL buffer");
    AEM_REQUIRE(G * ((K + group_size - 1) / group_size) < (1ll << 31) && N <= 65535ll * 128,
                "aem_quantize_q4: dimensions out of range");
    auto s = static_cast<cudaStream_t>(stream);
    const bool wf = w_dtype == AEM_F32, sf = scale_dtype == AEM_F32;
    if (wf)
        sf ? aem::launch_quantize<float, float>(w, G, K, N, group_size, q, scale, s)
           : aem::launch_quantize<float, __nv_bfloat16>(w, G, K, N, group_size, q, scale, s);
    else
        sf ? aem::launch_quantize<__nv_bfloat16, float>(w, G, K, N, group_size, q, scale, s)
           : aem::launch_quantize<__nv_bfloat16, __nv_bfloat16>(w, G, K, N, group_size, q, scale, s);
    AEM_CHECK_LAUNCH();
    aem::count_launches(1);
    return AEM_OK;
}

aem_status aem_q4weight_pack_device(const int8_t* q, const void* scale, aem_dtype scale_dtype,
                                    int64_t G, int64_t K, int64_t N, int group_size, void* stream,
                                    aem_q4weight_t* out) {
    return aem::pack_q4(q, scale, scale_dtype, G, K, N, group_size, static_cast<cudaStream_t>(stream), false, out);
}

aem_status aem_q4weight_pack_checked(const int8_t* q, const void* scale, aem_dtype scale_dtype,
                                     int64_t G, int64_t K, int64_t N, int group_size, void* stream,
                                     aem_q4weight_t* out) {
    return aem::pack_q4(q, scale, scale_dtype, G, K, N, group_size, static_cast<cudaStream_t>(stream), true, out);
}

aem_status aem_q4weight_pack(const int8_t* q, const void* scale, aem_dtype scale_dtype, int64_t G,
                             int64_t K, int64_t N, int group_size, int device, aem_q4weight_t* out) {
    AEM_REQUIRE(out != nullptr, "aem_q4weight_pack: out is NULL");
    *out = nullptr;
    AEM_TRY(aem::check_q4_shape("aem_q4weight_pack", G, K, N, group_size, scale_dtype));
    AEM_REQUIRE(q && scale, "aem_q4weight_pack: NULL buffer");
    const int64_t count = G * K * N, KB = (K + group_size - 1) / group_size;
    for (int64_t i = 0; i < count; ++i)
        AEM_REQUIRE(q[i] >= -7 && q[i] <= 7, "aem_q4weight_pack: q[%lld]=%d is outside [-7, 7]",
                    (long long)i, q[i]);
    if (!aem::is_sm100(device)) {
        set_error("aem_q4weight_pack: device %d is not an sm_100 (B200) GPU", device);
        return AEM_EUNSUPPORTED;
    }
    struct Device {  // the caller's device is current again at the end
        int before = 0;
        Device() { cudaGetDevice(&before); }
        ~Device() { cudaSetDevice(before); }
    } restore;
    AEM_TRY_CUDA(cudaSetDevice(device));
    const size_t sb = static_cast<size_t>(G * KB * N) * (scale_dtype == AEM_BF16 ? 2 : 4);
    int8_t* dq = nullptr;
    void* ds = nullptr;
    AEM_TRY_CUDA(cudaMalloc(&dq, static_cast<size_t>(count)));
    if (cudaMalloc(&ds, sb) != cudaSuccess) {
        cudaGetLastError();
        cudaFree(dq);
        set_error("aem_q4weight_pack: device allocation failed");
        return AEM_ENOMEM;
    }
    aem_status st = AEM_OK;
    if (cudaMemcpy(dq, q, static_cast<size_t>(count), cudaMemcpyHostToDevice) != cudaSuccess ||
        cudaMemcpy(ds, scale, sb, cudaMemcpyHostToDevice) != cudaSuccess) {
        set_error("aem_q4weight_pack: copy failed");
        st = AEM_ECUDA;
    }
    // waits, so the copies may go
    if (st == AEM_OK) st = aem::pack_q4(dq, ds, scale_dtype, G, K, N, group_size, nullptr, true, out);
    cudaFree(dq);
    cudaFree(ds);
    return st;
}

aem_status aem_q4weight_free(aem_q4weight_t wh) {
    if (!wh) return AEM_OK;
    auto* w = reinterpret_cast<aem::Q4Weight*>(wh);
    int prev = 0;
    cudaGetDevice(&prev);
    cudaSetDevice(w->device);
    cudaDeviceSynchronize();
    aem::free_q4(w);
    cudaSetDevice(prev);
    return AEM_OK;
}

aem_status aem_q4weight_shape(aem_q4weight_t wh, int64_t* G, int64_t* K, int64_t* N,
                              int* group_size) {
    AEM_REQUIRE(wh != nullptr, "aem_q4weight_shape: handle is NULL");
    auto* w = reinterpret_cast<aem::Q4Weight*>(wh);
    if (G) *G = w->G;
    if (K) *K = w->K;
    if (N) *N = w->N;
    if (group_size) *group_size = w->gs;
    return AEM_OK;
}

size_t aem_q4gemm_workspace(aem_q4weight_t wh, aem_dtype x_dtype, int64_t M, int grouped) {
    if (!wh || M < 1 || !aem::is_dtype(x_dtype)) return 0;
    return aem::q4_workspace(reinterpret_cast<aem::Q4Weight*>(wh), x_dtype == AEM_F32, M, grouped != 0);
}

aem_status aem_q4gemm(aem_q4weight_t wh, int64_t group, const void* x, aem_dtype x_dtype,
                      int64_t ldx, int64_t M, void* out, aem_dtype out_dtype, int64_t ldo,
                      void* workspace, size_t workspace_bytes, void* stream) {
    AEM_REQUIRE(wh != nullptr, "aem_q4gemm: weight handle is NULL");
    auto* w = reinterpret_cast<aem::Q4Weight*>(wh);
    AEM_REQUIRE(group >= 0 && group < w->G, "aem_q4gemm: group %lld out of range [0, %lld)",
                (long long)group, (long long)w->G);
    AEM_REQUIRE(M >= 0, "aem_q4gemm: M must be >= 0");
    AEM_REQUIRE(aem::is_dtype(x_dtype) && aem::is_dtype(out_dtype), "aem_q4gemm: bad dtype");
    AEM_REQUIRE(ldx >= 0 && ldo >= w->N, "aem_q4gemm: bad row stride");
    if (M == 0) return AEM_OK;
    AEM_REQUIRE(x && out, "aem_q4gemm: NULL buffer");
    aem::Q4Args a{};
    a.ldx = ldx;
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group = group;
    a.G = 1;
    a.out_bf16 = out_dtype == AEM_BF16;
    return aem::q4_any(w, "aem_q4gemm", a, x, x_dtype, workspace, workspace_bytes,
                           static_cast<cudaStream_t>(stream));
}

aem_status aem_grouped_q4gemm(aem_q4weight_t wh, const int32_t* group_rows, const void* x,
                              aem_dtype x_dtype, int64_t ldx, int64_t M, void* out,
                              aem_dtype out_dtype, int64_t ldo, int relu, void* workspace,
                              size_t workspace_bytes, void* stream) {
    AEM_REQUIRE(wh != nullptr, "aem_grouped_q4gemm: weight handle is NULL");
    auto* w = reinterpret_cast<aem::Q4Weight*>(wh);
    AEM_REQUIRE(w->G <= AEM_MAX_EXPERTS, "aem_grouped_q4gemm: %lld weight groups, at most %d",
                (long long)w->G, AEM_MAX_EXPERTS);
    AEM_REQUIRE(M >= 0 && M < (1ll << 31), "aem_grouped_q4gemm: M=%lld out of range", (long long)M);
    AEM_REQUIRE(aem::is_dtype(x_dtype) && aem::is_dtype(out_dtype), "aem_grouped_q4gemm: bad dtype");
    AEM_REQUIRE(ldx >= 0 && ldo >= w->N, "aem_grouped_q4gemm: bad row stride");
    if (M == 0) return AEM_OK;
    AEM_REQUIRE(group_rows && x && out, "aem_grouped_q4gemm: NULL buffer");
    aem::Q4Args a{};
    a.ldx = ldx;
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group_rows = group_rows;
    a.G = static_cast<int>(w->G);
    a.out_bf16 = out_dtype == AEM_BF16;
    a.relu = relu != 0;
    return aem::q4_any(w, "aem_grouped_q4gemm", a, x, x_dtype, workspace, workspace_bytes,
                           static_cast<cudaStream_t>(stream));
}

}  // extern "C"
