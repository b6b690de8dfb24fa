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
// [2^14, 2^15), x * rho = t_0 + t_1 + ... where t_j is what is left after
// t_0 .. t_{j-1}, truncated to e5m2's three significant bits (down to 2^-16).
// Three terms hold a bf16 value and eight a float32 value exactly unless its
// last bits lie below rho * |x| = 2^-16; what is cut off there is under 2^-30
// of the row's largest magnitude, below the rounding of a float32 sum that
// holds it.  Every product is exact, sums are float32 (tcgen05, accumulators
// in TMEM), the terms' sums are added and the scales multiply the result in
// float32: no rounded weight ever exists.
//
// What bounds it is the weight stream, K*N/2 bytes plus the scales.  Forms
// that could not keep up with it (4096 x 14336, 1 row): warp MMAs (mma.sync
// m16n8k16 occupies its sub-core's tensor pipe for 32 cycles: 16.6 us, 47.6
// for 64 rows), and bf16 operands for tcgen05 (7 logic operations and 4
// subtractions per 8 weights, the logic pipe the bound: 17.3 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <new>

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

constexpr int kThreads = 256, kWarps = 8;  // quantise, pack

// ------------------------------------------------------------------ quantise
// One block per (128 columns, scale group): warp w holds rows w, w+8, ... of
// the group in registers, 4 columns per lane, so w is read once; the column
// maxima meet in shared memory.  scale = max(amax / 7, 1e-12), rounded to
// the scale's type before q = clip(rint(w / scale), -7, 7) is taken with it
// (IEEE float32 division, ties to even).
template <typename WT, typename ST, int GS>
__global__ void __launch_bounds__(kThreads)
    quantize_q4_kernel(const WT* __restrict__ w, int64_t K, int64_t N, int64_t KB, bool vec,
                       int8_t* __restrict__ q, ST* __restrict__ scale) {
    constexpr int R = GS / kWarps;
    __shared__ float amax[kWarps][128];
    const int lane = threadIdx.x & 31, wi = threadIdx.x >> 5;
    const int64_t g = blockIdx.x / KB, b = blockIdx.x % KB;
    const int64_t n0 = blockIdx.y * 128ll + lane * 4, k0 = b * GS + wi;
    const WT* src = w + g * K * N;
    float v[R][4];
    float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t k = k0 + i * kWarps;
        v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
        if (k < K && n0 < N) {
            const WT* p = src + k * N + n0;
            if (vec) {
                if constexpr (sizeof(WT) == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(p);
                    v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(p);
                    v[i][0] = __uint_as_float(u.x << 16), v[i][1] = __uint_as_float(u.x & 0xffff0000u);
                    v[i][2] = __uint_as_float(u.y << 16), v[i][3] = __uint_as_float(u.y & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n0 + j < N) v[i][j] = static_cast<float>(p[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = fmaxf(m[j], fabsf(v[i][j]));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) amax[wi][lane * 4 + j] = m[j];
    __syncthreads();
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < kWarps; ++i) m[j] = fmaxf(m[j], amax[i][lane * 4 + j]);
        s[j] = fmaxf(__fdiv_rn(m[j], 7.0f), 1e-12f);
        if constexpr (sizeof(ST) == 2) s[j] = __bfloat162float(__float2bfloat16_rn(s[j]));
        if (wi == 0 && n0 + j < N) scale[(g * KB + b) * N + n0 + j] = static_cast<ST>(s[j]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t k = k0 + i * kWarps;
        if (k >= K || n0 >= N) continue;
        int8_t c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float r = fminf(fmaxf(rintf(__fdiv_rn(v[i][j], s[j])), -7.0f), 7.0f);
            c[j] = static_cast<int8_t>(static_cast<int>(r));
        }
        int8_t* p = q + (g * K + k) * N + n0;
        if (vec) {
            *reinterpret_cast<char4*>(p) = make_char4(c[0], c[1], c[2], c[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < N) p[j] = c[j];
        }
    }
}

// ------------------------------------------------------------------ pack
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
    const float* unscale;       // [M]: 2^9 / rho of a row of x
    void* out;
    const int32_t* group_rows;  // nullptr: one group of M rows, weight group `group`
    int64_t ldo, M, N, NC, NP;
    int64_t group;
    int* err;
    int G, block, S, rows;  // S: CTAs (one cluster) that split K; rows: rows of a row tile
    bool scale_bf16, out_bf16, relu;
};

constexpr int kTermsBf16 = 3, kTermsF32 = 8;

// Activations as the products read them, one block per row: out [M * terms]
// [KP] e5m2 bytes (KP = K rounded up to 128, zero padded), unscale [M].  An
// infinity or NaN is all in the first term.  e5m2 is the upper byte of an
// fp16, so truncating the fp16 truncates the term.
template <typename XT, int TERMS>
__global__ void __launch_bounds__(512)
    q4_terms_kernel(const XT* __restrict__ x, int64_t ldx, int64_t K, int64_t KP, bool vec,
                    uint8_t* __restrict__ out, float* __restrict__ unscale) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ uint32_t top[16];
    const XT* row = x + blockIdx.x * ldx;
    auto load4 = [&](int64_t k, float (&v)[4]) {
        if (vec && k + 4 <= K) {
            if constexpr (sizeof(XT) == 4) {
                const float4 f = *reinterpret_cast<const float4*>(row + k);
                v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(row + k);
                v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u);
                v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = k + i < K ? static_cast<float>(row[k + i]) : 0.0f;
        }
    };
    uint32_t mine = 0;  // magnitudes order as their bits do
    for (int64_t k = threadIdx.x * 4; k < K; k += 512 * 4) {
        float v[4];
        load4(k, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = __float_as_uint(v[i]) & 0x7fffffffu;
            if (u < 0x7f800000u) mine = max(mine, u);
        }
    }
    mine = __reduce_max_sync(~0u, mine);
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = mine;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) mine = max(mine, top[i]);
    // rho = 2^up, up = 14 - exponent, in two factors (it may be beyond float32)
    const int up = 141 - static_cast<int>(mine >> 23);
    const float f1 = __uint_as_float(static_cast<uint32_t>(127 + up / 2) << 23);
    const float f2 = __uint_as_float(static_cast<uint32_t>(127 + up - up / 2) << 23);
    if (threadIdx.x == 0) unscale[blockIdx.x] = ldexpf(1.0f, 9 - up);
    uint8_t* o = out + blockIdx.x * TERMS * KP;
    for (int64_t k = threadIdx.x * 4; k < KP; k += 512 * 4) {
        float v[4];
        load4(k, v);
        uint32_t t[TERMS];
#pragma unroll
        for (int j = 0; j < TERMS; ++j) t[j] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool finite = (__float_as_uint(v[i]) & 0x7f800000u) != 0x7f800000u;
            float r = v[i] * f1 * f2;
#pragma unroll
            for (int j = 0; j < TERMS; ++j) {
                const uint32_t h = __half_as_ushort(__float2half_rz(r)) & 0xff00u;
                t[j] |= (h >> 8) << (8 * i);
                r -= __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
            }
            if (!finite) {
                const uint32_t code = v[i] != v[i] ? 0x7fu : v[i] > 0.0f ? 0x7cu : 0xfcu;
#pragma unroll
                for (int j = 0; j < TERMS; ++j)
                    t[j] = (t[j] & ~(0xffu << (8 * i))) | (j == 0 ? code << (8 * i) : 0u);
            }
        }
#pragma unroll
        for (int j = 0; j < TERMS; ++j) *reinterpret_cast<uint32_t*>(o + j * KP + k) = t[j];
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

__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_u32(p, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void store_out(const Q4Args& a, int64_t m, int64_t n, float v) {
    if (a.relu && v < 0.0f) v = 0.0f;
    if (a.out_bf16)
        static_cast<__nv_bfloat16*>(a.out)[m * a.ldo + n] = __float2bfloat16_rn(v);
    else
        static_cast<float*>(a.out)[m * a.ldo + n] = v;
}

// Shape of the product kernel for COLS MMA columns, scale groups of GS k and
// TERMS columns a row.  A block of the packed weight is 128 channels x 128 k;
// a unit is what a warpgroup hands to the tensor core at once: a block, with
// one accumulator per scale group side by side, or half of one where a
// block's accumulators would not fit.
template <int COLS, int GS, int TERMS>
struct Q4Cfg {
    static constexpr int ROWS = COLS / TERMS;
    static constexpr int TW = 128;                     // TMEM columns of a warpgroup: 4 per SM
    static constexpr int FULL = GS == 128 ? 1 : 128 / GS;  // scale groups of a block
    static constexpr int UK = FULL * COLS <= 96 ? 128 : 64;  // k of a unit
    static constexpr int SUB = UK < GS ? 1 : UK / GS;  // accumulators per unit
    static constexpr int UA = UK / 4;                  // columns of a unit's weights
    static constexpr int ND = UA + 2 * SUB * COLS <= TW ? 2 : 1;  // accumulator buffers
    static constexpr int XB = COLS * 128;              // activation bytes of a block
    static constexpr int STAGE = XB + 8192 + (FULL * 512 + 1023) / 1024 * 1024;
    // an even ring: a stage always comes back to the warpgroup that saw its
    // previous phase, so no parity wait can mistake a phase for the one two back
    static constexpr int FIT = (113 * 1024 - 2048) / STAGE / 2 * 2;
    static constexpr int NS = FIT > 8 ? 8 : FIT;
    static constexpr int LD = 128 + 4;
    static constexpr int USED = 1024 + NS * STAGE + (2 * NS + 4) * 8 + 16;
    // two CTAs on an SM, never three: no CTA ever waits for tensor memory
    static constexpr int SMEM = USED > 78 * 1024 ? USED : 78 * 1024;
    static_assert(UA + ND * SUB * COLS <= TW && NS >= 4 && SMEM <= 113 * 1024, "budgets");
    static_assert(UK >= GS || UK == 128, "a scale group inside a unit");
    static_assert(NS * STAGE >= ROWS * LD * 4, "the sums fit the ring");
};
constexpr int kQ4Threads = 12 * 32;

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
//   warp 11     copies the activations, one TMA box per block (128-byte swizzle).
// Two accumulator buffers let the sums be taken back under the next unit's
// MMAs; where only one fits they are taken before the unit is handed over.
// The S CTAs of a cluster take parts of K; their sums are added in rank order.
// Every wait is bounded; a timeout sets the error word and ends all roles.
template <int COLS, int GS, int TERMS>
__global__ void __launch_bounds__(kQ4Threads, 2)
    q4_kernel(const __grid_constant__ CUtensorMap xmap, const Q4Args a) {
    using C = Q4Cfg<COLS, GS, TERMS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    float* fin = reinterpret_cast<float*>(ring);  // [ROWS][LD], after the loop
    uint64_t* in_full = reinterpret_cast<uint64_t*>(ring + C::NS * C::STAGE);
    uint64_t* in_empty = in_full + C::NS;
    uint64_t* a_full = in_empty + C::NS;  // [2]: a unit's weights are in tensor memory
    uint64_t* done = a_full + 2;          // [2]: its MMAs have finished
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t tile = blockIdx.x / a.S;
    const int ks = blockIdx.x % a.S;
    int64_t g, m0;
    int rows;
    if (!find_rows(a, blockIdx.y, &g, &m0, &rows)) return;  // the whole cluster alike
    const int p0 = static_cast<int>(a.NP * ks / a.S), np = static_cast<int>(a.NP * (ks + 1) / a.S) - p0;

    const uint8_t* src = a.w + ((g * a.NC + tile) * a.NP + p0) * a.block;
    auto copy_weights = [&](int p) {
        uint64_t* full = &in_full[p % C::NS];
        mbar_arrive_expect_tx(full, a.block);
        bulk_load(ring + p % C::NS * C::STAGE + C::XB, src + static_cast<int64_t>(p) * a.block, a.block, full);
    };
    if (w == 9) {
        tmem_alloc(tmem_slot, 2 * C::TW);
        tmem_relinquish();
    } else if (w == 10 && lane == 0) {
        // the first weights are on their way before the rest of the set-up
        for (int i = 0; i < C::NS; ++i) {
            mbar_init(&in_full[i], 2);   // both copies
            mbar_init(&in_empty[i], 4);  // the four warps of the block's warpgroup
        }
        for (int j = 0; j < 2; ++j) {
            mbar_init(&a_full[j], 4);
            mbar_init(&done[j], 1);
        }
        *abort_flag = 0;
        fence_barrier_init();
        for (int p = 0; p < min(np, C::NS); ++p) copy_weights(p);
    } else if (w == 11 && lane == 0) {
        tma_prefetch_desc(&xmap);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int wg = w < 8 ? w >> 2 : w & 1;  // the warpgroup a channel or MMA warp belongs to
    const uint32_t td = tmem + static_cast<uint32_t>(wg * C::TW);  // accumulators, then the unit's weights
    const uint32_t ta = td + C::ND * C::SUB * COLS;
    auto wait = [&](uint64_t* bar, int phase) {  // whole warps
        if (__all_sync(~0u, mbar_try_wait(bar, phase & 1))) return true;
        return __all_sync(~0u, mbar_wait_bounded(bar, phase & 1, abort_flag, a.err, ERR_GEMM_TIMEOUT)) != 0;
    };

    float acc[C::ROWS] = {};
    const int ch = threadIdx.x & 127;
    if (w < 8) {
        const uint32_t quarter = static_cast<uint32_t>(32 * (w & 3)) << 16;
        // RB rows' terms at a time, whole 8-column loads
        constexpr int RB = TERMS == kTermsF32 ? 2 : COLS == 16 ? 5 : 8, CB = (RB * TERMS + 7) / 8 * 8;
        auto take = [&](int u, const float (&s)[C::SUB]) {  // unit u's sums, scaled
#pragma unroll
            for (int j = 0; j < C::SUB; ++j)
#pragma unroll
                for (int r0 = 0; r0 < C::ROWS; r0 += RB) {
                    if (r0 >= rows) continue;
                    uint32_t r[CB];
                    const uint32_t at = td + quarter + (u % C::ND * C::SUB + j) * COLS + r0 * TERMS;
#pragma unroll
                    for (int c = 0; c < CB; c += 8) tc_ld_32x32b_x8(at + c, *reinterpret_cast<uint32_t(*)[8]>(r + c));
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < RB; ++i) {
                        if (r0 + i >= C::ROWS) continue;
                        float v = __uint_as_float(r[i * TERMS]);
#pragma unroll
                        for (int t = 1; t < TERMS; ++t) v += __uint_as_float(r[i * TERMS + t]);
                        acc[r0 + i] = fmaf(s[j], v, acc[r0 + i]);
                    }
                }
            tc_fence_before();
        };
        float s_prev[C::SUB];
        int u = 0;  // units of this warpgroup so far
        bool ok = true;
        for (int p = wg; ok && p < np; p += 2) {
            const uint8_t* st = ring + p % C::NS * C::STAGE + C::XB;
            if (!(ok = wait(&in_full[p % C::NS], p / C::NS))) break;
            float s[C::FULL];
#pragma unroll
            for (int j = 0; j < C::FULL; ++j)
                s[j] = a.scale_bf16
                           ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(st + 8192)[j * 128 + ch])
                           : reinterpret_cast<const float*>(st + 8192)[j * 128 + ch];
#pragma unroll
            for (int j = 0; j < 128 / C::UK; ++j) {
                uint32_t v[C::UA];
#pragma unroll
                for (int i = 0; i < C::UK / 32; ++i) {
                    const uint4 q = *reinterpret_cast<const uint4*>(st + (j * (C::UK / 32) + i) * 2048 + ch * 16);
                    const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[8 * i + 2 * e] = word[e] & 0x87878787u;
                        v[8 * i + 2 * e + 1] = __funnelshift_r(word[e], word[e], 4) & 0x87878787u;
                    }
                }
                if (u) {
                    // the unit before is done: its weights' columns, its
                    // accumulators and (at a block's start) its stage are free
                    if (!(ok = wait(&done[wg], u - 1))) break;
                    tc_fence_after();
                    if (j == 0 && lane == 0) mbar_arrive(&in_empty[(p - 2) % C::NS]);
                    if (C::ND == 1) take(u - 1, s_prev);
                }
                if constexpr (C::UA == 32)
                    tc_st_32x32b_x32(ta + quarter, v);
                else
                    tc_st_32x32b_x16(ta + quarter, v);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_full[wg]);
                if (C::ND == 2 && u) take(u - 1, s_prev);
#pragma unroll
                for (int i = 0; i < C::SUB; ++i) s_prev[i] = s[C::UK == 128 ? i : j * 64 / GS + i];
                ++u;
            }
        }
        if (ok && u && wait(&done[wg], u - 1)) {
            tc_fence_after();
            take(u - 1, s_prev);
        }
    } else if (w < 10) {
        const uint32_t idesc = idesc_e4m3_e5m2_f32(128, static_cast<uint32_t>((rows * TERMS + 15) & ~15));
        int u = 0;
        bool ok = true;
        for (int p = wg; ok && p < np; p += 2) {
            if (!(ok = wait(&in_full[p % C::NS], p / C::NS))) break;
            const uint64_t bd = smem_desc_sw128(smem_u32(ring + p % C::NS * C::STAGE));
#pragma unroll
            for (int j = 0; j < 128 / C::UK; ++j) {
                if (!(ok = wait(&a_full[wg], u))) break;
                tc_fence_after();
                const uint32_t d = td + static_cast<uint32_t>(u % C::ND * C::SUB * COLS);
#pragma unroll
                for (int m = 0; m < C::UK / 32; ++m)
                    tc_mma_f8_ts_elect(d + 32 * m / GS * COLS, ta + 8 * m, bd + 2 * (j * (C::UK / 32) + m), idesc,
                                       32 * m % GS ? 1u : 0u);
                tc_commit_elect(&done[wg]);
                ++u;
            }
        }
    } else if (lane == 0) {
        const bool weights = w == 10;
        if (!weights) asm volatile("griddepcontrol.wait;" ::: "memory");  // x is the terms kernel's
        int p = weights ? min(np, C::NS) : 0;
        for (; p < np; ++p) {
            uint64_t* full = &in_full[p % C::NS];
            if (!mbar_wait_bounded(&in_empty[p % C::NS], (p / C::NS & 1) ^ 1, abort_flag, a.err, ERR_GEMM_TIMEOUT))
                break;
            if (weights) {
                copy_weights(p);
            } else {
                mbar_arrive_expect_tx(full, C::XB);
                tma_load_2d(ring + p % C::NS * C::STAGE, &xmap, full, (p0 + p) * 128, static_cast<int>(m0 * TERMS));
            }
        }
        if (*abort_flag)  // a failed call leaves no copy in flight behind (bounded as well)
            for (int i = max(0, p - C::NS); i < p; ++i)
                for (int t = 0; t < 1 << 14 && !mbar_try_wait(&in_full[i % C::NS], i / C::NS & 1); ++t) {
                }
    }

    // every MMA has been waited for by the channel warps (or the call failed):
    // give the tensor memory back before any wait on another CTA
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (w == 9) tmem_dealloc(tmem, 2 * C::TW);
    for (int j = 0; j < 2; ++j) {  // the warpgroups' sums
        if (w < 8 && wg == j)
#pragma unroll
            for (int c = 0; c < C::ROWS; ++c)
                if (c < rows) fin[c * C::LD + ch] = j ? fin[c * C::LD + ch] + acc[c] : acc[c];
        __syncthreads();
    }
    if (a.S > 1) cluster_sync();
    asm volatile("griddepcontrol.wait;" ::: "memory");  // unscale is the terms kernel's
    for (int i = ks * kQ4Threads + threadIdx.x; i < rows * 128; i += a.S * kQ4Threads) {
        const int r = i >> 7, c = i & 127;
        const float* p = fin + r * C::LD + c;
        float v = 0.0f;
        for (int s = 0; s < a.S; ++s) v += s == ks ? *p : ld_cluster(p, s);
        if (tile * 128 + c < a.N) store_out(a, m0 + r, tile * 128 + c, v * a.unscale[m0 + r]);
    }
    if (a.S > 1) cluster_sync();  // the sums stay until every rank has read them
}

template <int COLS, int GS, int TERMS>
aem_status launch_q4(const CUtensorMap& xmap, const Q4Args& a, dim3 grid, cudaStream_t s) {
    using C = Q4Cfg<COLS, GS, TERMS>;
    auto kern = q4_kernel<COLS, GS, TERMS>;
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
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // starts under the terms kernel
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = a.S;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = a.S > 1 ? 2 : 1;
    AEM_TRY_CUDA(cudaLaunchKernelEx(&cfg, kern, xmap, a));
    count_launches(1);
    return AEM_OK;
}

template <int COLS, int TERMS>
aem_status launch_cols(const uint8_t* x, Q4Args a, int gs, int64_t slots, cudaStream_t s) {
    CUtensorMap xmap;
    AEM_TRY(make_tmap_2d(&xmap, x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.NP * 128, a.M * TERMS, 128, COLS,
                         CU_TENSOR_MAP_SWIZZLE_128B));
    // K is split until the CTAs fill the SMs: waves x (a CTA's own latency, as
    // long as about 8 blocks, and its blocks)
    const int64_t ctas = a.NC * slots, fit = 148 * 2;
    int64_t best = INT64_MAX;
    for (int S = 1; S <= 8 && S <= std::max<int64_t>(1, a.NP / 2); ++S) {
        const int64_t cost = (ctas * S + fit - 1) / fit * (8 + (a.NP + S - 1) / S);
        if (cost < best) {
            best = cost;
            a.S = S;
        }
    }
    const dim3 grid(static_cast<unsigned>(a.NC * a.S), static_cast<unsigned>(slots));
    if (gs == 128) return launch_q4<COLS, 128, TERMS>(xmap, a, grid, s);
    if (gs == 64) return launch_q4<COLS, 64, TERMS>(xmap, a, grid, s);
    if constexpr (COLS <= 48)  // the largest row tile has no room for groups of 32
        return launch_q4<COLS, 32, TERMS>(xmap, a, grid, s);
    set_error("q4 product: no such row tile");
    return AEM_EINVAL;
}

size_t q4_workspace(const Q4Weight* w, int terms, int64_t M) {
    return static_cast<size_t>(M) * terms * w->NP * 128 + static_cast<size_t>(M) * 4;
}

// x: the caller's rows.
template <typename XT, int TERMS>
aem_status q4_product(const Q4Weight* w, const char* what, Q4Args a, const XT* x, int64_t ldx,
                      void* workspace, size_t workspace_bytes, cudaStream_t s) {
    AEM_REQUIRE(current_device() == w->device, "%s: the weights are on device %d, the current one is %d",
                what, w->device, current_device());
    a.w = w->data;
    a.block = w->block;
    a.scale_bf16 = w->scale_bf16;
    a.N = w->N;
    a.NC = w->NC;
    a.NP = w->NP;
    a.err = device_error_word(w->device);
    AEM_REQUIRE(a.M * TERMS < (1ll << 31), "%s: M=%lld out of range", what, (long long)a.M);
    // columns of a row tile: as many as the rows (grouped: an average group's) need
    const int64_t groups = std::min<int64_t>(a.G, a.M);
    const int64_t want = a.group_rows ? (a.M + groups - 1) / groups : a.M;
    const int cols = want <= 16 / TERMS ? 16 : want <= 48 / TERMS || w->gs == 32 ? 48 : 96;
    a.rows = cols / TERMS;
    const int64_t slots = a.group_rows ? groups + a.M / a.rows : (a.M + a.rows - 1) / a.rows;
    AEM_REQUIRE(slots <= 65535, "%s: M=%lld rows are too many for one call", what, (long long)a.M);
    const size_t need = q4_workspace(w, TERMS, a.M);
    AEM_REQUIRE(!workspace || (workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                "%s: workspace of %zu bytes (%zu needed, 16-byte aligned)", what, workspace_bytes, need);
    void* own = nullptr;
    if (!workspace) {
        AEM_TRY_CUDA(cudaMallocAsync(&own, need, s));
        workspace = own;
    }
    auto* terms = static_cast<uint8_t*>(workspace);
    auto* unscale = reinterpret_cast<float*>(terms + static_cast<size_t>(a.M) * TERMS * w->NP * 128);
    a.unscale = unscale;
    const bool vec = reinterpret_cast<uintptr_t>(x) % (4 * sizeof(XT)) == 0 && ldx % 4 == 0;
    q4_terms_kernel<XT, TERMS><<<static_cast<unsigned>(a.M), 512, 0, s>>>(x, ldx, w->K, w->NP * 128, vec, terms,
                                                                          unscale);
    count_launches(1);
    const cudaError_t e = cudaGetLastError();
    aem_status st;
    if (e != cudaSuccess) {
        set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
        st = AEM_ECUDA;
    } else {
        st = cols == 16   ? launch_cols<16, TERMS>(terms, a, w->gs, slots, s)
             : cols == 48 ? launch_cols<48, TERMS>(terms, a, w->gs, slots, s)
                          : launch_cols<96, TERMS>(terms, a, w->gs, slots, s);
    }
    if (own) cudaFreeAsync(own, s);
    return st;
}

aem_status q4_any(const Q4Weight* w, const char* what, const Q4Args& a, const void* x, aem_dtype xd,
                  int64_t ldx, void* workspace, size_t bytes, cudaStream_t s) {
    if (xd == AEM_F32)
        return q4_product<float, kTermsF32>(w, what, a, static_cast<const float*>(x), ldx, workspace, bytes, s);
    return q4_product<__nv_bfloat16, kTermsBf16>(w, what, a, static_cast<const __nv_bfloat16*>(x), ldx, workspace,
                                                 bytes, s);
}

bool is_dtype(aem_dtype t) { return t == AEM_F32 || t == AEM_BF16; }
bool is_group(int gs) { return gs == 32 || gs == 64 || gs == 128; }

template <typename WT, typename ST>
void launch_quantize(const void* w, int64_t G, int64_t K, int64_t N, int gs, int8_t* q, void* scale,
                     cudaStream_t s) {
    const int64_t KB = (K + gs - 1) / gs;
    const dim3 grid(static_cast<unsigned>(G * KB), static_cast<unsigned>((N + 127) / 128));
    const bool vec = N % 4 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(q) % 4 == 0;
    auto* wt = static_cast<const WT*>(w);
    auto* st = static_cast<ST*>(scale);
    if (gs == 32)
        quantize_q4_kernel<WT, ST, 32><<<grid, kThreads, 0, s>>>(wt, K, N, KB, vec, q, st);
    else if (gs == 64)
        quantize_q4_kernel<WT, ST, 64><<<grid, kThreads, 0, s>>>(wt, K, N, KB, vec, q, st);
    else
        quantize_q4_kernel<WT, ST, 128><<<grid, kThreads, 0, s>>>(wt, K, N, KB, vec, q, st);
}

void free_q4(Q4Weight* w) {
    cudaFree(w->data);
    delete w;
}

aem_status check_q4_shape(const char* what, int64_t G, int64_t K, int64_t N, int gs, aem_dtype sd) {
    AEM_REQUIRE(G >= 1 && K >= 1 && N >= 1, "%s: G=%lld K=%lld N=%lld must be >= 1", what,
                (long long)G, (long long)K, (long long)N);
    AEM_REQUIRE(K < (1ll << 31) && N < (1ll << 31) && G < (1ll << 31) && G * N < (1ll << 40),
                "%s: dimensions out of range", what);
    AEM_REQUIRE(is_group(gs), "%s: group_size=%d is not 32, 64 or 128", what, gs);
    AEM_REQUIRE(is_dtype(sd), "%s: bad scale dtype", what);
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
    AEM_REQUIRE(out != nullptr, "aem_q4weight_pack: out is NULL");
    *out = nullptr;
    AEM_TRY(aem::check_q4_shape("aem_q4weight_pack", G, K, N, group_size, scale_dtype));
    AEM_REQUIRE(q && scale, "aem_q4weight_pack: NULL buffer");
    auto s = static_cast<cudaStream_t>(stream);
    int* err = aem::device_error_word(aem::current_device());
    auto* w = new (std::nothrow) aem::Q4Weight();
    if (!err || !w) {
        delete w;
        set_error("aem_q4weight_pack: out of memory");
        return AEM_ENOMEM;
    }
    w->device = aem::current_device();
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
    if (cudaMalloc(&w->data, static_cast<size_t>(blocks) * w->block) != cudaSuccess) {
        cudaGetLastError();
        aem::free_q4(w);
        set_error("aem_q4weight_pack: device allocation failed");
        return AEM_ENOMEM;
    }
    const unsigned g1 = static_cast<unsigned>(std::min<int64_t>(blocks * 2, 148 * 64));
    aem::pack_q4_kernel<<<g1, aem::kThreads, 0, s>>>(q, K, N, w->NC, w->NP, blocks * 512, w->block, w->data, err);
    const int64_t scales = blocks * per * 128;
    const unsigned g2 = static_cast<unsigned>(std::min<int64_t>((scales + 255) / 256, 148 * 64));
    if (w->scale_bf16)
        aem::pack_q4_scale_kernel<__nv_bfloat16><<<g2, aem::kThreads, 0, s>>>(
            static_cast<const __nv_bfloat16*>(scale), KB, N, w->NC, w->NP, scales, per, w->block, w->data);
    else
        aem::pack_q4_scale_kernel<float><<<g2, aem::kThreads, 0, s>>>(
            static_cast<const float*>(scale), KB, N, w->NC, w->NP, scales, per, w->block, w->data);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        aem::free_q4(w);
        set_error("aem_q4weight_pack: launch failed: %s", cudaGetErrorString(e));
        return AEM_ECUDA;
    }
    aem::count_launches(2);
    *out = reinterpret_cast<aem_q4weight_t>(w);
    return AEM_OK;
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
    if (st == AEM_OK)
        st = aem_q4weight_pack_device(dq, ds, scale_dtype, G, K, N, group_size, nullptr, out);
    if (st == AEM_OK && cudaDeviceSynchronize() != cudaSuccess) {
        set_error("aem_q4weight_pack: %s", cudaGetErrorString(cudaGetLastError()));
        st = AEM_ECUDA;
    }
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

size_t aem_q4gemm_workspace(aem_q4weight_t wh, aem_dtype x_dtype, int64_t M) {
    if (!wh || M < 1 || !aem::is_dtype(x_dtype)) return 0;
    return aem::q4_workspace(reinterpret_cast<aem::Q4Weight*>(wh), x_dtype == AEM_F32 ? aem::kTermsF32 : aem::kTermsBf16, M);
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
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group = group;
    a.G = 1;
    a.out_bf16 = out_dtype == AEM_BF16;
    return aem::q4_any(w, "aem_q4gemm", a, x, x_dtype, ldx, workspace, workspace_bytes,
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
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group_rows = group_rows;
    a.G = static_cast<int>(w->G);
    a.out_bf16 = out_dtype == AEM_BF16;
    a.relu = relu != 0;
    return aem::q4_any(w, "aem_grouped_q4gemm", a, x, x_dtype, ldx, workspace, workspace_bytes,
                           static_cast<cudaStream_t>(stream));
}

}  // extern "C"
