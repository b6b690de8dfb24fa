// 4-bit weights with group scales: quantisation, packing, and the products of
// a few activation rows with them (decode), dense and grouped by expert.
//
// Weight (k, n) of group g of G is q[g][k][n] * scale[g][k / gs][n] with q an
// integer in [-8, 7] and gs = 32, 64 or 128 consecutive k sharing a scale:
//   out[m, n] = sum_b scale[b, n] * sum_{k in block b} q[k, n] x[m, k]
// A 4-bit integer is exact in bf16, so each inner sum runs on the tensor cores
// (tcgen05, bf16 operands, float32 accumulators in TMEM) and the scale
// multiplies its float32 result: no rounded weight ever exists.  bf16 x enters
// as it is; float32 x enters as three bf16 terms that add up to it exactly
// (8 + 8 + 8 mantissa bits), in three MMA columns whose sums are added at the
// end.
//
// What bounds it is the weight stream, K*N/2 bytes plus the scales.  Warp MMAs
// (mma.sync) cannot keep up with it on this chip: one m16n8k16 occupies its
// sub-core's tensor pipe for 32 cycles, 12400 cycles for a 4096 x 14336
// weight and 8 columns, and the time grows with the columns (measured 16.6 us
// for 1 row, 47.6 us for 64).  So 128 channels are the M of a tcgen05.mma and
// the weights, converted in registers, are its A operand in tensor memory.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <new>

#include "common.cuh"
#include "runtime.h"

namespace aem {

// Packed 4-bit weight (device): [G][NC][NP] blocks of `block` bytes, NC =
// ceil(N / 128) channel blocks and NP = ceil(K / 128).  A block holds 128
// channels x 128 k and their scales, so one bulk copy brings both:
//   [2][2][128][16 B]  weights: 64-k tile, half of it, channel.  The word j
//                      (of 8) of a channel's tile holds k = 8j .. 8j + 7: the
//                      pair (8j + 2r, 8j + 2r + 1) at bits 4r and 16 + 4r, as
//                      q + 8; padding holds 8
//   [128 / gs][128]    scales in the caller's type; padding is zero
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
                if (v < -8 || v > 7) {
                    bad = true;
                    v = v < 0 ? -8 : 7;
                }
                word[j] |= static_cast<uint32_t>(v + 8) << (4 * (e >> 1) + 16 * (e & 1));
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

// Columns of the MMAs: the rows of x as they are (bf16), or three per row
// (float32: the terms that add up to it).
struct Q4Args {
    const uint8_t* w;
    void* out;
    const int32_t* group_rows;  // nullptr: one group of M rows, weight group `group`
    int64_t ldo, M, N, NC, NP;
    int64_t group;
    int* err;
    int G, block, S, rows, terms;  // S: CTAs (one cluster) that split K; rows: rows of a row tile
    bool scale_bf16, out_bf16, relu, dependent;
};

// Eight 4-bit weights -> four bf16 pairs.  0x4300 is bf16 128, whose last
// mantissa bit is 1: 0x4300 | nibble = 128 + nibble, and subtracting 136
// leaves q exactly.
__device__ __forceinline__ void unpack_q4(uint32_t w, uint32_t* a) {
    const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t v = ((w >> (4 * r)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
        a[r] = *reinterpret_cast<const uint32_t*>(&d);
    }
}

// Activations in the form the products read: [M * terms][KP] bf16, KP = K
// rounded up to 64, zero padded.  float32 gives three truncated terms v =
// t0 + t1 + t2 (8 mantissa bits each, every difference exact; an infinity or
// NaN is all in t0), bf16 is copied (rows that are not 16-byte aligned).
template <typename XT>
__global__ void __launch_bounds__(kThreads)
    q4_terms_kernel(const XT* __restrict__ x, int64_t ldx, int64_t M, int64_t K, int64_t KP,
                    __nv_bfloat16* __restrict__ out) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t total = M * KP;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t m = i / KP, k = i - m * KP;
        if constexpr (sizeof(XT) == 2) {
            out[i] = k < K ? x[m * ldx + k] : __float2bfloat16_rn(0.0f);
        } else {
            const float v = k < K ? x[m * ldx + k] : 0.0f;
            const uint32_t u = __float_as_uint(v);
            float r1 = v - __uint_as_float(u & 0xffff0000u);
            if ((u & 0x7f800000u) == 0x7f800000u) r1 = 0.0f;
            const float r2 = r1 - __uint_as_float(__float_as_uint(r1) & 0xffff0000u);
            const float t[3] = {v, r1, r2};
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                uint16_t h = static_cast<uint16_t>(__float_as_uint(t[j]) >> 16);
                if (j == 0 && v != v) h = 0x7fff;
                out[(3 * m + j) * KP + k] = __ushort_as_bfloat16(h);
            }
        }
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

// Shape of the product kernel for COLS MMA columns and scale groups of GS k.
// A block of the packed weight (128 channels x 128 k) is a pair of 64-k tiles;
// a unit is what a warpgroup hands to the tensor core at once: a pair, with
// one accumulator per scale group side by side, or one tile where a pair's
// accumulators would not fit.
template <int COLS, int GS>
struct Q4Cfg {
    static constexpr int TW = 128;                     // TMEM columns of a warpgroup: 4 per SM
    static constexpr int UT = GS == 32 && COLS == 32 ? 1 : 2;  // tiles per unit
    static constexpr int SUB = UT * 64 < GS ? 1 : UT * 64 / GS;  // accumulators per unit
    static constexpr int NSC = 128 / GS;               // scale groups of a pair
    static constexpr int ND = 32 * UT + 2 * SUB * COLS <= TW ? 2 : 1;  // accumulator buffers
    static constexpr int XB = COLS * 128;              // bytes of an activation tile
    // a pair's activations, then its block of weights and scales
    static constexpr int STAGE = 2 * XB + 8192 + (NSC * 512 + 1023) / 1024 * 1024;
    // an even ring: a stage always comes back to the warpgroup that saw its
    // previous phase, so no parity wait can mistake a phase for the one two back
    static constexpr int FIT = (113 * 1024 - 2048) / STAGE / 2 * 2;
    static constexpr int NS = FIT > 8 ? 8 : FIT;
    static constexpr int LD = 128 + 4;
    static constexpr int USED = 1024 + NS * STAGE + (2 * NS + 4) * 8 + 16;
    // two CTAs on an SM, never three: no CTA ever waits for tensor memory
    static constexpr int SMEM = USED > 78 * 1024 ? USED : 78 * 1024;
    static_assert(32 * UT + ND * SUB * COLS <= TW && NS >= 4 && SMEM <= 113 * 1024, "budgets");
    static_assert(NS * STAGE >= COLS * LD * 4, "the sums fit the ring");
};
constexpr int kQ4Threads = 12 * 32;

// A CTA computes 128 channels of one row tile over its part of K:
//   warps 0-7   two warpgroups, thread = channel = TMEM lane, that take the
//               pairs of 64-k tiles in turn.  Per unit: the channel's 4-bit
//               weights come from the shared-memory ring and go to tensor
//               memory as bf16 pairs (32 columns a tile) once the MMAs of the
//               unit before are done; then that unit's accumulators come back
//               and scale * sum is added to float32 registers.
//   warps 8-9   one per warpgroup, issue its MMAs (M = 128 channels, N =
//               columns, K = 16); one commit per unit.
//   warp 10     copies the weights, one bulk copy per pair.
//   warp 11     copies the activations, one TMA box per pair (128-byte swizzle).
// Four warpgroups share an SM (two CTAs).  Converting is what they compete
// for: 7 logic operations (half rate) and 4 subtractions per 8 weights, 224
// cycles of a scheduler per pair.  Two accumulator buffers let the sums be
// taken back under the next unit's MMAs; where only one fits they are taken
// before the unit is handed over.
// The S CTAs of a cluster take parts of K; their sums are added in rank order.
// Every wait is bounded; a timeout sets the error word and ends all roles.
template <int COLS, int GS>
__global__ void __launch_bounds__(kQ4Threads, 2)
    q4_kernel(const __grid_constant__ CUtensorMap xmap, const Q4Args a) {
    using C = Q4Cfg<COLS, GS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    float* fin = reinterpret_cast<float*>(ring);  // [COLS][LD], after the loop
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
    const int cols = rows * a.terms;
    const int p0 = static_cast<int>(a.NP * ks / a.S), np = static_cast<int>(a.NP * (ks + 1) / a.S) - p0;

    const uint8_t* src = a.w + ((g * a.NC + tile) * a.NP + p0) * a.block;
    auto copy_weights = [&](int p) {
        uint64_t* full = &in_full[p % C::NS];
        mbar_arrive_expect_tx(full, a.block);
        bulk_load(ring + p % C::NS * C::STAGE + 2 * C::XB, src + static_cast<int64_t>(p) * a.block, a.block, full);
    };
    auto copy_x = [&](int p) {
        uint64_t* full = &in_full[p % C::NS];
        mbar_arrive_expect_tx(full, 2 * C::XB);
        tma_load_3d(ring + p % C::NS * C::STAGE, &xmap, full, 0, static_cast<int>(m0 * a.terms), 2 * (p0 + p));
    };
    if (w == 9) {
        tmem_alloc(tmem_slot, 2 * C::TW);
        tmem_relinquish();
    } else if (w == 10 && lane == 0) {
        // the first weights are on their way before the rest of the set-up
        for (int i = 0; i < C::NS; ++i) {
            mbar_init(&in_full[i], 2);   // both copies
            mbar_init(&in_empty[i], 4);  // the four warps of the pair's warpgroup
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

    float acc[COLS] = {};
    const int ch = threadIdx.x & 127;
    if (w < 8) {
        const uint32_t quarter = static_cast<uint32_t>(32 * (w & 3)) << 16;
        auto take = [&](int u, const float (&s)[C::SUB]) {  // unit u's sums, scaled
#pragma unroll
            for (int j = 0; j < C::SUB; ++j)
#pragma unroll
                for (int c = 0; c < COLS; c += 16) {
                    if (c >= cols) continue;
                    uint32_t r[16];
                    tc_ld_32x32b_x16(td + quarter + (u % C::ND * C::SUB + j) * COLS + c, r);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[c + i] = fmaf(s[j], __uint_as_float(r[i]), acc[c + i]);
                }
            tc_fence_before();
        };
        float s_prev[C::SUB];
        int u = 0;  // units of this warpgroup so far
        bool ok = true;
        for (int p = wg; ok && p < np; p += 2) {
            const uint8_t* st = ring + p % C::NS * C::STAGE + 2 * C::XB;
            if (!(ok = wait(&in_full[p % C::NS], p / C::NS))) break;
            float s[C::NSC];
#pragma unroll
            for (int j = 0; j < C::NSC; ++j)
                s[j] = a.scale_bf16
                           ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(st + 8192)[j * 128 + ch])
                           : reinterpret_cast<const float*>(st + 8192)[j * 128 + ch];
            auto weights = [&](int i) { return *reinterpret_cast<const uint4*>(st + i * 2048 + ch * 16); };
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t v[16];
                if (C::ND == 2) {  // registers allow converting under the wait
                    const uint4 q0 = weights(2 * j);
                    unpack_q4(q0.x, v), unpack_q4(q0.y, v + 4), unpack_q4(q0.z, v + 8), unpack_q4(q0.w, v + 12);
                }
                if (u && (C::UT == 1 || j == 0)) {
                    // the unit before is done: its weights' columns, its
                    // accumulators and (at a pair's start) its stage are free
                    if (!(ok = wait(&done[wg], u - 1))) break;
                    tc_fence_after();
                    if (j == 0 && lane == 0) mbar_arrive(&in_empty[(p - 2) % C::NS]);
                    if (C::ND == 1) take(u - 1, s_prev);
                }
                if (C::ND == 1) {
                    const uint4 q0 = weights(2 * j);
                    unpack_q4(q0.x, v), unpack_q4(q0.y, v + 4), unpack_q4(q0.z, v + 8), unpack_q4(q0.w, v + 12);
                }
                const uint32_t at = ta + quarter + (C::UT == 2 ? 32 * j : 0);
                tc_st_32x32b_x16(at, v);
                const uint4 q1 = weights(2 * j + 1);
                unpack_q4(q1.x, v), unpack_q4(q1.y, v + 4), unpack_q4(q1.z, v + 8), unpack_q4(q1.w, v + 12);
                tc_st_32x32b_x16(at + 16, v);
                if (C::UT == 2 && j == 0) continue;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_full[wg]);
                if (C::ND == 2 && u) take(u - 1, s_prev);
#pragma unroll
                for (int i = 0; i < C::SUB; ++i) s_prev[i] = s[C::UT == 2 ? i : j * C::SUB + i];
                ++u;
            }
        }
        if (ok && u && wait(&done[wg], u - 1)) {
            tc_fence_after();
            take(u - 1, s_prev);
        }
    } else if (w < 10) {
        const uint32_t idesc = idesc_bf16_f32(128, static_cast<uint32_t>((cols + 15) & ~15));
        int u = 0;
        bool ok = true;
        for (int p = wg; ok && p < np; p += 2) {
            if (!(ok = wait(&in_full[p % C::NS], p / C::NS))) break;
            const uint64_t bd = smem_desc_sw128(smem_u32(ring + p % C::NS * C::STAGE));
#pragma unroll
            for (int j = 0; j < 2 / C::UT; ++j) {
                if (!(ok = wait(&a_full[wg], u))) break;
                tc_fence_after();
                const uint32_t d = td + static_cast<uint32_t>(u % C::ND * C::SUB * COLS);
#pragma unroll
                for (int m = 0; m < 4 * C::UT; ++m)
                    tc_mma_f16_ts_elect(d + 16 * m / GS * COLS, ta + 8 * m,
                                        bd + (j + m / 4) * (C::XB >> 4) + 2 * (m % 4), idesc,
                                        16 * m % GS ? 1u : 0u);
                tc_commit_elect(&done[wg]);
                ++u;
            }
        }
    } else if (lane == 0) {
        const bool weights = w == 10;
        if (!weights && a.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");  // x is the terms kernel's
        int p = weights ? min(np, C::NS) : 0;
        for (; p < np; ++p) {
            if (!mbar_wait_bounded(&in_empty[p % C::NS], (p / C::NS & 1) ^ 1, abort_flag, a.err, ERR_GEMM_TIMEOUT))
                break;
            if (weights)
                copy_weights(p);
            else
                copy_x(p);
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
            for (int c = 0; c < COLS; ++c)
                if (c < cols) fin[c * C::LD + ch] = j ? fin[c * C::LD + ch] + acc[c] : acc[c];
        __syncthreads();
    }
    if (a.S > 1) cluster_sync();
    for (int i = ks * kQ4Threads + threadIdx.x; i < rows * 128; i += a.S * kQ4Threads) {
        const int r = i >> 7, c = i & 127;
        float v = 0.0f;
        for (int s = 0; s < a.S; ++s)
            for (int j = 0; j < a.terms; ++j) {
                const float* p = fin + (r * a.terms + j) * C::LD + c;
                v += s == ks ? *p : ld_cluster(p, s);
            }
        if (tile * 128 + c < a.N) store_out(a, m0 + r, tile * 128 + c, v);
    }
    if (a.S > 1) cluster_sync();  // the sums stay until every rank has read them
}

template <int COLS, int GS>
aem_status launch_q4(const CUtensorMap& xmap, const Q4Args& a, dim3 grid, cudaStream_t s) {
    using C = Q4Cfg<COLS, GS>;
    auto kern = q4_kernel<COLS, GS>;
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
    if (a.S > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = a.S;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    if (a.dependent) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    AEM_TRY_CUDA(cudaLaunchKernelEx(&cfg, kern, xmap, a));
    count_launches(1);
    return AEM_OK;
}

template <int COLS>
aem_status launch_cols(const void* x, int64_t ldx, int64_t K, Q4Args a, int gs, int64_t slots,
                       cudaStream_t s) {
    CUtensorMap xmap;  // [K / 64][rows][64]: one box holds a pair of 64-k tiles
    AEM_TRY(make_tmap_3d(&xmap, x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 64, a.M * a.terms, K / 64, ldx * 2, 128,
                         64, COLS, 2, CU_TENSOR_MAP_SWIZZLE_128B));
    // K is split until the CTAs fill the SMs: waves x (a CTA's own latency, as
    // long as about 8 pairs, and its pairs)
    const int64_t ctas = a.NC * slots, fit = 148 * 2, pairs = a.NP;
    int64_t best = INT64_MAX;
    for (int S = 1; S <= 8 && S <= std::max<int64_t>(1, pairs / 2); ++S) {
        const int64_t cost = (ctas * S + fit - 1) / fit * (8 + (pairs + S - 1) / S);
        if (cost < best) {
            best = cost;
            a.S = S;
        }
    }
    const dim3 grid(static_cast<unsigned>(a.NC * a.S), static_cast<unsigned>(slots));
    return gs == 32   ? launch_q4<COLS, 32>(xmap, a, grid, s)
           : gs == 64 ? launch_q4<COLS, 64>(xmap, a, grid, s)
                      : launch_q4<COLS, 128>(xmap, a, grid, s);
}

// x: the caller's rows.
aem_status q4_product(const Q4Weight* w, const char* what, Q4Args a, const void* x, aem_dtype xd,
                      int64_t ldx, void* workspace, size_t workspace_bytes, cudaStream_t s) {
    AEM_REQUIRE(current_device() == w->device, "%s: the weights are on device %d, the current one is %d",
                what, w->device, current_device());
    a.w = w->data;
    a.block = w->block;
    a.scale_bf16 = w->scale_bf16;
    a.N = w->N;
    a.NC = w->NC;
    a.NP = w->NP;
    a.err = device_error_word(w->device);
    a.terms = xd == AEM_F32 ? 3 : 1;
    AEM_REQUIRE(a.M * a.terms < (1ll << 31), "%s: M=%lld out of range", what, (long long)a.M);
    // columns of a row tile: as many as the rows (grouped: an average group's) need, up to 32
    const int64_t groups = std::min<int64_t>(a.G, a.M);
    const int64_t want = (a.group_rows ? (a.M + groups - 1) / groups : a.M) * a.terms;
    const int cols = want <= 16 ? 16 : 32;
    a.rows = cols / a.terms;
    const int64_t slots = a.group_rows ? groups + a.M / a.rows : (a.M + a.rows - 1) / a.rows;
    AEM_REQUIRE(slots <= 65535, "%s: M=%lld rows are too many for one call", what, (long long)a.M);
    const int64_t K = w->K;
    int64_t KP = K;
    void* own = nullptr;
    if (xd != AEM_BF16 || K % 64 != 0 || (reinterpret_cast<uintptr_t>(x) & 15) != 0 || ldx % 8 != 0 || ldx < K) {
        KP = (K + 63) / 64 * 64;
        const size_t need = static_cast<size_t>(a.M) * a.terms * KP * 2;
        AEM_REQUIRE(!workspace || (workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                    "%s: workspace of %zu bytes (%zu needed, 16-byte aligned)", what, workspace_bytes, need);
        if (!workspace) {
            AEM_TRY_CUDA(cudaMallocAsync(&own, need, s));
            workspace = own;
        }
        auto* t = static_cast<__nv_bfloat16*>(workspace);
        const unsigned g = static_cast<unsigned>(std::min<int64_t>((a.M * KP + kThreads - 1) / kThreads, 148 * 8));
        if (xd == AEM_F32)
            q4_terms_kernel<float><<<g, kThreads, 0, s>>>(static_cast<const float*>(x), ldx, a.M, K, KP, t);
        else
            q4_terms_kernel<__nv_bfloat16><<<g, kThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(x), ldx,
                                                                  a.M, K, KP, t);
        count_launches(1);
        a.dependent = true;
        x = t;
        ldx = KP;
    }
    const cudaError_t e = cudaGetLastError();
    aem_status st;
    if (e != cudaSuccess) {
        set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
        st = AEM_ECUDA;
    } else {
        st = cols == 16 ? launch_cols<16>(x, ldx, KP, a, w->gs, slots, s)
                        : launch_cols<32>(x, ldx, KP, a, w->gs, slots, s);
    }
    if (own) cudaFreeAsync(own, s);
    return st;
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
        AEM_REQUIRE(q[i] >= -8 && q[i] <= 7, "aem_q4weight_pack: q[%lld]=%d is outside [-8, 7]",
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
    const int64_t KP = (reinterpret_cast<aem::Q4Weight*>(wh)->K + 63) / 64 * 64;
    return static_cast<size_t>(M) * (x_dtype == AEM_F32 ? 3 : 1) * KP * 2;
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
    return aem::q4_product(w, "aem_q4gemm", a, x, x_dtype, ldx, workspace, workspace_bytes,
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
    return aem::q4_product(w, "aem_grouped_q4gemm", a, x, x_dtype, ldx, workspace, workspace_bytes,
                           static_cast<cudaStream_t>(stream));
}

}  // extern "C"
