// Products of rows with 8-bit floating point weights, scales per block of 128:
//
//   out[m, n] = sum_b xs[m, b] ws[b, n / 128] sum_{k in block b} xq[m, k] wq[k, n]
//
// dense and grouped by expert, and with the transposed weight (the gradient of the
// rows: the sum runs over the channels).  A block's sum is four tcgen05 MMAs of
// K = 32 on e4m3 operands with float32 accumulators in TMEM; the block's scales
// differ from row to row, so its sum is taken back and added to float32 registers
// as one multiply-add per element.
//
// fp8_few_kernel: weights are the MMA's 128 rows (the channels), tokens its
// columns; the weight stream is what bounds few rows.  One bf16 row, 4096 x 14336:
// 15.4 us with its quantisation, 13.9 without, 4.2 TB/s of weights; 64 rows 17.8 us;
// 384 rows of 64 experts of 2048 x 1408 36 us, 5.1 TB/s.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "fp8.h"
#include "runtime.h"

namespace aem {
namespace {

using namespace aem::dev;

struct Fp8Args {
    const uint8_t* w;           // packed tiles
    const float* ws;            // their scales
    const float* xs;            // [M][lds]
    void* out;
    const int32_t* group_rows;  // nullptr: one group of M rows, weight group `group`
    int64_t lds, ldo, M, N;     // N: columns of out
    int64_t group, group_tiles; // tiles of a weight group
    int64_t out_step, sum_step; // tiles from one 128 of out's columns (of the sum) to the next
    int nb, kb, G, S, rows;     // 128-blocks of out's columns and of the sum; S: CTAs (one cluster) that split
                                // the sum; rows: rows of a row tile
    int out_bf16, relu, ovec, ovec16;  // ovec: out can be stored in vectors of 4; ovec16: of 16 bytes
    int* err;
};

// Row tile `slot` of the groups' row tiles: its group, first row and rows.
// Every warp searches alike.  Offsets are clamped to [0, M].
__device__ __forceinline__ bool find_rows(const Fp8Args& a, int slot, int64_t* g, int64_t* m0, int* rows) {
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

// a0 += s0 * v0, a1 += s1 * v1
__device__ __forceinline__ void fma2(float& a0, float& a1, float s0, float s1, uint32_t v0, uint32_t v1) {
    asm volatile("{\n.reg .b64 a, s, v;\nmov.b64 a, {%0, %1};\nmov.b64 s, {%2, %3};\nmov.b64 v, {%4, %5};\n"
                 "fma.rn.f32x2 a, s, v, a;\nmov.b64 {%0, %1}, a;\n}"
                 : "+f"(a0), "+f"(a1)
                 : "f"(s0), "f"(s1), "r"(v0), "r"(v1));
}

__device__ __forceinline__ void st_cluster(const float4* p, uint32_t rank, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mapa_u32(p, rank)), "f"(v.x),
                 "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}

__device__ __forceinline__ float relu_of(float v) { return v < 0.0f ? 0.0f : v; }  // keeps a NaN

// Four columns of a row of out.
__device__ __forceinline__ void store_out(const Fp8Args& a, int64_t m, int64_t n, float4 v) {
    if (a.relu) v = make_float4(relu_of(v.x), relu_of(v.y), relu_of(v.z), relu_of(v.w));
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

// Operand descriptor of a packed tile and its step along K for 32 more: K-major
// rows (32 bytes further), or MN-major (32 rows of 128 bytes further; the tile's 128
// elements of M or N are one atom wide, 8 rows of K follow 1024 bytes apart).
// Both have the same fields.
template <bool MN>
constexpr uint32_t kStep32 = MN ? 32 * 128 / 16 : 32 / 16;

// Few rows: a CTA computes 128 columns of out for a tile of TN rows over its part
// of the sum.
//   warps 0-7   thread = column of out = TMEM lane; warps 0-3 have the first half
//               of the rows, 4-7 the second.  Per block of 128: its accumulator
//               comes back and scale * sum is added to the row's register.
//   warp 8      issues the MMAs (M = 128, N = rows, K = 32), four per block
//   warp 9      copies the weights, one bulk copy of a 16 KB tile per block
//   warp 10     copies the rows, one TMA box per block, and leaves the products of
//               their scales with the block's beside them
// The S CTAs of a cluster take parts of the sum: each sends its sums to the rank
// that writes those rows, which adds them in rank order.
// Every wait is bounded; a timeout sets the error word and ends all roles.
constexpr int kFewThreads = 11 * 32;
template <int TN, bool ALONE>
struct FewCfg {
    static constexpr int CTAS = ALONE ? 1 : 2;  // on an SM
    static constexpr int ND = 4;                // accumulators in TMEM
    static constexpr int XB = TN * 128;
    static constexpr int STAGE = kFp8Tile + XB + TN * 4;
    static constexpr int MOST = ALONE ? 226 * 1024 : 113 * 1024;
    static constexpr int FIXED = 1024 + 512;  // alignment; barriers
    static constexpr int FIT = (MOST - FIXED) / STAGE;
    static constexpr int NS = FIT > 12 ? 12 : FIT;
    static constexpr int USED = FIXED + NS * STAGE;
    // so many CTAs on an SM and no more: no CTA ever waits for tensor memory
    static constexpr int LEAST = ALONE ? 116 * 1024 : 78 * 1024;
    static constexpr int SMEM = USED > LEAST ? USED : LEAST;
    static constexpr int COLS = ND * TN < 32 ? 32 : ND * TN;
    static_assert(COLS * CTAS <= 512 && NS >= 3, "budgets");
    // the CTA's sums [TN][128] and the cluster's [S][ceil(TN / S)][128], in the ring
    static_assert((TN + TN + 7) * 512 <= NS * (kFp8Tile + XB), "sums fit the ring");
};

template <int TN, bool ALONE, bool TRANS>
__global__ void __launch_bounds__(kFewThreads, ALONE ? 1 : 2)
    fp8_few_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ Fp8Args a) {
    using C = FewCfg<TN, ALONE>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    uint8_t* xring = ring + C::NS * kFp8Tile;
    float* sring = reinterpret_cast<float*>(xring + C::NS * C::XB);
    uint64_t* full = reinterpret_cast<uint64_t*>(sring + C::NS * TN);
    uint64_t* empty = full + C::NS;
    uint64_t* dfull = empty + C::NS;
    uint64_t* dempty = dfull + C::ND;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dempty + C::ND);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int tile = static_cast<int>(blockIdx.x) / a.S, ks = static_cast<int>(blockIdx.x) % a.S;
    int64_t g, m0;
    int rows;
    if (!find_rows(a, blockIdx.y, &g, &m0, &rows)) {  // the whole cluster alike
        asm volatile("griddepcontrol.wait;" ::: "memory");  // this grid ends after the one that makes the rows
        return;
    }
    const int p0 = static_cast<int>(static_cast<int64_t>(a.kb) * ks / a.S);
    const int np = static_cast<int>(static_cast<int64_t>(a.kb) * (ks + 1) / a.S) - p0;
    const int64_t t0 = g * a.group_tiles + tile * a.out_step + p0 * a.sum_step;  // the CTA's first tile
    auto copy_weights = [&](int u) {
        mbar_arrive_expect_tx(&full[u % C::NS], kFp8Tile);
        bulk_load(ring + u % C::NS * kFp8Tile, a.w + (t0 + u * a.sum_step) * kFp8Tile, kFp8Tile, &full[u % C::NS]);
    };
    if (w == 8) {
        tmem_alloc(tmem_slot, C::COLS);
        tmem_relinquish();
    } else if (w == 9 && lane == 0) {
        for (int i = 0; i < C::NS; ++i) {
            mbar_init(&full[i], 3);  // both copies' bytes and the scales
            mbar_init(&empty[i], 1 + 8);  // the MMAs and the warps that read the scales
        }
        for (int i = 0; i < C::ND; ++i) {
            mbar_init(&dfull[i], 1);
            mbar_init(&dempty[i], 8);
        }
        *abort_flag = 0;
        fence_barrier_init();
        // the first weights are on their way before the rest of the set-up
        for (int u = 0; u < min(np, C::NS); ++u) copy_weights(u);
    } else if (w == 10 && lane == 0) {
        tma_prefetch_desc(&xmap);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto wait = [&](uint64_t* bar, int phase) {  // whole warps
        if (__all_sync(~0u, mbar_try_wait(bar, phase & 1))) return true;
        return __all_sync(~0u, mbar_wait_bounded(bar, phase & 1, abort_flag, a.err, ERR_GEMM_TIMEOUT)) != 0;
    };

    constexpr int CPT = TN / 2;  // rows of a thread
    float acc[CPT] = {};
    if (w < 8) {
        const int h = w >> 2;
        const uint32_t at = tmem + (static_cast<uint32_t>(32 * (w & 3)) << 16) + h * CPT;
        for (int u = 0; u < np; ++u) {
            const int st = u % C::NS, b = u % C::ND;
            if (!wait(&full[st], u / C::NS) || !wait(&dfull[b], u / C::ND)) break;
            tc_fence_after();
            uint32_t d[CPT];
            if constexpr (CPT == 8)
                tc_ld_32x32b_x8(at + b * TN, d);
            else if constexpr (CPT == 16)
                tc_ld_32x32b_x16(at + b * TN, d);
            else
#pragma unroll
                for (int c = 0; c < CPT; c += 32)
                    tc_ld_32x32b_x32(at + b * TN + c, *reinterpret_cast<uint32_t(*)[32]>(d + c));
            tc_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&dempty[b]);
            const float4* sc = reinterpret_cast<const float4*>(sring + st * TN + h * CPT);
#pragma unroll
            for (int c = 0; c < CPT; c += 4) {
                const float4 s = sc[c / 4];
                fma2(acc[c], acc[c + 1], s.x, s.y, d[c], d[c + 1]);
                fma2(acc[c + 2], acc[c + 3], s.z, s.w, d[c + 2], d[c + 3]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
    } else if (w == 8) {
        const uint32_t idesc = idesc_e4m3_f32(128, static_cast<uint32_t>((rows + 15) & ~15), TRANS, false);
        for (int u = 0; u < np; ++u) {
            const int st = u % C::NS, b = u % C::ND;
            if (!wait(&full[st], u / C::NS) || !wait(&dempty[b], u / C::ND + 1)) break;
            tc_fence_after();
            const uint64_t ad = smem_desc_sw128(smem_u32(ring + st * kFp8Tile));
            const uint64_t bd = smem_desc_sw128(smem_u32(xring + st * C::XB));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                tc_mma_f8_elect(tmem + b * TN, ad + i * kStep32<TRANS>, bd + i * kStep32<false>, idesc, i ? 1u : 0u);
            tc_commit_elect(&empty[st]);
            tc_commit_elect(&dfull[b]);
        }
    } else if (w == 9) {
        if (lane == 0) {
            int u = min(np, C::NS);
            for (; u < np; ++u) {
                if (!mbar_wait_bounded(&empty[u % C::NS], (u / C::NS + 1) & 1, abort_flag, a.err, ERR_GEMM_TIMEOUT)) break;
                copy_weights(u);
            }
            if (*abort_flag)  // a failed call leaves no copy in flight behind (bounded as well)
                for (int i = max(0, u - C::NS); i < u; ++i)
                    for (int t = 0; t < 1 << 14 && !mbar_try_wait(&full[i % C::NS], i / C::NS & 1); ++t) {
                    }
        }
    } else {
        // scales: the weights' of 32 blocks, one a lane, and the rows' of a lane's rows,
        // four blocks at a time and four ahead
        constexpr int R = (TN + 31) / 32;
        float held = a.ws[t0 + min(lane, np - 1) * a.sum_step], now[R][4], next[R][4];
        asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows may be another kernel's
        const float* xs = a.xs + m0 * a.lds + p0;
        auto fetch = [&](int u) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) next[r][k] = xs[min(r * 32 + lane, rows - 1) * a.lds + min(u + k, np - 1)];
        };
        fetch(0);
        int u = 0;
        for (bool ok = true; ok && u < np;) {
            if (u && (u & 31) == 0) held = a.ws[t0 + min(u + lane, np - 1) * a.sum_step];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) now[r][k] = next[r][k];
            fetch(u + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (u >= np) break;
                const int st = u % C::NS;
                const float sw = __shfl_sync(~0u, held, u & 31);
                if (!(ok = wait(&empty[st], u / C::NS + 1))) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&full[st], C::XB);
                    tma_load_2d(xring + st * C::XB, &xmap, &full[st], (p0 + u) * 128, static_cast<int>(m0));
                }
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (r * 32 + lane < TN) sring[st * TN + r * 32 + lane] = now[r][k] * sw;
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[st]);
                ++u;
            }
        }
        if (lane == 0 && *abort_flag)
            for (int i = max(0, u - C::NS); i < u; ++i)
                for (int t = 0; t < 1 << 14 && !mbar_try_wait(&full[i % C::NS], i / C::NS & 1); ++t) {
                }
    }

    // every MMA has been waited for by the warps that read its sums (or the call
    // failed): give the tensor memory back before any wait on another CTA
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (w == 8) tmem_dealloc(tmem, C::COLS);
    float* fin = reinterpret_cast<float*>(ring);  // [TN][128]
    float* recv = fin + TN * 128;                 // [S][share][128]
    if (w < 8)
#pragma unroll
        for (int c = 0; c < CPT; ++c) fin[((w >> 2) * CPT + c) * 128 + (w & 3) * 32 + lane] = acc[c];
    __syncthreads();
    const int share = (rows + a.S - 1) / a.S;    // rows that a rank writes
    const int64_t n = tile * 128ll + lane * 4;  // a warp has a row, a lane four columns of it
    const float4* fin4 = reinterpret_cast<const float4*>(fin) + lane;
    float4* recv4 = reinterpret_cast<float4*>(recv) + lane;
    constexpr int WARPS = kFewThreads / 32;
    if (a.S == 1) {
        for (int r = w; r < rows; r += WARPS) store_out(a, m0 + r, n, fin4[r * 32]);
        return;
    }
    cluster_sync();  // the ranks' rings are free
    for (int r = w; r < rows; r += WARPS) {
        const int to = r / share;
        st_cluster(recv4 + (ks * share + r - to * share) * 32, to, fin4[r * 32]);
    }
    cluster_sync();
    for (int r = w; r < share && ks * share + r < rows; r += WARPS) {
        float4 v = recv4[r * 32];
        for (int s = 1; s < a.S; ++s) {
            const float4 u = recv4[(s * share + r) * 32];
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        store_out(a, m0 + ks * share + r, n, v);
    }
}

// Many rows: a pair of SMs computes 256 rows x 256 columns of out, one CTA 128
// rows of it.  Rows are the MMA's M (a thread has a row, so a block's two scales are
// one factor for all of its columns), the weights are its N, half of them in each
// CTA's shared memory, which halves what has to be read for them.  The pair is
// persistent over tiles.
//   warp 0      copies a block's rows and weights, 16 KB each, into the ring
//   warp 1      issues the pair's MMAs (M = 256, N = 256, K = 32) in CTA 0, four a
//               block, into one of two accumulators that fill tensor memory
//   warps 4-11  thread = row = TMEM lane; warps 4-7 have the first 128 columns, 8-11
//               the rest.  A block's accumulator comes back 16 columns at a time and
//               factor * sum is added to 128 registers; at the tile's end these are
//               left in shared memory
//   warps 2, 3  write them from there, whole rows of 128 columns, under the next tile
//               (a bulk copy of each row by the summing warps held those up for 3200
//               cycles a tile, 90 a copy: 98304 x 2048 x 1408 by 64 experts 342 us, so 309)
// 4096 x 4096 x 14336, rows quantised before: 220 us, 2.2 PFLOP/s.  The MMAs with
// their barriers alone take 155; what bounds it is the warps that take the sums back,
// about 700 cycles a block where the MMAs take 512 (264 are multiply-adds of the two
// warps that share a sub-core), and a tile's first and last block, which overlap with
// no other's MMAs.  For seconds on end it takes 249 us (258 a call with the rows'
// quantisation): the power limit (990 W) leaves 1.5 GHz.  Accumulators of half the width,
// four of them, wait twice as often: 261 us.
// The registers decide: 128 sums, 32 columns under way, and every variable more that
// was kept through the loop was moved about in it (32 columns a load 238 us, the next
// block's first columns ahead 231, pointers kept 245, one float4 of scales 225 instead of
// 220).
// Every wait is bounded; a timeout sets the error word and ends all roles of both CTAs.
constexpr int kManyThreads = 12 * 32, kManyStages = 4, kManyTile = 256;
constexpr int kManyStage = 2 * kFp8Tile;                      // of one CTA
constexpr int kManyPitch = 256 + 16;                          // a row's 256 bytes of out, in other banks than the next's
constexpr int kManyOut = 8 * 32 * kManyPitch;
constexpr int kManyScales = 2 * 256 * 16;                     // four blocks' scales of a thread's row, twice
// Registers of a thread of warps 0-3 and of warps 4-11: together what the block is launched with.
constexpr int kManyFewRegs = 40, kManyManyRegs = 232;
static_assert(kManyFewRegs * 128 + kManyManyRegs * 256 <= 168 * kManyThreads, "register shares");
constexpr int kBand = 16;  // row tiles that share the columns' weights before the next ones come

// Shared memory of a CTA, in bytes from a 1024-byte boundary on.  Addresses are this
// boundary's 32 bits and a constant: the sums leave few registers for anything else.
constexpr int kManyOutAt = kManyStages * kManyStage, kManyScalesAt = kManyOutAt + kManyOut;
constexpr int kManyFullAt = kManyScalesAt + kManyScales;             // [stages], used in CTA 0
constexpr int kManyEmptyAt = kManyFullAt + 8 * kManyStages;          // [stages]
constexpr int kManyDoneAt = kManyEmptyAt + 8 * kManyStages;          // [2]: an accumulator's sums are there
constexpr int kManyFreeAt = kManyDoneAt + 16;                        // [2]: they have been read; used in CTA 0
constexpr int kManyStagedAt = kManyFreeAt + 16;                      // [2]: results of 128 columns lie in shared memory
constexpr int kManyCopiedAt = kManyStagedAt + 16;                    // [2]: they have been read from there
constexpr int kManySlotAt = kManyCopiedAt + 16, kManyAbortAt = kManySlotAt + 4;
constexpr int kManyRowsAt = kManySlotAt + 16, kManyTilesAt = kManyRowsAt + (AEM_MAX_EXPERTS + 1) * 4;
// A pair's first tiles, looked up side by side at the start: three roles ask for each
// one, and of 64 groups a search takes some 500 cycles.
constexpr int kManyKept = 256, kManyKeptAt = (kManyTilesAt + (AEM_MAX_EXPERTS + 1) * 4 + 15) / 16 * 16;
constexpr int kManySmem = 1024 + kManyKeptAt + kManyKept * 16;
static_assert(kManyKept <= kManyThreads && kManySmem <= 227 * 1024, "a thread looks a tile up; shared memory");

__device__ __forceinline__ int lds_int(uint32_t at) {
    int v;
    asm volatile("ld.volatile.shared.s32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ void sts_int(uint32_t at, int v) {
    asm volatile("st.volatile.shared.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
// Whether the phase with `parity` is complete: at once, or after a while.
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint32_t cluster_address(uint32_t at, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
// An arrival of the warp's first lane at a barrier of the cluster, without a branch.
__device__ __forceinline__ void arrive_first_lane(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .u32 l;\n\t"
        "mov.u32 l, %%laneid;\n\t"
        "setp.eq.u32 p, l, 0;\n\t"
        "@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar)
        : "memory");
}
// Bounded wait of a whole warp that, on giving up, raises the abort flag of both CTAs.
// `done`: what a look at the barrier ahead of time saw (a look takes some 60 cycles).
__device__ __forceinline__ bool pair_wait(uint32_t bar, uint32_t parity, bool done, uint32_t sb, int* err) {
    if (__all_sync(~0u, done)) return true;
    uint64_t t0 = 0;
    for (int i = 0;; ++i) {  // the clock is read now and then: it is slow
        if (__all_sync(~0u, bar_try(bar, parity))) return true;
        if (i & 31) continue;
        if (__any_sync(~0u, lds_int(sb + kManyAbortAt) != 0)) return false;
        if (i == 0) continue;
        const uint64_t t = globaltimer_ns();
        if (t0 == 0) t0 = t;
        if (__any_sync(~0u, t - t0 > 2000000000ull)) {
            for (uint32_t r = 0; r < 2; ++r)
                asm volatile("st.shared::cluster.u32 [%0], 1;" ::"r"(cluster_address(sb + kManyAbortAt, r)) : "memory");
            atomicOr(err, ERR_GEMM_TIMEOUT);
            return false;
        }
    }
}

// 16 columns: acc += f * d.  (Two columns an instruction: beside 128 single ones a
// block, the MMAs take half as long again.)
__device__ __forceinline__ void add_columns(float* acc, float f, const uint32_t (&d)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 2)
        asm volatile("{\n.reg .b64 a, f, v;\nmov.b64 a, {%0, %1};\nmov.b64 f, {%2, %2};\nmov.b64 v, {%3, %4};\n"
                     "fma.rn.f32x2 a, f, v, a;\nmov.b64 {%0, %1}, a;\n}"
                     : "+f"(acc[i]), "+f"(acc[i + 1])
                     : "f"(f), "r"(d[i]), "r"(d[i + 1]));
}

__device__ __forceinline__ uint32_t bf16x2_of(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

struct ManyTile {
    int64_t t0;    // first weight tile of the pair's columns
    int m0, rows;  // first row and number of rows
    int col;       // first 128-block of columns
};
struct ManyKept {
    int m0, rows, col, g;  // the same with the group
};
__device__ __forceinline__ ManyKept find_tile(const Fp8Args& a, int t, uint32_t sb) {
    int lo = 0, hi = a.G;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (lds_int(sb + kManyTilesAt + mid * 4) <= t) lo = mid; else hi = mid;
    }
    const int first = lds_int(sb + kManyTilesAt + lo * 4), nc = (a.nb + 1) / 2;
    const int r = t - first, n = (lds_int(sb + kManyTilesAt + lo * 4 + 4) - first) / nc;
    const int band = r / (kBand * nc), in = r - band * kBand * nc, high = min(kBand, n - band * kBand);
    const int row = lds_int(sb + kManyRowsAt + lo * 4), end = lds_int(sb + kManyRowsAt + lo * 4 + 4);
    ManyKept o;
    o.col = in / high * 2;
    o.m0 = row + (band * kBand + in % high) * kManyTile;
    o.rows = min(kManyTile, end - o.m0);
    o.g = lo;
    return o;
}
// Tile t, the pair's turn-th.
__device__ __forceinline__ ManyTile many_tile(const Fp8Args& a, int t, int turn, uint32_t sb) {
    ManyKept k;
    if (turn < kManyKept)
        asm volatile("ld.volatile.shared.v4.s32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(k.m0), "=r"(k.rows), "=r"(k.col), "=r"(k.g)
                     : "r"(sb + kManyKeptAt + turn * 16));
    else
        k = find_tile(a, t, sb);
    return {(a.group_rows ? k.g : a.group) * a.group_tiles, k.m0, k.rows, k.col};
}

template <bool TRANS, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kManyThreads, 1)
    fp8_many_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                    const __grid_constant__ Fp8Args a) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sb = (smem_u32(smem_raw) + 1023) & ~1023u;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const uint32_t cta = cluster_rank();
    const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);
    if (w == 0 && lane == 0) {
        auto init = [&](uint32_t at, uint32_t count) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sb + at), "r"(count) : "memory");
        };
        for (int i = 0; i < kManyStages; ++i) {
            init(kManyFullAt + 8 * i, 1);
            init(kManyEmptyAt + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            init(kManyDoneAt + 8 * i, 1);
            init(kManyFreeAt + 8 * i, 16);  // the warps of both CTAs that read it
            init(kManyStagedAt + 8 * i, 4);
            init(kManyCopiedAt + 8 * i, 32);
        }
        sts_int(sb + kManyAbortAt, 0);
        fence_barrier_init();
        tma_prefetch_desc(&xmap);
        tma_prefetch_desc(&wmap);
    } else if (w == 1) {  // the same warp of both CTAs
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(sb + kManySlotAt)
                     : "memory");
        tmem_relinquish_pair();
    } else if (w == 2) {
        // first rows and first tiles of the groups, 32 groups at a time
        const int nc = (a.nb + 1) / 2, M = static_cast<int>(a.M);
        int before = 0;
        for (int i = 0; i < a.G; i += 32) {
            int lo = 0, hi = 0;
            if (i + lane < a.G) {
                lo = a.group_rows ? min(max(a.group_rows[i + lane], 0), M) : 0;
                hi = a.group_rows ? min(max(a.group_rows[i + lane + 1], 0), M) : M;
            }
            const int n = hi > lo ? (hi - lo + kManyTile - 1) / kManyTile * nc : 0;
            int s = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(~0u, s, o);
                if (lane >= o) s += v;
            }
            if (i + lane < a.G) {
                sts_int(sb + kManyRowsAt + (i + lane) * 4, lo);
                sts_int(sb + kManyTilesAt + (i + lane) * 4, before + s - n);
                if (i + lane == a.G - 1) {
                    sts_int(sb + kManyRowsAt + a.G * 4, hi);
                    sts_int(sb + kManyTilesAt + a.G * 4, before + s);
                }
            }
            before += __shfl_sync(~0u, s, 31);
        }
    }
    tc_fence_before();
    __syncthreads();
    const int total = lds_int(sb + kManyTilesAt + a.G * 4);
    if (const int i = threadIdx.x; i < kManyKept && pair + i * pairs < total) {
        const ManyKept k = find_tile(a, pair + i * pairs, sb);
        asm volatile("st.volatile.shared.v4.s32 [%0], {%1, %2, %3, %4};" ::"r"(sb + kManyKeptAt + i * 16), "r"(k.m0),
                     "r"(k.rows), "r"(k.col), "r"(k.g)
                     : "memory");
    }
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are there before any remote arrival
    tc_fence_after();
    const uint32_t tmem = static_cast<uint32_t>(lds_int(sb + kManySlotAt));

    if (w < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyFewRegs));
        if (w == 0) {
            asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows may be another kernel's
            // both CTAs' bytes complete on CTA 0's barrier
            const uint32_t full = cluster_address(sb + kManyFullAt, 0);
            auto load = [&](uint32_t to, const CUtensorMap* map, uint32_t bar, int x, int y) {
                asm volatile(
                    "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
                    " [%0], [%1, {%3, %4}], [%2];" ::"r"(to),
                    "l"(map), "r"(bar), "r"(x), "r"(y)
                    : "memory");
            };
            int st = 0;
            uint32_t phase = 0;
            int issued = 0;
            bool ok = true;
            for (int t = pair, turn = 0; ok && t < total; t += pairs, ++turn) {
                const ManyTile z = many_tile(a, t, turn, sb);
                // an odd number of blocks: the last pair's second half takes the last block
                // again, its results are not stored
                int tile = static_cast<int>((z.t0 + min(z.col + static_cast<int>(cta), a.nb - 1) * a.out_step) * 128);
                const int row = z.m0 + static_cast<int>(cta) * 128, step = static_cast<int>(a.sum_step * 128);
                for (int u = 0; u < a.kb; ++u, tile += step) {
                    if (!(ok = pair_wait(sb + kManyEmptyAt + 8 * st, phase ^ 1, false, sb, a.err))) break;
                    if (lane == 0) {
                        const uint32_t to = sb + st * kManyStage;
                        if (cta == 0)
                            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                                             sb + kManyFullAt + 8 * st),
                                         "r"(2 * kManyStage)
                                         : "memory");
                        load(to, &xmap, full + 8 * st, u * 128, row);
                        load(to + kFp8Tile, &wmap, full + 8 * st, 0, tile);
                    }
                    ++issued;
                    if (++st == kManyStages) st = 0, phase ^= 1;
                }
            }
            if (!ok && cta == 0 && lane == 0)  // a failed call leaves no copy in flight behind (bounded as well)
                for (int i = max(0, issued - kManyStages); i < issued; ++i)
                    for (int n = 0; n < 1 << 14 && !bar_try(sb + kManyFullAt + 8 * (i % kManyStages),
                                                            i / kManyStages & 1); ++n) {
                    }
        } else if (w >= 2) {
            // results of a tile's first or last 128 columns, from shared memory to out
            const int half = w - 2;
            constexpr int ES = BF16 ? 2 : 4, PER = 256 / ES;  // columns of a piece
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair, turn = 0; ok && t < total; t += pairs, ++turn) {
                const ManyTile z = many_tile(a, t, turn, sb);
                const int64_t n = (z.col + half) * 128ll;
                const int left = static_cast<int>(min(static_cast<int64_t>(128), a.N - n));
                if (left <= 0 || !(a.ovec16 && left * ES % 16 == 0)) continue;
                const int first = static_cast<int>(cta) * 128 + (lane >> 4);
                const int rows = min(128, z.rows - static_cast<int>(cta) * 128);
                uint8_t* to = static_cast<uint8_t*>(a.out) + ((z.m0 + first) * a.ldo + n) * ES + (lane & 15) * 16;
                const uint32_t piece = sb + kManyOutAt + (half * 128 + (lane >> 4)) * kManyPitch + (lane & 15) * 16;
                const int64_t step = 2 * a.ldo * ES;
                for (int c = 0; c < left; c += PER) {
                    if (!(ok = pair_wait(sb + kManyStagedAt + 8 * half, phase, false, sb, a.err))) break;
                    phase ^= 1;
                    const bool inside = c + (lane & 15) * (16 / ES) < left;
                    uint8_t* dst = to + c * ES;
                    // two whole rows at a time, the next two on their way
#pragma unroll 1
                    for (int r = 0; r < rows; r += 4) {
                        uint32_t v[2][4];
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(v[k][0]), "=r"(v[k][1]), "=r"(v[k][2]), "=r"(v[k][3])
                                         : "r"(piece + (r + 2 * k) * kManyPitch)
                                         : "memory");
#pragma unroll
                        for (int k = 0; k < 2; ++k, dst += step)
                            if (inside && r + 2 * k + (lane >> 4) < rows)
                                *reinterpret_cast<uint4*>(dst) = make_uint4(v[k][0], v[k][1], v[k][2], v[k][3]);
                    }
                    __syncwarp();
                    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sb + kManyCopiedAt + 8 * half)
                                 : "memory");
                }
            }
        } else if (w == 1 && cta == 0) {
            constexpr uint32_t idesc = idesc_e4m3_f32(256, 256, false, TRANS);
            auto commit = [&](uint32_t bar) {  // to the barrier's place in both CTAs
                asm volatile(
                    "{\n\t.reg .pred e;\n\t"
                    "elect.sync _|e, 0xffffffff;\n\t"
                    "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
                    " [%0], %1;\n\t}" ::"r"(bar),
                    "h"(static_cast<uint16_t>(3))
                    : "memory");
            };
            int st = 0;
            uint32_t phase = 0, used = 0;  // used: bit b: parity of the uses of accumulator b
            bool ok = true, seen = false;  // seen: the next block's operands
            for (int t = pair; ok && t < total; t += pairs)
                for (int u = 0; u < a.kb; ++u) {
                    const uint32_t b = u & 1, parity = (used >> b & 1) ^ 1;
                    const bool free = bar_test(sb + kManyFreeAt + 8 * b, parity);
                    if (!(ok = pair_wait(sb + kManyFullAt + 8 * st, phase, seen, sb, a.err) &&
                               pair_wait(sb + kManyFreeAt + 8 * b, parity, free, sb, a.err)))
                        break;
                    used ^= 1u << b;
                    tc_fence_after();
                    const uint64_t ad = smem_desc_sw128(sb + st * kManyStage);
                    const uint64_t bd = smem_desc_sw128(sb + st * kManyStage + kFp8Tile);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        tc_mma_f8_pair_elect(tmem + b * 256, ad + i * kStep32<false>, bd + i * kStep32<TRANS>, idesc,
                                             i ? 1u : 0u);
                    commit(sb + kManyDoneAt + 8 * b);
                    commit(sb + kManyEmptyAt + 8 * st);
                    if (++st == kManyStages) st = 0, phase ^= 1;
                    seen = bar_test(sb + kManyFullAt + 8 * st, phase);
                }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyManyRegs));
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const uint32_t mine = sb + kManyScalesAt + (threadIdx.x - 128) * 16;
        const uint32_t at = tmem + (static_cast<uint32_t>(32 * (w & 3)) << 16) + ((w - 4) >> 2) * 128;
        const uint32_t free_at = cluster_address(sb + kManyFreeAt, 0);
        uint32_t used = 0;
        bool ok = true, seen = false;  // seen: the next block's sums are there
        // where the scales of the thread's row (rows behind the tile's compute something
        // that nobody stores) and of the warp's columns begin
        auto scales_of = [&](int t, int turn, const float*& xs, const float*& ws) {
            const ManyTile z = many_tile(a, t, turn, sb);
            xs = a.xs + min(static_cast<int64_t>(z.m0) + static_cast<int>(cta) * 128 + (w & 3) * 32 + lane, a.M - 1) * a.lds;
            ws = a.ws + z.t0 + min(z.col + ((w - 4) >> 2), a.nb - 1) * a.out_step;
        };
        // the row's scales of blocks u to u + 3 on their way to shared memory
        auto fetch = [&](const float* xs, int u) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 16;\ncp.async.commit_group;" ::"r"(mine + (u & 4) * 1024),
                         "l"(xs + u)
                         : "memory");
        };
        float held = 0.0f;  // the weight scales of 32 blocks, one a lane
        // a tile's first scales, asked for before the last tile's results are written
        auto fetch_first = [&](int t, int turn) {
            if (t >= total) return;
            const float *xs, *ws;
            scales_of(t, turn, xs, ws);
            fetch(xs, 0);
            held = ws[min(lane, a.kb - 1) * a.sum_step];
        };
        fetch_first(pair, 0);
#pragma unroll 1
        for (int t = pair, turn = 0; ok && t < total; t += pairs, ++turn) {
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
            {
                const float *xs, *ws;
                scales_of(t, turn, xs, ws);
                // block u in accumulator b
                auto block = [&](int u, uint32_t b) {
                    ok &= pair_wait(sb + kManyDoneAt + 8 * b, used >> b & 1, seen, sb, a.err);
                    used ^= 1u << b;
                    tc_fence_after();
                    uint32_t d[2][16];  // 16 columns on their way while the last 16 are added
                    tc_ld_32x32b_x16(at + b * 256, d[0]);
                    float f;
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(mine + (u & 4) * 1024 + (u & 3) * 4) : "memory");
                    f *= __shfl_sync(~0u, held, u & 31);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        tc_wait_ld();
                        if (c < 7) {
                            tc_ld_32x32b_x16(at + b * 256 + (c + 1) * 16, d[(c + 1) & 1]);
                        } else {
                            tc_fence_before();
                            __syncwarp();
                            arrive_first_lane(free_at + b * 8);
                            seen = bar_test(sb + kManyDoneAt + 8 * (b ^ 1), used >> (b ^ 1) & 1);
                        }
                        add_columns(acc + c * 16, f, d[c & 1]);
                    }
                };
                int u = 0;
                auto next_four = [&]() {
                    if (u && (u & 31) == 0) held = ws[min(u + lane, a.kb - 1) * a.sum_step];
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    if (u + 4 < a.kb) fetch(xs, u + 4);
                };
                // four blocks a round, so that few branches are left between their sums
#pragma unroll 1
                for (; u + 4 <= a.kb; u += 4) {
                    next_four();
                    block(u, 0);
                    block(u + 1, 1);
                    block(u + 2, 0);
                    block(u + 3, 1);
                }
                if (u < a.kb) {
                    next_four();
#pragma unroll 1
                    for (; u < a.kb; ++u) block(u, u & 1);
                }
                if (a.kb & 1) seen = false;  // the next tile begins with accumulator 0 again
            }
            fetch_first(t + pairs, turn + 1);
            const ManyTile z = many_tile(a, t, turn, sb);  // (kept from before, it would cost the sums registers)
            const int r = static_cast<int>(cta) * 128 + (w & 3) * 32 + lane;
            const int64_t n = (z.col + ((w - 4) >> 2)) * 128ll, left = min(static_cast<int64_t>(128), a.N - n);
            if (!ok || left <= 0) continue;
            constexpr int ES = BF16 ? 2 : 4, PER = 256 / ES;  // columns of a piece
            uint8_t* to = static_cast<uint8_t*>(a.out) + ((z.m0 + r) * a.ldo + n) * ES;
            auto column = [&](int i) { return a.relu ? relu_of(acc[i]) : acc[i]; };
            if (!(a.ovec16 && left * ES % 16 == 0)) {
                if (r < z.rows)
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (i < left) {
                            if constexpr (BF16)
                                reinterpret_cast<__nv_bfloat16*>(to)[i] = __float2bfloat16_rn(column(i));
                            else
                                reinterpret_cast<float*>(to)[i] = column(i);
                        }
                continue;
            }
            // 256 bytes of a row at a time, left in shared memory for the warp that copies
            const uint32_t piece = sb + kManyOutAt + ((w - 4) * 32 + lane) * kManyPitch;
#pragma unroll
            for (int c = 0; c < 128; c += PER) {
                ok &= pair_wait(sb + kManyCopiedAt + 8 * ((w - 4) >> 2), (used >> 2 & 1) ^ 1, false, sb, a.err);
                used ^= 4;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    uint32_t v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if constexpr (BF16)
                            v[k] = bf16x2_of(column(8 * i + 2 * k), column(8 * i + 2 * k + 1));
                        else
                            v[k] = __float_as_uint(column(c + 4 * i + k));
                    }
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(piece + 16 * i), "r"(v[0]), "r"(v[1]),
                                 "r"(v[2]), "r"(v[3])
                                 : "memory");
                }
                __syncwarp();
                arrive_first_lane(cluster_address(sb + kManyStagedAt + 8 * ((w - 4) >> 2), cta));
                if (c + PER >= left) break;
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }

    // the pair's MMAs, commits and remote arrivals are done
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    if (w == 1) tmem_dealloc_pair(tmem, 512);
}

// Rows of out outside every group.
__global__ void __launch_bounds__(256)
    zero_rest_kernel(const int32_t* __restrict__ group_rows, int G, int64_t M, int64_t N, int64_t ldo, int bf16, void* out) {
    const int64_t first = min(max(static_cast<int64_t>(group_rows[0]), int64_t{0}), M);
    const int64_t last = min(max(static_cast<int64_t>(group_rows[G]), int64_t{0}), M);
    for (int64_t r = blockIdx.x; r < first + M - last; r += gridDim.x) {
        const int64_t m = r < first ? r : last + r - first;
        for (int64_t n = threadIdx.x; n < N; n += blockDim.x) {
            if (bf16)
                static_cast<__nv_bfloat16*>(out)[m * ldo + n] = __float2bfloat16_rn(0.0f);
            else
                static_cast<float*>(out)[m * ldo + n] = 0.0f;
        }
    }
}

constexpr int kSMs = 148;

// What a product takes, in units of 10 ns, from its CTAs (pairs), the blocks of the
// sum and the rows of a tile.  Neither counts the bytes of out: they were measured with
// sums of 16 blocks and more or few rows; with a sum of one or two blocks and many
// columns the stores decide, and which kernel is the faster one there was not measured.
//
// Few rows: CTAs (at most 8, one cluster) split the sum.  Row tiles of 16 and 32
// share an SM by twos while there are more CTAs than SMs, the wider ones have one to
// themselves.  One row, 4096 x 4096 (32 tiles): 1, 2, 4, 8 CTAs a tile 12.8, 9.4, 7.3,
// 8.1 us; 14336 x 4096: 38.8, 22.1, 14.8, 13.9; 4096 x 14336 (112 tiles): 14.3, 13.9,
// 17.5, 24.2.  128 rows, 4096 x 4096: 21.1, 16.7, 13.8, 32.1.
int64_t few_cost(int64_t ctas, int64_t blocks, int rows, int* split) {
    int64_t least = INT64_MAX;
    for (int S = 1; S <= 8 && (S == 1 || blocks >= 2 * S); ++S) {
        const int64_t each = (blocks + S - 1) / S, n = ctas * S;
        int64_t cost;
        if (rows <= 32)
            cost = n <= kSMs ? 530 + 30 * each : (n + 2 * kSMs - 1) / (2 * kSMs) * (720 + 45 * each);
        else
            cost = (n + kSMs - 1) / kSMs * (700 + (S > 1 ? 200 : 0) + (rows <= 64 ? 34 : 55) * each);
        if (cost < least) {
            least = cost;
            *split = S;
        }
    }
    return least;
}
// Many rows: persistent pairs.  4096 x 14336 (56 tiles), 64, 128, 256 and 384 rows:
// 23.4, 23.4, 23.4 and 41.1 us, the kernel for few rows 20.6, 24.1, 45.8 and 65.7; 14336
// x 4096 (16 tiles) 55 to 56 us, the other 19.4, 25.4, 35.6 and 76.7.  64 experts of 2048
// x 1408 with 32, 64, 96, 128 and 256 rows each: 60, 62, 63, 64 and 67 us, the other 44,
// 67, 74, 79 and 141.
int64_t many_cost(int64_t tiles, int64_t blocks, int pairs) {
    return 600 + (tiles + pairs - 1) / pairs * (320 + 41 * blocks);
}

template <int TN, bool ALONE>
aem_status launch_few(Fp8Args a, const void* q, int64_t ldq, int64_t cols, bool transposed, bool dependent,
                      int64_t slots, cudaStream_t s) {
    using C = FewCfg<TN, ALONE>;
    CUtensorMap xmap{};
    AEM_TRY(make_tmap_2d_u8(&xmap, q, cols, a.M, ldq, TN, CU_TENSOR_MAP_SWIZZLE_128B));
    auto kern = transposed ? fp8_few_kernel<TN, ALONE, true> : fp8_few_kernel<TN, ALONE, false>;
    static std::atomic<uint64_t> ready[2];  // bit per device: the shared memory opt-in is done
    const uint64_t bit = 1ull << (current_device() & 63);
    if (!(ready[transposed].load(std::memory_order_relaxed) & bit)) {
        AEM_TRY_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        ready[transposed].fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.nb * a.S), static_cast<unsigned>(slots));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    int n = 0;
    if (dependent) {  // starts under the kernel that quantises the rows
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

// Pairs of SMs that can run the kernel at once (0: it cannot).
int max_pairs(int device) {
    static std::atomic<int> cache[64];
    const int known = cache[device & 63].load(std::memory_order_relaxed);
    if (known) return known - 1;
    int n = 0;
    for (auto kern : {fp8_many_kernel<false, false>, fp8_many_kernel<false, true>, fp8_many_kernel<true, false>,
                      fp8_many_kernel<true, true>}) {
        cudaFuncAttributes f;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(2 * 512);
        cfg.blockDim = dim3(kManyThreads);
        cfg.dynamicSmemBytes = kManySmem;
        // a launch with fewer registers could not share them out as the kernel does
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kManySmem) != cudaSuccess ||
            cudaFuncGetAttributes(&f, kern) != cudaSuccess ||
            f.numRegs * kManyThreads < kManyFewRegs * 128 + kManyManyRegs * 256 ||
            cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
            cudaGetLastError();
            n = 0;
            break;
        }
    }
    cache[device & 63].store(n + 1, std::memory_order_relaxed);
    return n;
}

aem_status launch_many(const Fp8Args& a, const Fp8Weight* w, const void* q, int64_t ldq, int64_t cols, bool transposed,
                       bool dependent, int64_t row_tiles, cudaStream_t s) {
    CUtensorMap xmap{}, wmap{};
    AEM_TRY(make_tmap_2d_u8(&xmap, q, cols, a.M, ldq, 128, CU_TENSOR_MAP_SWIZZLE_128B));
    AEM_TRY(make_tmap_2d_u8(&wmap, w->data, 128, w->G * w->NC * w->KC * 128, 128, 128, CU_TENSOR_MAP_SWIZZLE_NONE));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<int64_t>(max_pairs(w->device), row_tiles * ((a.nb + 1) / 2))));
    cfg.blockDim = dim3(kManyThreads);
    cfg.dynamicSmemBytes = kManySmem;
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;  // starts under the kernel that quantises the rows
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = dependent ? 1 : 0;
    auto kern = transposed ? (a.out_bf16 ? fp8_many_kernel<true, true> : fp8_many_kernel<true, false>)
                           : (a.out_bf16 ? fp8_many_kernel<false, true> : fp8_many_kernel<false, false>);
    AEM_TRY_CUDA(cudaLaunchKernelEx(&cfg, kern, xmap, wmap, a));
    count_launches(1);
    return AEM_OK;
}

// Quantised rows in a workspace: bytes, then scales.
struct Scratch {
    int64_t ldq, lds;
    size_t scale_at, bytes;
};
Scratch scratch_of(int64_t M, int64_t cols) {
    Scratch z;
    z.ldq = (cols + 15) / 16 * 16;
    z.lds = ((cols + 127) / 128 + 3) / 4 * 4;
    z.scale_at = align_up(static_cast<size_t>(M) * z.ldq, 16);
    z.bytes = z.scale_at + static_cast<size_t>(M) * z.lds * sizeof(float);
    return z;
}

struct Rows {  // the caller's x
    const void* x;
    aem_dtype dtype;
    int64_t ldx;
    const float* scale;
    int64_t lds;
};

aem_status fp8_product(const Fp8Weight* w, const char* what, Fp8Args a, Rows x, bool transposed, int zero_rest,
                       void* workspace, size_t workspace_bytes, cudaStream_t s) {
    AEM_REQUIRE(current_device() == w->device, "%s: the weights are on device %d, the current one is %d", what,
                w->device, current_device());
    const int64_t cols = transposed ? w->N : w->K;
    a.N = transposed ? w->K : w->N;
    AEM_REQUIRE(a.ldo >= a.N, "%s: bad row stride of out", what);
    a.w = w->data;
    a.ws = w->scale;
    a.group_tiles = w->NC * w->KC;
    a.out_step = transposed ? 1 : w->KC;
    a.sum_step = transposed ? w->KC : 1;
    a.nb = static_cast<int>(transposed ? w->KC : w->NC);
    a.kb = static_cast<int>(transposed ? w->NC : w->KC);
    a.ovec = reinterpret_cast<uintptr_t>(a.out) % (a.out_bf16 ? 8 : 16) == 0 && a.ldo % 4 == 0;
    a.ovec16 = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.ldo % (a.out_bf16 ? 8 : 4) == 0;
    a.err = device_error_word(w->device);
    if (!a.err) {
        set_error("%s: no device error word", what);
        return AEM_ENOMEM;
    }
    const int64_t n = std::min<int64_t>(a.G, a.M), want = (a.M + n - 1) / n;
    a.rows = want <= 16 ? 16 : want <= 32 ? 32 : want <= 64 ? 64 : 128;
    // (the groups' sizes are not known here: all as large as the average.  Where a few
    // groups have most rows their weights pass once for each tile of the average's size)
    const int64_t cost = few_cost(n * ((want + a.rows - 1) / a.rows) * a.nb, a.kb, a.rows, &a.S);
    const int pairs = want > 32 ? max_pairs(w->device) : 0;
    const bool many = pairs > 0 && (a.M > 65535ll * 64 ||  // (more row tiles than a grid of the other kernel has)
                                    many_cost(n * ((want + kManyTile - 1) / kManyTile) * ((a.nb + 1) / 2), a.kb, pairs) < cost);
    if (many) a.rows = kManyTile;
    // row tiles at most: n groups with rows have up to n + (M - n) / rows
    const int64_t slots = a.group_rows ? n + (a.M - n) / a.rows : (a.M + a.rows - 1) / a.rows;
    AEM_REQUIRE((many || slots <= 65535) && slots * ((a.nb + 1) / 2) < (1ll << 31),
                "%s: M=%lld rows are too many for one call", what, (long long)a.M);
    void* own = nullptr;
    const bool make = x.dtype != AEM_E4M3;
    if (make) {
        const Scratch z = scratch_of(a.M, cols);
        AEM_REQUIRE(!workspace || (workspace_bytes >= z.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                    "%s: workspace of %zu bytes (%zu needed, 16-byte aligned)", what, workspace_bytes, z.bytes);
        if (!workspace) {
            AEM_TRY_CUDA(cudaMallocAsync(&own, z.bytes, s));
            workspace = own;
        }
        auto* q = static_cast<uint8_t*>(workspace);
        auto* sc = reinterpret_cast<float*>(q + z.scale_at);
        const aem_status st = launch_quantize_fp8(what, x.x, x.dtype, x.ldx, a.M, cols, q, z.ldq, sc, z.lds, s);
        if (st != AEM_OK) {
            if (own) cudaFreeAsync(own, s);
            return st;
        }
        x = {q, AEM_E4M3, z.ldq, sc, z.lds};
    }
    a.xs = x.scale;
    a.lds = x.lds;
    aem_status st = many             ? launch_many(a, w, x.x, x.ldx, cols, transposed, make, slots, s)
                    : a.rows == 16   ? launch_few<16, false>(a, x.x, x.ldx, cols, transposed, make, slots, s)
                    : a.rows == 32   ? launch_few<32, false>(a, x.x, x.ldx, cols, transposed, make, slots, s)
                    : a.rows == 64   ? launch_few<64, true>(a, x.x, x.ldx, cols, transposed, make, slots, s)
                                     : launch_few<128, true>(a, x.x, x.ldx, cols, transposed, make, slots, s);
    if (own) cudaFreeAsync(own, s);
    AEM_TRY(st);
    if (zero_rest) {
        const auto grid = static_cast<unsigned>(std::min<int64_t>(a.M, kSMs * 8));
        zero_rest_kernel<<<grid, 256, 0, s>>>(a.group_rows, a.G, a.M, a.N, a.ldo, a.out_bf16, a.out);
        AEM_CHECK_LAUNCH();
        count_launches(1);
    }
    return AEM_OK;
}

// Rows are indexed in 32 bits, a tile past the last one included.
aem_status check_most_rows(const char* what, int64_t M) {
    AEM_REQUIRE(M >= 0, "%s: M must be >= 0", what);
    AEM_REQUIRE(M < (1ll << 31) - kManyTile, "%s: M=%lld rows are too many for one call", what, (long long)M);
    return AEM_OK;
}

aem_status check_rows(const char* what, const Rows& x, int64_t cols, int64_t M) {
    AEM_REQUIRE(x.dtype == AEM_F32 || x.dtype == AEM_BF16 || x.dtype == AEM_E4M3, "%s: bad dtype", what);
    AEM_REQUIRE(x.ldx >= 0 && x.lds >= 0, "%s: bad row stride", what);
    if (x.dtype == AEM_E4M3) {
        AEM_REQUIRE(x.ldx >= cols && x.ldx % 16 == 0 && x.lds >= (cols + 127) / 128 && x.lds % 4 == 0,
                    "%s: bad row stride of e4m3 rows or their scales", what);
        AEM_REQUIRE(M == 0 || x.scale, "%s: e4m3 rows without scales", what);
        AEM_REQUIRE(reinterpret_cast<uintptr_t>(x.x) % 16 == 0 && reinterpret_cast<uintptr_t>(x.scale) % 16 == 0,
                    "%s: e4m3 rows and their scales must be 16-byte aligned", what);
    } else {
        AEM_REQUIRE(!x.scale, "%s: scales are for e4m3 rows", what);
    }
    return AEM_OK;
}

}  // namespace
}  // namespace aem

using aem::set_error;

extern "C" {

size_t aem_fp8gemm_workspace(aem_fp8weight_t wh, aem_dtype x_dtype, int64_t M, int transposed) {
    if (!wh || M < 1 || (x_dtype != AEM_F32 && x_dtype != AEM_BF16)) return 0;
    auto* w = reinterpret_cast<aem::Fp8Weight*>(wh);
    return aem::scratch_of(M, transposed ? w->N : w->K).bytes;
}

aem_status aem_fp8gemm(aem_fp8weight_t wh, int64_t group, int transposed, const void* x, aem_dtype x_dtype,
                       int64_t ldx, const float* x_scale, int64_t lds, int64_t M, void* out, aem_dtype out_dtype,
                       int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    AEM_REQUIRE(wh != nullptr, "aem_fp8gemm: weight handle is NULL");
    AEM_TRY(aem::check_most_rows("aem_fp8gemm", M));
    auto* w = reinterpret_cast<aem::Fp8Weight*>(wh);
    AEM_REQUIRE(group >= 0 && group < w->G, "aem_fp8gemm: group %lld out of range [0, %lld)", (long long)group,
                (long long)w->G);
    AEM_REQUIRE(out_dtype == AEM_F32 || out_dtype == AEM_BF16, "aem_fp8gemm: bad dtype");
    const aem::Rows rows{x, x_dtype, ldx, x_scale, lds};
    AEM_TRY(aem::check_rows("aem_fp8gemm", rows, transposed ? w->N : w->K, M));
    if (M == 0) return AEM_OK;
    AEM_REQUIRE(x && out, "aem_fp8gemm: NULL buffer");
    aem::Fp8Args a{};
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group = group;
    a.G = 1;
    a.out_bf16 = out_dtype == AEM_BF16;
    return aem::fp8_product(w, "aem_fp8gemm", a, rows, transposed != 0, 0, workspace, workspace_bytes,
                            static_cast<cudaStream_t>(stream));
}

aem_status aem_grouped_fp8gemm(aem_fp8weight_t wh, const int32_t* group_rows, int transposed, const void* x,
                               aem_dtype x_dtype, int64_t ldx, const float* x_scale, int64_t lds, int64_t M, void* out,
                               aem_dtype out_dtype, int64_t ldo, int relu, int zero_rest, void* workspace,
                               size_t workspace_bytes, void* stream) {
    AEM_REQUIRE(wh != nullptr, "aem_grouped_fp8gemm: weight handle is NULL");
    AEM_TRY(aem::check_most_rows("aem_grouped_fp8gemm", M));
    auto* w = reinterpret_cast<aem::Fp8Weight*>(wh);
    AEM_REQUIRE(w->G <= AEM_MAX_EXPERTS, "aem_grouped_fp8gemm: %lld weight groups, at most %d", (long long)w->G,
                AEM_MAX_EXPERTS);
    AEM_REQUIRE(out_dtype == AEM_F32 || out_dtype == AEM_BF16, "aem_grouped_fp8gemm: bad dtype");
    const aem::Rows rows{x, x_dtype, ldx, x_scale, lds};
    AEM_TRY(aem::check_rows("aem_grouped_fp8gemm", rows, transposed ? w->N : w->K, M));
    if (M == 0) return AEM_OK;
    AEM_REQUIRE(group_rows && x && out, "aem_grouped_fp8gemm: NULL buffer");
    aem::Fp8Args a{};
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group_rows = group_rows;
    a.G = static_cast<int>(w->G);
    a.out_bf16 = out_dtype == AEM_BF16;
    a.relu = relu != 0;
    return aem::fp8_product(w, "aem_grouped_fp8gemm", a, rows, transposed != 0, zero_rest, workspace, workspace_bytes,
                            static_cast<cudaStream_t>(stream));
}

}  // extern "C"
