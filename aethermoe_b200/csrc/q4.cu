// 4-bit weights with group scales: quantisation, packing, and the products of
// a few activation rows with them (decode), dense and grouped by expert.
//
// Weight (k, n) of group g of G is q[g][k][n] * scale[g][k / gs][n] with q an
// integer in [-8, 7] and gs = 32, 64 or 128 consecutive k sharing a scale:
//   out[m, n] = sum_b scale[b, n] * sum_{k in block b} q[k, n] x[m, k]
// A 4-bit integer is exact in bf16, so each inner sum runs on warp MMAs
// (bf16 operands, float32 accumulators) and the scale multiplies its float32
// result: no rounded weight ever exists.  bf16 x enters as it is; float32 x
// enters as three bf16 terms that add up to it exactly (8 + 8 + 8 mantissa
// bits), in three MMA columns whose sums are added at the end.
//
// What bounds it is the weight stream, K*N/2 bytes plus the scales, so the
// layout serves that stream: a tile of 16 channels x 64 k is 512 contiguous
// bytes, 16 per lane, and those 16 bytes are the lane's own A fragments of
// four m16n8k16 MMAs -- one 16-byte load, no shared memory, no shuffles.
#include <cuda_bf16.h>

#include <algorithm>
#include <new>

#include "common.cuh"
#include "runtime.h"

namespace aem {

// Packed 4-bit weight (device).  q: [G][NT][KT][32][16 B] with NT = channels
// in tiles of 16 (an even number), KT = ceil(K/64).  In a tile lane
// l = 4*c + t holds the weights of channels c and c+8 at
// k = 32h + 8t + 4(i & 1) + {0..3} for its words i = 0..3, h = i >> 1: nibble
// pair r of a word (bits 4r and 16 + 4r) is A register r of MMA i, i.e. the
// k offsets {0,1} (r < 2) or {2,3} of channel c + 8*(r & 1).  The nibble is
// q + 8; padding holds 8.  scale: [G][KB][NT][8][2], channel c of a tile
// beside channel c + 8, in the caller's type, padding zero.
struct Q4Weight {
    int device = 0;
    int64_t G = 0, K = 0, N = 0, NT = 0, KT = 0, KB = 0;
    int gs = 0;
    bool scale_bf16 = false;
    uint4* q = nullptr;
    void* scale = nullptr;
};

namespace {

constexpr int kThreads = 256, kWarps = 8;

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
    pack_q4_kernel(const int8_t* __restrict__ q, int64_t K, int64_t N, int64_t NT, int64_t KT,
                   int64_t tiles, uint4* __restrict__ out, int* err) {
    const int lane = threadIdx.x & 31, c = lane >> 2, t = lane & 3;
    bool bad = false;
    for (int64_t tile = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5); tile < tiles;
         tile += static_cast<int64_t>(gridDim.x) * kWarps) {
        const int64_t kt = tile % KT, nt = tile / KT % NT, g = tile / KT / NT;
        uint32_t word[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            word[i] = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    const int64_t k = kt * 64 + 32 * (i >> 1) + 8 * t + 4 * (i & 1) + 2 * (r >> 1) + hi;
                    const int64_t n = nt * 16 + c + 8 * (r & 1);
                    int v = k < K && n < N ? q[(g * K + k) * N + n] : 0;
                    if (v < -8 || v > 7) {
                        bad = true;
                        v = v < 0 ? -8 : 7;
                    }
                    word[i] |= static_cast<uint32_t>(v + 8) << (4 * r + 16 * hi);
                }
        }
        out[tile * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
    }
    if (bad) atomicOr(err, ERR_Q4_VALUE);
}

template <typename ST>
__global__ void __launch_bounds__(kThreads)
    pack_q4_scale_kernel(const ST* __restrict__ s, int64_t GB, int64_t N, int64_t NT,
                         ST* __restrict__ out) {
    const int64_t total = GB * NT * 16;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t b = i / (NT * 16), r = i % (NT * 16);
        const int64_t n = r / 16 * 16 + (r & 1) * 8 + (r % 16) / 2;
        out[i] = n < N ? s[b * N + n] : ST(0.0f);
    }
}

// ------------------------------------------------------------------ product
struct Q4Args {
    const uint4* q;
    const void* scale;
    const void* x;
    void* out;
    const int32_t* group_rows;  // nullptr: one group of M rows, weight group `group`
    int64_t ldx, ldo, M, K, N, NT, KT, KB;
    int64_t group;
    int G, gs, S, rows;  // S: CTAs (one cluster) that split K; rows: rows of a row tile
    bool scale_bf16, out_bf16, relu;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight 4-bit weights -> four bf16 pairs.  0x4300 is bf16 128, whose last
// mantissa bit is 1: 0x4300 | nibble = 128 + nibble, and subtracting 136
// leaves q exactly.
__device__ __forceinline__ void unpack_q4(uint32_t w, uint32_t (&a)[4]) {
    const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t v = ((w >> (4 * r)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
        a[r] = *reinterpret_cast<const uint32_t*>(&d);
    }
}

// Upper halves of two float32 bit patterns as a bf16 pair.
__device__ __forceinline__ uint32_t pack_hi(float a, float b) {
    return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}

// Term `m1, m2` of a float32: masks 0, 0 give v (its upper half is the first
// term), ~0, 0 what the first term leaves, ~0, ~0 what the first two leave
// (truncated terms: the differences are exact).  An infinity is all in the
// first term.
__device__ __forceinline__ float f32_term(float v, uint32_t m1, uint32_t m2) {
    float r = v - __uint_as_float(__float_as_uint(v) & m1);
    r = r - __uint_as_float(__float_as_uint(r) & m2);
    return r == r || m1 == 0 ? r : 0.0f;
}

// The lane's B fragments of one 64-k tile and one 8-column tile: b[i] of MMA
// i.  p: the column's activation row (nullptr: column unused, zeros).
template <bool F32, bool FAST>
__device__ __forceinline__ void load_x(const void* p, int64_t k0, int64_t K, uint32_t m1,
                                       uint32_t m2, uint32_t (&b)[4][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t k = k0 + 32 * h;
        uint32_t u[4] = {0, 0, 0, 0};
        if constexpr (FAST) {  // 16-byte rows, K a multiple of 8
            if (p && k < K) {
                if constexpr (F32) {
                    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + k);
                    const float4 lo = __ldg(f), hi = __ldg(f + 1);
                    u[0] = pack_hi(f32_term(lo.x, m1, m2), f32_term(lo.y, m1, m2));
                    u[1] = pack_hi(f32_term(lo.z, m1, m2), f32_term(lo.w, m1, m2));
                    u[2] = pack_hi(f32_term(hi.x, m1, m2), f32_term(hi.y, m1, m2));
                    u[3] = pack_hi(f32_term(hi.z, m1, m2), f32_term(hi.w, m1, m2));
                } else {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + k));
                    u[0] = v.x, u[1] = v.y, u[2] = v.z, u[3] = v.w;
                }
            }
        } else if (p) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float e[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int64_t kk = k + 2 * i + j;
                    if constexpr (F32)
                        e[j] = kk < K ? f32_term(static_cast<const float*>(p)[kk], m1, m2) : 0.0f;
                    else
                        e[j] = kk < K ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[kk]) : 0.0f;
                }
                u[i] = pack_hi(e[0], e[1]);
            }
        }
        b[2 * h][0] = u[0], b[2 * h][1] = u[1], b[2 * h + 1][0] = u[2], b[2 * h + 1][1] = u[3];
    }
}

// Row tile `slot` of the groups' row tiles: its group, first row and rows.
// Every warp searches alike.  Offsets are clamped to [0, M].
__device__ __forceinline__ bool find_rows(const Q4Args& a, int64_t slot, int64_t* g, int64_t* m0,
                                          int* rows) {
    if (!a.group_rows) {
        *g = a.group;
        *m0 = slot * a.rows;
        *rows = static_cast<int>(min(static_cast<int64_t>(a.rows), a.M - *m0));
        return *rows > 0;
    }
    const int lane = threadIdx.x & 31;
    int64_t before = 0;
    for (int e0 = 0; e0 < a.G; e0 += 32) {
        const int e = e0 + lane;
        const int64_t lo = e < a.G ? min(max(static_cast<int64_t>(a.group_rows[e]), 0l), a.M) : 0;
        const int64_t hi = e < a.G ? min(max(static_cast<int64_t>(a.group_rows[e + 1]), 0l), a.M) : 0;
        const int n = hi > lo ? static_cast<int>((hi - lo + a.rows - 1) / a.rows) : 0;
        int s = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, s, o);
            if (lane >= o) s += v;
        }
        const int64_t first = before + s - n;
        const unsigned hit = __ballot_sync(~0u, slot >= first && slot < first + n);
        if (hit) {
            const int l = __ffs(hit) - 1;
            const int64_t m = lo + (slot - first) * a.rows;
            const int r = static_cast<int>(min(static_cast<int64_t>(a.rows), hi - m));
            *g = e0 + l;
            *m0 = __shfl_sync(~0u, m, l);
            *rows = __shfl_sync(~0u, r, l);
            return true;
        }
        before += __shfl_sync(~0u, s, 31);
    }
    return false;
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
    uint32_t at;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(dev::smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// A CTA computes 32 channels of one row tile; its 8 warps (and the S CTAs of
// its cluster) split K and their float32 sums are added in a fixed order.
// NT: 8-column tiles; G32: scale groups of 32 (two per 64-k tile).
template <int NT, bool F32, bool FAST, bool G32>
__global__ void __launch_bounds__(kThreads) q4_kernel(const Q4Args a) {
    constexpr int PF = 4;  // weight tiles in flight
    constexpr int NS = G32 ? 2 : 1;
    __shared__ float red[kWarps][NT * 4 * 32];
    __shared__ float fin[32][NT * 8 + 1];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t tile = blockIdx.x / a.S;
    const int ks = blockIdx.x % a.S;
    int64_t g, m0;
    int rows;
    if (!find_rows(a, blockIdx.y, &g, &m0, &rows)) return;

    // columns of this lane: B column 8*nt + lane/4
    const void* xp[NT];
    uint32_t m1[NT], m2[NT];
    const int t8 = 8 * (lane & 3);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int col = 8 * nt + (lane >> 2);
        const int r = F32 ? col / 3 : col, term = F32 ? col % 3 : 0;
        m1[nt] = term > 0 ? 0xffff0000u : 0u;
        m2[nt] = term > 1 ? 0xffff0000u : 0u;
        xp[nt] = nullptr;
        if (r < rows) {
            const int64_t off = (m0 + r) * a.ldx;
            xp[nt] = F32 ? static_cast<const void*>(static_cast<const float*>(a.x) + off)
                         : static_cast<const void*>(static_cast<const __nv_bfloat16*>(a.x) + off);
        }
    }

    // this warp's 64-k tiles, whole scale groups
    const int gran = a.gs > 64 ? a.gs / 64 : 1;
    const int64_t units = (a.KT + gran - 1) / gran;
    const int64_t part = ks * kWarps + w, parts = a.S * kWarps;
    const int kt0 = static_cast<int>(units * part / parts * gran);
    const int kt1 = static_cast<int>(min(units * (part + 1) / parts * gran, a.KT));

    const uint4* wq = a.q + ((g * a.NT + tile * 2) * a.KT) * 32 + lane;
    const int64_t wstep = a.KT * 32;  // to the second 16 channels
    const char* sp = static_cast<const char*>(a.scale);
    const int64_t sbase = ((g * a.KB) * a.NT + tile * 2) * 16 + (lane >> 2) * 2;

    uint4 wr[PF][2];
    uint2 sr[PF][2][NS];
    auto fetch = [&](int slot, int kt) {
        if (kt >= kt1) return;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            wr[slot][c] = __ldg(wq + static_cast<int64_t>(kt) * 32 + c * wstep);
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int64_t b = G32 ? min(static_cast<int64_t>(2 * kt + j), a.KB - 1) : static_cast<int64_t>(kt) * 64 / a.gs;
                const int64_t at = sbase + b * a.NT * 16 + c * 16;
                if (a.scale_bf16)
                    sr[slot][c][j].x = __ldg(reinterpret_cast<const uint32_t*>(sp + at * 2));
                else
                    sr[slot][c][j] = __ldg(reinterpret_cast<const uint2*>(sp + at * 4));
            }
        }
    };
    float acc[2][NT][4] = {}, sum[2][NT][4] = {};
    auto apply = [&](int slot, int j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint2 u = sr[slot][c][j];
            const float s0 = __uint_as_float(a.scale_bf16 ? u.x << 16 : u.x);
            const float s1 = __uint_as_float(a.scale_bf16 ? u.x & 0xffff0000u : u.y);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[c][nt][i] = fmaf(i < 2 ? s0 : s1, sum[c][nt][i], acc[c][nt][i]);
                    sum[c][nt][i] = 0.0f;
                }
        }
    };
#pragma unroll
    for (int i = 0; i < PF; ++i) fetch(i, kt0 + i);
    for (int kb = kt0; kb < kt1; kb += PF) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int kt = kb + i;
            if (kt >= kt1) break;
            uint32_t wa[2][4][4];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                unpack_q4(wr[i][c].x, wa[c][0]);
                unpack_q4(wr[i][c].y, wa[c][1]);
                unpack_q4(wr[i][c].z, wa[c][2]);
                unpack_q4(wr[i][c].w, wa[c][3]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                uint32_t b[4][2];
                load_x<F32, FAST>(xp[nt], static_cast<int64_t>(kt) * 64 + t8, a.K, m1[nt], m2[nt], b);
                if constexpr (G32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float p[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_bf16(p, wa[c][2 * h], b[2 * h][0], b[2 * h][1]);
                            mma_bf16(p, wa[c][2 * h + 1], b[2 * h + 1][0], b[2 * h + 1][1]);
                            const uint2 u = sr[i][c][h < NS ? h : 0];
                            const float s0 = __uint_as_float(a.scale_bf16 ? u.x << 16 : u.x);
                            const float s1 = __uint_as_float(a.scale_bf16 ? u.x & 0xffff0000u : u.y);
                            acc[c][nt][0] = fmaf(s0, p[0], acc[c][nt][0]);
                            acc[c][nt][1] = fmaf(s0, p[1], acc[c][nt][1]);
                            acc[c][nt][2] = fmaf(s1, p[2], acc[c][nt][2]);
                            acc[c][nt][3] = fmaf(s1, p[3], acc[c][nt][3]);
                        }
                } else {
#pragma unroll
                    for (int m = 0; m < 4; ++m)
#pragma unroll
                        for (int c = 0; c < 2; ++c) mma_bf16(sum[c][nt], wa[c][m], b[m][0], b[m][1]);
                }
            }
            if constexpr (!G32)
                if ((kt + 1) % gran == 0 || kt + 1 == kt1) apply(i, 0);
            fetch(i, kt + PF);
        }
    }

    // the warps' sums, in warp order, into fin[channel][column]
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        if (c) __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[w][(nt * 4 + i) * 32 + lane] = acc[c][nt][i];
        __syncthreads();
        for (int i = threadIdx.x; i < NT * 4 * 32; i += kThreads) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < kWarps; ++j) s += red[j][i];
            const int l = i & 31, e = (i >> 5) & 3, nt = i >> 7;
            fin[c * 16 + (l >> 2) + 8 * (e >> 1)][nt * 8 + 2 * (l & 3) + (e & 1)] = s;
        }
    }
    __syncthreads();
    if (a.S > 1) cluster_barrier();
    if (ks == 0) {
        for (int i = threadIdx.x; i < rows * 32; i += kThreads) {
            const int r = i >> 5, ch = i & 31;
            const int64_t n = tile * 32 + ch;
            float v = 0.0f;
            for (int s = 0; s < a.S; ++s)
#pragma unroll
                for (int j = 0; j < (F32 ? 3 : 1); ++j) {
                    const float* p = &fin[ch][F32 ? 3 * r + j : r];
                    v += s == 0 ? *p : ld_cluster(p, s);
                }
            if (n >= a.N) continue;
            if (a.relu && v < 0.0f) v = 0.0f;
            if (a.out_bf16)
                static_cast<__nv_bfloat16*>(a.out)[(m0 + r) * a.ldo + n] = __float2bfloat16_rn(v);
            else
                static_cast<float*>(a.out)[(m0 + r) * a.ldo + n] = v;
        }
    }
    if (a.S > 1) cluster_barrier();  // the others' fin stays until rank 0 has read it
}

template <int NT, bool F32>
aem_status launch_nt(const Q4Args& a, bool fast, dim3 grid, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = a.S;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = a.S > 1 ? 1 : 0;
    if (a.gs == 32)
        AEM_TRY_CUDA(fast ? cudaLaunchKernelEx(&cfg, q4_kernel<NT, F32, true, true>, a)
                          : cudaLaunchKernelEx(&cfg, q4_kernel<NT, F32, false, true>, a));
    else
        AEM_TRY_CUDA(fast ? cudaLaunchKernelEx(&cfg, q4_kernel<NT, F32, true, false>, a)
                          : cudaLaunchKernelEx(&cfg, q4_kernel<NT, F32, false, false>, a));
    count_launches(1);
    return AEM_OK;
}

template <bool F32>
aem_status launch_q4(Q4Args a, bool fast, int64_t want_rows, cudaStream_t s) {
    // columns of a row tile: as many as the rows need, up to 64
    constexpr int per = F32 ? 3 : 1;
    int nt = 8;
    for (int n : {1, 2, 4})
        if (want_rows * per <= 8 * n) {
            nt = n;
            break;
        }
    a.rows = 8 * nt / per;
    const int64_t slots = a.group_rows
                              ? std::min<int64_t>(a.G, a.M) + a.M / a.rows
                              : (a.M + a.rows - 1) / a.rows;
    AEM_REQUIRE(slots <= 65535, "q4 product: M=%lld rows are too many for one call", (long long)a.M);
    const int64_t tiles = a.NT / 2, ctas = tiles * slots;
    a.S = 1;
    while (a.S < 8 && ctas * a.S < 148 * 2 && a.KT >= 2 * kWarps * a.S) a.S *= 2;
    AEM_REQUIRE(tiles * a.S < (1ll << 31), "q4 product: N=%lld out of range", (long long)a.N);
    const dim3 grid(static_cast<unsigned>(tiles * a.S), static_cast<unsigned>(slots));
    switch (nt) {
        case 1: return launch_nt<1, F32>(a, fast, grid, s);
        case 2: return launch_nt<2, F32>(a, fast, grid, s);
        case 4: return launch_nt<4, F32>(a, fast, grid, s);
        default: return launch_nt<8, F32>(a, fast, grid, s);
    }
}

aem_status q4_product(const Q4Weight* w, const char* what, Q4Args a, aem_dtype xd, cudaStream_t s) {
    AEM_REQUIRE(current_device() == w->device, "%s: the weights are on device %d, the current one is %d",
                what, w->device, current_device());
    a.q = w->q;
    a.scale = w->scale;
    a.K = w->K;
    a.N = w->N;
    a.NT = w->NT;
    a.KT = w->KT;
    a.KB = w->KB;
    a.gs = w->gs;
    a.scale_bf16 = w->scale_bf16;
    const int es = xd == AEM_F32 ? 4 : 2;
    const bool fast = a.K % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (a.ldx * es) % 16 == 0;
    // grouped: the rows that a group has on average
    const int64_t want = a.group_rows ? (a.M + std::min<int64_t>(a.G, a.M) - 1) / std::min<int64_t>(a.G, a.M) : a.M;
    return xd == AEM_F32 ? launch_q4<true>(a, fast, want, s) : launch_q4<false>(a, fast, want, s);
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
    cudaFree(w->q);
    cudaFree(w->scale);
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
    w->NT = (N + 31) / 32 * 2;
    w->KT = (K + 63) / 64;
    w->KB = (K + group_size - 1) / group_size;
    w->gs = group_size;
    w->scale_bf16 = scale_dtype == AEM_BF16;
    const int64_t tiles = G * w->NT * w->KT, scales = G * w->KB * w->NT * 16;
    if (cudaMalloc(&w->q, static_cast<size_t>(tiles) * 512) != cudaSuccess ||
        cudaMalloc(&w->scale, static_cast<size_t>(scales) * (w->scale_bf16 ? 2 : 4)) != cudaSuccess) {
        cudaGetLastError();
        aem::free_q4(w);
        set_error("aem_q4weight_pack: device allocation failed");
        return AEM_ENOMEM;
    }
    aem::pack_q4_kernel<<<static_cast<unsigned>(std::min<int64_t>((tiles + 7) / 8, 148 * 64)),
                          aem::kThreads, 0, s>>>(q, K, N, w->NT, w->KT, tiles, w->q, err);
    const unsigned gr = static_cast<unsigned>(std::min<int64_t>((scales + 255) / 256, 148 * 64));
    if (w->scale_bf16)
        aem::pack_q4_scale_kernel<__nv_bfloat16><<<gr, aem::kThreads, 0, s>>>(
            static_cast<const __nv_bfloat16*>(scale), G * w->KB, N, w->NT,
            static_cast<__nv_bfloat16*>(w->scale));
    else
        aem::pack_q4_scale_kernel<float><<<gr, aem::kThreads, 0, s>>>(
            static_cast<const float*>(scale), G * w->KB, N, w->NT, static_cast<float*>(w->scale));
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

aem_status aem_q4gemm(aem_q4weight_t wh, int64_t group, const void* x, aem_dtype x_dtype,
                      int64_t ldx, int64_t M, void* out, aem_dtype out_dtype, int64_t ldo,
                      void* stream) {
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
    a.x = x;
    a.ldx = ldx;
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group = group;
    a.G = 1;
    a.out_bf16 = out_dtype == AEM_BF16;
    return aem::q4_product(w, "aem_q4gemm", a, x_dtype, static_cast<cudaStream_t>(stream));
}

aem_status aem_grouped_q4gemm(aem_q4weight_t wh, const int32_t* group_rows, const void* x,
                              aem_dtype x_dtype, int64_t ldx, int64_t M, void* out,
                              aem_dtype out_dtype, int64_t ldo, int relu, void* stream) {
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
    a.x = x;
    a.ldx = ldx;
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group_rows = group_rows;
    a.G = static_cast<int>(w->G);
    a.out_bf16 = out_dtype == AEM_BF16;
    a.relu = relu != 0;
    return aem::q4_product(w, "aem_grouped_q4gemm", a, x_dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
