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
// q + 8; padding holds 8.  scale: [G][KB][NT/2][8][4], channels c, c+8, c+16,
// c+24 of 32 side by side, in the caller's type, padding zero.
struct Q4Weight {
    int device = 0;
    int64_t G = 0, K = 0, N = 0, NT = 0, KT = 0, KB = 0;
    int gs = 0;
    bool scale_bf16 = false;
    uint4* q = nullptr;
    void* scale = nullptr;
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
        const int64_t n = r / 32 * 32 + (r & 3) * 8 + (r % 32) / 4;
        out[i] = n < N ? s[b * N + n] : ST(0.0f);
    }
}

// ------------------------------------------------------------------ product
// Columns of the MMAs: the rows of x as they are (bf16), or three per row
// (float32: the terms that add up to it).
struct Q4Args {
    const uint4* q;
    const void* scale;
    const __nv_bfloat16* x;     // [M * terms][ldx], 16-byte rows, readable to a multiple of 8 k
    void* out;
    const int32_t* group_rows;  // nullptr: one group of M rows, weight group `group`
    int64_t ldx, ldo, M, K, N, NT, KT, KB;
    int64_t group;
    int G, S, rows, terms;  // S: CTAs (one cluster) that split K; rows: rows of a row tile
    bool out_bf16, relu, dependent;
};

template <bool ZERO>
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    if constexpr (ZERO)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
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

// Activations in the form the products read: [M * terms][KP] bf16, KP = K
// rounded up to 8, zero padded.  float32 gives three truncated terms v =
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

// The scales of one lane and scale group: channels c, c+8, c+16, c+24 of 32.
template <typename ST>
struct Scales;
template <>
struct Scales<float> {
    float4 v;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        v = __ldg(reinterpret_cast<const float4*>(p) + i);
    }
    __device__ __forceinline__ float get(int c, int hi) const {
        return c ? (hi ? v.w : v.z) : (hi ? v.y : v.x);
    }
};
template <>
struct Scales<__nv_bfloat16> {
    uint2 v;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        v = __ldg(reinterpret_cast<const uint2*>(p) + i);
    }
    __device__ __forceinline__ float get(int c, int hi) const {
        const uint32_t u = c ? v.y : v.x;
        return __uint_as_float(hi ? u & 0xffff0000u : u << 16);
    }
};

// The weight stream of one warp: 32 channels, 64-k tiles [kt0, kt1), PF tiles
// in flight in registers.
constexpr int PF = 4;
template <int GS, typename ST>
struct Stream {
    static constexpr int NS = GS == 32 ? 2 : 1;
    uint4 w[PF][2];
    Scales<ST> s[PF][NS];
    const uint4* wp;
    const void* sp;
    int64_t wstep, s0, sstep;
    int kt1;
    int64_t last;

    __device__ __forceinline__ void start(const Q4Args& a, int64_t g, int64_t pair, int end) {
        const int lane = threadIdx.x & 31;
        wp = a.q + (g * a.NT + pair * 2) * a.KT * 32 + lane;
        wstep = a.KT * 32;
        sp = a.scale;
        s0 = (g * a.KB * (a.NT / 2) + pair) * 8 + (lane >> 2);
        sstep = a.NT / 2 * 8;
        kt1 = end;
        last = a.KB - 1;
    }
    __device__ __forceinline__ void fetch(int slot, int kt) {
        if (kt >= kt1) return;
        w[slot][0] = __ldg(wp + static_cast<int64_t>(kt) * 32);
        w[slot][1] = __ldg(wp + static_cast<int64_t>(kt) * 32 + wstep);
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int64_t b = GS == 32 ? min(static_cast<int64_t>(2 * kt + j), last) : kt / (GS / 64);
            s[slot][j].load(sp, s0 + b * sstep);
        }
    }
};

// One 64-k tile: NT column tiles of B fragments from `b(nt, h)` (uint4: MMAs
// 2h and 2h+1) times the 32 channels of w, scaled into acc.  FIRST / LAST:
// the tile opens / closes a scale group (GS >= 64).
template <int NT, int GS, typename ST, typename B>
__device__ __forceinline__ void tile_product(const uint4 (&w)[2], const Scales<ST>* s, bool first,
                                             bool last, float (&acc)[2][NT][4],
                                             float (&sum)[2][NT][4], B b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t wa[2][2][4];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            unpack_q4(h ? w[c].z : w[c].x, wa[c][0]);
            unpack_q4(h ? w[c].w : w[c].y, wa[c][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint4 x = b(nt, h);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if constexpr (GS == 32) {
                    float p[4];
                    mma_bf16<true>(p, wa[c][0], x.x, x.y);
                    mma_bf16<false>(p, wa[c][1], x.z, x.w);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[c][nt][i] = fmaf(s[h].get(c, i >> 1), p[i], acc[c][nt][i]);
                } else {
                    if (h == 0 && first)
                        mma_bf16<true>(sum[c][nt], wa[c][0], x.x, x.y);
                    else
                        mma_bf16<false>(sum[c][nt], wa[c][0], x.x, x.y);
                    mma_bf16<false>(sum[c][nt], wa[c][1], x.z, x.w);
                    if (h == 1 && last)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[c][nt][i] = fmaf(s[0].get(c, i >> 1), sum[c][nt][i], acc[c][nt][i]);
                }
            }
        }
    }
}

__device__ __forceinline__ void store_out(const Q4Args& a, int64_t m, int64_t n, float v) {
    if (a.relu && v < 0.0f) v = 0.0f;
    if (a.out_bf16)
        static_cast<__nv_bfloat16*>(a.out)[m * a.ldo + n] = __float2bfloat16_rn(v);
    else
        static_cast<float*>(a.out)[m * a.ldo + n] = v;
}

// Part `part` of `parts` of the 64-k tiles, cut at scale groups.
__device__ __forceinline__ void k_range(const Q4Args& a, int gran, int64_t part, int64_t parts,
                                        int* kt0, int* kt1) {
    const int64_t units = (a.KT + gran - 1) / gran;
    *kt0 = static_cast<int>(units * part / parts * gran);
    *kt1 = static_cast<int>(min(units * (part + 1) / parts * gran, a.KT));
}

// Few columns (8 NT <= 16): a CTA computes 32 channels, its 4 warps (and the S
// CTAs of its cluster) split K, and their float32 sums meet in a fixed order.
// Each warp reads the B fragments of its own k straight from x (cached), one
// tile ahead.
template <int NT, int GS, typename ST>
__global__ void __launch_bounds__(128) q4_narrow_kernel(const Q4Args a) {
    constexpr int W = 4;
    __shared__ float red[W][NT * 8 * 32];
    __shared__ float fin[32][NT * 8 + 1];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t tile = blockIdx.x / a.S;
    const int ks = blockIdx.x % a.S;
    int64_t g, m0;
    int rows;
    if (!find_rows(a, blockIdx.y, &g, &m0, &rows)) return;
    int kt0, kt1;
    k_range(a, GS > 64 ? GS / 64 : 1, ks * W + w, a.S * W, &kt0, &kt1);
    Stream<GS, ST> st;
    st.start(a, g, tile, kt1);
#pragma unroll
    for (int i = 0; i < PF; ++i) st.fetch(i, kt0 + i);
    if (a.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");  // x is the terms kernel's

    const __nv_bfloat16* xp[NT];
    const int t8 = 8 * (lane & 3);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int col = 8 * nt + (lane >> 2);
        xp[nt] = col < rows * a.terms ? a.x + (m0 * a.terms + col) * a.ldx : nullptr;
    }
    uint4 xb[2][NT][2];
    auto load_x = [&](int slot, int kt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t k = kt * 64ll + 32 * h + t8;
                xb[slot][nt][h] = make_uint4(0, 0, 0, 0);
                if (xp[nt] && kt < kt1 && k < a.K)
                    xb[slot][nt][h] = *reinterpret_cast<const uint4*>(xp[nt] + k);
            }
    };
    float acc[2][NT][4] = {}, sum[2][NT][4] = {};
    load_x(0, kt0);
    for (int kb = kt0; kb < kt1; kb += PF) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int kt = kb + i;
            if (kt >= kt1) break;
            load_x((i + 1) & 1, kt + 1);
            const uint4 wt[2] = {st.w[i][0], st.w[i][1]};
            Scales<ST> sc[Stream<GS, ST>::NS];
#pragma unroll
            for (int j = 0; j < Stream<GS, ST>::NS; ++j) sc[j] = st.s[i][j];
            st.fetch(i, kt + PF);
            const bool first = GS <= 64 || i % 2 == 0;
            const bool last = GS <= 64 || i % 2 == 1 || kt + 1 == kt1;
            tile_product<NT, GS, ST>(wt, sc, first, last, acc, sum,
                                     [&](int nt, int h) { return xb[i & 1][nt][h]; });
        }
    }

    // the warps' sums, in warp order, into fin[channel][column]
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[w][((c * NT + nt) * 4 + i) * 32 + lane] = acc[c][nt][i];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 8 * 32; i += 128) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) s += red[j][i];
        const int l = i & 31, e = (i >> 5) & 3, cn = i >> 7, c = cn / NT, nt = cn % NT;
        fin[c * 16 + (l >> 2) + 8 * (e >> 1)][nt * 8 + 2 * (l & 3) + (e & 1)] = s;
    }
    __syncthreads();
    if (a.S > 1) cluster_barrier();
    if (ks == 0)
        for (int i = threadIdx.x; i < rows * 32; i += 128) {
            const int r = i >> 5, ch = i & 31;
            const int64_t n = tile * 32 + ch;
            float v = 0.0f;
            for (int s = 0; s < a.S; ++s)
                for (int j = 0; j < a.terms; ++j) {
                    const float* p = &fin[ch][r * a.terms + j];
                    v += s == 0 ? *p : ld_cluster(p, s);
                }
            if (n < a.N) store_out(a, m0 + r, n, v);
        }
    if (a.S > 1) cluster_barrier();  // the others' fin stays until rank 0 has read it
}

// Many columns: a CTA computes 128 channels, 32 per warp; the B fragments of a
// 64-k tile are copied once per CTA into a shared-memory ring, in the order
// the lanes read them (16 bytes a lane, no bank conflicts).  The S CTAs of
// the cluster split K; each adds up its share of the channels in rank order.
template <int NT, int GS, typename ST>
__global__ void __launch_bounds__(128) q4_wide_kernel(const Q4Args a) {
    constexpr int W = 4, COLS = 8 * NT, LD = W * 32 + 4;
    constexpr int kRing = PF * NT * 64 * 16, kFin = COLS * LD * 4;
    __shared__ __align__(16) char smem[kRing > kFin ? kRing : kFin];
    auto* ring = reinterpret_cast<uint4*>(smem);  // [PF][NT][2][32]
    auto* fin = reinterpret_cast<float*>(smem);   // [COLS][LD], after the loop
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t tile = blockIdx.x / a.S;
    const int ks = blockIdx.x % a.S;
    int64_t g, m0;
    int rows;
    if (!find_rows(a, blockIdx.y, &g, &m0, &rows)) return;
    int kt0, kt1;
    k_range(a, GS > 64 ? GS / 64 : 1, ks, a.S, &kt0, &kt1);
    const int64_t pair = tile * W + w;
    const bool mine = pair < a.NT / 2;
    Stream<GS, ST> st;
    st.start(a, g, mine ? pair : 0, mine ? kt1 : kt0);
#pragma unroll
    for (int i = 0; i < PF; ++i) st.fetch(i, kt0 + i);
    if (a.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");

    constexpr int COPIES = NT / 2;  // 16-byte pieces per thread: NT * 64 / 128
    const __nv_bfloat16* src[COPIES];
    int koff[COPIES];
#pragma unroll
    for (int j = 0; j < COPIES; ++j) {
        const int i = threadIdx.x + 128 * j, l = i & 31;
        const int col = 8 * (i >> 6) + (l >> 2);
        koff[j] = 32 * ((i >> 5) & 1) + 8 * (l & 3);
        src[j] = col < rows * a.terms ? a.x + (m0 * a.terms + col) * a.ldx : nullptr;
    }
    auto copy_x = [&](int slot, int kt) {
        if (kt < kt1)
#pragma unroll
            for (int j = 0; j < COPIES; ++j) {
                const int64_t k = kt * 64ll + koff[j];
                const bool on = src[j] && k < a.K;
                const uint32_t to = dev::smem_u32(ring + slot * NT * 64 + threadIdx.x + 128 * j);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to),
                             "l"(on ? src[j] + k : a.x), "r"(on ? 16 : 0)
                             : "memory");
            }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float acc[2][NT][4] = {}, sum[2][NT][4] = {};
#pragma unroll
    for (int i = 0; i < PF - 1; ++i) copy_x(i, kt0 + i);
    for (int kb = kt0; kb < kt1; kb += PF) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int kt = kb + i;
            if (kt >= kt1) break;
            asm volatile("cp.async.wait_group %0;" ::"n"(PF - 2) : "memory");
            __syncthreads();  // tile kt has landed; every warp is past tile kt - 1
            copy_x((i + PF - 1) % PF, kt + PF - 1);
            const uint4 wt[2] = {st.w[i][0], st.w[i][1]};
            Scales<ST> sc[Stream<GS, ST>::NS];
#pragma unroll
            for (int j = 0; j < Stream<GS, ST>::NS; ++j) sc[j] = st.s[i][j];
            st.fetch(i, kt + PF);
            const bool first = GS <= 64 || i % 2 == 0;
            const bool last = GS <= 64 || i % 2 == 1 || kt + 1 == kt1;
            if (mine)
                tile_product<NT, GS, ST>(wt, sc, first, last, acc, sum, [&](int nt, int h) {
                    return ring[((i * NT + nt) * 2 + h) * 32 + lane];
                });
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                fin[(nt * 8 + 2 * (lane & 3) + (i & 1)) * LD + w * 32 + c * 16 + (lane >> 2) + 8 * (i >> 1)] =
                    acc[c][nt][i];
    __syncthreads();
    if (a.S > 1) cluster_barrier();
    for (int i = ks * 128 + threadIdx.x; i < rows * W * 32; i += a.S * 128) {
        const int r = i / (W * 32), ch = i % (W * 32);
        const int64_t n = tile * W * 32 + ch;
        float v = 0.0f;
        for (int s = 0; s < a.S; ++s)
            for (int j = 0; j < a.terms; ++j) {
                const float* p = fin + (r * a.terms + j) * LD + ch;
                v += s == ks ? *p : ld_cluster(p, s);
            }
        if (n < a.N) store_out(a, m0 + r, n, v);
    }
    if (a.S > 1) cluster_barrier();
}

template <int NT, int GS, typename ST>
aem_status launch_q4(const Q4Args& a, dim3 grid, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(128);
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
    if constexpr (NT <= 2)
        AEM_TRY_CUDA(cudaLaunchKernelEx(&cfg, q4_narrow_kernel<NT, GS, ST>, a));
    else
        AEM_TRY_CUDA(cudaLaunchKernelEx(&cfg, q4_wide_kernel<NT, GS, ST>, a));
    count_launches(1);
    return AEM_OK;
}

template <int NT>
aem_status launch_nt(const Q4Args& a, int gs, bool sb, dim3 grid, cudaStream_t s) {
    if (sb)
        return gs == 32   ? launch_q4<NT, 32, __nv_bfloat16>(a, grid, s)
               : gs == 64 ? launch_q4<NT, 64, __nv_bfloat16>(a, grid, s)
                          : launch_q4<NT, 128, __nv_bfloat16>(a, grid, s);
    return gs == 32   ? launch_q4<NT, 32, float>(a, grid, s)
           : gs == 64 ? launch_q4<NT, 64, float>(a, grid, s)
                      : launch_q4<NT, 128, float>(a, grid, s);
}

// x: the caller's rows; a.x and a.terms are set here.
aem_status q4_product(const Q4Weight* w, const char* what, Q4Args a, const void* x, aem_dtype xd,
                      void* workspace, size_t workspace_bytes, cudaStream_t s) {
    AEM_REQUIRE(current_device() == w->device, "%s: the weights are on device %d, the current one is %d",
                what, w->device, current_device());
    a.q = w->q;
    a.scale = w->scale;
    a.K = w->K;
    a.N = w->N;
    a.NT = w->NT;
    a.KT = w->KT;
    a.KB = w->KB;
    a.terms = xd == AEM_F32 ? 3 : 1;
    const bool as_is = xd == AEM_BF16 && a.K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
                       a.ldx % 8 == 0;
    void* own = nullptr;
    if (as_is) {
        a.x = static_cast<const __nv_bfloat16*>(x);
    } else {
        const int64_t KP = (a.K + 7) / 8 * 8;
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
            q4_terms_kernel<float><<<g, kThreads, 0, s>>>(static_cast<const float*>(x), a.ldx, a.M, a.K, KP, t);
        else
            q4_terms_kernel<__nv_bfloat16><<<g, kThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(x), a.ldx,
                                                                  a.M, a.K, KP, t);
        AEM_CHECK_LAUNCH();
        count_launches(1);
        a.x = t;
        a.ldx = KP;
        a.dependent = true;
    }
    // columns of a row tile: as many as the rows (grouped: an average group's) need, up to 64
    const int64_t groups = std::min<int64_t>(a.G, a.M);
    const int64_t want = (a.group_rows ? (a.M + groups - 1) / groups : a.M) * a.terms;
    const int nt = want <= 8 ? 1 : want <= 16 ? 2 : want <= 32 ? 4 : 8;
    a.rows = 8 * nt / a.terms;
    const int64_t slots = a.group_rows ? groups + a.M / a.rows : (a.M + a.rows - 1) / a.rows;
    const int64_t per = nt <= 2 ? 1 : 4, tiles = (a.NT / 2 + per - 1) / per, ctas = tiles * slots;
    const int64_t kparts = nt <= 2 ? 4 : 1;  // K shares inside a CTA
    a.S = 1;
    while (a.S < 8 && ctas * a.S < 148 * 2 && a.KT >= 4 * kparts * a.S) a.S *= 2;
    aem_status st = AEM_OK;
    const dim3 grid(static_cast<unsigned>(tiles * a.S), static_cast<unsigned>(slots));
    if (slots > 65535) {
        set_error("%s: M=%lld rows are too many for one call", what, (long long)a.M);
        st = AEM_EINVAL;
    } else if (nt == 1) {
        st = launch_nt<1>(a, w->gs, w->scale_bf16, grid, s);
    } else if (nt == 2) {
        st = launch_nt<2>(a, w->gs, w->scale_bf16, grid, s);
    } else if (nt == 4) {
        st = launch_nt<4>(a, w->gs, w->scale_bf16, grid, s);
    } else {
        st = launch_nt<8>(a, w->gs, w->scale_bf16, grid, s);
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

size_t aem_q4gemm_workspace(aem_q4weight_t wh, aem_dtype x_dtype, int64_t M) {
    if (!wh || M < 1 || !aem::is_dtype(x_dtype)) return 0;
    const int64_t KP = (reinterpret_cast<aem::Q4Weight*>(wh)->K + 7) / 8 * 8;
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
    a.ldx = ldx;
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.group = group;
    a.G = 1;
    a.out_bf16 = out_dtype == AEM_BF16;
    return aem::q4_product(w, "aem_q4gemm", a, x, x_dtype, workspace, workspace_bytes,
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
    return aem::q4_product(w, "aem_grouped_q4gemm", a, x, x_dtype, workspace, workspace_bytes,
                           static_cast<cudaStream_t>(stream));
}

}  // extern "C"
