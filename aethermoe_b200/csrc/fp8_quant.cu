// Quantisation to 8-bit floating point (e4m3) in blocks of 128, rows and weights,
// and the packing of the weights.
//
// A block's scale is max(amax / 448, 2^-126) and q = e4m3(x / scale), both IEEE
// float32 divisions, so that a block's largest magnitude becomes the largest e4m3
// value.  448 (1 + 2^-23) is the most that the quotient can be, which rounds to
// 448.  Memory bound: 2 or 4 bytes read and one written per element; each element
// is read once and stays in registers between the maximum and the quotient.
#include <cuda_bf16.h>

#include <algorithm>
#include <new>

#include "common.cuh"
#include "fp8.h"
#include "runtime.h"

namespace aem {
namespace {

constexpr int kThreads = 256;

// Two quotients x / s, rounded as IEEE division does: with r = 1/s rounded and
// q = x r, the residual x - s q is exact in a fused multiply-add, and q + r (x - s q)
// is the rounded quotient (P. Markstein, IBM J. Res. Dev. 34, 1990).  The residual
// has to stay normal, which holds for s in [2^-90, 2^126): a quotient that e4m3
// does not round to zero is 2^-11 at least, so x is 2^-101.  It is rounded downward, so
// that one of zero is -0 and a quotient of either zero keeps its sign.
__device__ __forceinline__ void quotient2(float x0, float x1, float s, float r, float& q0, float& q1) {
    asm("{\n.reg .b64 x, s, n, r, q, e;\nmov.b64 x, {%2, %3};\nmov.b64 n, {%5, %5};\nmov.b64 r, {%4, %4};\n"
        "mul.rn.f32x2 q, x, r;\nfma.rm.f32x2 e, n, q, x;\nfma.rn.f32x2 q, e, r, q;\nmov.b64 {%0, %1}, q;\n}"
        : "=f"(q0), "=f"(q1)
        : "f"(x0), "f"(x1), "f"(r), "f"(-s));
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t v;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(hi), "f"(lo));
    return v;
}
// The same for one, divided by 448: exact where nothing is subnormal.
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    const float a = __uint_as_float(amax_bits);  // a NaN's bits are above infinity's
    if (a >= 0x1p-90f && a <= 0x1.fffffep+127f) {
        constexpr float r = 1.0f / 448.0f;  // rounded
        const float q = a * r;
        return fmaf(fmaf(-448.0f, q, a), r, q);
    }
    const float s = __fdiv_rn(a, 448.0f);
    return s < 0x1p-126f ? 0x1p-126f : s;
}
// N values of one block, N even, to N bytes.
template <int N>
__device__ __forceinline__ void to_e4m3(const float (&v)[N], float s, uint32_t (&o)[N / 4]) {
    float q[N];
    if (s >= 0x1p-90f && s < 0x1p126f) {
        const float r = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < N; i += 2) quotient2(v[i], v[i + 1], s, r, q[i], q[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = __fdiv_rn(v[i], s);
    }
#pragma unroll
    for (int i = 0; i < N; i += 4) o[i / 4] = e4m3x2(q[i], q[i + 1]) | e4m3x2(q[i + 2], q[i + 3]) << 16;
}

// 8 elements of a row from k on as they lie in memory, zero past K.
template <typename XT>
struct Eight {
    uint32_t w[2 * sizeof(XT)];
    template <bool VEC>
    __device__ __forceinline__ void load(const XT* row, int64_t k, int64_t K) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(2 * sizeof(XT)); ++i) w[i] = 0;
        if (VEC && k + 8 <= K) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(XT)) / 2; ++i) {
                const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(row + k) + 16 * i);
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < K) {
                if constexpr (sizeof(XT) == 4)
                    w[i] = __float_as_uint(row[k + i]);
                else
                    w[i / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(row[k + i])) << (16 * (i & 1));
            }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(XT) == 4) return __uint_as_float(w[i]);
        return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
    // Bits of the largest magnitude, a NaN's above everything.
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < static_cast<int>(2 * sizeof(XT)); ++i)
            m = sizeof(XT) == 4 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
        return sizeof(XT) == 4 ? m : max(m & 0xffff0000u, m << 16);
    }
};

// 8 lanes share a block, twice 8 elements each, 64 apart, so that a load's lanes lie
// side by side; they take kHeld blocks that follow one another, all of their loads
// in flight at once.  The divisions of a block's scale are shared by 16 elements (16
// lanes of 8 each: 98304 x 2048 bf16 in 147 us, so in 108, 5.6 TB/s; float32 rows at
// 6.8).
template <typename XT>
constexpr int kHeld = sizeof(XT) == 2 ? 2 : 1;
template <typename XT, bool VEC>
__global__ void __launch_bounds__(kThreads)
    quantize_fp8_kernel(const XT* __restrict__ x, int64_t ldx, int64_t blocks, int64_t K, int64_t KB,
                        uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale, int64_t lds) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int HELD = kHeld<XT>;
    const int sub = threadIdx.x & 7;
    const int64_t first = (blockIdx.x * static_cast<int64_t>(kThreads / 8) + (threadIdx.x >> 3)) * HELD;
    // (a 32-bit division where it will do)
    int64_t m = first < (1ll << 31) && KB < (1ll << 31) ? static_cast<uint32_t>(first) / static_cast<uint32_t>(KB) : first / KB;
    int64_t b = first - m * KB;
    int64_t row[HELD], kb[HELD];
    Eight<XT> v[HELD][2];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        row[i] = m;
        kb[i] = b;
        const int64_t end = first + i < blocks ? K : 0;
        v[i][0].template load<VEC>(x + m * ldx, b * 128 + sub * 8, end);
        v[i][1].template load<VEC>(x + m * ldx, b * 128 + 64 + sub * 8, end);
        if (++b == KB) b = 0, ++m;
    }
    const int64_t end = (K + 15) / 16 * 16;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        uint32_t top = max(v[i][0].top(), v[i][1].top());
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
        if (first + i >= blocks) continue;
        const float s = block_scale(top);
        float f[16];
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = v[i][j / 8].get(j % 8);
        to_e4m3(f, s, o);
        const int64_t k = kb[i] * 128 + sub * 8;
        uint8_t* to = q + row[i] * ldq + k;
        if (k < end) *reinterpret_cast<uint2*>(to) = make_uint2(o[0], o[1]);
        if (k + 64 < end) *reinterpret_cast<uint2*>(to + 64) = make_uint2(o[2], o[3]);
        if (sub == 0) scale[row[i] * lds + kb[i]] = s;
    }
}

// A block of 128 x 128 weights per thread block, in registers between its maximum
// and its quotients: a lane has 16 bytes of a row at a time.  Memory bound: 4096 x
// 14336 float32 in 51 us, 5.8 TB/s.
template <typename WT, bool VEC>
__global__ void __launch_bounds__(kThreads, sizeof(WT) == 4 ? 3 : 4)
    quantize_fp8_weight_kernel(const WT* __restrict__ w, int64_t K, int64_t N, int64_t KB, int64_t NB,
                               uint8_t* __restrict__ q, float* __restrict__ scale) {
    constexpr int CL = 16 / sizeof(WT), LANES = 128 / CL, STEP = kThreads / LANES, R = 128 / STEP;
    __shared__ uint32_t tops[kThreads / 32];
    const int64_t g = blockIdx.x / (KB * NB), t = blockIdx.x % (KB * NB), kb = t / NB, nb = t % NB;
    const int64_t n = nb * 128 + threadIdx.x % LANES * CL, k0 = kb * 128 + threadIdx.x / LANES;
    const int64_t at = (g * K + k0) * N + n;
    uint32_t v[R][4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0;
        if (k0 + i * STEP >= K || n >= N) continue;
        const WT* p = w + at + static_cast<int64_t>(i) * STEP * N;
        if constexpr (VEC) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            v[i][0] = u.x, v[i][1] = u.y, v[i][2] = u.z, v[i][3] = u.w;
        } else {
#pragma unroll
            for (int j = 0; j < CL; ++j)
                if (n + j < N) {
                    if constexpr (sizeof(WT) == 4)
                        v[i][j] = __float_as_uint(p[j]);
                    else
                        v[i][j / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(p[j])) << (16 * (j & 1));
                }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            top = sizeof(WT) == 4 ? max(top, v[i][j] & 0x7fffffffu) : __vmaxu2(top, v[i][j] & 0x7fff7fffu);
    if (sizeof(WT) == 2) top = max(top & 0xffff0000u, top << 16);
    top = __reduce_max_sync(~0u, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) top = max(top, tops[i]);
    const float s = block_scale(top);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (k0 + i * STEP >= K || n >= N) continue;
        float f[CL];
        uint32_t o[CL / 4];
#pragma unroll
        for (int j = 0; j < CL; ++j)
            f[j] = sizeof(WT) == 4 ? __uint_as_float(v[i][j % 4])
                                   : __uint_as_float(j & 1 ? v[i][j / 2] & 0xffff0000u : v[i][j / 2] << 16);
        to_e4m3(f, s, o);
        uint8_t* p = q + at + static_cast<int64_t>(i) * STEP * N;
        if constexpr (VEC && CL == 8) {
            *reinterpret_cast<uint2*>(p) = make_uint2(o[0], o[1]);
        } else if constexpr (VEC) {
            *reinterpret_cast<uint32_t*>(p) = o[0];
        } else {
#pragma unroll
            for (int j = 0; j < CL; ++j)
                if (n + j < N) p[j] = static_cast<uint8_t>(o[j / 4] >> (8 * (j & 3)));
        }
    }
}

// Once per weight: a tile of 128 k x 128 channels turned round, 4 x 4 bytes at a time
// in registers and the rest in shared memory, where a row of 4-byte pieces of k
// belongs to a channel.
template <bool VEC>
__global__ void __launch_bounds__(kThreads)
    pack_fp8_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale, int64_t K, int64_t N, int64_t NC,
                    int64_t KC, uint8_t* __restrict__ out, float* __restrict__ out_scale) {
    __shared__ uint32_t tile[128][33];  // [channel][piece of 4 k]
    const int64_t g = blockIdx.x / (NC * KC), t = blockIdx.x % (NC * KC), nc = t / KC, kc = t % KC;
    const int n0 = threadIdx.x % 32 * 4;
    for (int p = threadIdx.x / 32; p < 32; p += kThreads / 32) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t k = kc * 128 + p * 4 + i, n = nc * 128 + n0;
            const uint8_t* from = q + (g * K + k) * N + n;
            v[i] = 0;
            if (k >= K) continue;
            if (VEC && n < N) {
                v[i] = *reinterpret_cast<const uint32_t*>(from);
            } else if (!VEC) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < N) v[i] |= static_cast<uint32_t>(from[j]) << (8 * j);
            }
        }
        const uint32_t a = __byte_perm(v[0], v[1], 0x5140), b = __byte_perm(v[2], v[3], 0x5140);
        const uint32_t c = __byte_perm(v[0], v[1], 0x7362), d = __byte_perm(v[2], v[3], 0x7362);
        tile[n0][p] = __byte_perm(a, b, 0x5410);
        tile[n0 + 1][p] = __byte_perm(a, b, 0x7632);
        tile[n0 + 2][p] = __byte_perm(c, d, 0x5410);
        tile[n0 + 3][p] = __byte_perm(c, d, 0x7632);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * 8; i += kThreads) {
        const int n = i >> 3, c = i & 7;
        *reinterpret_cast<uint4*>(out + blockIdx.x * static_cast<int64_t>(kFp8Tile) + n * 128 + ((c ^ (n & 7)) << 4)) =
            make_uint4(tile[n][4 * c], tile[n][4 * c + 1], tile[n][4 * c + 2], tile[n][4 * c + 3]);
    }
    if (threadIdx.x == 0) out_scale[blockIdx.x] = scale[(g * KC + kc) * NC + nc];
}

aem_status check_weight_shape(const char* what, int64_t G, int64_t K, int64_t N) {
    AEM_REQUIRE(G >= 1 && K >= 1 && N >= 1, "%s: G=%lld K=%lld N=%lld must be >= 1", what, (long long)G, (long long)K,
                (long long)N);
    AEM_REQUIRE(K < (1ll << 30) && N < (1ll << 30) && G < (1ll << 30) &&
                    G * ((K + 127) / 128) < (1ll << 31) && G * ((K + 127) / 128) * ((N + 127) / 128) < (1ll << 24),
                "%s: dimensions out of range", what);
    return AEM_OK;
}

void free_fp8(Fp8Weight* w) {
    cudaFree(w->data);
    delete w;
}

aem_status pack_fp8(const uint8_t* q, const float* scale, int64_t G, int64_t K, int64_t N, cudaStream_t s,
                    aem_fp8weight_t* out) {
    auto* w = new (std::nothrow) Fp8Weight();
    if (!w) {
        set_error("aem_fp8weight_pack: out of memory");
        return AEM_ENOMEM;
    }
    w->device = current_device();
    w->G = G;
    w->K = K;
    w->N = N;
    w->NC = (N + 127) / 128;
    w->KC = (K + 127) / 128;
    const int64_t tiles = G * w->NC * w->KC;
    if (cudaMalloc(&w->data, static_cast<size_t>(tiles) * (kFp8Tile + sizeof(float))) != cudaSuccess) {
        cudaGetLastError();
        free_fp8(w);
        set_error("aem_fp8weight_pack: device allocation failed");
        return AEM_ENOMEM;
    }
    w->scale = reinterpret_cast<float*>(w->data + tiles * kFp8Tile);
    auto kern = N % 4 == 0 && reinterpret_cast<uintptr_t>(q) % 4 == 0 ? pack_fp8_kernel<true> : pack_fp8_kernel<false>;
    kern<<<static_cast<unsigned>(tiles), kThreads, 0, s>>>(q, scale, K, N, w->NC, w->KC, w->data, w->scale);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        free_fp8(w);
        set_error("aem_fp8weight_pack: %s", cudaGetErrorString(e));
        return AEM_ECUDA;
    }
    count_launches(1);
    *out = reinterpret_cast<aem_fp8weight_t>(w);
    return AEM_OK;
}

}  // namespace

aem_status launch_quantize_fp8(const char* what, const void* x, aem_dtype dtype, int64_t ldx, int64_t M, int64_t K,
                               uint8_t* q, int64_t ldq, float* scale, int64_t lds, cudaStream_t s) {
    const int64_t KB = (K + 127) / 128, blocks = M * KB, per = kThreads / 8 * (dtype == AEM_F32 ? kHeld<float> : kHeld<__nv_bfloat16>);
    AEM_REQUIRE((blocks + per - 1) / per < (1ll << 31), "%s: M=%lld out of range", what, (long long)M);
    const auto grid = static_cast<unsigned>((blocks + per - 1) / per);
    const int es = dtype == AEM_F32 ? 4 : 2;
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * es % 16 == 0;
    auto go = [&](auto* p) {
        using XT = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        if (vec)
            quantize_fp8_kernel<XT, true><<<grid, kThreads, 0, s>>>(p, ldx, blocks, K, KB, q, ldq, scale, lds);
        else
            quantize_fp8_kernel<XT, false><<<grid, kThreads, 0, s>>>(p, ldx, blocks, K, KB, q, ldq, scale, lds);
    };
    if (dtype == AEM_F32)
        go(static_cast<const float*>(x));
    else
        go(static_cast<const __nv_bfloat16*>(x));
    AEM_CHECK_LAUNCH();
    count_launches(1);
    return AEM_OK;
}

}  // namespace aem

using aem::set_error;

extern "C" {

aem_status aem_quantize_fp8(const void* x, aem_dtype dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* q,
                            int64_t ldq, float* scale, int64_t lds, void* stream) {
    AEM_REQUIRE(dtype == AEM_F32 || dtype == AEM_BF16, "aem_quantize_fp8: bad dtype");
    AEM_REQUIRE(M >= 0 && K >= 1 && M < (1ll << 40) && K < (1ll << 30), "aem_quantize_fp8: M=%lld K=%lld out of range",
                (long long)M, (long long)K);
    AEM_REQUIRE(ldx >= 0 && ldq >= K && ldq % 16 == 0 && lds >= (K + 127) / 128 && lds % 4 == 0,
                "aem_quantize_fp8: bad row stride");
    if (M == 0) return AEM_OK;
    AEM_REQUIRE(x && q && scale, "aem_quantize_fp8: NULL buffer");
    AEM_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(scale) % 16 == 0,
                "aem_quantize_fp8: q and scale must be 16-byte aligned");
    return aem::launch_quantize_fp8("aem_quantize_fp8", x, dtype, ldx, M, K, q, ldq, scale, lds,
                                    static_cast<cudaStream_t>(stream));
}

aem_status aem_quantize_fp8_weight(const void* w, aem_dtype dtype, int64_t G, int64_t K, int64_t N, uint8_t* q,
                                   float* scale, void* stream) {
    AEM_TRY(aem::check_weight_shape("aem_quantize_fp8_weight", G, K, N));
    AEM_REQUIRE(dtype == AEM_F32 || dtype == AEM_BF16, "aem_quantize_fp8_weight: bad dtype");
    AEM_REQUIRE(w && q && scale, "aem_quantize_fp8_weight: NULL buffer");
    const int64_t KB = (K + 127) / 128, NB = (N + 127) / 128;
    const auto grid = static_cast<unsigned>(G * KB * NB);
    auto s = static_cast<cudaStream_t>(stream);
    const int cl = dtype == AEM_F32 ? 4 : 8;
    const bool vec = N % cl == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % cl == 0;
    auto go = [&](auto* p) {
        using WT = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        if (vec)
            aem::quantize_fp8_weight_kernel<WT, true><<<grid, aem::kThreads, 0, s>>>(p, K, N, KB, NB, q, scale);
        else
            aem::quantize_fp8_weight_kernel<WT, false><<<grid, aem::kThreads, 0, s>>>(p, K, N, KB, NB, q, scale);
    };
    if (dtype == AEM_F32)
        go(static_cast<const float*>(w));
    else
        go(static_cast<const __nv_bfloat16*>(w));
    AEM_CHECK_LAUNCH();
    aem::count_launches(1);
    return AEM_OK;
}

aem_status aem_fp8weight_pack_device(const uint8_t* q, const float* scale, int64_t G, int64_t K, int64_t N,
                                     void* stream, aem_fp8weight_t* out) {
    AEM_REQUIRE(out != nullptr, "aem_fp8weight_pack: out is NULL");
    *out = nullptr;
    AEM_TRY(aem::check_weight_shape("aem_fp8weight_pack", G, K, N));
    AEM_REQUIRE(q && scale, "aem_fp8weight_pack: NULL buffer");
    return aem::pack_fp8(q, scale, G, K, N, static_cast<cudaStream_t>(stream), out);
}

aem_status aem_fp8weight_pack(const uint8_t* q, const float* scale, int64_t G, int64_t K, int64_t N, int device,
                              aem_fp8weight_t* out) {
    AEM_REQUIRE(out != nullptr, "aem_fp8weight_pack: out is NULL");
    *out = nullptr;
    AEM_TRY(aem::check_weight_shape("aem_fp8weight_pack", G, K, N));
    AEM_REQUIRE(q && scale, "aem_fp8weight_pack: NULL buffer");
    if (!aem::is_sm100(device)) {
        set_error("aem_fp8weight_pack: device %d is not an sm_100 (B200) GPU", device);
        return AEM_EUNSUPPORTED;
    }
    struct Device {  // the caller's device is current again at the end
        int before = 0;
        Device() { cudaGetDevice(&before); }
        ~Device() { cudaSetDevice(before); }
    } restore;
    AEM_TRY_CUDA(cudaSetDevice(device));
    const size_t qb = static_cast<size_t>(G * K * N);
    const size_t sb = static_cast<size_t>(G * ((K + 127) / 128) * ((N + 127) / 128)) * sizeof(float);
    uint8_t* dq = nullptr;
    float* ds = nullptr;
    AEM_TRY_CUDA(cudaMalloc(&dq, qb));
    if (cudaMalloc(&ds, sb) != cudaSuccess) {
        cudaGetLastError();
        cudaFree(dq);
        set_error("aem_fp8weight_pack: device allocation failed");
        return AEM_ENOMEM;
    }
    aem_status st = AEM_OK;
    if (cudaMemcpy(dq, q, qb, cudaMemcpyHostToDevice) != cudaSuccess ||
        cudaMemcpy(ds, scale, sb, cudaMemcpyHostToDevice) != cudaSuccess) {
        set_error("aem_fp8weight_pack: copy failed");
        st = AEM_ECUDA;
    }
    if (st == AEM_OK) st = aem::pack_fp8(dq, ds, G, K, N, nullptr, out);
    if (st == AEM_OK && cudaStreamSynchronize(nullptr) != cudaSuccess) {
        set_error("aem_fp8weight_pack: packing failed");
        aem::free_fp8(reinterpret_cast<aem::Fp8Weight*>(*out));
        *out = nullptr;
        st = AEM_ECUDA;
    }
    cudaFree(dq);
    cudaFree(ds);
    return st;
}

aem_status aem_fp8weight_free(aem_fp8weight_t wh) {
    if (!wh) return AEM_OK;
    auto* w = reinterpret_cast<aem::Fp8Weight*>(wh);
    int prev = 0;
    cudaGetDevice(&prev);
    cudaSetDevice(w->device);
    cudaDeviceSynchronize();
    aem::free_fp8(w);
    cudaSetDevice(prev);
    return AEM_OK;
}

aem_status aem_fp8weight_shape(aem_fp8weight_t wh, int64_t* G, int64_t* K, int64_t* N) {
    AEM_REQUIRE(wh != nullptr, "aem_fp8weight_shape: handle is NULL");
    auto* w = reinterpret_cast<aem::Fp8Weight*>(wh);
    if (G) *G = w->G;
    if (K) *K = w->K;
    if (N) *N = w->N;
    return AEM_OK;
}

}  // extern "C"
