// Routing of tokens to experts from their logits: softmax or sigmoid scores, a
// balance bias, groups of experts, top-k and renormalised weights, with the
// gradient of the weights.
//
// Row x[E] with bias b[E], s = softmax(x) or 1 / (1 + exp(-x)):
//   key_e  = s_e + b_e, or x_e without a bias (the order of the scores is the logits')
//   a group's value is the sum of its group_top (1 or 2) largest keys (scores, where
//   two are summed without a bias); the top_groups largest groups are kept, and of
//   their experts the k largest keys; ties go to the lower index
//   v_j = s[id_j], w_j = scale v_j or scale v_j / (sum v + 1e-20)
//
// The order has to be the one of 64-bit arithmetic, so that it depends on no
// rounding of a float32 exp or sum.  Keys are computed in float32 beside a bound
// on their error; wherever two keys that decide the order (neighbours among the
// k + 1 largest, the last group kept and the first dropped) are nearer than their
// bounds, the warp chooses again with keys in 64 bits.  With normally distributed
// logits that is a row in some hundred.  Logits themselves need no bound.
//
// A row lies across LANES lanes, 8 neighbouring experts a lane, so a lane's order
// is the experts' and up to 32 rows share a warp.  What has to be moved is T*E
// logits and 8 T*k bytes.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "runtime.h"

namespace aem {
namespace {

constexpr int kV = 8;             // experts of a lane
constexpr int kRouteWarps = 8;    // of a block
constexpr int kRouteThreads = 32 * kRouteWarps;

struct RouteArgs {
    const void* logits;
    const float* bias;
    const int32_t* ids_in;      // backward
    const float* grad;          // backward: of the weights
    void* grad_logits;
    int32_t* ids;
    float* weights;
    int64_t ld, T, ldi, ldg, ldo;
    float scale;
    int E, k, groups, top_groups, group_top, size, size_inv;  // size: experts of a group
    int sigmoid, renorm, vec, ovec;
    int* err;
};

// ---- segments: the LANES lanes of a row
template <int LANES, typename T, typename F>
__device__ __forceinline__ T seg_reduce(T v, F f) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(~0u, v, o));
    return v;
}
template <int LANES>
__device__ __forceinline__ float seg_sum(float v) {
    return seg_reduce<LANES>(v, [](float a, float b) { return a + b; });
}
template <int LANES>
__device__ __forceinline__ double seg_sum(double v) {
    return seg_reduce<LANES>(v, [](double a, double b) { return a + b; });
}
template <int LANES>
__device__ __forceinline__ float seg_max(float v) {
    return seg_reduce<LANES>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int LANES>
__device__ __forceinline__ uint32_t seg_max(uint32_t v) {
    if constexpr (LANES == 32) return __reduce_max_sync(~0u, v);
    return seg_reduce<LANES>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int LANES>
__device__ __forceinline__ unsigned long long seg_max(unsigned long long v) {
    return seg_reduce<LANES>(v, [](unsigned long long a, unsigned long long b) { return max(a, b); });
}

// ---- keys as unsigned numbers in the same order: NaN above everything, both
// zeros alike, 0 for "cannot be chosen" (the key -inf)
__device__ __forceinline__ uint32_t rank_of(float v) {
    if (v != v) return ~0u;
    if (v == -INFINITY) return 0;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ (u >> 31 ? ~0u : 0x80000000u);
}
__device__ __forceinline__ unsigned long long rank_of(double v) {
    if (v != v) return ~0ull;
    if (v == -INFINITY) return 0;
    const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
    return u ^ (u >> 63 ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ float value_of(uint32_t r) {
    return r == ~0u ? NAN : r == 0 ? -INFINITY : __uint_as_float(r ^ (r >> 31 ? 0x80000000u : ~0u));
}
__device__ __forceinline__ double value_of(unsigned long long r) {
    return r == ~0ull ? NAN
           : r == 0   ? -INFINITY
                      : __longlong_as_double(static_cast<long long>(r ^ (r >> 63 ? 0x8000000000000000ull : ~0ull)));
}

template <typename F>
struct Rank;
template <>
struct Rank<float> {
    using type = uint32_t;
};
template <>
struct Rank<double> {
    using type = unsigned long long;
};

// A float32 key's distance from the real one: the score's relative error is
// under 2^-19 (exp: 2 ulp, its argument: |x - m| 2^-24 for |x - m| <= 32, further
// down the score is under 2^-46 and the last term holds it; the sum of 256: 11
// halves of an ulp; the quotient 2), and the sum with the bias is rounded once.
__device__ __forceinline__ float slack(float score, float key) {
    return fmaf(0x1p-19f, score, fmaf(0x1p-23f, fabsf(key), 0x1p-64f));
}

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// Scores of a lane's experts; a row without any finite logit has zeros.
template <int LANES, typename F>
__device__ __forceinline__ void scores(const float (&x)[kV], bool sigmoid, F (&s)[kV]) {
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const F t = exp_of(-fabs(static_cast<F>(x[i])));
            s[i] = (x[i] < 0.0f ? t : F(1)) / (F(1) + t);
        }
        return;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kV; ++i) m = fmaxf(m, x[i]);
    m = seg_max<LANES>(m);
    if (m == -INFINITY) m = 0.0f;
    F z = 0;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
        s[i] = exp_of(static_cast<F>(x[i]) - static_cast<F>(m));
        z += s[i];
    }
    z = seg_sum<LANES>(z);
    const F r = z == F(0) ? F(0) : F(1) / z;
#pragma unroll
    for (int i = 0; i < kV; ++i) s[i] *= r;
}

struct RouteShared {
    double by[kRouteWarps][256];     // a warp's rows: values of the experts (or float)
    double value[kRouteWarps][256];  // of the groups
    int32_t ids[kRouteWarps][256];   // [row][k]: LANES * 8 >= k
    float v[kRouteWarps][256];
};

// Chooses from keys (and, for groups, from `by`) and leaves ids and `take`n
// values in shared memory.  CERT: returns whether a decision was nearer than the
// keys' slack.
template <int LANES, typename F, bool CERT>
__device__ __forceinline__ bool choose(const RouteArgs& a, const F (&key)[kV], const F (&by)[kV], const F (&s)[kV],
                                       const float (&take)[kV], RouteShared& sh) {
    using U = typename Rank<F>::type;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, sub = lane % LANES, row = lane / LANES;
    bool near = false;
    U u[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) u[i] = rank_of(key[i]);
    if (a.groups > 1) {
        F* val = reinterpret_cast<F*>(sh.by[w]) + row * LANES * kV;
        F* gv = reinterpret_cast<F*>(sh.value[w]) + row * LANES * kV;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kV; ++i) val[sub * kV + i] = by[i];
        __syncwarp();
        for (int g = sub; g < a.groups; g += LANES) {
            U first = 0, second = 0;
            for (int i = 0, at = g % a.size; i < a.size; ++i) {  // lanes start apart: other banks
                const U r = rank_of(val[g * a.size + at]);
                second = max(second, min(first, r));
                first = max(first, r);
                if (++at == a.size) at = 0;
            }
            F t = value_of(first);
            if (a.group_top == 2 && second) t += value_of(second);
            gv[g] = t;
        }
        __syncwarp();
        uint32_t kept[8] = {};  // a bit per group
        F least = INFINITY, most = -INFINITY;
        for (int g = sub; g < a.groups; g += LANES) {
            const U mine = rank_of(gv[g]);
            int before = 0;
            for (int h = 0; h < a.groups; ++h) {
                const U other = rank_of(gv[h]);
                before += other > mine || (other == mine && h < g);
            }
            if (before < a.top_groups) {
                least = gv[g] < least ? gv[g] : least;
#pragma unroll
                for (int i = 0; i < 8; ++i) kept[i] |= g >> 5 == i ? 1u << (g & 31) : 0u;
            } else {
                most = gv[g] > most ? gv[g] : most;
            }
        }
        if constexpr (CERT) {
            least = -seg_max<LANES>(-least);
            most = seg_max<LANES>(most);
            // a value is the sum of one or two keys of at most these sizes
            float top = 0.0f, largest = 0.0f;
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                top = fmaxf(top, s[i]);
                if (by[i] != -INFINITY) largest = fmaxf(largest, fabsf(by[i]));
            }
            top = seg_max<LANES>(top);
            largest = seg_max<LANES>(largest);
            const float e = 4.0f * slack(top, largest) + 0x1p-22f * largest;
            near |= most > -INFINITY && !(least - most > e);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i * 32 < a.groups) kept[i] = seg_reduce<LANES>(kept[i], [](uint32_t p, uint32_t q) { return p | q; });
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const int g = (sub * kV + i) * a.size_inv >> 16;
            uint32_t bits = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) bits = g >> 5 == j ? kept[j] : bits;
            if (!(bits >> (g & 31) & 1)) u[i] = 0;
        }
    }
    U best = 0;
#pragma unroll
    for (int i = 0; i < kV; ++i) best = max(best, u[i]);
    const unsigned segment = (LANES == 32 ? ~0u : (1u << LANES) - 1) << (row * LANES);
    float last_key = INFINITY, last_score = 0.0f;
    for (int j = 0; j < a.k + (CERT ? 1 : 0); ++j) {
        const U m = seg_max<LANES>(best);
        const int owner = __ffs(__ballot_sync(~0u, best == m) & segment) - 1;
        int at = kV;
        float score = 0.0f;
#pragma unroll
        for (int i = kV - 1; i >= 0; --i)
            if (u[i] == m) at = i;
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < kV; ++i)
            if (i == at) {
                t = take[i];
                if (CERT) score = s[i];
                if (lane == owner) u[i] = 0;
            }
        if (j < a.k && lane == owner) {
            sh.ids[w][row * a.k + j] = m ? sub * kV + at : -1;
            sh.v[w][row * a.k + j] = t;
        }
        best = 0;
#pragma unroll
        for (int i = 0; i < kV; ++i) best = max(best, u[i]);
        if constexpr (CERT) {
            score = __shfl_sync(~0u, score, owner);
            const float k = value_of(m);
            if (a.bias && j > 0 && m) near |= !(last_key - k > slack(score, k) + slack(last_score, last_key));
            last_key = k;
            last_score = score;
        }
    }
    __syncwarp();
    return near;
}

template <typename LT>
__device__ __forceinline__ void load_row(const RouteArgs& a, int64_t t, int e0, float (&x)[kV]) {
#pragma unroll
    for (int i = 0; i < kV; ++i) x[i] = -INFINITY;
    if (t >= a.T) return;
    const LT* p = static_cast<const LT*>(a.logits) + t * a.ld + e0;
    if (a.vec) {
        if (e0 >= a.E) return;
        if constexpr (sizeof(LT) == 4) {
            const float4 u = *reinterpret_cast<const float4*>(p), v = *reinterpret_cast<const float4*>(p + 4);
            x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(q[i] << 16);
                x[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kV; ++i)
        if (e0 + i < a.E) x[i] = static_cast<float>(p[i]);
}

// The choice again with keys in 64 bits (rare: kept apart from the registers of
// the ordinary path).
template <int LANES>
__device__ __noinline__ void choose_exactly(const RouteArgs& a, const float (&x)[kV], const float (&take)[kV],
                                            RouteShared& sh) {
    const int e0 = (threadIdx.x & 31) % LANES * kV;
    double s[kV], key[kV], by[kV];
    scores<LANES>(x, a.sigmoid, s);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
        const float b = a.bias && e0 + i < a.E ? a.bias[e0 + i] : 0.0f;
        const bool none = x[i] == -INFINITY || b == -INFINITY;
        key[i] = none ? -INFINITY : a.bias ? s[i] + static_cast<double>(b) : static_cast<double>(x[i]);
        by[i] = none ? -INFINITY : a.bias ? key[i] : s[i];
    }
    choose<LANES, double, false>(a, key, by, s, take, sh);
}

template <int LANES, typename LT>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const RouteArgs a) {
    __shared__ RouteShared sh;
    constexpr int ROWS = 32 / LANES;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, sub = lane % LANES, row = lane / LANES, e0 = sub * kV;
    const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kRouteWarps + w) * ROWS;
    if (t0 >= a.T) return;
    float x[kV], s[kV], key[kV], by[kV], take[kV];
    load_row<LT>(a, t0 + row, e0, x);
    // renormalised softmax weights are the softmax of the chosen logits
    const bool of_logits = a.renorm && !a.sigmoid, two = a.groups > 1 && a.group_top == 2;
    const bool scored = !of_logits || a.bias || two;
    if (scored) scores<LANES>(x, a.sigmoid, s);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
        if (!scored) s[i] = 0.0f;
        const float b = a.bias && e0 + i < a.E ? a.bias[e0 + i] : 0.0f;
        const bool none = x[i] == -INFINITY || b == -INFINITY;
        key[i] = none ? -INFINITY : a.bias ? s[i] + b : x[i];
        by[i] = none ? -INFINITY : a.bias ? key[i] : two ? s[i] : x[i];
        take[i] = of_logits ? (s[i] == s[i] ? x[i] : s[i]) : s[i];
    }
    if (a.bias || two) {
        if (__any_sync(~0u, choose<LANES, float, true>(a, key, by, s, take, sh))) choose_exactly<LANES>(a, x, take, sh);
    } else {
        choose<LANES, float, false>(a, key, by, s, take, sh);
    }
    // weights: the sums over a row's k in the order of the slots
    const int n = static_cast<int>(min(static_cast<int64_t>(ROWS), a.T - t0)) * a.k;
    for (int i = lane; i < n; i += 32) {
        const int r0 = i / a.k * a.k;
        const int id = sh.ids[w][i];
        float v = sh.v[w][i];
        if (of_logits) {
            float m = -INFINITY, z = 0.0f;
            for (int j = r0; j < r0 + a.k; ++j)
                if (sh.ids[w][j] >= 0) m = fmaxf(m, sh.v[w][j]);
            for (int j = r0; j < r0 + a.k; ++j)
                if (sh.ids[w][j] >= 0) z += expf(sh.v[w][j] - m);
            v = expf(v - m) / z;
        } else if (a.renorm) {
            float z = 0.0f;
            for (int j = r0; j < r0 + a.k; ++j)
                if (sh.ids[w][j] >= 0) z += sh.v[w][j];
            v /= z + 1e-20f;
        }
        a.ids[t0 * a.k + i] = id;
        a.weights[t0 * a.k + i] = id >= 0 ? v * a.scale : 0.0f;
    }
}

// Gradient.  With c = scale, g = dL/dw, and sums over the slots with an expert:
//   softmax                   dx_e = c s_e ([e chosen] g_e - sum_j g_j s_j)
//   softmax, renormalised     dx_j = c q_j (g_j - sum_i g_i q_i), q = softmax of the chosen
//   sigmoid                   dx_j = c g_j s_j (1 - s_j)
//   sigmoid, renormalised     dx_j = c (g_j - sum_i g_i v_i / D) / D s_j (1 - s_j), D = sum v + 1e-20
// and zero for the experts that were not chosen, in the last three.  A slot's
// term is computed by a lane and left in shared memory; every lane adds the terms
// of its own experts in the order of the slots.
template <int LANES, typename LT>
__global__ void __launch_bounds__(kRouteThreads) route_backward_kernel(const RouteArgs a) {
    __shared__ int32_t s_ids[kRouteWarps][256];
    __shared__ float s_x[kRouteWarps][256], s_g[kRouteWarps][256];
    constexpr int ROWS = 32 / LANES;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, sub = lane % LANES, row = lane / LANES, e0 = sub * kV;
    const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kRouteWarps + w) * ROWS;
    if (t0 >= a.T) return;
    const int64_t t = t0 + row;
    const bool all = !a.sigmoid && !a.renorm;
    float x[kV], s[kV];
    if (all) load_row<LT>(a, t, e0, x);
    const int n = static_cast<int>(min(static_cast<int64_t>(ROWS), a.T - t0)) * a.k;
    for (int i = lane; i < n; i += 32) {
        const int64_t r = t0 + i / a.k;
        const int j = i % a.k;
        const int id = a.ids_in[r * a.ldi + j];
        const bool on = id >= 0 && id < a.E;
        if (id >= a.E) atomicOr(a.err, ERR_ROUTE_EXPERT);
        s_ids[w][i] = on ? id : -1;
        s_x[w][i] = on ? static_cast<float>(static_cast<const LT*>(a.logits)[r * a.ld + id]) : 0.0f;
        s_g[w][i] = on ? a.grad[r * a.ldg + j] * a.scale : 0.0f;
    }
    __syncwarp();
    float dot = 0.0f;
    if (all) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kV; ++i) m = fmaxf(m, x[i]);
        m = seg_max<LANES>(m);
        if (m == -INFINITY) m = 0.0f;
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            s[i] = expf(x[i] - m);
            z += s[i];
        }
        z = seg_sum<LANES>(z);
        const float r = z == 0.0f ? 0.0f : 1.0f / z;
#pragma unroll
        for (int i = 0; i < kV; ++i) s[i] *= r;
        if (t < a.T)
            for (int j = sub; j < a.k; j += LANES)
                if (s_ids[w][row * a.k + j] >= 0) dot += s_g[w][row * a.k + j] * (expf(s_x[w][row * a.k + j] - m) * r);
        dot = seg_sum<LANES>(dot);
    } else {
        float d[8];  // a lane's slots: n <= 256
        int at = 0;
        for (int i = lane; i < n; i += 32, ++at) {
            const int r0 = i / a.k * a.k;
            float v = 0.0f;
            if (s_ids[w][i] >= 0) {
                const float g = s_g[w][i];
                if (a.sigmoid) {
                    const float e = expf(-fabsf(s_x[w][i])), q = 1.0f / (1.0f + e);
                    const float up = s_x[w][i] < 0.0f ? e * q : q, down = s_x[w][i] < 0.0f ? q : e * q;
                    v = g;
                    if (a.renorm) {
                        float z = 0.0f, p = 0.0f;
                        for (int j = r0; j < r0 + a.k; ++j)
                            if (s_ids[w][j] >= 0) {
                                const float f = expf(-fabsf(s_x[w][j]));
                                z += (s_x[w][j] < 0.0f ? f : 1.0f) / (1.0f + f);
                            }
                        z += 1e-20f;
                        for (int j = r0; j < r0 + a.k; ++j)
                            if (s_ids[w][j] >= 0) {
                                const float f = expf(-fabsf(s_x[w][j]));
                                p = fmaf(s_g[w][j], (s_x[w][j] < 0.0f ? f : 1.0f) / (1.0f + f) / z, p);
                            }
                        v = (g - p) / z;
                    }
                    v *= up * down;
                } else {
                    float m = -INFINITY, z = 0.0f, p = 0.0f;
                    for (int j = r0; j < r0 + a.k; ++j)
                        if (s_ids[w][j] >= 0) m = fmaxf(m, s_x[w][j]);
                    for (int j = r0; j < r0 + a.k; ++j)
                        if (s_ids[w][j] >= 0) z += expf(s_x[w][j] - m);
                    for (int j = r0; j < r0 + a.k; ++j)
                        if (s_ids[w][j] >= 0) p = fmaf(s_g[w][j], expf(s_x[w][j] - m) / z, p);
                    v = expf(s_x[w][i] - m) / z * (g - p);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j == at) d[j] = v;
        }
        __syncwarp();
        at = 0;
        for (int i = lane; i < n; i += 32, ++at)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j == at) s_g[w][i] = d[j];
        __syncwarp();
    }
    if (t >= a.T || e0 >= a.E) return;
    float sum[kV] = {};
    for (int j = 0; j < a.k; ++j) {
        const int id = s_ids[w][row * a.k + j];
        if (id < e0 || id >= e0 + kV) continue;
        const float g = s_g[w][row * a.k + j];
#pragma unroll
        for (int i = 0; i < kV; ++i) sum[i] += id == e0 + i ? g : 0.0f;
    }
    if (all)
#pragma unroll
        for (int i = 0; i < kV; ++i) sum[i] = s[i] * (sum[i] - dot);
    LT* p = static_cast<LT*>(a.grad_logits) + t * a.ldo + e0;
    if (a.ovec) {
        if constexpr (sizeof(LT) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(sum[0], sum[1], sum[2], sum[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
        } else {
            __nv_bfloat162 h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(sum[2 * i], sum[2 * i + 1]);
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kV; ++i)
        if (e0 + i < a.E) p[i] = static_cast<LT>(sum[i]);
}

// Lanes of a row: 8 experts each.
template <typename F>
void with_lanes(int E, F f) {
    if (E <= 8)
        f(std::integral_constant<int, 1>{});
    else if (E <= 16)
        f(std::integral_constant<int, 2>{});
    else if (E <= 32)
        f(std::integral_constant<int, 4>{});
    else if (E <= 64)
        f(std::integral_constant<int, 8>{});
    else if (E <= 128)
        f(std::integral_constant<int, 16>{});
    else
        f(std::integral_constant<int, 32>{});
}

aem_status check_route(const char* what, const aem_route_config* c, aem_dtype dtype, int64_t ld, int64_t T, int E) {
    AEM_REQUIRE(c != nullptr, "%s: config is NULL", what);
    AEM_REQUIRE(c->score == AEM_SCORE_SOFTMAX || c->score == AEM_SCORE_SIGMOID, "%s: bad score %d", what, (int)c->score);
    AEM_REQUIRE(dtype == AEM_F32 || dtype == AEM_BF16, "%s: bad dtype", what);
    AEM_REQUIRE(E >= 1 && E <= AEM_MAX_EXPERTS, "%s: E=%d outside [1, %d]", what, E, AEM_MAX_EXPERTS);
    AEM_REQUIRE(c->groups >= 1 && E % c->groups == 0, "%s: %d groups do not divide %d experts", what, c->groups, E);
    AEM_REQUIRE(c->top_groups >= 1 && c->top_groups <= c->groups, "%s: top_groups=%d outside [1, %d]", what,
                c->top_groups, c->groups);
    AEM_REQUIRE(c->group_top == 1 || c->group_top == 2, "%s: group_top=%d is not 1 or 2", what, c->group_top);
    AEM_REQUIRE(c->k >= 1 && c->k <= AEM_MAX_TOPK && c->k <= E / c->groups * c->top_groups,
                "%s: k=%d outside [1, min(%d, %d)]", what, c->k, AEM_MAX_TOPK, E / c->groups * c->top_groups);
    AEM_REQUIRE(c->scale == c->scale, "%s: scale is NaN", what);
    AEM_REQUIRE(ld >= 0, "%s: bad row stride", what);
    AEM_REQUIRE(T >= 0 && T < (1ll << 40) / E, "%s: T=%lld out of range", what, (long long)T);
    return AEM_OK;
}

RouteArgs route_args(const aem_route_config* c, const void* logits, aem_dtype dtype, int64_t ld, int64_t T, int E) {
    RouteArgs a{};
    a.logits = logits;
    a.ld = ld;
    a.T = T;
    a.E = E;
    a.k = c->k;
    a.groups = c->top_groups == c->groups ? 1 : c->groups;  // all kept: no groups
    a.top_groups = c->top_groups;
    a.group_top = c->group_top;
    a.size = E / c->groups;
    a.size_inv = (65536 + a.size - 1) / a.size;  // e * size_inv >> 16 == e / size for e < 256
    a.scale = c->scale;
    a.sigmoid = c->score == AEM_SCORE_SIGMOID;
    a.renorm = c->renormalize != 0;
    const int es = dtype == AEM_F32 ? 4 : 2;
    a.vec = E % kV == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld * es % 16 == 0;
    return a;
}

aem_status route_grid(const char* what, int64_t T, int rows, unsigned* blocks) {
    const int64_t n = (T + rows * kRouteWarps - 1) / (rows * kRouteWarps);
    AEM_REQUIRE(n < (1ll << 31), "%s: T=%lld out of range", what, (long long)T);
    *blocks = static_cast<unsigned>(n);
    return AEM_OK;
}

}  // namespace
}  // namespace aem

using aem::set_error;

extern "C" {

aem_status aem_route_tokens(const aem_route_config* config, const void* logits, aem_dtype dtype, int64_t ld,
                            int64_t T, int E, const float* bias, int32_t* ids, float* weights, void* stream) {
    AEM_TRY(aem::check_route("aem_route_tokens", config, dtype, ld, T, E));
    if (T == 0) return AEM_OK;
    AEM_REQUIRE(logits && ids && weights, "aem_route_tokens: NULL buffer");
    aem::RouteArgs a = aem::route_args(config, logits, dtype, ld, T, E);
    a.bias = bias;
    a.ids = ids;
    a.weights = weights;
    aem_status st = AEM_OK;
    aem::with_lanes(E, [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        unsigned blocks;
        st = aem::route_grid("aem_route_tokens", T, 32 / L, &blocks);
        if (st != AEM_OK) return;
        auto s = static_cast<cudaStream_t>(stream);
        if (dtype == AEM_F32)
            aem::route_kernel<L, float><<<blocks, aem::kRouteThreads, 0, s>>>(a);
        else
            aem::route_kernel<L, __nv_bfloat16><<<blocks, aem::kRouteThreads, 0, s>>>(a);
    });
    AEM_TRY(st);
    AEM_CHECK_LAUNCH();
    aem::count_launches(1);
    return AEM_OK;
}

aem_status aem_route_tokens_backward(const aem_route_config* config, const float* grad_weights, int64_t ldg,
                                     const void* logits, aem_dtype dtype, int64_t ld, int64_t T, int E,
                                     const int32_t* ids, int64_t ldi, void* grad_logits, int64_t ldo, void* stream) {
    AEM_TRY(aem::check_route("aem_route_tokens_backward", config, dtype, ld, T, E));
    AEM_REQUIRE(ldg >= 0 && ldi >= 0 && ldo >= E, "aem_route_tokens_backward: bad row stride");
    if (T == 0) return AEM_OK;
    AEM_REQUIRE(grad_weights && logits && ids && grad_logits, "aem_route_tokens_backward: NULL buffer");
    aem::RouteArgs a = aem::route_args(config, logits, dtype, ld, T, E);
    a.grad = grad_weights;
    a.ldg = ldg;
    a.ids_in = ids;
    a.ldi = ldi;
    a.grad_logits = grad_logits;
    a.ldo = ldo;
    a.err = aem::device_error_word(aem::current_device());
    if (!a.err) {
        set_error("aem_route_tokens_backward: no device error word");
        return AEM_ENOMEM;
    }
    a.ovec = E % aem::kV == 0 && reinterpret_cast<uintptr_t>(grad_logits) % 16 == 0 &&
             ldo * (dtype == AEM_F32 ? 4 : 2) % 16 == 0;
    aem_status st = AEM_OK;
    aem::with_lanes(E, [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        unsigned blocks;
        st = aem::route_grid("aem_route_tokens_backward", T, 32 / L, &blocks);
        if (st != AEM_OK) return;
        auto s = static_cast<cudaStream_t>(stream);
        if (dtype == AEM_F32)
            aem::route_backward_kernel<L, float><<<blocks, aem::kRouteThreads, 0, s>>>(a);
        else
            aem::route_backward_kernel<L, __nv_bfloat16><<<blocks, aem::kRouteThreads, 0, s>>>(a);
    });
    AEM_TRY(st);
    AEM_CHECK_LAUNCH();
    aem::count_launches(1);
    return AEM_OK;
}

}  // extern "C"
