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
// on their error (route_bounds.h); wherever two keys that decide the order (neighbours
// among the k + 1 largest, the last group kept and the first dropped) are nearer than
// their bounds, the warp decides with keys in 64 bits: those of the chosen experts where
// only their order is open (with normally distributed logits and 256 experts, top-8,
// sigmoid with a bias, a row in 2400), else of all of them (an eighth of those rows; a
// call with such a row takes 5 us longer, and when all took that way 16383 rows took
// 38 us instead of 32).  Logits themselves need no bound.
//
// A row lies across LANES lanes, 8 neighbouring experts a lane, so a lane's order
// is the experts' and up to 32 rows share a warp.  A lane sorts its experts once
// and leaves them in shared memory; a choice is then the maximum of the lanes'
// first ones, and the lane that had it moves on to its next (looking through all 8
// again for every choice took 29 us where this takes 24: 16384 rows of 256, top-8).
// Groups of whole lanes take their two largest from the sorted lists; others are
// read through shared memory.  What has to be moved is T*E logits and 8 T*k bytes,
// but a choice of k costs k warp-wide maxima, and those bound it.  256 float32 logits,
// top-8: 1 row 3.6 us softmax and 4.9 sigmoid with bias and 8 groups, 16383 rows 23
// and 32 us, 262144 rows 307 and 447 us (0.9 and 0.6 TB/s of logits).
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "route_bounds.h"
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
    int E, k, groups, top_groups, group_top, size;  // size: experts of a group
    int size_inv, k_inv;                            // n * inv >> 16 == n / (size, k) for n < 256
    int sigmoid, renorm, vec, bvec, ovec;  // rows, the bias, gradients can be moved in 16 bytes
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
// (a NaN wins where a warp is one row; every caller's results are NaN then anyway, or
// none comes here)
template <int LANES>
__device__ __forceinline__ float seg_max(float v) {
    if constexpr (LANES == 32) return value_of(__reduce_max_sync(~0u, rank_of(v)));
    return seg_reduce<LANES>(v, [](float a, float b) { return fmaxf(a, b); });
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

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
// (1 <= b <= 2; a reciprocal of 2 ulp, and a step that takes the quotient's rest)
__device__ __forceinline__ float quotient(float a, float b) {
    const float r = __fdividef(1.0f, b), q = a * r;
    return fmaf(fmaf(-q, b, a), r, q);
}
__device__ __forceinline__ double quotient(double a, double b) { return a / b; }

// Scores of a lane's experts; a row without any finite logit has zeros.
template <int LANES, typename F>
__device__ __forceinline__ void scores(const float (&x)[kV], bool sigmoid, F (&s)[kV]) {
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const F t = exp_of(-fabs(static_cast<F>(x[i])));
            s[i] = quotient(x[i] < 0.0f ? t : F(1), F(1) + t);
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

// A warp's rows.
struct RouteShared {
    unsigned long long list[kRouteWarps][kV][32];  // the lanes' experts, sorted: ranks and indices
    float take[kRouteWarps][256];                  // what becomes of a chosen expert
    int32_t ids[kRouteWarps][256];                 // [row][k]: LANES * 8 >= k
    double value[kRouteWarps][32];                 // of groups of whole lanes, chosen exactly
    uint32_t rank[kRouteWarps][256 + 32];          // [row][k + 1]: of the chosen and of the next one
};
// Groups that are not whole lanes (or not a power of two of them): values of the
// experts and of the groups.
struct GroupShared {
    double by[kRouteWarps][256], value[kRouteWarps][256];
};

// A rank and its expert's place in the lane; larger ones come first.
__device__ __forceinline__ unsigned long long entry_of(uint32_t rank, int i) {
    return static_cast<unsigned long long>(rank) << 32 | static_cast<uint32_t>(7 - i);
}
template <typename T>
__device__ __forceinline__ void order2(T& a, T& b) {
    const T hi = max(a, b), lo = min(a, b);
    a = hi, b = lo;
}
// 8 values in falling order: 19 exchanges.
template <typename T>
__device__ __forceinline__ void sort8(T (&v)[8]) {
    order2(v[0], v[1]), order2(v[2], v[3]), order2(v[4], v[5]), order2(v[6], v[7]);
    order2(v[0], v[2]), order2(v[1], v[3]), order2(v[4], v[6]), order2(v[5], v[7]);
    order2(v[1], v[2]), order2(v[5], v[6]), order2(v[0], v[4]), order2(v[3], v[7]);
    order2(v[1], v[5]), order2(v[2], v[6]);
    order2(v[1], v[4]), order2(v[3], v[6]);
    order2(v[2], v[4]), order2(v[3], v[5]);
    order2(v[3], v[4]);
}

// Which of the row's groups stay, for any size: keys of the others become -inf.
// Returns whether the last that stayed and the first that did not are nearer than
// `e`, the slack of the values.
template <int LANES, typename F>
__device__ __forceinline__ bool keep_groups(const RouteArgs& a, F (&key)[kV], const F (&by)[kV], float e, void* vals,
                                            void* values) {
    using U = typename Rank<F>::type;
    const int lane = threadIdx.x & 31, sub = lane % LANES, row = lane / LANES;
    F* val = static_cast<F*>(vals) + row * LANES * kV;
    F* gv = static_cast<F*>(values) + row * a.groups;
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
    bool near = false;
    if constexpr (sizeof(F) == 4) {
        least = -seg_max<LANES>(-least);
        most = seg_max<LANES>(most);
        near = e > 0.0f && most > -INFINITY && !(least - most > e);
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
        if (!(bits >> (g & 31) & 1)) key[i] = -INFINITY;
    }
    return near;
}

// The same for groups of whole lanes, `span` (a power of two) of them, from the
// lane's two largest values: returns whether the lane's group stays.
template <int LANES, typename F>
__device__ __forceinline__ bool keep_lanes(const RouteArgs& a, int span, F first, F second, float e, bool& near) {
    using U = typename Rank<F>::type;
    const int lane = threadIdx.x & 31, base = lane & ~(LANES - 1), mine = lane & ~(span - 1);
    U p = rank_of(first), q = a.group_top == 2 ? rank_of(second) : 0;
    for (int o = 1; o < span; o <<= 1) {
        const U r = __shfl_xor_sync(~0u, p, o), t = __shfl_xor_sync(~0u, q, o);
        q = max(max(q, t), min(p, r));
        p = max(p, r);
    }
    F v = value_of(p);
    if (a.group_top == 2 && q) v += value_of(q);
    const U rank = rank_of(v);
    int before = 0;
    for (int g = 0; g < a.groups; ++g) {
        const int at = base + g * span;
        const U other = __shfl_sync(~0u, rank, at);
        before += other > rank || (other == rank && at < mine);
    }
    const bool stays = before < a.top_groups && lane - base < a.groups * span;
    if constexpr (sizeof(F) == 4) {
        const bool real = lane - base < a.groups * span;
        const float least = -seg_max<LANES>(stays && v == v ? -v : -INFINITY);
        const float most = seg_max<LANES>(real && !stays ? v : -INFINITY);
        near |= e > 0.0f && most > -INFINITY && !(least - most > e);
    }
    return stays;
}

// The k largest of the lanes' sorted lists in shared memory, `on` whether the lane
// takes part; their ids and, with a bound on the keys' errors (CERT), what is nearer
// than that and so open.  `score` bounds the errors of
// all the row's scores.
template <int LANES, bool CERT>
__device__ __forceinline__ int extract(const RouteArgs& a, bool on, float score, RouteShared& sh) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, sub = lane % LANES, row = lane / LANES;
    const unsigned segment = (LANES == 32 ? ~0u : (1u << LANES) - 1) << (row * LANES);
    unsigned long long head = on ? sh.list[w][0][lane] : 0;
    // of the lane's list; past its end for a lane of a dropped group, which has the
    // row's maximum too once nothing is left (rank 0) and must not move on
    int next = on ? 1 : kV;
    uint32_t* ranks = &sh.rank[w][row * (a.k + 1)];
    int32_t* ids = &sh.ids[w][row * a.k];
    for (int j = 0; j < a.k + (CERT ? 1 : 0); ++j) {
        const uint32_t rank = static_cast<uint32_t>(head >> 32);
        const uint32_t m = seg_max<LANES>(rank);
        if (lane == __ffs(__ballot_sync(~0u, rank == m) & segment) - 1) {
            const int id = m ? sub * kV + 7 - static_cast<int>(head & 7) : -1;
            if (j < a.k) ids[j] = id;
            if constexpr (CERT) {
                ranks[j] = m;
            }
            head = next < kV ? sh.list[w][next][lane] : 0;
            ++next;
        }
    }
    __syncwarp();
    int open = 0;
    if constexpr (CERT) {
        const float* take = &sh.take[w][row * LANES * kV];
        for (int j = sub; j < a.k; j += LANES) {
            if (ranks[j + 1] == 0) break;
            const float key = value_of(ranks[j]), then = value_of(ranks[j + 1]);
            const float slack = key_slack(a.sigmoid, take[ids[j]], key);
            if (j + 1 == a.k)
                open |= open_at_end(key, slack, then, score);
            else if (!(key - then > slack + key_slack(a.sigmoid, take[ids[j + 1]], then)))
                open |= OPEN_ORDER;
        }
    }
    return open;
}

// The chosen experts in the order of their keys in 64 bits, where it is known that
// they are the ones: a slot a lane (k <= LANES, sigmoid scores with a bias).
template <int LANES, typename LT>
__device__ __noinline__ void order_exactly(const RouteArgs& a, int64_t t0, int32_t* ids) {
    const int lane = threadIdx.x & 31, sub = lane % LANES, row = lane / LANES;
    const bool slot = sub < a.k && t0 + row < a.T;
    ids += row * a.k;
    const int id = slot ? ids[sub] : -1;
    unsigned long long rank = 0;
    if (id >= 0) {
        const double v = static_cast<float>(static_cast<const LT*>(a.logits)[(t0 + row) * a.ld + id]), t = exp(-fabs(v));
        rank = rank_of((v < 0.0 ? t : 1.0) / (1.0 + t) + static_cast<double>(a.bias[id]));
    }
    int at = 0;
    for (int i = 0; i < a.k; ++i) {
        const unsigned long long other = __shfl_sync(~0u, rank, row * LANES + i);
        const int that = __shfl_sync(~0u, id, row * LANES + i);
        at += other > rank || (other == rank && (that < id || (that == id && i < sub)));
    }
    __syncwarp();
    if (slot) ids[at] = id;
    __syncwarp();
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

// The choice again with keys in 64 bits.  It is rare and apart from the registers of
// the ordinary path, so it fetches the logits again: handed over they would lie in
// memory for every warp (262144 x 256 sigmoid with a bias: 407 us, so 397).
template <int LANES, typename LT>
__device__ __noinline__ void choose_exactly(const RouteArgs& a, int64_t t0, RouteShared& sh, double* values) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, sub = lane % LANES, row = lane / LANES, e0 = sub * kV;
    const unsigned segment = (LANES == 32 ? ~0u : (1u << LANES) - 1) << (row * LANES);
    float x[kV];
    load_row<LT>(a, t0 + row, e0, x);
    double s[kV], key[kV], by[kV];
    scores<LANES>(x, a.sigmoid, s);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
        const float b = a.bias && e0 + i < a.E ? a.bias[e0 + i] : 0.0f;
        const bool none = x[i] == -INFINITY || b == -INFINITY;
        key[i] = none ? -INFINITY : a.bias ? s[i] + static_cast<double>(b) : static_cast<double>(x[i]);
        by[i] = none ? -INFINITY : a.bias ? key[i] : a.group_top == 2 ? s[i] : key[i];
    }
    // the lists are no longer needed
    if (a.groups > 1) keep_groups<LANES, double>(a, key, by, 0.0f, &sh.list[w][0][0], values);
    unsigned long long u[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) u[i] = rank_of(key[i]);
    for (int j = 0; j < a.k; ++j) {
        unsigned long long best = 0;
#pragma unroll
        for (int i = 0; i < kV; ++i) best = max(best, u[i]);
        const unsigned long long m = seg_max<LANES>(best);
        const int owner = __ffs(__ballot_sync(~0u, best == m) & segment) - 1;
        if (lane == owner) {
            int at = kV;
#pragma unroll
            for (int i = kV - 1; i >= 0; --i) at = u[i] == m ? i : at;
#pragma unroll
            for (int i = 0; i < kV; ++i) u[i] = i == at ? 0 : u[i];
            sh.ids[w][row * a.k + j] = m ? e0 + at : -1;
        }
        __syncwarp();
    }
}

// Any groups that are not whole lanes go through shared memory (ANY).
template <int LANES, typename LT, bool ANY>
__global__ void __launch_bounds__(kRouteThreads, 4) route_kernel(const RouteArgs a) {
    extern __shared__ uint8_t dynamic[];
    __shared__ RouteShared sh;
    auto& gsh = *reinterpret_cast<GroupShared*>(dynamic);  // ANY
    constexpr int ROWS = 32 / LANES;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, sub = lane % LANES, row = lane / LANES, e0 = sub * kV;
    const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kRouteWarps + w) * ROWS;
    if (t0 >= a.T) return;
    float x[kV], s[kV], key[kV];
    load_row<LT>(a, t0 + row, e0, x);
    // renormalised softmax weights are the softmax of the chosen logits
    const bool of_logits = a.renorm && !a.sigmoid, two = a.groups > 1 && a.group_top == 2;
    const bool scored = !of_logits || a.bias || two;
    if (scored) scores<LANES>(x, a.sigmoid, s);
    bool nan = false;  // a NaN among the scores is one in all of them
    float b[kV] = {};
    if (a.bvec && e0 < a.E) {
        const float4 u = *reinterpret_cast<const float4*>(a.bias + e0), v = *reinterpret_cast<const float4*>(a.bias + e0 + 4);
        b[0] = u.x, b[1] = u.y, b[2] = u.z, b[3] = u.w, b[4] = v.x, b[5] = v.y, b[6] = v.z, b[7] = v.w;
    } else if (a.bias) {
#pragma unroll
        for (int i = 0; i < kV; ++i) b[i] = e0 + i < a.E ? a.bias[e0 + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kV; ++i) {
        if (!scored) s[i] = 0.0f;
        const bool none = x[i] == -INFINITY || b[i] == -INFINITY;
        key[i] = none ? -INFINITY : a.bias ? s[i] + b[i] : x[i];
        nan |= s[i] != s[i];
    }
    const bool sure = !a.bias && !two;  // keys are the logits themselves
    float e = 0.0f;                     // slack of a group's value
    // the bound of any score's error in the row
    auto any_score = [&]() {
        float top = 0.0f;
        if (!a.sigmoid) {
#pragma unroll
            for (int i = 0; i < kV; ++i) top = fmaxf(top, s[i]);
            // (none is negative: their bits have the same order)
            top = __uint_as_float(seg_max<LANES>(__float_as_uint(top)));
        }
        return score_slack(a.sigmoid, top);
    };
    if (!sure && a.groups > 1) {
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < kV; ++i)
            if (key[i] != -INFINITY) largest = fmaxf(largest, fabsf(a.bias ? key[i] : s[i]));
        e = group_slack(any_score(), __uint_as_float(seg_max<LANES>(__float_as_uint(largest))));
    }
    bool near = false, on = true;
    if constexpr (ANY) {
        float by[kV];
#pragma unroll
        for (int i = 0; i < kV; ++i) by[i] = key[i] == -INFINITY ? -INFINITY : a.bias ? key[i] : two ? s[i] : key[i];
        near = keep_groups<LANES, float>(a, key, by, e, gsh.by[w], gsh.value[w]);
    }
    unsigned long long v[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] = entry_of(rank_of(key[i]), i);
    // what becomes of an expert: its score, for the bound and for the weights (a
    // logit where they are the softmax of the chosen logits)
#pragma unroll
    for (int i = 0; i < kV; i += 4)
        *reinterpret_cast<float4*>(&sh.take[w][lane * kV + i]) =
            of_logits && !a.bias && !nan ? make_float4(x[i], x[i + 1], x[i + 2], x[i + 3])
                                         : make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
    sort8(v);
#pragma unroll
    for (int i = 0; i < kV; ++i) sh.list[w][i][lane] = v[i];
    __syncwarp();
    if (!ANY && a.groups > 1) {
        float first = value_of(static_cast<uint32_t>(v[0] >> 32)), second = value_of(static_cast<uint32_t>(v[1] >> 32));
        if (!a.bias && two) {  // values are scores, in the same order
            const float* mine = &sh.take[w][lane * kV];
            if (of_logits && !nan) {
                // (their logits lie there; the scores are in registers)
                float p = -INFINITY, q = -INFINITY;
                const int i0 = 7 - static_cast<int>(v[0] & 7), i1 = 7 - static_cast<int>(v[1] & 7);
#pragma unroll
                for (int i = 0; i < kV; ++i) p = i == i0 ? s[i] : p, q = i == i1 ? s[i] : q;
                first = first == -INFINITY ? first : p;
                second = second == -INFINITY ? second : q;
            } else {
                first = first == -INFINITY ? first : mine[7 - static_cast<int>(v[0] & 7)];
                second = second == -INFINITY ? second : mine[7 - static_cast<int>(v[1] & 7)];
            }
        }
        on = keep_lanes<LANES, float>(a, a.size / kV, first, second, e, near);
    }
    int open = near ? OPEN_SET : 0;
    if (a.bias) {
        open |= extract<LANES, true>(a, on, any_score(), sh);
    } else {
        extract<LANES, false>(a, on, 0.0f, sh);
    }
    int decide = 0;
    if (!sure) {
        // (Lanes leave the comparisons one after the other.  A reduction of the bits, put
        // right behind them by the compiler, did not see all lanes in rows of 8 experts.)
        __syncwarp();
        if (__any_sync(~0u, open & (OPEN_ORDER | OPEN_SET)))
            decide = to_decide(OPEN_ORDER | (__any_sync(~0u, open & OPEN_SET) ? OPEN_SET : 0) |
                               (__any_sync(~0u, open & OPEN_BEHIND) ? OPEN_BEHIND : 0));
    }
    if (decide == 1 && a.sigmoid && a.k <= LANES)
        order_exactly<LANES, LT>(a, t0, sh.ids[w]);
    else if (decide)
        choose_exactly<LANES, LT>(a, t0, sh, ANY ? gsh.value[w] : sh.value[w]);
    if (of_logits && a.bias) {  // the scores have been compared
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kV; ++i) sh.take[w][lane * kV + i] = nan ? s[i] : x[i];
        __syncwarp();
    }
    // weights: the sums over a row's k in the order of the slots
    const int n = static_cast<int>(min(static_cast<int64_t>(ROWS), a.T - t0)) * a.k;
    for (int i = lane; i < n; i += 32) {
        const int r = i * a.k_inv >> 16, r0 = r * a.k;
        const float* take = &sh.take[w][r * LANES * kV];
        const int id = sh.ids[w][i];
        float v = id >= 0 ? take[id] : 0.0f;
        if (of_logits) {
            float m = -INFINITY, z = 0.0f;
            for (int j = r0; j < r0 + a.k; ++j)
                if (sh.ids[w][j] >= 0) m = fmaxf(m, take[sh.ids[w][j]]);
            for (int j = r0; j < r0 + a.k; ++j)
                if (sh.ids[w][j] >= 0) z += expf(take[sh.ids[w][j]] - m);
            v = expf(v - m) / z;
        } else if (a.renorm) {
            float z = 0.0f;
            for (int j = r0; j < r0 + a.k; ++j)
                if (sh.ids[w][j] >= 0) z += take[sh.ids[w][j]];
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
// and zero for the experts that were not chosen, in the last three.  A lane has a
// slot: it leaves what the row's sums need in shared memory, takes the sums from
// there in the slots' order, and leaves its term at its expert; of slots with the
// same expert the first one adds the others' terms.  Then every lane writes its own 8
// experts, or, where the chosen ones alone have a gradient, pieces of whole lines.  There
// a warp has four rows, so that its lanes have slots: 16383 rows of 256 float32, top-8,
// in 6.3 us, one row a warp 9.8.  262144 such rows take 90 us (2.9 TB/s written, 0.8
// read), with the sums over all experts 173 us (3.1 TB/s), 55 to 60% of what a copy
// reaches: a warp's ids, the logits that they name, the sums and the stores follow one
// another, and it does this once.
template <int LANES, typename LT, int RB>
__global__ void __launch_bounds__(kRouteThreads / (RB > 1 ? 2 : 1)) route_backward_kernel(const RouteArgs a) {
    constexpr int WARPS = kRouteWarps / (RB > 1 ? 2 : 1), ROWS = 32 / LANES * RB;  // RB rows of a lane
    __shared__ int32_t s_ids[WARPS][256];
    __shared__ float s_p[WARPS][256], s_g[WARPS][256], s_term[WARPS][256];
    __shared__ __align__(16) float s_row[WARPS][256 * RB];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, sub = lane % LANES, row = lane / LANES, e0 = sub * kV;
    const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * WARPS + w) * ROWS;
    if (t0 >= a.T) return;
    const int64_t t = t0 + row;
    const bool all = RB == 1 && !a.sigmoid && !a.renorm;
    const int n = static_cast<int>(min(static_cast<int64_t>(ROWS), a.T - t0)) * a.k;
    float s[kV], m = 0.0f, r = 0.0f;
    if (all) {
        float x[kV], z = 0.0f;
        load_row<LT>(a, t, e0, x);
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kV; ++i) m = fmaxf(m, x[i]);
        m = seg_max<LANES>(m);
        if (m == -INFINITY) m = 0.0f;
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            s[i] = expf(x[i] - m);
            z += s[i];
        }
        z = seg_sum<LANES>(z);
        r = z == 0.0f ? 0.0f : 1.0f / z;
#pragma unroll
        for (int i = 0; i < kV; ++i) s[i] *= r;
    }
#pragma unroll
    for (int i = 0; i < kV * RB; i += 4)
        *reinterpret_cast<float4*>(&s_row[w][lane * 4 + i * 32]) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // a slot's id, gradient and score (softmax, renormalised: its logit)
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + lane, q = min(i, n - 1) * a.k_inv >> 16;
        // the row's largest logit and its sum, from its lanes
        const float mq = __shfl_sync(~0u, m, q * LANES), rq = __shfl_sync(~0u, r, q * LANES);
        if (i >= n) continue;
        const int id = a.ids_in[(t0 + q) * a.ldi + i - q * a.k];
        const float g = a.grad[(t0 + q) * a.ldg + i - q * a.k] * a.scale;
        const bool on = id >= 0 && id < a.E;
        if (id >= a.E) atomicOr(a.err, ERR_ROUTE_EXPERT);
        const float x = on ? static_cast<float>(static_cast<const LT*>(a.logits)[(t0 + q) * a.ld + id]) : 0.0f;
        s_ids[w][i] = on ? id : -1;
        s_g[w][i] = on ? g : 0.0f;
        if (a.sigmoid) {
            const float e = expf(-fabsf(x)), f = 1.0f / (1.0f + e);
            s_p[w][i] = on ? (x < 0.0f ? e * f : f) : 0.0f;
            s_term[w][i] = x < 0.0f ? f : e * f;  // 1 - s
        } else {
            s_p[w][i] = !on ? (all ? 0.0f : -INFINITY) : all ? expf(x - mq) * rq : x;
        }
    }
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
        const int j0 = (i * a.k_inv >> 16) * a.k, j1 = j0 + a.k;
        const float g = s_g[w][i], p = s_p[w][i];
        if (a.sigmoid) {
            float v = g;
            if (a.renorm) {
                float z = 0.0f, sum = 0.0f;
                for (int j = j0; j < j1; ++j) z += s_p[w][j];
                z += 1e-20f;
                const float f = 1.0f / z;
                for (int j = j0; j < j1; ++j) sum = fmaf(s_g[w][j], s_p[w][j] * f, sum);
                v = (g - sum) * f;
            }
            s_term[w][i] *= v * p;
        } else if (a.renorm) {
            float top = -INFINITY, z = 0.0f, sum = 0.0f;
            for (int j = j0; j < j1; ++j) top = fmaxf(top, s_p[w][j]);
            if (top == -INFINITY) top = 0.0f;
            for (int j = j0; j < j1; ++j) {
                const float q = expf(s_p[w][j] - top);
                z += q;
                sum = fmaf(s_g[w][j], q, sum);
            }
            s_term[w][i] = expf(p - top) / z * (g - sum / z);
        } else {
            s_term[w][i] = g;
        }
    }
    float dot = 0.0f;
    if (all) {
        if (t < a.T)
            for (int j = sub; j < a.k; j += LANES) dot = fmaf(s_g[w][row * a.k + j], s_p[w][row * a.k + j], dot);
        dot = seg_sum<LANES>(dot);
    }
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
        const int q = i * a.k_inv >> 16, id = s_ids[w][i], j0 = q * a.k;
        bool first = id >= 0;
        float v = 0.0f;
        for (int j = j0; j < j0 + a.k; ++j) {
            const bool same = s_ids[w][j] == id;
            first &= !(same && j < i);
            v += same ? s_term[w][j] : 0.0f;
        }
        if (first) s_row[w][q * LANES * kV + id] = v;
    }
    __syncwarp();
    if (!all && sizeof(LT) == 4 && a.ovec) {  // nothing is in registers: whole lines at once
#pragma unroll
        for (int q = 0; q < RB; ++q) {
            const int64_t t = t0 + q * (32 / LANES) + row;
            if (t >= a.T) return;
#pragma unroll
            for (int e = sub * 4; e < LANES * kV; e += LANES * 4)
                if (e < a.E)
                    *reinterpret_cast<float4*>(static_cast<float*>(a.grad_logits) + t * a.ldo + e) =
                        *reinterpret_cast<const float4*>(&s_row[w][q * 256 + row * LANES * kV + e]);
        }
        return;
    }
    if (e0 >= a.E) return;
#pragma unroll
    for (int q = 0; q < RB; ++q) {
        const int64_t t = t0 + q * (32 / LANES) + row;
        if (t >= a.T) return;
        float sum[kV];
#pragma unroll
        for (int i = 0; i < kV; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(&s_row[w][q * 256 + lane * kV + i]);
            sum[i] = v.x, sum[i + 1] = v.y, sum[i + 2] = v.z, sum[i + 3] = v.w;
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
            continue;
        }
#pragma unroll
        for (int i = 0; i < kV; ++i)
            if (e0 + i < a.E) p[i] = static_cast<LT>(sum[i]);
    }
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
    a.size_inv = (65536 + a.size - 1) / a.size;
    a.k_inv = (65536 + a.k - 1) / a.k;
    a.scale = c->scale;
    a.sigmoid = c->score == AEM_SCORE_SIGMOID;
    a.renorm = c->renormalize != 0;
    const int es = dtype == AEM_F32 ? 4 : 2;
    a.vec = E % kV == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld * es % 16 == 0;
    return a;
}

aem_status route_grid(const char* what, int64_t T, int rows, int warps, unsigned* blocks) {
    const int64_t n = (T + rows * warps - 1) / (rows * warps);
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
    a.bvec = bias && E % aem::kV == 0 && reinterpret_cast<uintptr_t>(bias) % 16 == 0;
    a.ids = ids;
    a.weights = weights;
    aem_status st = AEM_OK;
    aem::with_lanes(E, [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        unsigned blocks;
        st = aem::route_grid("aem_route_tokens", T, 32 / L, aem::kRouteWarps, &blocks);
        if (st != AEM_OK) return;
        auto s = static_cast<cudaStream_t>(stream);
        const int span = a.size / aem::kV;
        const bool any = a.groups > 1 && (a.size % aem::kV != 0 || (span & (span - 1)) != 0);
        auto go = [&](auto kern, auto any_groups) {
            constexpr bool ANY = decltype(any_groups)::value;
            if constexpr (ANY) {
                static std::atomic<uint64_t> kernels[2];  // per dtype (the kernels have one type), a bit per
                auto& ready = kernels[dtype];             // device: the shared memory opt-in is done
                const uint64_t bit = 1ull << (aem::current_device() & 63);
                if (!(ready.load(std::memory_order_relaxed) & bit)) {
                    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                               static_cast<int>(sizeof(aem::GroupShared)));
                    if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
                }
            }
            kern<<<blocks, aem::kRouteThreads, ANY ? sizeof(aem::GroupShared) : 0, s>>>(a);
        };
        const std::true_type yes;
        const std::false_type no;
        if (dtype == AEM_F32)
            any ? go(aem::route_kernel<L, float, true>, yes) : go(aem::route_kernel<L, float, false>, no);
        else
            any ? go(aem::route_kernel<L, __nv_bfloat16, true>, yes) : go(aem::route_kernel<L, __nv_bfloat16, false>, no);
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
        auto s = static_cast<cudaStream_t>(stream);
        auto go = [&](auto rows) {
            constexpr int RB = decltype(rows)::value;
            st = aem::route_grid("aem_route_tokens_backward", T, 32 / L * RB, aem::kRouteWarps / (RB > 1 ? 2 : 1), &blocks);
            if (st != AEM_OK) return;
            const int threads = aem::kRouteThreads / (RB > 1 ? 2 : 1);
            if (dtype == AEM_F32)
                aem::route_backward_kernel<L, float, RB><<<blocks, threads, 0, s>>>(a);
            else
                aem::route_backward_kernel<L, __nv_bfloat16, RB><<<blocks, threads, 0, s>>>(a);
        };
        // four rows a warp; with softmax scores of all experts a row's are in registers
        constexpr int RB = L == 32 ? 4 : L == 16 ? 2 : 1;
        if (a.sigmoid || a.renorm)
            go(std::integral_constant<int, RB>{});
        else
            go(std::integral_constant<int, 1>{});
    });
    AEM_TRY(st);
    AEM_CHECK_LAUNCH();
    aem::count_launches(1);
    return AEM_OK;
}

}  // extern "C"
