// Token dispatch and combine around expert products, and their gradients.
//
// A unit u = t*k + j is slot j of token t with expert id e = ids[t, j]; ids
// below 0 mean no expert.  The sort is a stable counting sort of the units by
// expert (units of one expert stay in increasing u):
//   starts[e]  = number of units with an expert below e
//   row_of[u]  = starts[e] + number of units v < u with the same expert
//   unit_of[row_of[u]] = u
// dispatch            rows[row_of[t, j]]  = x[t]
// dispatch, backward  grad_x[t]           = sum_j grad_rows[row_of[t, j]]
// combine             out[t]              = sum_j w[t, j] rows[row_of[t, j]]
// combine, backward   grad_rows[row_of[t, j]] = w[t, j] grad_out[t]
//                     grad_w[t, j]            = <grad_out[t], rows[row_of[t, j]]>
// Sums run in float32 in increasing j (over d: a fixed tree), and no kernel
// uses floating atomics, so results do not change from call to call.  All of
// it is bound by memory: every row crosses HBM once in each direction that
// the formula names.  16384 tokens of 2048 bf16, 6 of 64 experts: dispatch 86.5
// us (5.4 TB/s, six sevenths of it writes), combine 73 (6.4 TB/s), its backward
// pass for 8191 tokens 75.5 (5.6 TB/s); for one token a call is its launch (2.9
// us on the device).
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "runtime.h"

namespace aem {

namespace {

constexpr int kThreads = 256, kWarps = 8;
// Units that one block ranks: 8 per thread.  Batches of at most kFusedUnits
// are sorted again by every block of the moving kernel, one launch instead of
// three: 48 units of 2048 bf16 3.4 us (three kernels 6.1), 1024 units of 4096
// 7.9 (10.5).
constexpr int kBlockUnits = 2048, kFusedUnits = 1024;

struct Ids {
    const int32_t* p;
    int64_t st, sk;  // element strides of tokens and slots
    int k, E;
};

// Expert of unit u, or E for none.  An id of E or more is reported.
__device__ __forceinline__ int unit_expert(const Ids& ids, int64_t u, int* err) {
    const uint32_t t = static_cast<uint32_t>(u) / static_cast<uint32_t>(ids.k);  // u < 2^31
    const int id = ids.p[t * ids.st + (u - t * ids.k) * ids.sk];
    if (id >= ids.E) atomicOr(err, ERR_ROUTE_EXPERT);
    return id >= 0 && id < ids.E ? id : ids.E;
}

// Exclusive scan over the block's 256 threads; *total receives the sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(~0u, s, o);
        if (lane >= o) s += n;
    }
    if (lane == 31) warp_sums[w] = s;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        const int x = warp_sums[i];
        if (i < w) before += x;
        all += x;
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

struct SortSmem {
    int hist[kWarps][AEM_MAX_EXPERTS];
    int warp_sums[kWarps];
};

// Ranks units [u0, u0 + n) of the block (n <= 32 * kWarps * ITERS): warp w
// owns a contiguous range, and inside 32 units the lanes with equal experts
// find each other by a warp match, so ranks follow the unit order.
// `first(e)` gives the row of the block's first unit of expert e.
// key[i] = expert (E: none) and row[i] of unit
// u0 + w*32*iters + 32*i + lane; returns iters.
template <int ITERS, typename First>
__device__ __forceinline__ int rank_units(const Ids& ids, int64_t u0, int n, SortSmem& sm,
                                          int (&key)[ITERS], int (&row)[ITERS], int* err,
                                          First first) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int iters = (n + 32 * kWarps - 1) / (32 * kWarps);
    for (int i = threadIdx.x; i < kWarps * AEM_MAX_EXPERTS; i += kThreads) (&sm.hist[0][0])[i] = 0;
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int l = (w * iters + i) * 32 + lane;
        key[i] = i < iters && l < n ? unit_expert(ids, u0 + l, err) : ids.E;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        row[i] = -1;
        if (i >= iters) continue;
        const unsigned same = __match_any_sync(~0u, key[i]);
        const unsigned below = same & ((1u << lane) - 1);
        if (key[i] < ids.E) row[i] = sm.hist[w][key[i]] + __popc(below);
        __syncwarp();
        if (key[i] < ids.E && below == 0) sm.hist[w][key[i]] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    int mine = 0;
    if (threadIdx.x < ids.E)
        for (int i = 0; i < kWarps; ++i) mine += sm.hist[i][threadIdx.x];
    int base = first(mine);
    if (threadIdx.x < ids.E)
        for (int i = 0; i < kWarps; ++i) {
            const int c = sm.hist[i][threadIdx.x];
            sm.hist[i][threadIdx.x] = base;
            base += c;
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
        if (row[i] >= 0) row[i] += sm.hist[w][key[i]];
    return iters;
}

struct SortOut {
    int32_t* starts;
    int32_t* row_of;
    int32_t* unit_of;
    int64_t U;
};

struct MoveArgs {
    const char* x;  // nullptr: sort only
    char* rows;
    int64_t ldx, ldr;  // bytes
    int cols;          // vectors per row
};

// rows[dest[t*k + j]] = x[t0 + t] for nt tokens; the (token, vector) pairs are
// taken from pair i0 in strides of `step`.  Each vector of x is read once and
// stored k times.
template <typename V>
__device__ __forceinline__ void move_flat(const MoveArgs& m, int64_t t0, int nt, int i0, int step,
                                          int k, const int* dest) {
    int t = i0 / m.cols, c = i0 % m.cols;
    const int dt = step / m.cols, dc = step % m.cols;
    while (t < nt) {
        const int64_t b = static_cast<int64_t>(c) * sizeof(V);
        const V v = *reinterpret_cast<const V*>(m.x + (t0 + t) * m.ldx + b);
        for (int j = 0; j < k; ++j) {
            const int r = dest[t * k + j];
            if (r >= 0) *reinterpret_cast<V*>(m.rows + r * m.ldr + b) = v;
        }
        t += dt;
        c += dc;
        if (c >= m.cols) {
            c -= m.cols;
            ++t;
        }
    }
}

// The same for a block's own tokens: a warp per token, four vectors a lane in
// flight, where a row has enough of them (short rows go flat).  At 16384 tokens
// (above): 90 us, 100 with one vector in flight.
template <typename V>
__device__ __forceinline__ void move_rows(const MoveArgs& m, int64_t t0, int nt, int k,
                                          const int* dest) {
    if (m.cols < 64) return move_flat<V>(m, t0, nt, threadIdx.x, kThreads, k, dest);
    constexpr int U = 4;
    const int lane = threadIdx.x & 31;
    for (int t = threadIdx.x >> 5; t < nt; t += kWarps) {
        const char* x = m.x + (t0 + t) * m.ldx + lane * sizeof(V);
        int c = lane;
        for (; c + 32 * (U - 1) < m.cols; c += 32 * U, x += 32 * U * sizeof(V)) {
            V v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const V*>(x + u * 32 * sizeof(V));
            for (int j = 0; j < k; ++j) {
                const int r = dest[t * k + j];
                if (r < 0) continue;
                char* to = m.rows + r * m.ldr + static_cast<int64_t>(c) * sizeof(V);
#pragma unroll
                for (int u = 0; u < U; ++u) *reinterpret_cast<V*>(to + u * 32 * sizeof(V)) = v[u];
            }
        }
        for (; c < m.cols; c += 32, x += 32 * sizeof(V)) {
            const V v = *reinterpret_cast<const V*>(x);
            for (int j = 0; j < k; ++j) {
                const int r = dest[t * k + j];
                if (r >= 0) *reinterpret_cast<V*>(m.rows + r * m.ldr + static_cast<int64_t>(c) * sizeof(V)) = v;
            }
        }
    }
}

// Rows that no unit has are zero.
template <typename V>
__device__ __forceinline__ void zero_rows(const MoveArgs& m, int64_t first, int64_t U) {
    const int64_t n = (U - first) * m.cols;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t r = i / m.cols;
        *reinterpret_cast<V*>(m.rows + (first + r) * m.ldr + (i - r * m.cols) * sizeof(V)) = V{};
    }
}

// At most kFusedUnits units: every block sorts all of them and moves its own
// share of the (token, vector) pairs; block 0 writes the order.
template <typename V>
__global__ void __launch_bounds__(kThreads)
    dispatch_small_kernel(Ids ids, SortOut so, MoveArgs m, int* err) {
    __shared__ SortSmem sm;
    __shared__ int dest[kFusedUnits];
    constexpr int ITERS = kFusedUnits / kThreads;
    int key[ITERS], row[ITERS], total = 0;
    const int n = static_cast<int>(so.U);
    const bool out = blockIdx.x == 0;
    const int iters = rank_units<ITERS>(ids, 0, n, sm, key, row, err, [&](int mine) {
        const int s = block_scan(mine, sm.warp_sums, &total);
        if (out && threadIdx.x < ids.E) so.starts[threadIdx.x] = s;
        return s;
    });
    if (out && threadIdx.x == 0) so.starts[ids.E] = total;
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int l = ((threadIdx.x >> 5) * iters + i) * 32 + (threadIdx.x & 31);
        if (i >= iters || l >= n) continue;
        dest[l] = row[i];
        if (out) {
            so.row_of[l] = row[i];
            if (row[i] >= 0) so.unit_of[row[i]] = l;
        }
    }
    if (out)
        for (int r = total + threadIdx.x; r < n; r += kThreads) so.unit_of[r] = -1;
    if (!m.x) return;
    __syncthreads();
    move_flat<V>(m, 0, n / ids.k, blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads, ids.k,
                 dest);
    zero_rows<V>(m, total, n);
}

// Larger batches, chunks of tc tokens: (1) units of each expert per chunk,
// counts[e][chunk]; (2) each expert's exclusive scan over the chunks, its sum
// in totals[e]; (3) ranks inside the chunk, the order, and the moved rows.
__global__ void __launch_bounds__(kThreads)
    sort_count_kernel(Ids ids, int64_t U, int tc, int C, int* counts, int* err) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ int hist[AEM_MAX_EXPERTS];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t u0 = blockIdx.x * static_cast<int64_t>(tc) * ids.k;
    const int n = static_cast<int>(min(static_cast<int64_t>(tc) * ids.k, U - u0));
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int e = unit_expert(ids, u0 + i, err);
        if (e < ids.E) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    if (threadIdx.x < ids.E) counts[static_cast<int64_t>(threadIdx.x) * C + blockIdx.x] = hist[threadIdx.x];
}

__global__ void __launch_bounds__(kThreads) sort_scan_kernel(int C, int* counts, int* totals) {
    asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
    __shared__ int ws[kWarps];
    int* c = counts + static_cast<int64_t>(blockIdx.x) * C;
    int carry = 0;
    for (int i0 = 0; i0 < C; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        const int v = i < C ? c[i] : 0;
        int sum;
        const int before = block_scan(v, ws, &sum);
        if (i < C) c[i] = carry + before;
        carry += sum;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <typename V>
__global__ void __launch_bounds__(kThreads)
    sort_move_kernel(Ids ids, SortOut so, int tc, int C, const int* counts,
                     const int* totals, MoveArgs m, int* err) {
    __shared__ SortSmem sm;
    __shared__ int dest[kBlockUnits];
    constexpr int ITERS = kBlockUnits / kThreads;
    int key[ITERS], row[ITERS], total = 0;
    const int64_t u0 = blockIdx.x * static_cast<int64_t>(tc) * ids.k;
    const int n = static_cast<int>(min(static_cast<int64_t>(tc) * ids.k, so.U - u0));
    const int iters = rank_units<ITERS>(ids, u0, n, sm, key, row, err, [&](int) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // the scan's sums
        const bool e = threadIdx.x < ids.E;
        const int s = block_scan(e ? totals[threadIdx.x] : 0, sm.warp_sums, &total);
        if (blockIdx.x == 0 && e) so.starts[threadIdx.x] = s;
        return e ? s + counts[static_cast<int64_t>(threadIdx.x) * C + blockIdx.x] : 0;
    });
    if (blockIdx.x == 0 && threadIdx.x == 0) so.starts[ids.E] = total;
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
        const int l = ((threadIdx.x >> 5) * iters + i) * 32 + (threadIdx.x & 31);
        if (i >= iters || l >= n) continue;
        dest[l] = row[i];
        so.row_of[u0 + l] = row[i];
        if (row[i] >= 0) so.unit_of[row[i]] = static_cast<int>(u0 + l);
    }
    for (int64_t r = total + blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; r < so.U;
         r += static_cast<int64_t>(gridDim.x) * kThreads)
        so.unit_of[r] = -1;
    if (!m.x) return;
    __syncthreads();
    move_rows<V>(m, u0 / ids.k, n / ids.k, ids.k, dest);
    zero_rows<V>(m, total, so.U);
}

// Rows moved by an order that exists already.
template <typename V>
__global__ void __launch_bounds__(kThreads)
    move_kernel(const int32_t* __restrict__ row_of, const int32_t* __restrict__ total, int64_t T,
                int k, int tc, MoveArgs m, int* err) {
    __shared__ int dest[kBlockUnits];
    const int64_t t0 = blockIdx.x * static_cast<int64_t>(tc), U = T * k;
    const int nt = static_cast<int>(min(static_cast<int64_t>(tc), T - t0));
    for (int i = threadIdx.x; i < nt * k; i += kThreads) {
        int r = row_of[t0 * k + i];
        if (r >= U) {
            atomicOr(err, ERR_ROW_INDEX);
            r = -1;
        }
        dest[i] = r;
    }
    __syncthreads();
    move_rows<V>(m, t0, nt, k, dest);
    zero_rows<V>(m, max(0, *total), U);
}

// ------------------------------------------------------------------ combine
// VE consecutive elements (8 or 4: 16 bytes of the widest type; or one) as
// they lie in memory; with 8 float32 elements a lane, two loads half a line
// apart, dispatch's backward pass took 40.2 us instead of 34.4.  Loads are kept
// apart from their conversion and made without conditions (a row that does not
// count is replaced by row 0 and dropped afterwards): a load inside a branch is
// waited for inside it, and the rows of a token would come one after the other
// (the backward pass 163 us instead of 76, the forward one 87 instead of 77).
template <typename T, int VE>
struct Vec {
    static constexpr int W = VE == 1 ? 1 : VE * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VE == 1) {
            if constexpr (sizeof(T) == 2)
                w[0] = static_cast<uint32_t>(__bfloat16_as_ushort(p[0])) << 16;
            else
                w[0] = __float_as_uint(p[0]);
        } else {
            if constexpr (W == 2) {
                const uint2 u = *reinterpret_cast<const uint2*>(p);
                w[0] = u.x, w[1] = u.y;
            }
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                const uint4 u = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (VE == 1 || sizeof(T) == 4) return __uint_as_float(w[i]);
        // bf16 is the upper half of a float32
        return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
};
template <typename T, int VE>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VE]) {
    if constexpr (VE == 1) {
        if constexpr (sizeof(T) == 2)
            p[0] = __float2bfloat16_rn(v[0]);
        else
            p[0] = v[0];
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VE / 4; ++i)
            reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
        uint32_t h[VE / 2];
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            h[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
        if constexpr (VE == 4)
            *reinterpret_cast<uint2*>(p) = make_uint2(h[0], h[1]);
        else
            *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
    }
}

// Rows of units j0 .. j0 + KB of a token (-1: none, or past its units, which
// is reported).
template <int KB>
__device__ __forceinline__ void unit_rows(const int32_t* at, int j0, int k, int64_t U, int* err,
                                          int (&r)[KB]) {
#pragma unroll
    for (int j = 0; j < KB; ++j) r[j] = at[min(j0 + j, k - 1)];
#pragma unroll
    for (int j = 0; j < KB; ++j) {
        if (r[j] >= U) {
            atomicOr(err, ERR_ROW_INDEX);
            r[j] = -1;
        }
        if (j0 + j >= k) r[j] = -1;
    }
}

struct CombineArgs {
    const void* rows;
    const float* weights;  // nullptr: every weight is 1
    const int32_t* row_of;
    void* out;
    int64_t ldr, ldw, ldo, T;
    int k, cols;  // cols: vectors of VE elements per row
    int* err;
};

// One thread per (token, vector): tpt threads of a block share a token, KB
// units' rows are in flight at a time.  At most 16 blocks an SM, which go on to
// further tokens: 72.6 us (16384 tokens), 76.1 with 64 blocks an SM.
template <typename RT, typename OT, int VE, int KB>
__global__ void __launch_bounds__(kThreads) combine_units_kernel(CombineArgs a, int tpt) {
    const int per = kThreads / tpt, lane = threadIdx.x % tpt;
    const int64_t U = a.T * a.k;
    for (int64_t t = blockIdx.x * static_cast<int64_t>(per) + threadIdx.x / tpt; t < a.T;
         t += static_cast<int64_t>(gridDim.x) * per) {
        const int32_t* at = a.row_of + t * a.k;
        for (int c = lane; c < a.cols; c += tpt) {
            float acc[VE] = {};
            for (int j0 = 0; j0 < a.k; j0 += KB) {
                int r[KB];
                unit_rows<KB>(at, j0, a.k, U, a.err, r);
                Vec<RT, VE> x[KB];
                float w[KB];
#pragma unroll
                for (int j = 0; j < KB; ++j)
                    x[j].load(static_cast<const RT*>(a.rows) + max(r[j], 0) * a.ldr + static_cast<int64_t>(c) * VE);
#pragma unroll
                for (int j = 0; j < KB; ++j)
                    w[j] = a.weights ? a.weights[t * a.ldw + min(j0 + j, a.k - 1)] : 1.0f;
#pragma unroll
                for (int j = 0; j < KB; ++j)
                    if (r[j] >= 0)
#pragma unroll
                        for (int i = 0; i < VE; ++i) acc[i] = fmaf(w[j], x[j].get(i), acc[i]);
            }
            store_vec<OT, VE>(static_cast<OT*>(a.out) + t * a.ldo + static_cast<int64_t>(c) * VE, acc);
        }
    }
}

struct CombineGradArgs {
    const void* grad_out;
    const void* rows;      // nullptr: no gradient of the weights
    const float* weights;  // nullptr: every weight is 1
    const int32_t* row_of;
    const int32_t* total;  // starts[E]
    void* grad_rows;       // nullptr: not wanted
    float* grad_weights;   // nullptr: not wanted
    int64_t ldg, ldr, ldw, ldgr, T;
    int k, cols;
    int* err;
};

// wpt warps of a block share a token; KB units at a time keep their rows in
// flight and their dot products in registers.
template <typename GT, typename RT, int VE, int KB>
__global__ void __launch_bounds__(kThreads, sizeof(RT) == 2 ? 3 : 2) combine_grad_kernel(CombineGradArgs a, int wpt) {
    __shared__ float part[kWarps][KB];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = kWarps / wpt, wt = w % wpt;
    const int64_t U = a.T * a.k;
    for (int64_t tb = blockIdx.x * static_cast<int64_t>(per); tb < a.T;
         tb += static_cast<int64_t>(gridDim.x) * per) {
        const bool on = tb + w / wpt < a.T;
        const int64_t t = on ? tb + w / wpt : a.T - 1;
        for (int j0 = 0; j0 < a.k; j0 += KB) {
            float dot[KB] = {}, wj[KB];
            int r[KB];
            unit_rows<KB>(a.row_of + t * a.k, j0, a.k, U, a.err, r);
#pragma unroll
            for (int j = 0; j < KB; ++j)
                wj[j] = a.weights ? a.weights[t * a.ldw + min(j0 + j, a.k - 1)] : 1.0f;
            if (on)
                for (int c = wt * 32 + lane; c < a.cols; c += wpt * 32) {
                    const int64_t at = static_cast<int64_t>(c) * VE;
                    Vec<GT, VE> g;
                    Vec<RT, VE> x[KB];
                    g.load(static_cast<const GT*>(a.grad_out) + t * a.ldg + at);
                    if (a.grad_weights)
#pragma unroll
                        for (int j = 0; j < KB; ++j)
                            x[j].load(static_cast<const RT*>(a.rows) + max(r[j], 0) * a.ldr + at);
                    if (a.grad_rows)
#pragma unroll
                        for (int j = 0; j < KB; ++j) {
                            if (r[j] < 0) continue;
                            float y[VE];
#pragma unroll
                            for (int i = 0; i < VE; ++i) y[i] = wj[j] * g.get(i);
                            store_vec<RT, VE>(static_cast<RT*>(a.grad_rows) + r[j] * a.ldgr + at, y);
                        }
                    if (a.grad_weights)
#pragma unroll
                        for (int j = 0; j < KB; ++j)
#pragma unroll
                            for (int i = 0; i < VE; ++i) dot[j] = fmaf(g.get(i), x[j].get(i), dot[j]);
                }
            if (!a.grad_weights) continue;
#pragma unroll
            for (int j = 0; j < KB; ++j) {
#pragma unroll
                for (int o = 16; o; o >>= 1) dot[j] += __shfl_xor_sync(~0u, dot[j], o);
                if (lane == 0) part[w][j] = r[j] < 0 ? 0.0f : dot[j];
            }
            __syncthreads();
            if (wt == 0 && lane < KB && j0 + lane < a.k && on) {
                float s = 0.0f;
                for (int i = 0; i < wpt; ++i) s += part[w + i][lane];
                a.grad_weights[t * a.k + j0 + lane] = s;
            }
            __syncthreads();
        }
    }
    if (a.grad_rows) {  // rows that no unit has
        const int64_t first = max(0, *a.total), n = (U - first) * a.cols;
        for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n;
             i += static_cast<int64_t>(gridDim.x) * kThreads) {
            const int64_t r = i / a.cols;
            const float z[VE] = {};
            store_vec<RT, VE>(static_cast<RT*>(a.grad_rows) + (first + r) * a.ldgr + (i - r * a.cols) * VE, z);
        }
    }
}

// ------------------------------------------------------------------ host side
// Chunks of the three-kernel sort: about 8 a SM.  16384 tokens: 86 us, 92.5
// with 4 (the last ones run alone), 90 with 16 (more to scan).
struct Plan {
    int tc = 0, C = 0;
};
Plan plan_of(int64_t T, int k) {
    Plan p;
    const int64_t want = (T + 148 * 8 - 1) / (148 * 8);
    p.tc = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, kBlockUnits / k)));
    p.C = static_cast<int>((T + p.tc - 1) / p.tc);
    return p;
}

// Largest of 16, 8, 4, 2 that divides all of the bits or'ed into v.
int vec_bytes(uint64_t v) {
    for (int b : {16, 8, 4})
        if (v % b == 0) return b;
    return 2;
}

template <typename F>
void with_vec(int bytes, F f) {
    if (bytes == 16)
        f(uint4{});
    else if (bytes == 8)
        f(uint2{});
    else if (bytes == 4)
        f(uint32_t{});
    else
        f(uint16_t{});
}

// Units whose rows a thread keeps in flight.
template <typename F>
void with_units(int k, F f) {
    if (k == 1)
        f(std::integral_constant<int, 1>{});
    else if (k == 2)
        f(std::integral_constant<int, 2>{});
    else if (k <= 4)
        f(std::integral_constant<int, 4>{});
    else if (k <= 6)
        f(std::integral_constant<int, 6>{});
    else
        f(std::integral_constant<int, 8>{});
}

aem_status sort_and_move(const Ids& ids, const SortOut& so, int64_t T, MoveArgs m, int vb,
                         void* ws, cudaStream_t s) {
    int* err = device_error_word(current_device());
    if (!err) {
        set_error("token sort: no device error word");
        return AEM_ENOMEM;
    }
    if (so.U <= kFusedUnits) {
        const int64_t work = m.x ? so.U * m.cols : 1;
        const unsigned g = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((work + kThreads - 1) / kThreads, 148 * 2)));
        with_vec(vb, [&](auto v) {
            dispatch_small_kernel<decltype(v)><<<g, kThreads, 0, s>>>(ids, so, m, err);
        });
        AEM_CHECK_LAUNCH();
        count_launches(1);
        return AEM_OK;
    }
    const Plan p = plan_of(T, ids.k);
    int* counts = static_cast<int*>(ws);
    int* totals = counts + static_cast<int64_t>(p.C) * ids.E;
    sort_count_kernel<<<p.C, kThreads, 0, s>>>(ids, so.U, p.tc, p.C, counts, err);
    AEM_CHECK_LAUNCH();
    // the scan and the ranking start under their predecessors and wait for
    // them where they read their results
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(ids.E);
    AEM_TRY_CUDA(cudaLaunchKernelEx(&cfg, sort_scan_kernel, p.C, counts, totals));
    cfg.gridDim = dim3(p.C);
    cudaError_t e = cudaSuccess;
    with_vec(vb, [&](auto v) {
        e = cudaLaunchKernelEx(&cfg, sort_move_kernel<decltype(v)>, ids, so, p.tc, p.C,
                               static_cast<const int*>(counts), static_cast<const int*>(totals), m, err);
    });
    AEM_TRY_CUDA(e);
    count_launches(3);
    return AEM_OK;
}

int elem(aem_dtype t) { return t == AEM_F32 ? 4 : 2; }
bool is_dtype(aem_dtype t) { return t == AEM_F32 || t == AEM_BF16; }

// A power of two of threads for one token's cols vectors: all of them at
// once when the batch is small, else the widest that leaves at most an
// eighth of the threads idle in the last round.
int threads_per_token(int64_t T, int cols) {
    int full = 8;
    while (full < cols && full < kThreads) full *= 2;
    if (T * full <= 148 * 1024) return full;
    for (int w = full; w > 8; w /= 2)
        if ((cols + w - 1) / w * w * 8 <= cols * 9) return w;
    return full;
}

}  // namespace

}  // namespace aem

using aem::set_error;

extern "C" {

size_t aem_token_sort_workspace(int64_t T, int k, int E) {
    if (T < 1 || k < 1 || k > AEM_MAX_TOPK || E < 1 || E > AEM_MAX_EXPERTS || T * k <= aem::kFusedUnits) return 0;
    return sizeof(int) * (static_cast<size_t>(aem::plan_of(T, k).C) + 1) * E;
}

aem_status aem_dispatch(const void* x, aem_dtype dtype, int64_t ldx, int64_t d, const int32_t* ids,
                        int64_t T, int k, int64_t stride_t, int64_t stride_k, int E, void* rows,
                        int64_t ldr, int32_t* starts, int32_t* row_of, int32_t* unit_of,
                        void* workspace, size_t workspace_bytes, void* stream) {
    const bool move = x != nullptr || rows != nullptr;
    AEM_REQUIRE(T >= 0, "aem_dispatch: T=%lld must be >= 0", (long long)T);
    AEM_REQUIRE(E >= 1 && E <= AEM_MAX_EXPERTS, "aem_dispatch: num_experts=%d outside [1, %d]", E,
                AEM_MAX_EXPERTS);
    AEM_REQUIRE(k >= 1 && k <= AEM_MAX_TOPK, "aem_dispatch: k=%d outside [1, %d]", k, AEM_MAX_TOPK);
    AEM_REQUIRE(T < (1ll << 31) / k, "aem_dispatch: T*k=%lld*%d exceeds 2^31 - 1", (long long)T, k);
    AEM_REQUIRE(starts != nullptr, "aem_dispatch: NULL starts");
    auto s = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        AEM_TRY_CUDA(cudaMemsetAsync(starts, 0, sizeof(int32_t) * (E + 1), s));
        return AEM_OK;
    }
    AEM_REQUIRE(ids && row_of && unit_of, "aem_dispatch: NULL buffer");
    AEM_REQUIRE(stride_t >= 0 && stride_k >= 0, "aem_dispatch: negative stride of the expert ids");
    aem::MoveArgs m{};
    int vb = 16;
    if (move) {
        AEM_REQUIRE(x && rows, "aem_dispatch: NULL buffer");
        AEM_REQUIRE(aem::is_dtype(dtype), "aem_dispatch: bad dtype");
        const int es = aem::elem(dtype);
        AEM_REQUIRE(d >= 1 && d < (1ll << 28), "aem_dispatch: d=%lld out of range", (long long)d);
        AEM_REQUIRE(ldx >= 0 && ldr >= d, "aem_dispatch: bad row stride");
        vb = aem::vec_bytes(reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows) |
                            static_cast<uint64_t>(d * es) | static_cast<uint64_t>(ldx * es) |
                            static_cast<uint64_t>(ldr * es));
        m.x = static_cast<const char*>(x);
        m.rows = static_cast<char*>(rows);
        m.ldx = ldx * es;
        m.ldr = ldr * es;
        m.cols = static_cast<int>(d * es / vb);
    }
    const size_t need = aem_token_sort_workspace(T, k, E);
    AEM_REQUIRE(!workspace || workspace_bytes >= need,
                "aem_dispatch: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    void* own = nullptr;
    if (!workspace && need) {
        AEM_TRY_CUDA(cudaMallocAsync(&own, need, s));
        workspace = own;
    }
    const aem_status st = aem::sort_and_move({ids, stride_t, stride_k, k, E},
                                             {starts, row_of, unit_of, T * k}, T, m, vb, workspace, s);
    if (own) cudaFreeAsync(own, s);
    return st;
}

aem_status aem_token_sort(const int32_t* ids, int64_t T, int k, int64_t stride_t, int64_t stride_k,
                          int E, int32_t* starts, int32_t* row_of, int32_t* unit_of,
                          void* workspace, size_t workspace_bytes, void* stream) {
    return aem_dispatch(nullptr, AEM_F32, 0, 0, ids, T, k, stride_t, stride_k, E, nullptr, 0,
                        starts, row_of, unit_of, workspace, workspace_bytes, stream);
}

aem_status aem_dispatch_rows(const void* x, aem_dtype dtype, int64_t ldx, int64_t d,
                             const int32_t* row_of, const int32_t* starts, int64_t T, int k, int E,
                             void* rows, int64_t ldr, void* stream) {
    AEM_REQUIRE(T >= 0 && k >= 1 && k <= AEM_MAX_TOPK && T < (1ll << 31) / k,
                "aem_dispatch_rows: T=%lld, k=%d out of range", (long long)T, k);
    AEM_REQUIRE(E >= 1 && E <= AEM_MAX_EXPERTS, "aem_dispatch_rows: num_experts=%d outside [1, %d]",
                E, AEM_MAX_EXPERTS);
    AEM_REQUIRE(aem::is_dtype(dtype), "aem_dispatch_rows: bad dtype");
    AEM_REQUIRE(d >= 1 && d < (1ll << 28), "aem_dispatch_rows: d=%lld out of range", (long long)d);
    AEM_REQUIRE(ldx >= 0 && ldr >= d, "aem_dispatch_rows: bad row stride");
    if (T == 0) return AEM_OK;
    AEM_REQUIRE(x && row_of && starts && rows, "aem_dispatch_rows: NULL buffer");
    int* err = aem::device_error_word(aem::current_device());
    if (!err) {
        set_error("aem_dispatch_rows: no device error word");
        return AEM_ENOMEM;
    }
    const int es = aem::elem(dtype);
    const int vb = aem::vec_bytes(reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows) |
                                  static_cast<uint64_t>(d * es) | static_cast<uint64_t>(ldx * es) |
                                  static_cast<uint64_t>(ldr * es));
    aem::MoveArgs m{static_cast<const char*>(x), static_cast<char*>(rows), ldx * es, ldr * es,
                    static_cast<int>(d * es / vb)};
    const aem::Plan p = aem::plan_of(T, k);
    aem::with_vec(vb, [&](auto v) {
        aem::move_kernel<decltype(v)><<<p.C, aem::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            row_of, starts + E, T, k, p.tc, m, err);
    });
    AEM_CHECK_LAUNCH();
    aem::count_launches(1);
    return AEM_OK;
}

aem_status aem_combine(const void* rows, aem_dtype rows_dtype, int64_t ldr, const float* weights,
                       int64_t ldw, const int32_t* row_of, int64_t T, int k, int64_t d, void* out,
                       aem_dtype out_dtype, int64_t ldo, void* stream) {
    AEM_REQUIRE(T >= 0 && k >= 1 && k <= AEM_MAX_TOPK && T < (1ll << 31) / k,
                "aem_combine: T=%lld, k=%d out of range", (long long)T, k);
    AEM_REQUIRE(aem::is_dtype(rows_dtype) && aem::is_dtype(out_dtype), "aem_combine: bad dtype");
    AEM_REQUIRE(d >= 1 && d < (1ll << 28), "aem_combine: d=%lld out of range", (long long)d);
    AEM_REQUIRE(ldr >= 0 && ldo >= d && (!weights || ldw >= 0), "aem_combine: bad row stride");
    if (T == 0) return AEM_OK;
    AEM_REQUIRE(rows && row_of && out, "aem_combine: NULL buffer");
    int* err = aem::device_error_word(aem::current_device());
    if (!err) {
        set_error("aem_combine: no device error word");
        return AEM_ENOMEM;
    }
    const uint64_t bits = reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(out) |
                          static_cast<uint64_t>(ldr * aem::elem(rows_dtype)) |
                          static_cast<uint64_t>(ldo * aem::elem(out_dtype));
    const bool vec = bits % 16 == 0 && d % 8 == 0;
    const int ve = rows_dtype == AEM_F32 ? 4 : 8;
    aem::CombineArgs a{rows, weights, row_of, out, ldr, ldw, ldo, T, k,
                       static_cast<int>(vec ? d / ve : d), err};
    const int tpt = aem::threads_per_token(T, a.cols);
    const int64_t per = aem::kThreads / tpt;
    const unsigned g = static_cast<unsigned>(std::min<int64_t>((T + per - 1) / per, 148 * 16));
    auto s = static_cast<cudaStream_t>(stream);
    auto go = [&](auto r, auto o) {
        using RT = decltype(r);
        using OT = decltype(o);
        if (!vec)
            aem::combine_units_kernel<RT, OT, 1, 4><<<g, aem::kThreads, 0, s>>>(a, tpt);
        else
            aem::with_units(k, [&](auto kb) {
                aem::combine_units_kernel<RT, OT, (sizeof(RT) == 4 ? 4 : 8), decltype(kb)::value><<<g, aem::kThreads, 0, s>>>(a, tpt);
            });
    };
    const __nv_bfloat16 h{};
    if (rows_dtype == AEM_BF16)
        out_dtype == AEM_BF16 ? go(h, h) : go(h, 0.0f);
    else
        out_dtype == AEM_BF16 ? go(0.0f, h) : go(0.0f, 0.0f);
    AEM_CHECK_LAUNCH();
    aem::count_launches(1);
    return AEM_OK;
}

aem_status aem_dispatch_backward(const void* grad_rows, aem_dtype rows_dtype, int64_t ldr,
                                 const int32_t* row_of, int64_t T, int k, int64_t d, void* grad_x,
                                 aem_dtype x_dtype, int64_t ldx, void* stream) {
    return aem_combine(grad_rows, rows_dtype, ldr, nullptr, 0, row_of, T, k, d, grad_x, x_dtype,
                       ldx, stream);
}

aem_status aem_combine_backward(const void* grad_out, aem_dtype out_dtype, int64_t ldg,
                                const void* rows, aem_dtype rows_dtype, int64_t ldr,
                                const float* weights, int64_t ldw, const int32_t* row_of,
                                const int32_t* starts, int64_t T, int k, int E, int64_t d,
                                void* grad_rows, int64_t ldgr, float* grad_weights, void* stream) {
    AEM_REQUIRE(T >= 0 && k >= 1 && k <= AEM_MAX_TOPK && T < (1ll << 31) / k,
                "aem_combine_backward: T=%lld, k=%d out of range", (long long)T, k);
    AEM_REQUIRE(E >= 1 && E <= AEM_MAX_EXPERTS,
                "aem_combine_backward: num_experts=%d outside [1, %d]", E, AEM_MAX_EXPERTS);
    AEM_REQUIRE(aem::is_dtype(rows_dtype) && aem::is_dtype(out_dtype),
                "aem_combine_backward: bad dtype");
    AEM_REQUIRE(d >= 1 && d < (1ll << 28), "aem_combine_backward: d=%lld out of range",
                (long long)d);
    AEM_REQUIRE(ldg >= 0 && (!grad_weights || ldr >= 0) && (!grad_rows || ldgr >= d) &&
                    (!weights || ldw >= 0),
                "aem_combine_backward: bad row stride");
    if (T == 0) return AEM_OK;
    AEM_REQUIRE(grad_rows || grad_weights, "aem_combine_backward: no gradient wanted");
    AEM_REQUIRE(grad_out && row_of && starts && (rows || !grad_weights),
                "aem_combine_backward: NULL buffer");
    int* err = aem::device_error_word(aem::current_device());
    if (!err) {
        set_error("aem_combine_backward: no device error word");
        return AEM_ENOMEM;
    }
    uint64_t bits = reinterpret_cast<uintptr_t>(grad_out) | static_cast<uint64_t>(ldg * aem::elem(out_dtype));
    if (grad_weights)
        bits |= reinterpret_cast<uintptr_t>(rows) | static_cast<uint64_t>(ldr * aem::elem(rows_dtype));
    if (grad_rows)
        bits |= reinterpret_cast<uintptr_t>(grad_rows) | static_cast<uint64_t>(ldgr * aem::elem(rows_dtype));
    const bool vec = bits % 16 == 0 && d % 8 == 0;
    const int ve = rows_dtype == AEM_F32 || out_dtype == AEM_F32 ? 4 : 8;
    aem::CombineGradArgs a{grad_out, rows, weights, row_of, starts + E, grad_rows, grad_weights,
                           ldg, ldr, ldw, ldgr, T, k, static_cast<int>(vec ? d / ve : d), err};
    int wpt = 1;  // more warps for a token while the batch leaves SMs idle
    while (wpt < aem::kWarps && T * wpt < 148 * 16 && a.cols > 32 * wpt) wpt *= 2;
    const int64_t per = aem::kWarps / wpt;
    const unsigned g = static_cast<unsigned>(std::min<int64_t>((T + per - 1) / per, 148 * 64));
    auto s = static_cast<cudaStream_t>(stream);
    auto go = [&](auto o, auto r) {
        using GT = decltype(o);
        using RT = decltype(r);
        if (!vec)
            aem::combine_grad_kernel<GT, RT, 1, 4><<<g, aem::kThreads, 0, s>>>(a, wpt);
        else
            aem::with_units(k, [&](auto kb) {
                aem::combine_grad_kernel<GT, RT, (sizeof(GT) + sizeof(RT) > 4 ? 4 : 8), decltype(kb)::value><<<g, aem::kThreads, 0, s>>>(a, wpt);
            });
    };
    const __nv_bfloat16 h{};
    if (out_dtype == AEM_BF16)
        rows_dtype == AEM_BF16 ? go(h, h) : go(h, 0.0f);
    else
        rows_dtype == AEM_BF16 ? go(0.0f, h) : go(0.0f, 0.0f);
    AEM_CHECK_LAUNCH();
    aem::count_launches(1);
    return AEM_OK;
}

}  // extern "C"
