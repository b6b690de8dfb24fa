// 8-bit floating point weights and the kernels' launchers (internal).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "aem.h"

namespace aem {

constexpr int kFp8Tile = 128 * 128;   // bytes of a packed tile

// Packed e4m3 weight (device): [G][NC][KC] tiles of 128 channels x 128 k, NC =
// ceil(N / 128), KC = ceil(K / 128).  A tile is 128 rows (channels) of 128 bytes
// (k) in the 128-byte swizzle that the MMA reads: 16-byte chunk c of row r lies at
// chunk c ^ (r & 7).  One bulk copy brings it, and it serves both directions: the
// product sums over k (K-major rows), the gradient over the channels (MN-major).
// scale [G][NC][KC] float32.  Padding is zero.
struct Fp8Weight {
    int device = 0;
    int64_t G = 0, K = 0, N = 0, NC = 0, KC = 0;
    uint8_t* data = nullptr;
    float* scale = nullptr;
};

// e4m3 rows: [M] rows of `ld` bytes (a multiple of 16) and lds scales (a multiple of 4).
aem_status launch_quantize_fp8(const char* what, const void* x, aem_dtype dtype, int64_t ldx, int64_t M, int64_t K,
                               uint8_t* q, int64_t ldq, float* scale, int64_t lds, cudaStream_t s);

}  // namespace aem
