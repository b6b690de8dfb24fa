// How far the routing's float32 keys are from the real ones (internal).  Functions of
// numbers alone, for the kernel and for tests on the host.
#pragma once

#include <math.h>

#ifdef __CUDACC__
#define AEM_BOUND __host__ __device__ __forceinline__
#else
#define AEM_BOUND inline
#endif

namespace aem {

// A float32 key's distance from the real one.  A sigmoid's relative error, from
// exp's 2 ulp (at most 2^-22, which reach the quotient by the factor 1 - s), the sum's
// 2^-24 and the quotient's, is under 2^-24 (2 + 4 (1 - s)).  A softmax's score has that
// of its exponential, whose argument rounds by |x - m| 2^-24, of the sum of 256 (13
// additions) and of two products: (|x - m| + 19) 2^-24, so under 2^-18 for |x - m| <=
// 45, and further down it is under 2^-64 altogether.  The sum with the bias is rounded
// once.  One or two hundredths more cover the bound's own roundings.
AEM_BOUND float key_slack(bool sigmoid, float score, float key) {
    const float by = sigmoid ? fmaf(score, -0x1p-22f, 6.02f * 0x1p-24f) : 0x1p-18f;
    return fmaf(by, score, fmaf(1.01f * 0x1p-24f, fabsf(key), 0x1p-64f));
}

// The most that the scores' part of it can be in a row whose largest score is `top`:
// a sigmoid's, s (6.02 - 4 s), is largest in the middle, 2.265 at s = 0.7525, whatever
// the row's largest; a softmax's grows with the score.
AEM_BOUND float score_slack(bool sigmoid, float top) {
    return sigmoid ? 2.27f * 0x1p-24f + 0x1p-64f : fmaf(0x1p-18f, top, 0x1p-64f);
}

// How far apart two groups' values have to be: two keys each, none larger than
// `largest`, whose sums are rounded.
AEM_BOUND float group_slack(float score, float largest) {
    return 4.0f * fmaf(1.01f * 0x1p-24f, largest, score) + 0x1p-22f * largest;
}

// What the keys leave open, as bits that the rows of a warp put together.
enum : int {
    OPEN_ORDER = 1,   // of two chosen ones that follow one another
    OPEN_SET = 2,     // the last chosen one or the next
    OPEN_BEHIND = 4,  // the next one or another chosen one, should that be open with the last
};

// The last chosen key (with its slack) and the next one.  An expert behind the next one
// may have a larger error than it, and an earlier chosen one than the last: `score` at
// most, apart from the rounding of its key.  Keys in falling order whose neighbours'
// bounds are apart prove that all earlier ones lie above the last; where that is not so
// (OPEN_ORDER), only OPEN_BEHIND shows whether they lie above the next.
AEM_BOUND int open_at_end(float key, float slack, float then, float score) {
    const float behind = fmaf(1.01f * 0x1p-24f, fabsf(then), score);
    const float ahead = fmaf(1.01f * 0x1p-24f, fabsf(key), score);
    return (key - then > slack + behind ? 0 : OPEN_SET) | (key - then > ahead + behind ? 0 : OPEN_BEHIND);
}

// 0: nothing has to be decided in 64 bits; 1: the order of the chosen ones; 2: who they are.
AEM_BOUND int to_decide(int open) {
    if (!(open & (OPEN_ORDER | OPEN_SET))) return 0;
    return open == OPEN_ORDER ? 1 : 2;
}

}  // namespace aem
