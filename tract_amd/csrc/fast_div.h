// Division of indices by a number that only the launch knows.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace trocm {
namespace {

// n / d for 0 <= n < 2^31 as a product: mul = floor(2^(31 + l) / d) + 1, l = ceil(log2 d).  (A division by a number that only the launch
// knows is some 40 dependent instructions; a workgroup with one tile to read spent a third of its time on five of them.)
struct FastDiv {
    uint32_t d, mul, shift;
    __device__ __forceinline__ int by(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};
FastDiv fast_div(int64_t d) {
    FastDiv f;
    uint32_t l = 0;
    if (d < 1) d = 1;
    while ((1ll << l) < d) l++;
    f.d = (uint32_t)d, f.shift = 31 + l;
    f.mul = (uint32_t)(((unsigned __int128)1 << f.shift) / (uint64_t)d + 1);
    return f;
}

}  // namespace
}  // namespace trocm
