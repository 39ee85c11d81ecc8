// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, 1994): (n + high half of n * mul) >> shift
#pragma once

struct FastDiv {
    unsigned mul, shift;
};
static inline FastDiv fast_div(unsigned d) {
    FastDiv v = {0u, 0u};
    while ((1ull << v.shift) < d) ++v.shift;
    v.mul = (unsigned)(((1ull << 32) * ((1ull << v.shift) - d)) / d + 1);
    return v;
}
__device__ __forceinline__ unsigned fast_over(unsigned n, FastDiv d) { return (__umulhi(n, d.mul) + n) >> d.shift; }
__device__ __forceinline__ int fast_over(int n, FastDiv d) { return (int)fast_over((unsigned)n, d); }
