// Places in a cache of keys and values in pages, for the kernels that write and read it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kutacc_hip.h"

namespace kutacc_dev {

// n / d for 0 <= n < 2^31 and a fixed 0 < d < 2^31 by one 64-bit product: with 2^(s - 1) < d <= 2^s and m = floor(2^(31 + s) / d) + 1, m d lies between 2^(31 + s) and
// 2^(31 + s) + 2^s, and floor(n m / 2^(31 + s)) is the quotient (T. Granlund and P. L. Montgomery, Division by invariant integers using multiplication, 1994, theorem 4.2).
struct Divisor {
    uint32_t d, m;
    int shift;

    static Divisor of(uint32_t d)
    {
        int s = 0;
        while (((uint64_t)1 << s) < d) {
            ++s;
        }
        return {d, d == 1 ? 0u : (uint32_t)((((uint64_t)1 << (31 + s)) / d) + 1), 31 + s};
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return d == 1 ? n : (uint32_t)(((uint64_t)n * m) >> shift); }
};

// first, one past the last, of a sequence's tokens among `tokens`, whatever the array holds
struct TokenRange {
    int first, end;
};
__device__ __forceinline__ TokenRange tokens_of(const int32_t *query_starts, int s, int tokens)
{
    const int first = min(max(query_starts[s], 0), tokens);
    return {first, max(first, min(query_starts[s + 1], tokens))};
}

} // namespace kutacc_dev
