// Shared by the readout kernels (readout_spikes.hip, readout_scan.hip, readout_logprobs.hip): the types that values are kept in.
// Arithmetic is in 32 bits throughout; 16-bit types are what is read and, rounded once, what is written.
#pragma once

#include "common.hpp"

namespace bmtk {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// division by a number known on the host: n / d for 0 <= n < 2^31.  With 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d) (at most 2^32 - 1 but
// for d = 1, which is looked after apart) the excess m d - 2^(31+s) is below d <= 2^s, so that n m / 2^(31+s) is off by less than 1 / d.
struct FastDiv {
    uint32_t d, m, s;
};
inline FastDiv fast_div(uint32_t d)
{
    FastDiv f{d, 0, 0};
    while ((1ull << f.s) < d) ++f.s;
    if (d > 1) f.m = (uint32_t)(((1ull << (31 + f.s)) + d - 1) / d);
    return f;
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv &f)
{
    return f.d == 1 ? n : (uint32_t)(((uint64_t)n * f.m) >> (31 + f.s));
}

inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline size_t type_size(int dtype) { return dtype == BMTK_F32 ? 4 : 2; }

// f(T()) for the type that a dtype code names; the code has been looked at
#define BMTK_BY_TYPE(dtype, T, ...)                        \
    do {                                                   \
        if ((dtype) == BMTK_F32) {                         \
            typedef float T;                               \
            __VA_ARGS__;                                   \
        } else if ((dtype) == BMTK_BF16) {                 \
            typedef bmtk::bf16 T;                          \
            __VA_ARGS__;                                   \
        } else {                                           \
            typedef bmtk::f16 T;                           \
            __VA_ARGS__;                                   \
        }                                                  \
    } while (0)

}  // namespace bmtk
