// Sixteen consecutive elements of a row, by 16-byte loads of whole registers (structs of elements are taken apart
// by the compiler, and a branch beside them then leaves loads of two bytes), and as float32.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace gtvec {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// float, _Float16 or __bf16; 16-byte aligned.
template <typename T>
struct Dims16 {
    u32x4 w[sizeof(T)];  // (2 registers' worth of 16 bytes for halves, 4 for floats)
    static constexpr int N = (int)sizeof(T);
    __device__ inline void load(const T *p) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = ((const u32x4 *)p)[i];
    }
    __device__ inline float get(int e) const {  // e: a constant after unrolling
        if constexpr (__is_same(T, float)) {
            const uint32_t u = w[e >> 2][e & 3];
            return __uint_as_float(u);
        } else {
            const uint32_t u = w[e >> 3][(e >> 1) & 3], h = e & 1 ? u >> 16 : u & 0xffffu;
            if constexpr (__is_same(T, _Float16)) return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
            else return __uint_as_float(h << 16);
        }
    }
};

}  // namespace gtvec
