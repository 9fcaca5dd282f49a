// Layout of the 8-bit block cache: codes of one byte (int8, or float8 e4m3) whose value is code x scale, one
// scale for each block of N = 32, 64 or 128 tokens of a sequence and kv head, for K and V apart.  Only whole
// blocks are quantized; the tokens after the last whole block (the tail, fewer than N) stay float32 until
// their block is full, so what the cache holds depends on the tokens alone, not on how they were appended.
//
// The scale is a power of two, the smallest that brings the block's largest magnitude within the type (127,
// 448).  Quantizing is then exact but for the one rounding to the type, a block that is quantized again under
// the same scale keeps its codes, and the values are exact in float16 and bfloat16 (their range aside).  It
// costs int8 up to one bit against the scale amax / 127: the rounding is half a step of 2^-6 to 2^-7 of amax.
//
// Codes lie in the order in which the matrix instruction v_mfma_f32_16x16x32 takes them, so that a wavefront's
// loads are contiguous 1 KiB runs and nothing passes through LDS on the way (lane l = 16 g + m):
//   K: tiles of 16 tokens; the 16 bytes at 16 l of KiB i are dims 16 (4i + g) .. +15 of token m, the A
//      operands (keys x dims) of two instructions;
//   V: units of 64 tokens; the 16 bytes at 16 l of KiB i are dim 16 i + m of tokens 16 kb + 4g + r at byte 4 kb + r
//      (kb, r < 4), the A operands (dims x keys) of two, whose keys are those of which lane l holds the
//      probabilities when the score product ends.
// int8 codes are kept as code + 128 (the bytes that place themselves under a float16 exponent).
// Dims are padded with zeros to Dp, a multiple of 64 (one of 64, 128 or 256).  Plain arithmetic that a host
// program can check.
#pragma once

#include <cstdint>

#ifndef __host__
#define GT_KVB_FN constexpr
#else
#define GT_KVB_FN __host__ __device__ constexpr
#endif

namespace gtkvb {

constexpr int kUnit = 64;        // tokens of a unit
constexpr int kMaxDim = 256;
constexpr int kMaxBlock = 128;

GT_KVB_FN inline int padded_dim(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// Byte of (token t, dim d) in the codes of one sequence and head.
GT_KVB_FN inline int64_t k_at(int64_t t, int d, int Dp) {
    return (t >> 4) * 16 * Dp + (d >> 4) * 256 + (t & 15) * 16 + (d & 15);
}
GT_KVB_FN inline int64_t v_at(int64_t t, int d, int Dp) {
    const int kk = (int)(t & 63);
    return (t >> 6) * 64 * Dp + (d >> 4) * 1024 + ((kk >> 2) & 3) * 256 + (d & 15) * 16 + (kk >> 4) * 4 + (kk & 3);
}

// Whether token p waits in the tail of a cache that holds `held` tokens: row p - (held >> shift << shift), below
// the tokens of a block (1 << shift).  A workgroup's span of 64 tokens may begin before that row 0.
GT_KVB_FN inline bool in_tail(int p, int held, int shift) { return p < held && p >= held >> shift << shift; }

// The scale's exponent for a block whose largest magnitude has the float32 bits `bits` (finite): the smallest
// e >= -126 with amax <= top * 2^e, top 127 (int8) or 448 (e4m3).
GT_KVB_FN inline int scale_exponent(uint32_t bits, bool e4m3) {
    const int x = (int)(bits >> 23) - 126;  // amax = f * 2^x, f in [0.5, 1), below that when subnormal
    const uint32_t frac = bits & 0x7fffffu;  // 127 = (127/128) 2^7, 448 = (7/8) 2^9
    const int e = e4m3 ? x - 9 + (frac > 0x600000u) : x - 7 + (frac > 0x7e0000u);
    return e < -126 ? -126 : e;
}

}  // namespace gtkvb
