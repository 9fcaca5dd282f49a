// Attention over the 8-bit block cache (kv_blocks.h), straight from the codes: decode steps, the several tokens of a
// draft that are checked together, and prompts that are too short to fill the GPU otherwise.
//
//   s[r, t] = scale q_r . k_t,  p = softmax over the keys that row r sees,  o_r = sum_t p[r, t] v_t
// with k_t = code x 2^a, v_t = code x 2^c, a and c a block's exponents.  HBM-bound: K and V are read once, a
// byte a value.
//
// Rows: the G query heads of a kv head times the L tokens, r = head * L + token, are the 16 columns of the matrix
// instruction; more than 16 take further workgroups over the same keys (two or four tiles of columns in a
// workgroup, which decode the keys once for all, left one wavefront per SIMD and took longer: D128 32 rows of S1024
// 19 against 16.5 us, 128 rows of S4096 42 against 35).  A workgroup owns a span of 64-token units (a split of the
// sequence), its wavefronts take them in turn, each with its own running maximum and sum; they are joined
// once at the end, and the last split of a row group to finish joins the splits (partials in uncached memory, as
// in decode_merge.h).
//
// Products on v_mfma_f32_16x16x32_f16, float32 sums.  Codes become float16 exactly: int8 (kept as code + 128) by placing
// two bytes under exponent bytes (1024 + 128 + code) and subtracting 1152, e4m3 by the hardware's conversion.
// Score S^T = K.Q^T: float16 queries are their own operand; bfloat16 and float32 rows are scaled by a power of
// two to a largest magnitude in [1, 2) and enter as one operand (bfloat16: exact, but for elements below 2^-14
// of the largest, which keep 2^-25 of it) or as two, x = hi + lo (float32: off by 2^-25 of the largest).
// P.V: the weights enter as p' = p 2^(c - r), the reference r following the largest p 2^c so that p' <= 1 and
// what float16 loses below 2^-14 is small against the largest term, whatever the blocks' scales.  float16 and
// bfloat16 results take p' rounded to float16 (2^-12 of each term), float32 results take hi + lo.
//
// The tail is one or two more units, of the operands that the append has left: a token's row (K and V) divided
// by its own power of two, as float16 hi + lo, which carry 22 bits (elements below 2^-14 of the row's largest: what
// is left of 2^-25 of it).  A token with an infinity or NaN has operands
// of zero and a NaN for a scale, which only the rows that see it meet.  (Formed here, from the float32 tokens, they
// took 30 us of a decode step, in loads one after the other.)
//
// Measured (GPU time, int8, float16 queries, D128): one token, B16 Hkv8 S8192 46 us, 5.8 TB/s of codes, the rate at which
// memory is read; B4 S4096 13 us, latency (6.5 us from the start to the first unit's results, 3 the joining of
// splits, 2 the tail); five tokens B8 S4096 21.8 us and 32 tokens B4 S4096 27, the vector ALU: 64 keys take a
// wavefront some 500 instructions beside 32 matrix instructions, half of them for making float16 of the codes.
#pragma once

#include "attn_common.h"
#include "gt_internal.h"
#include "kv_blocks.h"
#include "mfma_util.h"
#include "vec_dims.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <type_traits>

namespace gtkvb {

using gtmfma::fast_exp2;
using gtmfma::half8;
using gtmfma::f32x4;
using gtmfma::kLn2;
using gtmfma::kLog2e;
using gtmfma::u32x4;
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr int kColumns = 16;  // rows of a workgroup

struct AttnArgs {
    const void *q;
    int64_t q_sb, q_sh, q_sl;  // element strides; dims contiguous
    void *o;                   // dense (B, H, L, D) of q's type
    float *lse;                // (B, H, L) or null
    const uint8_t *k, *v;
    const float *ks, *vs;  // scales
    const _Float16 *kt, *vt;  // the tail's operands, hi then lo
    const float *kts, *vts;   // and scales
    const int32_t *len;
    float scale;
    int causal, q_vec;  // q_vec: query rows in aligned 16-byte pieces, D a multiple of 16
    int B, H, Hkv, L, D;
    int shift;  // log2 of the tokens of a block
    int64_t units;  // of a slice
    int nsplit, span;  // splits, units of each
    float *part_o, *part_ml;  // (rows, nsplit, Dp), (rows, nsplit, 2)
    int *counters;
};

// max over the four lanes 16 g + m of one m
__device__ inline float max_g(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    return gtmfma::xhalf_max(v);
}
__device__ inline float sum_g(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    return gtmfma::xhalf_sum(v);
}
__device__ inline float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
// e with 2^e <= a < 2^(e+1), kept within what pow2 and its reciprocal reach; 0 for a zero, infinity or NaN
__device__ inline int exponent_of(float a) {
    if (!(a > 0.0f) || !(a < INFINITY)) return 0;
    return min(max((int)(__float_as_uint(a) >> 23) - 127, -126), 126);
}

// The exponent of a scale (a power of two), NaN for a NaN.
__device__ inline float exponent_bits(uint32_t b) { return (b >> 23 & 255) == 255 ? NAN : (float)((int)(b >> 23) - 127); }

// Eight codes as float16.
template <bool E4M3>
__device__ inline half8 decode8(uint32_t w0, uint32_t w1) {
    half2v h[4];
    if constexpr (E4M3) {
        h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false);
        h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true);
        h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false);
        h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true);
    } else {
        // bytes code + 128 under 0x64: 1024 + 128 + code
        const half2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
        constexpr uint32_t k64 = 0x64646464u;
        h[0] = __builtin_bit_cast(half2v, (uint32_t)__builtin_amdgcn_perm(k64, w0, 0x04010400u)) - off;
        h[1] = __builtin_bit_cast(half2v, (uint32_t)__builtin_amdgcn_perm(k64, w0, 0x04030402u)) - off;
        h[2] = __builtin_bit_cast(half2v, (uint32_t)__builtin_amdgcn_perm(k64, w1, 0x04010400u)) - off;
        h[3] = __builtin_bit_cast(half2v, (uint32_t)__builtin_amdgcn_perm(k64, w1, 0x04030402u)) - off;
    }
    const u32x4 r = {__builtin_bit_cast(uint32_t, h[0]), __builtin_bit_cast(uint32_t, h[1]),
                     __builtin_bit_cast(uint32_t, h[2]), __builtin_bit_cast(uint32_t, h[3])};
    return __builtin_bit_cast(half8, r);
}

__device__ inline f32x4 mma(half8 a, half8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// x * inv as hi (+ lo) float16
__device__ inline void split8(const float *x, float inv, half8 &hi, half8 &lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float y = x[e] * inv;
        hi[e] = (_Float16)y;
        lo[e] = (_Float16)(y - (float)hi[e]);
    }
}

// A query row as lane (n, g) holds it: dims 16 (4i + g) .. +15 of its column's.  vec: aligned 16-byte pieces, D a
// multiple of 16.
template <typename QT, int NI>
struct QueryRow {
    gtvec::Dims16<QT> raw[NI];
    __device__ inline void load(const QT *row, int D, bool vec, int g) {
        if (!vec) return;
#pragma unroll
        for (int i = 0; i < NI; ++i) raw[i].load(row + (16 * (4 * i + g) < D ? 16 * (4 * i + g) : 0));
    }
};

// Its B operands, operand j the eight dims from 8j on of the sixteen.  Returns the row's scale (the operands are the
// row divided by it).
template <typename QT, int NI>
__device__ inline float query_operands(const QueryRow<QT, NI> &q, const QT *row, int D, bool vec, int g, half8 (*hi)[2], half8 (*lo)[2]) {
    constexpr bool F16 = __is_same(QT, _Float16);
    if constexpr (F16) {
        if (vec) {  // its own operand
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const u32x4 w = q.raw[i].w[j];
                    hi[i][j] = __builtin_bit_cast(half8, 16 * (4 * i + g) < D ? w : u32x4{0u, 0u, 0u, 0u});
                }
            return 1.0f;
        }
    }
    float x[NI][16];
    if (vec) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[i][e] = 16 * (4 * i + g) < D ? q.raw[i].get(e) : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = 16 * (4 * i + g) + e;
                x[i][e] = d < D ? (float)row[d] : 0.0f;
            }
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[i][e]));
    int e2 = 0;
    if constexpr (!F16) e2 = exponent_of(max_g(amax));
    const float inv = F16 ? 1.0f : pow2(-e2);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) split8(x[i] + 8 * j, inv, hi[i][j], lo[i][j]);
    return pow2(e2);
}

// Joins the splits of rows row0 .. row0 + n - 1; uncached partials (see decode_merge.h), each load a round trip
// to the memory: the (max, sum) pairs of all rows first, into LDS, then every thread four dims of a row, eight
// splits in flight.  lds: n * nsplit floats.
template <typename TO, int NI, int W>
__device__ inline void merge_splits(const AttnArgs &a, int64_t row0, int n, float *lds) {
    constexpr int Dp = 64 * NI, PIECES = Dp / 4;
    __shared__ float s_inv[kColumns];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, ns = a.nsplit;  // ns <= 64
    constexpr int RW = (kColumns + W - 1) / W;
    float mi[RW], li[RW];  // rows w, w + W, ...: split `lane`
#pragma unroll
    for (int k = 0; k < RW; ++k) {
        const int r = w + W * k;
        const float *ml = a.part_ml + ((row0 + min(r, n - 1)) * ns + min(lane, ns - 1)) * 2;
        if (r < n) {
            mi[k] = lane < ns ? ml[0] : -INFINITY;
            li[k] = lane < ns ? ml[1] : 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < RW; ++k) {
        const int r = w + W * k;
        if (r >= n) break;
        float M = mi[k];
        for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        // (a split without a key has max -inf and sum 0; one whose keys are NaN has a NaN sum)
        const float wi = mi[k] == -INFINITY ? 0.0f : fast_exp2(mi[k] - M);
        float L = li[k] != li[k] ? li[k] : wi * li[k];
        for (int o = 32; o >= 1; o >>= 1) L += __shfl_xor(L, o, 64);
        if (lane < ns) lds[r * ns + lane] = wi;
        if (lane == 0) {
            s_inv[r] = L == 0.0f ? 0.0f : 1.0f / L;
            if (a.lse) a.lse[row0 + r] = L == 0.0f ? INFINITY : (M + log2f(L)) * kLn2;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n * PIECES; e += 64 * W) {
        const int r = e / PIECES, d = 4 * (e % PIECES);
        const float *po = a.part_o + (row0 + r) * ns * Dp + d;
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int U = 8;
        for (int s0 = 0; s0 < ns; s0 += U) {
            f32x4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = *(const f32x4 *)(po + (int64_t)min(s0 + u, ns - 1) * Dp);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float ws = s0 + u < ns ? lds[r * ns + s0 + u] : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = ws == 0.0f ? acc[i] : fmaf(ws, x[u][i], acc[i]);
            }
        }
        const float inv = s_inv[r];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < a.D) ((TO *)a.o)[(row0 + r) * a.D + d + i] = (TO)(acc[i] * inv);
    }
}

// LDS of a launch: the wavefronts' rows on their way to being joined, or the splits' weights.
GT_KVB_FN inline int64_t attn_lds_floats(int rows, int Dp, int nsplit, int waves) {
    const int64_t join = waves / 2 * (int64_t)rows * (Dp + 4), merge = (int64_t)rows * nsplit;
    return join > merge ? join : merge;
}

template <typename QT, int NI, bool E4M3, int W>
__global__ __launch_bounds__(64 * W, NI <= 2 ? 2 : 1) void attn_kv_blocks_kernel(AttnArgs a) {
    constexpr bool F32 = __is_same(QT, float);
    constexpr int Dp = 64 * NI, DT = 4 * NI;
    constexpr int OP = Dp + 4;  // pitch of the rows to be joined
    extern __shared__ __attribute__((aligned(16))) float s_o[];  // [W / 2][row]
    __shared__ float s_m[W][kColumns], s_l[W][kColumns], s_M[kColumns], s_L[kColumns];
    __shared__ int s_last;

    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // row groups outermost: those of one slice land on the same XCD (workgroups are dealt round robin) when the slices
    // are a multiple of 8, and share its L2
    const int64_t x = blockIdx.x, slices = (int64_t)a.B * a.Hkv, bg = x % slices, b = bg / a.Hkv, kvh = bg - b * a.Hkv;
    const int rg = (int)(x / slices), G = a.H / a.Hkv, rows = G * a.L;
    const int r0 = rg * kColumns, nr = min(kColumns, rows - r0);
    const int len = a.len[b], full = len >> a.shift << a.shift;
    // keys from `seen` on are seen by no row of the group (with few tokens that is less than a unit)
    int seen = len;
    if (a.causal && a.L > kUnit) {
        const int h0 = r0 / a.L, last = r0 + nr - 1;
        seen = len - a.L + (last >= (h0 + 1) * a.L ? a.L : last - h0 * a.L + 1);
    }
    const int tail = min(len, seen) - full;

    // ---- whole blocks: the first unit's loads are on their way while the queries are made ready ----
    const int u0 = blockIdx.y * a.span, held = min(u0 + a.span, (full + kUnit - 1) / kUnit), u1 = min(held, (seen + kUnit - 1) / kUnit);
    const int64_t from = (bg * a.units + u0) * kUnit * Dp;
    // buffer loads of a unit each, a lane's 16 bytes: past the last unit the buffer is empty, they return zeros and fetch
    // nothing.  (Places are in the buffer's address and the lanes' offsets: a uniform offset is not checked.)
    auto buffer = [&](const uint8_t *codes, int u) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)(codes + from + (int64_t)(u - u0) * (kUnit * Dp)), 0, u < u1 ? kUnit * Dp : 0, 0x00027000);
    };
    const int64_t nblk = a.units * kUnit >> a.shift;
    const float *sc = ((lane & 4) ? a.vs : a.ks) + bg * nblk;  // lanes 0..3 hold K's scales, 4..7 V's
    u32x4 rk[DT], rv[DT];
    float rs = 0.0f;
    constexpr int kNonTemporal = 2;
    auto load_unit = [&](u32x4 *to, const uint8_t *codes, int u) {
        const auto r = buffer(codes, u);
        int at = 16 * lane;
        asm volatile("" : "+v"(at));  // (the offsets are not kept in registers from unit to unit)
#pragma unroll
        for (int t = 0; t < DT; ++t) to[t] = __builtin_amdgcn_raw_buffer_load_b128(r, at + 1024 * t, 0, kNonTemporal);
    };
    auto load_k = [&](int u) {
        load_unit(rk, a.k, u);
        rs = sc[min((u * kUnit + 16 * (lane & 3)) >> a.shift, (int)nblk - 1)];
    };
    auto load_v = [&](int u) { load_unit(rv, a.v, u); };
    if (u0 + w < u1) {
        load_k(u0 + w);
        load_v(u0 + w);
    }
    __builtin_amdgcn_sched_barrier(0);

    // the column's query, and the first key that it does not see
    half8 qh[NI][2], ql[NI][2];
    float f;
    int lim;
    {
        const int r = r0 + min(n, nr - 1), hh = r / a.L, l = r - hh * a.L;
        const QT *row = (const QT *)a.q + b * a.q_sb + (kvh * G + hh) * a.q_sh + l * a.q_sl;
        QueryRow<QT, NI> q;
        q.load(row, a.D, a.q_vec, g);
        f = query_operands<QT, NI>(q, row, a.D, a.q_vec, g, qh, ql) * a.scale * kLog2e;
        lim = n < nr ? (a.causal ? len - a.L + l + 1 : len) : 0;
    }
    const int lim_all = a.causal ? len - a.L + 1 : len;  // keys below it are seen by every row

    float m = -INFINITY, mv = -INFINITY, lsum = 0.0f;  // running max of s and of s + c, sum of 2^(s - m)
    f32x4 acc[DT];                                     // sum of 2^(s + c - mv) code
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // The softmax step over 64 keys from k0 on: c holds the column's products with the codes of keys 16 kb + 4g + i,
    // ksc and vexp(kb, i) a key's scale and V exponent (PER_KEY: they differ within a kb); every key at or above
    // `end` is not there.  Leaves p' as operands and rescales the sums.
    f32x4 c[4];
    half8 ph[2], pl[2];
    auto softmax = [&](auto per_key, int k0, int end, auto &&ksc, auto &&vexp) {
        constexpr bool PER_KEY = decltype(per_key)::value;
        const bool all = !PER_KEY && k0 + kUnit <= min(lim_all, end);
        float cm = -INFINITY, cv = -INFINITY;
        if (all) {
            // every row sees every key: the scales are positive, so a kb's largest s is its largest product's
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const float s = fmaxf(fmaxf(c[kb][0], c[kb][1]), fmaxf(c[kb][2], c[kb][3])) * (f * ksc(kb, 0));
                cm = fmaxf(cm, s);
                cv = fmaxf(cv, s + vexp(kb, 0));
            }
        } else {
#pragma unroll
            for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s = c[kb][i] * (f * ksc(kb, i));
                    c[kb][i] = k0 + 16 * kb + 4 * g + i < min(lim, end) ? s : -INFINITY;
                    cm = fmaxf(cm, c[kb][i]);
                    cv = fmaxf(cv, c[kb][i] + vexp(kb, i));
                }
        }
        const float mn = fmaxf(m, max_g(cm)), vn = fmaxf(mv, max_g(cv));
        const float ms = mn == -INFINITY ? 0.0f : mn;
        const float alpha = mn == -INFINITY ? 1.0f : fast_exp2(m - mn);
        const float beta = vn == -INFINITY ? 1.0f : fast_exp2(mv - vn);
        const float shift = (vn == -INFINITY ? 0.0f : vn) - ms;
        m = mn;
        mv = vn;
        float sum = 0.0f;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            const float fk = f * ksc(kb, 0);
            float up = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = fast_exp2(all ? fmaf(c[kb][i], fk, -ms) : c[kb][i] - ms);
                sum += p;
                // 2^(c - r): where it passes 2^100, p is 0 or next to it; a NaN (a block that holds one) stays
                if (i == 0 || PER_KEY) {
                    const float e = vexp(kb, i) - shift;
                    up = fast_exp2(e > 100.0f ? 100.0f : e);
                }
                float pv = p * up;
                if (!all) pv = p == 0.0f ? 0.0f : pv;  // (a key that is not seen adds nothing, NaN or not)
                const int at = 4 * (kb & 1) + i;
                const _Float16 hi = (_Float16)pv;
                ph[kb >> 1][at] = hi;
                if constexpr (F32) pl[kb >> 1][at] = (_Float16)(pv - (float)hi);
            }
        }
        lsum = fmaf(lsum, alpha, sum_g(sum));
        if (__builtin_amdgcn_ballot_w64(beta != 1.0f) != 0) {
#pragma unroll
            for (int t = 0; t < DT; ++t) acc[t] *= beta;
        }
    };

    float sk[4], ev[4];
    auto scores = [&]() {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            sk[kb] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(rs), kb));
            ev[kb] = exponent_bits(__builtin_amdgcn_readlane(__float_as_uint(rs), 4 + kb));
            __builtin_amdgcn_sched_barrier(0);  // (one tile's operands at a time: registers)
            c[kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const half8 ka = decode8<E4M3>(rk[kb * NI + i][2 * j], rk[kb * NI + i][2 * j + 1]);
                    if constexpr (F32) c[kb] = mma(ka, ql[i][j], c[kb]);
                    c[kb] = mma(ka, qh[i][j], c[kb]);
                }
        }
    };
    auto values = [&]() {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const half8 va = decode8<E4M3>(rv[t][2 * j], rv[t][2 * j + 1]);
                if constexpr (F32) acc[t] = mma(va, pl[j], acc[t]);
                acc[t] = mma(va, ph[j], acc[t]);
            }
        }
    };
    // the next unit's K is on its way during the softmax and P.V, its V during the next scores
    for (int u = u0 + w; u < u1; u += W) {
        scores();
        load_k(u + W);
        softmax(std::false_type{}, u * kUnit, full, [&](int kb, int) { return sk[kb]; }, [&](int kb, int) { return ev[kb]; });
        values();
        load_v(u + W);
    }

    // ---- the tail: by the last split that has units, as its next ones ----
    const int nu = max(held - u0, 0);
    const bool mine = full == 0 ? blockIdx.y == 0 : nu > 0 && held * kUnit >= full;
    const int room = max(1 << a.shift, kUnit);  // tokens of a plane of operands
    for (int tu = 0; mine && tu * kUnit < tail; ++tu) {
        if ((nu + tu) % W != w) continue;
        const int t0 = tu * kUnit;
        const _Float16 *kt = a.kt + (bg * 2 * room + t0) * Dp + 16 * lane, *vt = a.vt + (bg * 2 * room + t0) * Dp + 16 * lane;
        const int64_t lo_at = (int64_t)room * Dp;
        f32x4 ksc[4], vex[4];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            ksc[kb] = *(const f32x4 *)(a.kts + bg * room + t0 + 16 * kb + 4 * g);
            const f32x4 vs = *(const f32x4 *)(a.vts + bg * room + t0 + 16 * kb + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) vex[kb][i] = exponent_bits(__float_as_uint(vs[i]));
            c[kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (kb == 2) __builtin_amdgcn_sched_barrier(0);  // (two tiles' operands at a time: registers)
            if (t0 + 16 * kb >= tail) continue;
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const half8 hi = *(const half8 *)(kt + kb * 16 * Dp + 1024 * i + 8 * j);
                    const half8 lo = *(const half8 *)(kt + lo_at + kb * 16 * Dp + 1024 * i + 8 * j);
                    if constexpr (F32) c[kb] = mma(hi, ql[i][j], c[kb]);
                    c[kb] = mma(lo, qh[i][j], c[kb]);
                    c[kb] = mma(hi, qh[i][j], c[kb]);
                }
        }
        softmax(std::true_type{}, full + t0, len, [&](int kb, int i) { return ksc[kb][i]; }, [&](int kb, int i) { return vex[kb][i]; });
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (j == 0 && t % 4 == 0) __builtin_amdgcn_sched_barrier(0);
                if (t0 + 32 * j >= tail) continue;  // (operand j: tokens 32 j .. +31)
                const half8 hi = *(const half8 *)(vt + 1024 * t + 8 * j), lo = *(const half8 *)(vt + lo_at + 1024 * t + 8 * j);
                if constexpr (F32) acc[t] = mma(hi, pl[j], acc[t]);
                acc[t] = mma(lo, ph[j], acc[t]);
                acc[t] = mma(hi, ph[j], acc[t]);
            }
    }

    // ---- join the wavefronts, in order ----
    if (g == 0) {
        s_m[w][n] = m;
        s_l[w][n] = lsum;
    }
    __syncthreads();
    if (threadIdx.x < kColumns) {
        const int col = threadIdx.x;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int ww = 0; ww < W; ++ww) M = fmaxf(M, s_m[ww][col]);
#pragma unroll
        for (int ww = 0; ww < W; ++ww) {
            const float lw = s_l[ww][col];
            L += s_m[ww][col] == -INFINITY ? (lw != lw ? lw : 0.0f) : fast_exp2(s_m[ww][col] - M) * lw;
        }
        s_M[col] = M;
        s_L[col] = L;
    }
    __syncthreads();
    // the second half of the waves leave theirs, the first add their own
#pragma unroll
    for (int half = 1; half >= 0; --half) {
        if (w / (W / 2) == half && n < nr) {
            const float M = s_M[n];
            const float to = mv == -INFINITY ? 0.0f : fast_exp2(mv - (M == -INFINITY ? 0.0f : M));
            const bool bad = lsum != lsum;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                f32x4 y = acc[t] * to;
                if (bad) y = f32x4{NAN, NAN, NAN, NAN};
                f32x4 *o = (f32x4 *)&s_o[(w % (W / 2) * nr + n) * OP + 16 * t + 4 * g];
                *o = half == 0 ? *o + y : y;
            }
        }
        __syncthreads();
    }
    const int64_t row0 = (b * a.H + kvh * G) * a.L + r0;
    for (int e = threadIdx.x; e < nr * Dp; e += 64 * W) {
        const int col = e / Dp, d = e - col * Dp;
        const float M = s_M[col], L = s_L[col];
        float o = 0.0f;
#pragma unroll
        for (int h = 0; h < W / 2; ++h) o += s_o[(h * nr + col) * OP + d];
        const int64_t row = row0 + col;
        if (a.nsplit == 1) {
            if (d < a.D) ((QT *)a.o)[row * a.D + d] = (QT)(L == 0.0f ? 0.0f : o / L);
            if (a.lse && d == 0) a.lse[row] = L == 0.0f ? INFINITY : (M + log2f(L)) * kLn2;
        } else {
            const int64_t pr = row * a.nsplit + blockIdx.y;
            a.part_o[pr * Dp + d] = o;
            if (d == 0) {
                a.part_ml[2 * pr] = M;
                a.part_ml[2 * pr + 1] = L;
            }
        }
    }
    if (a.nsplit == 1) return;
    // every split writes its partial; the last one to arrive joins them (partials and counters are uncached)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        s_last = __hip_atomic_fetch_add(&a.counters[x], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.nsplit - 1;
    __syncthreads();
    if (!s_last) return;
    merge_splits<QT, NI, W>(a, row0, nr, s_o);
    if (threadIdx.x == 0) __hip_atomic_store(&a.counters[x], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The kernel for head sizes padded to Dp and workgroups of 4 or (Dp up to 128) 8 wavefronts.
template <typename QT>
inline const void *attn_kernel(int Dp, bool e4m3, int waves) {
#define GT_K(NI, W) (e4m3 ? (const void *)attn_kv_blocks_kernel<QT, NI, true, W> : (const void *)attn_kv_blocks_kernel<QT, NI, false, W>)
    if (Dp == 256) return GT_K(4, 4);
    if (waves == 8) return Dp == 64 ? GT_K(1, 8) : GT_K(2, 8);
    return Dp == 64 ? GT_K(1, 4) : GT_K(2, 4);
#undef GT_K
}

const void *attn_kernel_f16(int Dp, bool e4m3, int waves);
const void *attn_kernel_bf16(int Dp, bool e4m3, int waves);
const void *attn_kernel_f32(int Dp, bool e4m3, int waves);

}  // namespace gtkvb
