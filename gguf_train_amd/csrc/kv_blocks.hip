// The 8-bit block cache (kv_blocks.h): appending tokens (quantizing the blocks that become full) and reading
// back the values that it stands for.
//
// Append, bound by HBM (the rows once, a byte per value back): a workgroup owns a block of one sequence and
// head.  It reads the block's rows twice, for the largest magnitude and to quantize, the second time from the
// caches (a block of 32 tokens and 128 dims is 8 KiB of float16).
// Read, bound by HBM (mostly the values written): a workgroup stages a unit of 64 tokens' codes in LDS, from
// which each thread gathers 8 dims of a token.

#include "gt_internal.h"
#include "kv_blocks.h"

#include <algorithm>

namespace {

using namespace gtkvb;

constexpr int kThreads = 256;

template <typename T>
__device__ inline float to_f(T x) {
    return (float)x;
}
// A finite value stays finite: amax rounds up to a code's value, past float16's largest for amax near it.
template <typename T>
__device__ inline T from_f(float x) {
    if constexpr (__is_same(T, _Float16)) x = fabsf(x) < INFINITY && fabsf(x) > 65504.0f ? copysignf(65504.0f, x) : x;
    return (T)x;
}

// 16 dims of a row from d0 on as float32, zeros from D on; VEC: contiguous, 16-byte aligned, D % 16 == 0.
template <typename T, bool VEC>
__device__ inline void load16(const T *row, int64_t sd, int d0, int D, float *v) {
    if constexpr (VEC) {
        struct alignas(16) P {
            T e[16 / sizeof(T)];
        };
        constexpr int PER = 16 / sizeof(T);
        if (d0 >= D) {  // padding
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = 0.0f;
            return;
        }
#pragma unroll
        for (int j = 0; j < 16 / PER; ++j) {
            const P p = *(const P *)(row + d0 + j * PER);
#pragma unroll
            for (int e = 0; e < PER; ++e) v[j * PER + e] = to_f(p.e[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = d0 + e < D ? to_f(row[(int64_t)(d0 + e) * sd]) : 0.0f;
    }
}

// Four values already divided by the scale, as codes (round to nearest even).
template <bool E4M3>
__device__ inline uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
        return (uint32_t)w;
    } else {
        auto q = [](float x) { return (uint32_t)(int)rintf(x) & 0xffu; };
        return q(a) | q(b) << 8 | q(c) << 16 | q(d) << 24;
    }
}

struct AppendArgs {
    const void *src[2];
    int64_t st[2][4];  // element strides (B, Hkv, T, D)
    uint8_t *codes[2];
    float *scales[2], *tail[2];
    const int32_t *pos;    // tokens held before, per sequence; null: none
    const int32_t *count;  // tokens appended, per sequence; null: T
    int32_t *pos_next;     // tokens held afterwards, or null
    int T, Hkv, N, D, Dp;
    int64_t units;         // of 64 tokens per sequence and head
};

// grid: (blocks that an append can fill, at least 1, B * Hkv, K and V)
template <typename T, bool E4M3, bool VEC>
__global__ __launch_bounds__(kThreads) void kv_blocks_append_kernel(AppendArgs a) {
    const int z = blockIdx.z, N = a.N, D = a.D, Dp = a.Dp, tid = threadIdx.x;
    const int64_t bg = blockIdx.y, b = bg / a.Hkv, g = bg - b * a.Hkv;
    const int held = a.pos ? a.pos[b] : 0, more = a.count ? a.count[b] : a.T;
    const int first = held / N, whole = (held + more) / N;  // whole: blocks full afterwards
    const int blk = first + (int)blockIdx.x;
    const T *src = (const T *)a.src[z] + b * a.st[z][0] + g * a.st[z][1];
    float *tail = a.tail[z] + bg * N * D;
    __shared__ float s_max[kThreads / 64];
    if (a.pos_next && tid == 0 && g == 0 && z == 0 && blockIdx.x == 0) a.pos_next[b] = held + more;

    // 16 dims from d0 on of the block's token t: from the tail, where they have been waiting, or from the source
    auto load = [&](int t, int d0, float *v) {
        const int p = blk * N + t;
        if (p < held) {
            const float *row = tail + (int64_t)t * D;
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = d0 + e < D ? row[d0 + e] : 0.0f;
        } else {
            load16<T, VEC>(src + (int64_t)(p - held) * a.st[z][2], a.st[z][3], d0, D, v);
        }
    };
    const int chunks = Dp / 16;
    if (blk < whole) {
        float amax = 0.0f;
        bool odd = false;  // an infinity or NaN among them
        for (int i = tid; i < N * chunks; i += kThreads) {
            float v[16];
            load(i / chunks, i % chunks * 16, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                amax = fmaxf(amax, fabsf(v[e]));
                odd = odd || !(fabsf(v[e]) < INFINITY);
            }
        }
        amax = odd ? INFINITY : amax;
        for (int m = 32; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));
        if ((tid & 63) == 0) s_max[tid >> 6] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        const bool bad = amax == INFINITY;
        const int e2 = bad ? 0 : scale_exponent(__float_as_uint(amax), E4M3);
        // (a block with an infinity or NaN has no scale: all of it reads as NaN)
        if (tid == 0) a.scales[z][bg * (a.units * kUnit / N) + blk] = bad ? NAN : __uint_as_float((uint32_t)(e2 + 127) << 23);
        const float inv = bad ? 0.0f : __uint_as_float((uint32_t)(127 - e2) << 23);
        uint8_t *codes = a.codes[z] + bg * a.units * kUnit * Dp;
        if (z == 0) {
            for (int i = tid; i < N * chunks; i += kThreads) {
                // 16 threads next to each other write the 16 tokens of a tile's chunk
                const int t = (i / (16 * chunks)) * 16 + (i & 15), c = (i / 16) % chunks;
                float v[16];
                load(t, 16 * c, v);
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    w[j] = bad ? 0u : encode4<E4M3>(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv);
                *(uint4 *)(codes + k_at((int64_t)blk * N + t, 16 * c, Dp)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            // a dim of four tokens is four bytes in a row
            for (int i = tid; i < N / 4 * Dp; i += kThreads) {
                const int d = i % Dp, t = i / Dp * 4;
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int p = blk * N + t + j;
                    v[j] = d >= D ? 0.0f
                           : p < held ? tail[(int64_t)(t + j) * D + d]
                                      : to_f(src[(int64_t)(p - held) * a.st[z][2] + (int64_t)d * a.st[z][3]]);
                }
                const uint32_t w = bad ? 0u : encode4<E4M3>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                *(uint32_t *)(codes + v_at((int64_t)blk * N + t, d, Dp)) = w;
            }
        }
    }
    if (blockIdx.x != 0) return;
    // the tokens after the last whole block; the old tail has been read above
    __syncthreads();
    const int from = max(held, whole * N), rows = held + more - from;
    for (int i = tid; i < rows * D; i += kThreads) {
        const int r = i / D, d = i - r * D;
        tail[(int64_t)(from - whole * N + r) * D + d] = to_f(src[(int64_t)(from + r - held) * a.st[z][2] + (int64_t)d * a.st[z][3]]);
    }
}

// 8 codes as values.
template <bool E4M3>
__device__ inline void decode4(uint32_t w, float *v) {
    if constexpr (E4M3) {
        v[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
        v[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
        v[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
        v[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)(int8_t)(w >> (8 * j));
    }
}

struct ReadArgs {
    const uint8_t *codes[2];
    const float *scales[2], *tail[2];
    void *out[2];            // dense (B, Hkv, rows, D)
    const int32_t *len;      // tokens held per sequence
    const int64_t *kept;     // (B, Hkv, rows) tokens to read, or null: 0, 1, ...
    int rows, Hkv, N, D, Dp;
    int64_t units;
};

// grid: (units of 64 rows, B * Hkv, K and V); rows past what is held are zero
template <typename TO, bool E4M3, bool GATHER>
__global__ __launch_bounds__(kThreads) void kv_blocks_read_kernel(ReadArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t raw[GATHER ? 16 : kUnit * kMaxDim];
    const int z = blockIdx.z, N = a.N, D = a.D, Dp = a.Dp, tid = threadIdx.x;
    const int64_t bg = blockIdx.y, b = bg / a.Hkv;
    const int r0 = blockIdx.x * kUnit, held = a.len[b], full = held / N * N;
    const uint8_t *codes = a.codes[z] + bg * a.units * kUnit * Dp;
    const float *scales = a.scales[z] + bg * (a.units * kUnit / N);
    const float *tail = a.tail[z] + bg * N * D;
    TO *out = (TO *)a.out[z] + bg * (int64_t)a.rows * D;
    if constexpr (!GATHER) {
        if (r0 < full) {
            for (int i = tid; i < kUnit * Dp / 16; i += kThreads)
                *(uint4 *)(raw + 16 * i) = *(const uint4 *)(codes + (int64_t)r0 * Dp + 16 * i);
        }
        __syncthreads();
    }
    const int groups = Dp / 8, n = min(kUnit, a.rows - r0);
    for (int i = tid; i < n * groups; i += kThreads) {
        const int r = i / groups, d0 = i % groups * 8;
        if (d0 >= D) continue;
        int64_t t = r0 + r;
        if constexpr (GATHER) t = a.kept[bg * a.rows + t];
        float v[8];
        if (t < 0 || t >= held) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        } else if (t >= full) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = d0 + e < D ? tail[(t - full) * D + d0 + e] : 0.0f;
        } else {
            uint32_t w[2];
            const uint8_t *base = GATHER ? codes : raw;
            const int64_t tt = GATHER ? t : r;
            if (z == 0) {
                const uint2 q = *(const uint2 *)(base + k_at(tt, d0, Dp));
                w[0] = q.x;
                w[1] = q.y;
            } else {
                const uint8_t *p = base + v_at(tt, d0, Dp);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    w[j] = p[64 * j] | (uint32_t)p[64 * j + 16] << 8 | (uint32_t)p[64 * j + 32] << 16 | (uint32_t)p[64 * j + 48] << 24;
            }
            const float s = scales[t / N];
            decode4<E4M3>(w[0], v);
            decode4<E4M3>(w[1], v + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= s;
        }
        TO *o = out + (int64_t)(r0 + r) * D + d0;
        if (D % 8 == 0) {
            struct alignas(sizeof(TO) * 8 < 16 ? sizeof(TO) * 8 : 16) P {
                TO e[8];
            } p;
#pragma unroll
            for (int e = 0; e < 8; ++e) p.e[e] = from_f<TO>(v[e]);
            *(P *)o = p;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (d0 + e < D) o[e] = from_f<TO>(v[e]);
        }
    }
}

template <typename T>
hipError_t launch_append(const AppendArgs &a, bool e4m3, bool vec, dim3 grid, hipStream_t s) {
    if (e4m3) {
        if (vec) hipLaunchKernelGGL((kv_blocks_append_kernel<T, true, true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((kv_blocks_append_kernel<T, true, false>), grid, dim3(kThreads), 0, s, a);
    } else {
        if (vec) hipLaunchKernelGGL((kv_blocks_append_kernel<T, false, true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((kv_blocks_append_kernel<T, false, false>), grid, dim3(kThreads), 0, s, a);
    }
    return hipGetLastError();
}

template <typename TO>
hipError_t launch_read(const ReadArgs &a, bool e4m3, dim3 grid, hipStream_t s) {
    if (a.kept) {
        if (e4m3) hipLaunchKernelGGL((kv_blocks_read_kernel<TO, true, true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((kv_blocks_read_kernel<TO, false, true>), grid, dim3(kThreads), 0, s, a);
    } else {
        if (e4m3) hipLaunchKernelGGL((kv_blocks_read_kernel<TO, true, false>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((kv_blocks_read_kernel<TO, false, false>), grid, dim3(kThreads), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t gt_launch_kv_blocks_append(const gt_kv_blocks &c, const void *const *src, int src_dtype,
                                      const int64_t *const *strides, const int32_t *pos, const int32_t *count,
                                      int32_t *pos_next, int64_t T, int64_t blocks, hipStream_t s) {
    AppendArgs a{};
    bool vec = c.D % 16 == 0;
    const int64_t es = src_dtype == GT_F32 ? 4 : 2;
    for (int z = 0; z < 2; ++z) {
        a.src[z] = src[z];
        for (int i = 0; i < 4; ++i) a.st[z][i] = strides[z][i];
        a.codes[z] = (uint8_t *)c.codes[z];
        a.scales[z] = c.scales[z];
        a.tail[z] = c.tail[z];
        vec = vec && strides[z][3] == 1 && (uintptr_t)src[z] % 16 == 0;
        for (int i = 0; i < 3; ++i) vec = vec && strides[z][i] * es % 16 == 0;
    }
    a.pos = pos;
    a.count = count;
    a.pos_next = pos_next;
    a.T = (int)T;
    a.Hkv = (int)c.Hkv;
    a.N = c.N;
    a.D = (int)c.D;
    a.Dp = c.Dp;
    a.units = c.units;
    const int64_t bg = c.B * c.Hkv;
    if (bg > 65535 || blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)std::max<int64_t>(blocks, 1), (unsigned)bg, 2);
    switch (src_dtype) {
        case GT_F32: return launch_append<float>(a, c.e4m3, vec, grid, s);
        case GT_F16: return launch_append<_Float16>(a, c.e4m3, vec, grid, s);
        case GT_BF16: return launch_append<__bf16>(a, c.e4m3, vec, grid, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t gt_launch_kv_blocks_read(const gt_kv_blocks &c, const int32_t *len, const int64_t *kept, int64_t rows,
                                    void *k, void *v, int dtype, hipStream_t s) {
    if (rows <= 0) return hipSuccess;
    ReadArgs a{};
    for (int z = 0; z < 2; ++z) {
        a.codes[z] = (const uint8_t *)c.codes[z];
        a.scales[z] = c.scales[z];
        a.tail[z] = c.tail[z];
    }
    a.out[0] = k;
    a.out[1] = v;
    a.len = len;
    a.kept = kept;
    a.rows = (int)rows;
    a.Hkv = (int)c.Hkv;
    a.N = c.N;
    a.D = (int)c.D;
    a.Dp = c.Dp;
    a.units = c.units;
    const int64_t bg = c.B * c.Hkv;
    if (bg > 65535) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)((rows + kUnit - 1) / kUnit), (unsigned)bg, 2);
    switch (dtype) {
        case GT_F32: return launch_read<float>(a, c.e4m3, grid, s);
        case GT_F16: return launch_read<_Float16>(a, c.e4m3, grid, s);
        case GT_BF16: return launch_read<__bf16>(a, c.e4m3, grid, s);
        default: return hipErrorInvalidValue;
    }
}
