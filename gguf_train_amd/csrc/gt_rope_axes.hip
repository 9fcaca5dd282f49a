// Rotary positions with several axes (time, height, width of an image or video patch).  Pair i < n_dims/2
// of the row at token (b, s) turns by
//   angle = freq_scale * pos[axis(i), b, s] * freq_base^(-2 i / n_dims),
// the frequency that one-axis RoPE gives the pair, at the position of the axis the pair belongs to:
// the axes' sections one after the other, or (interleaved) pair i to axis i % A while i / A is below
// that axis' section, to axis 0 otherwise.  y_lo = x_lo c - x_hi s, y_hi = x_lo s + x_hi c; the backward
// is the inverse rotation, (c, -s).  NORMAL pairs elements (2i, 2i+1), NeoX (i, i + n_dims/2); elements from
// n_dims on pass through.
//
// Angles are formed in float64 as turns, angle / 2 pi, whose whole part is dropped before the float32
// sincospif: a float32 angle of position 60000 is off by 2^-9 and a bfloat16 result by a step.  The
// rotation runs in float32 (float64 inputs: in float64) and is rounded once.
//
// Bound: HBM, each element read and written once.  A workgroup owns R rows (tokens) of a chunk of the
// heads: their angles are formed once, into LDS, and turn every head's rows, so a thread spends about four
// angles (some 100 instructions each) on the 2 H 16-byte pieces of its heads, and no table passes through
// memory.  A thread loads both halves of its pairs, so each byte is requested once.  bfloat16 D128 H64 S8192 (268 MB):
// 50 us, 5.4 TB/s; H32 S4096 (67 MB) 14 us; a decode step 4.6 us, the latency of one workgroup.

#include "gt_internal.h"
#include "gt_rope_math.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int kThreads = 256;
constexpr int kAngles = 512;       // angles of a workgroup's rows, about
constexpr int64_t kWorkgroups = 2048;  // enough workgroups to fill the GPU several times over
// (us for 256, 512 and 1024 angles: bfloat16 D128 H32 S4096 15.2, 14.2, 16.5; B2 H16 S2048 9.7, 9.7, 12.7; H64 S8192 52,
// 50, 48; B2 H32 S4096 25.4, 24.4, 25.8.  4096 workgroups with 512: 16.1, 13.6, 47, 23.5)

struct Args {
    const void *x;
    int64_t sb, sh, ss, sd;  // element strides of x (B, H, S, D)
    void *y;                 // dense (B, H, S, D)
    const void *pos;
    int64_t pa, pb, ps;  // element strides of pos (A, B, S)
    double log2_step;    // the frequency of pair i is first * 2^(-i * log2_step) turns per position
    double first;
    int64_t rows;  // B * S
    int S, H, D, half, rows_per, heads_per;
    int axes, interleaved;
    int sections[4];
    int neox, backward;
};

template <typename T>
struct Wide {
    typedef float F;
    typedef float2 F2;
};
template <>
struct Wide<double> {
    typedef double F;
    typedef double2 F2;
};

__device__ inline int axis_of(const Args &a, int i) {
    if (a.interleaved) {
        const int n = i % a.axes;
        return i / a.axes < a.sections[n] ? n : 0;
    }
    int n = 0, end = a.sections[0];
    while (i >= end) end += a.sections[++n];  // i < half, the sections' sum
    return n;
}

__device__ inline float2 sin_cos_turns(double t, float2) {
    float s, c;
    sincospif(2.0f * (float)t, &s, &c);  // |2t| <= 1
    return make_float2(c, s);
}
__device__ inline double2 sin_cos_turns(double t, double2) {
    double s, c;
    sincospi(2.0 * t, &s, &c);
    return make_double2(c, s);
}

__device__ inline float rot_lo(float lo, float hi, float2 cs) { return rope_rot_lo(lo, hi, cs); }
__device__ inline float rot_hi(float lo, float hi, float2 cs) { return rope_rot_hi(lo, hi, cs); }
__device__ inline double rot_lo(double lo, double hi, double2 cs) { return fma(lo, cs.x, -(hi * cs.y)); }
__device__ inline double rot_hi(double lo, double hi, double2 cs) { return fma(hi, cs.x, lo * cs.y); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Piece {
    T e[VEC];
};

// P: the positions' type.  Piece u of a row: u < half / VEC is VEC pairs, the elements [a, a + VEC) and [b, b +
// VEC) (NeoX: the pairs' lower and upper halves; NORMAL: the pairs in order); the others pass through.
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(Args a) {
    typedef typename Wide<T>::F F;
    typedef typename Wide<T>::F2 F2;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    double *freq = (double *)lds;                                      // [half]
    F2 *turn = (F2 *)(lds + (size_t)((a.half + 1) & ~1) * sizeof(double));  // [rows_per][half]
    int64_t *xoff = (int64_t *)(turn + (size_t)a.rows_per * a.half);   // [rows_per]
    int64_t *yoff = xoff + a.rows_per;
    const int64_t r0 = (int64_t)blockIdx.x * a.rows_per;
    const int nr = (int)min((int64_t)a.rows_per, a.rows - r0);
    for (int i = threadIdx.x; i < a.half; i += kThreads) freq[i] = a.first * exp2(-(double)i * a.log2_step);
    for (int r = threadIdx.x; r < nr; r += kThreads) {
        const int64_t b = (r0 + r) / a.S, s = r0 + r - b * a.S;
        xoff[r] = b * a.sb + s * a.ss;
        yoff[r] = (b * a.H * a.S + s) * a.D;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nr * a.half; e += kThreads) {
        const int r = e / a.half, i = e - r * a.half;
        const int64_t b = (r0 + r) / a.S, s = r0 + r - b * a.S;
        double t = (double)((const P *)a.pos)[axis_of(a, i) * a.pa + b * a.pb + s * a.ps] * freq[i];
        t -= rint(t);
        F2 cs = sin_cos_turns(t, F2{});
        if (a.backward) cs.y = -cs.y;
        turn[e] = cs;
    }
    __syncthreads();
    const int pairs = a.half / VEC, units = pairs + (a.D - 2 * a.half) / VEC;
    const int h0 = blockIdx.y * a.heads_per, nh = min(a.heads_per, a.H - h0);
    for (int n = threadIdx.x; n < nh * nr * units; n += kThreads) {
        const int hr = n / units, u = n - hr * units, h = hr / nr, r = hr - h * nr;
        const T *xr = (const T *)a.x + xoff[r] + (h0 + h) * a.sh;
        T *yr = (T *)a.y + yoff[r] + (int64_t)(h0 + h) * a.S * a.D;
        typedef Piece<T, VEC> V;
        auto load = [&](int d) {
            V v;
            if constexpr (VEC == 1) v.e[0] = xr[d * a.sd];
            else v = *(const V *)(xr + d);
            return v;
        };
        if (u >= pairs) {
            const int d = 2 * a.half + (u - pairs) * VEC;
            *(V *)(yr + d) = load(d);
            continue;
        }
        const int p0 = u * VEC, lo = a.neox ? p0 : 2 * p0, hi = a.neox ? p0 + a.half : 2 * p0 + VEC;
        V va = load(lo), vb = load(hi);
        const F2 *cs = turn + r * a.half + p0;
        V oa, ob;
        if (a.neox) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                oa.e[j] = (T)rot_lo((F)va.e[j], (F)vb.e[j], cs[j]);
                ob.e[j] = (T)rot_hi((F)va.e[j], (F)vb.e[j], cs[j]);
            }
        } else if constexpr (VEC == 1) {
            oa.e[0] = (T)rot_lo((F)va.e[0], (F)vb.e[0], cs[0]);
            ob.e[0] = (T)rot_hi((F)va.e[0], (F)vb.e[0], cs[0]);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
                oa.e[j] = (T)rot_lo((F)va.e[j], (F)va.e[j + 1], cs[j / 2]);
                oa.e[j + 1] = (T)rot_hi((F)va.e[j], (F)va.e[j + 1], cs[j / 2]);
                ob.e[j] = (T)rot_lo((F)vb.e[j], (F)vb.e[j + 1], cs[VEC / 2 + j / 2]);
                ob.e[j + 1] = (T)rot_hi((F)vb.e[j], (F)vb.e[j + 1], cs[VEC / 2 + j / 2]);
            }
        }
        *(V *)(yr + lo) = oa;
        *(V *)(yr + hi) = ob;
    }
}

template <typename T, typename P, int VEC>
hipError_t launch(const Args &a, size_t lds, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((rope_axes_kernel<T, P, VEC>), grid, dim3(kThreads), lds, s, a);
    return hipGetLastError();
}

template <typename T, typename P>
hipError_t dispatch(Args a, int64_t B, hipStream_t s) {
    // rows and heads of a workgroup: about kAngles angles for as many heads as leave the GPU filled
    a.rows = B * a.S;
    a.rows_per = (int)std::min<int64_t>(a.rows, std::max(1, kAngles / a.half));
    const int64_t tiles = (a.rows + a.rows_per - 1) / a.rows_per;
    if (tiles > 0x7fffffff) return hipErrorInvalidConfiguration;
    int64_t chunks = std::min<int64_t>(a.H, std::max<int64_t>(1, kWorkgroups / tiles));
    // (nr * heads * pieces stays an int: at most a few thousand rows' elements)
    chunks = std::max<int64_t>(chunks, ((int64_t)a.rows_per * a.H * a.D + (1 << 30) - 1) >> 30);
    chunks = std::max<int64_t>(chunks, (a.H + 65534) / 65535);
    a.heads_per = (int)((a.H + chunks - 1) / chunks);
    const int64_t gy = (a.H + a.heads_per - 1) / a.heads_per;
    if (gy > 65535) return hipErrorInvalidConfiguration;
    typedef typename Wide<T>::F2 F2;
    const size_t lds = (size_t)((a.half + 1) & ~1) * sizeof(double) + (size_t)a.rows_per * a.half * sizeof(F2) +
                       (size_t)a.rows_per * 2 * sizeof(int64_t);
    const dim3 grid((unsigned)tiles, (unsigned)gy);
    // pieces of 16 bytes where every one is aligned and on one side of each border
    constexpr int V = 16 / (int)sizeof(T);
    const bool vec = a.sd == 1 && a.half % V == 0 && a.D % V == 0 && a.sb % V == 0 && a.sh % V == 0 && a.ss % V == 0 &&
                     (uintptr_t)a.x % 16 == 0;
    if (vec) return launch<T, P, V>(a, lds, grid, s);
    return launch<T, P, 1>(a, lds, grid, s);
}

template <typename T>
hipError_t dispatch_pos(const Args &a, int pos_dtype, int64_t B, hipStream_t s) {
    switch (pos_dtype) {
        case GT_I32: return dispatch<T, int32_t>(a, B, s);
        case GT_I64: return dispatch<T, int64_t>(a, B, s);
        case GT_F32: return dispatch<T, float>(a, B, s);
        case GT_F64: return dispatch<T, double>(a, B, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t gt_launch_rope_axes(const gt_rope_axes_args &r, hipStream_t s) {
    if (r.B * r.H * r.S * r.D <= 0) return hipSuccess;
    if (r.S > 0x7fffffff || r.H > 0x7fffffff || r.D > kRopeAxesMaxDim) return hipErrorInvalidValue;
    Args a{};
    a.x = r.x;
    a.sb = r.x_strides[0];
    a.sh = r.x_strides[1];
    a.ss = r.x_strides[2];
    a.sd = r.x_strides[3];
    a.y = r.y;
    a.pos = r.pos;
    a.pa = r.pos_strides[0];
    a.pb = r.pos_strides[1];
    a.ps = r.pos_strides[2];
    a.log2_step = 2.0 * std::log2(r.freq_base) / r.n_dims;
    a.first = r.freq_scale / 6.283185307179586;
    a.S = (int)r.S;
    a.H = (int)r.H;
    a.D = (int)r.D;
    a.half = r.n_dims / 2;
    a.axes = r.n_axes;
    a.interleaved = r.interleaved;
    for (int i = 0; i < r.n_axes; ++i) a.sections[i] = r.sections[i];
    a.neox = r.mode == 2;
    a.backward = r.backward;
    switch (r.dtype) {
        case GT_F32: return dispatch_pos<float>(a, r.pos_dtype, r.B, s);
        case GT_F16: return dispatch_pos<_Float16>(a, r.pos_dtype, r.B, s);
        case GT_BF16: return dispatch_pos<__bf16>(a, r.pos_dtype, r.B, s);
        case GT_F64: return dispatch_pos<double>(a, r.pos_dtype, r.B, s);
        default: return hipErrorInvalidValue;
    }
}
