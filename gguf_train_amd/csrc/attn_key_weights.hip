// The attention weight that a cache's tokens receive: for a call's queries over the cache (B, Hkv, cap, D),
//   a[b, g, t] <- f a[b, g, t] + sum over the group's heads h and the rows l of exp(scale q_hl . k_t - lse_hl),
// the column sums of the softmax that the attention of the same call has just formed, from its log-sum-exp.
//
// Bound: at few rows the keys, read once more (half the attention's bytes, much of it from the caches); at many
// the products.  A wavefront owns 16 TW keys, whose operands stay in registers while it walks the rows in
// columns of 16 (row r = head * L + token): S^T = K.Q^T on v_mfma_f32_16x16x32_f16, exp, a sum per lane, and at
// the end a sum over the 16 lanes of a key's row.  One writer per sum, so no atomics and the same bits each time;
// where few wavefronts meet many rows the columns are split, and a second launch adds the splits in order.
//
// Measured (B4 H32/8 D128 S4096): a float16 cache, one row 9.8 us (3.4 TB/s of keys), int8 and 32 rows of a head 15.7:
// latency, some 8 us before the first column (length, keys, queries, one after the other) and 1 us a column; with
// each tile's products in a branch of its own and a tail's lo operands in registers for every wavefront it was 17.6.
//
// Operands as attn_kv_blocks.h has them: codes are exact in float16; other rows of keys (bfloat16, float32,
// Q8_0 values, a block cache's tail) are divided by their own power of two and enter as float16 hi, or as
// hi + lo where they hold more bits than float16 (float32, Q8_0); float32 queries as hi + lo.

#include "attn_kv_blocks.h"

#include <cmath>
#include <type_traits>

namespace {

using namespace gtkvb;

constexpr int kWaves = 4;

enum Source { kInt8, kE4m3, kF16, kBf16, kF32, kQ8, kAny };  // kAny: float rows not in whole aligned pieces of 16 dims

struct Args {
    const void *q;
    int64_t q_sb, q_sh, q_sl;
    const char *k;  // rows (B, Hkv, cap); the codes of a block cache
    int64_t row_bytes, cap;
    const float *ks;       // a block cache's scales, and its tail's operands and scales
    const _Float16 *kt;
    const float *kts;
    int shift;  // log2 of the tokens of a block
    int64_t units;
    const float *lse;
    const int32_t *len;
    float *sums;   // (B, Hkv, cap)
    float *parts;  // (splits, B, Hkv, max_len), or null: one split writes sums
    int64_t max_len;
    float keep;
    float scale;
    int causal, q_vec, k_dtype;
    int H, Hkv, L, D;
    int col_tiles, span;  // columns of 16 rows in all, and per split
};

// Dims d0 .. d0 + 15 of a row of keys as they lie in memory, from an address inside the row whatever d0 (no branch
// around a load: all of a wavefront's are in flight together), and then as values.
template <int KIND>
struct KeyDims {
    typedef std::conditional_t<KIND == kF32, float, std::conditional_t<KIND == kBf16, __bf16, _Float16>> T;
    gtvec::Dims16<T> piece;
    __device__ void load(const char *row, int d0, int, int D) { piece.load((const T *)row + (d0 < D ? d0 : 0)); }
    __device__ void values(int d0, int D, float *x) const {  // zeros from D on
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = d0 < D ? piece.get(e) : 0.0f;
    }
};
template <>
struct KeyDims<kQ8> {  // half a block of 32: its scale, and 16 codes in steps of 2 bytes
    uint16_t w[8], scale;
    __device__ void load(const char *row, int d0, int, int D) {
        const int d = d0 < D ? d0 : 0;
        const uint8_t *blk = (const uint8_t *)row + (d >> 5) * 34;
        scale = *(const uint16_t *)blk;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = *(const uint16_t *)(blk + 2 + (d & 31) + 2 * e);
    }
    __device__ void values(int d0, int D, float *x) const {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            x[e] = d0 < D ? (float)__builtin_bit_cast(_Float16, scale) * (float)(int8_t)(w[e / 2] >> (8 * (e & 1))) : 0.0f;
    }
};
template <>
struct KeyDims<kAny> {
    float v[16];
    __device__ void load(const char *row, int d0, int dtype, int D) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int d = min(d0 + e, D - 1);
            v[e] = dtype == GT_F32 ? ((const float *)row)[d] : dtype == GT_F16 ? (float)((const _Float16 *)row)[d] : (float)((const __bf16 *)row)[d];
        }
    }
    __device__ void values(int d0, int D, float *x) const {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = d0 + e < D ? v[e] : 0.0f;
    }
};

// The A operands of a key row of which this lane holds dims 16 (4i + g) .. +15, and the row's scale (the same in the
// four lanes).
template <int KIND, int NI>
__device__ inline float key_operands(const KeyDims<KIND> *raw, int D, int g, half8 (*hi)[2], half8 (*lo)[2]) {
    if constexpr (KIND == kF16) {  // its own operand
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const u32x4 w = raw[i].piece.w[j];
                hi[i][j] = __builtin_bit_cast(half8, 16 * (4 * i + g) < D ? w : u32x4{0u, 0u, 0u, 0u});
            }
        return 1.0f;
    }
    float x[NI][16];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        raw[i].values(16 * (4 * i + g), D, x[i]);
#pragma unroll
        for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[i][e]) < INFINITY ? fabsf(x[i][e]) : INFINITY);
    }
    amax = max_g(amax);
    const bool odd = amax == INFINITY;  // (an infinity or NaN: the key's scores are NaN, and no other key's)
    const int e2 = exponent_of(amax);
    const float inv = pow2(-e2);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[i][e] = odd ? 0.0f : x[i][e];
#pragma unroll
        for (int j = 0; j < 2; ++j) split8(x[i] + 8 * j, inv, hi[i][j], lo[i][j]);
    }
    return odd ? NAN : pow2(e2);
}

// grid: (wavefronts' keys / 4, B * Hkv, column splits).  (Two wavefronts a SIMD: without that bound the products' results
// go through accumulation registers, and a float32 cache's kernel takes more than half of a SIMD's registers.)
template <typename QT, int SRC, int NI, int TW>
__global__ __launch_bounds__(64 * kWaves, NI <= 2 ? 2 : 1) void attn_key_weights_kernel(Args a) {
    constexpr bool CODES = SRC == kInt8 || SRC == kE4m3;
    constexpr bool KLO = SRC == kF32 || SRC == kQ8 || SRC == kAny;  // keys of more bits than float16
    constexpr bool QLO = __is_same(QT, float);
    constexpr int Dp = 64 * NI;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t bg = blockIdx.y, b = bg / a.Hkv, kvh = bg - b * a.Hkv;
    const int len = a.len[b], full = CODES ? len >> a.shift << a.shift : 0;
    // (the last keys first: the workgroups with fewer keys than the others)
    const int k0 = ((int)(gridDim.x - 1 - blockIdx.x) * kWaves + w) * 16 * TW;
    if (k0 >= len) return;

    // the keys' operands; the lo ones of a block cache, which only its tail has, wait in LDS (a lane's own)
    half8 kh[TW][NI][2], kl[CODES ? 1 : TW][NI][2];
    __shared__ half8 s_lo[CODES ? kWaves : 1][CODES ? TW : 1][NI][2][64];
    float ksc[TW][4];
    const bool tail = CODES && k0 + 16 * TW > full;
    KeyDims<CODES ? kF32 : SRC> raw[CODES ? 1 : TW][NI];
    if constexpr (!CODES) {
#pragma unroll
        for (int kb = 0; kb < TW; ++kb)
#pragma unroll
            for (int i = 0; i < NI; ++i)  // (tokens that are not there: the last one, left out below)
                raw[kb][i].load(a.k + (bg * a.cap + min(k0 + 16 * kb + n, len - 1)) * a.row_bytes, 16 * (4 * i + g), a.k_dtype, a.D);
    }
#pragma unroll
    for (int kb = 0; kb < TW; ++kb) {
        const int t0 = k0 + 16 * kb;
        if (CODES && t0 < full) {  // (a whole block is a multiple of 16 tokens)
            const uint8_t *p = (const uint8_t *)a.k + bg * a.units * kUnit * Dp + (int64_t)t0 * Dp + 16 * lane;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const u32x4 r = *(const u32x4 *)(p + 1024 * i);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    kh[kb][i][j] = decode8<SRC == kE4m3>(r[2 * j], r[2 * j + 1]);
                    if (tail) s_lo[w][kb][i][j][lane] = half8{0, 0, 0, 0, 0, 0, 0, 0};
                }
            }
            const float s = a.ks[bg * (a.units * kUnit >> a.shift) + (t0 >> a.shift)];
#pragma unroll
            for (int i = 0; i < 4; ++i) ksc[kb][i] = s;
        } else if constexpr (CODES) {
            const int room = max(1 << a.shift, kUnit), at = min(t0 - full, room - 16);  // (the last tiles may hold no token)
            const _Float16 *p = a.kt + (bg * 2 * room + at) * Dp + 16 * lane;
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    kh[kb][i][j] = *(const half8 *)(p + 1024 * i + 8 * j);
                    s_lo[w][kb][i][j][lane] = *(const half8 *)(p + (int64_t)room * Dp + 1024 * i + 8 * j);
                }
            const f32x4 s = *(const f32x4 *)(a.kts + bg * room + at + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) ksc[kb][i] = s[i];
        } else {
            const float s = key_operands<SRC, NI>(raw[kb], a.D, g, kh[kb], kl[CODES ? 0 : kb]);
#pragma unroll
            for (int i = 0; i < 4; ++i) ksc[kb][i] = __shfl(s, 4 * g + i, 64);
        }
    }

    float sum[TW][4];
#pragma unroll
    for (int kb = 0; kb < TW; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[kb][i] = 0.0f;
    const int G = a.H / a.Hkv, rows = G * a.L;
    const int c0 = blockIdx.z * a.span, c1 = min(c0 + a.span, a.col_tiles);
    // a column's query and log-sum-exp, on their way while the column before is worked on
    QueryRow<QT, NI> q;
    const QT *row;
    int lim;
    float lse;
    int hh = (16 * c0 + n) / a.L, l = 16 * c0 + n - hh * a.L;  // the next column's head and token
    const int heads16 = 16 / a.L, tokens16 = 16 - heads16 * a.L;
    auto load = [&]() {
        const int h = min(hh, G - 1);  // (past the last row: some row, which sees no key)
        lim = hh < G ? (a.causal ? len - a.L + l + 1 : len) : 0;
        row = (const QT *)a.q + b * a.q_sb + (kvh * G + h) * a.q_sh + l * a.q_sl;
        q.load(row, a.D, a.q_vec, g);
        lse = a.lse[(b * a.H + kvh * G + h) * a.L + l];
        l += tokens16;
        hh += heads16;
        if (l >= a.L) l -= a.L, ++hh;
    };
    if (c0 < c1) load();
    for (int ct = c0; ct < c1; ++ct) {
        half8 qh[NI][2], ql[NI][2];
        const float f = query_operands<QT, NI>(q, row, a.D, a.q_vec, g, qh, ql) * a.scale * kLog2e, ls = lse * kLog2e;
        const int seen = lim;
        if (ct + 1 < c1) load();
        if (__builtin_amdgcn_ballot_w64(seen > k0) == 0) continue;
        const bool all = __builtin_amdgcn_ballot_w64(seen >= k0 + 16 * TW) == ~0ull;
        // the tiles' products side by side: each tile's own follow one another
        f32x4 c[TW];
#pragma unroll
        for (int kb = 0; kb < TW; ++kb) c[kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        auto products = [&](auto with_lo) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int kb = 0; kb < TW; ++kb) {
                        if constexpr (QLO) c[kb] = mma(kh[kb][i][j], ql[i][j], c[kb]);
                        if constexpr (decltype(with_lo)::value) c[kb] = mma(s_lo[w][kb][i][j][lane], qh[i][j], c[kb]);
                        if constexpr (KLO) c[kb] = mma(kl[kb][i][j], qh[i][j], c[kb]);
                        c[kb] = mma(kh[kb][i][j], qh[i][j], c[kb]);
                    }
        };
        if constexpr (CODES) {
            if (tail) products(std::true_type{});
            else products(std::false_type{});
        } else {
            products(std::false_type{});
        }
#pragma unroll
        for (int kb = 0; kb < TW; ++kb)
#pragma unroll
            for (int i = 0; i < 4; ++i) c[kb][i] = fast_exp2(fmaf(c[kb][i], f * ksc[kb][i], -ls));
        if (all) {
#pragma unroll
            for (int kb = 0; kb < TW; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[kb][i] += c[kb][i];
        } else {
#pragma unroll
            for (int kb = 0; kb < TW; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[kb][i] += k0 + 16 * kb + 4 * g + i < seen ? c[kb][i] : 0.0f;
        }
    }
#pragma unroll
    for (int kb = 0; kb < TW; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float s = sum[kb][i];
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o, 64);
            const int t = k0 + 16 * kb + 4 * g + i;
            if (n != 0 || t >= len) continue;
            if (a.parts) a.parts[((int64_t)blockIdx.z * gridDim.y + bg) * a.max_len + t] = s;
            else {
                float *o = a.sums + bg * a.cap + t;
                *o = a.keep == 0.0f ? s : fmaf(a.keep, *o, s);
            }
        }
}

__global__ void add_parts_kernel(const float *parts, int splits, int64_t max_len, const int32_t *len, float *sums, float keep,
                                 int Hkv, int64_t cap) {
    const int64_t bg = blockIdx.y, t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= len[bg / Hkv]) return;
    float s = 0.0f;
    for (int z = 0; z < splits; ++z) s += parts[((int64_t)z * gridDim.y + bg) * max_len + t];
    float *o = sums + bg * cap + t;
    *o = keep == 0.0f ? s : fmaf(keep, *o, s);
}

template <typename QT, int SRC>
const void *kernel_d(int Dp) {
    switch (Dp) {
        case 64: return (const void *)attn_key_weights_kernel<QT, SRC, 1, 4>;
        case 128: return (const void *)attn_key_weights_kernel<QT, SRC, 2, 4>;
        default: return (const void *)attn_key_weights_kernel<QT, SRC, 4, 2>;
    }
}

template <typename QT>
const void *kernel_src(int src, int Dp) {
    switch (src) {
        case kInt8: return kernel_d<QT, kInt8>(Dp);
        case kE4m3: return kernel_d<QT, kE4m3>(Dp);
        case kF16: return kernel_d<QT, kF16>(Dp);
        case kBf16: return kernel_d<QT, kBf16>(Dp);
        case kF32: return kernel_d<QT, kF32>(Dp);
        case kQ8: return kernel_d<QT, kQ8>(Dp);
        default: return kernel_d<QT, kAny>(Dp);
    }
}

}  // namespace

hipError_t gt_launch_key_weights(const gt_key_weights &r, int dev, hipStream_t s) {
    if (r.B * r.Hkv > 65535 || r.D > kMaxDim) return hipErrorInvalidConfiguration;
    Args a{};
    a.q = r.q;
    a.q_sb = r.q_strides[0];
    a.q_sh = r.q_strides[1];
    a.q_sl = r.q_strides[2];
    a.cap = r.cap;
    a.lse = r.lse;
    a.len = r.len;
    a.sums = r.sums;
    a.keep = r.keep;
    a.scale = r.scale;
    a.causal = r.causal;
    const int64_t per16 = r.q_dtype == GT_F32 ? 4 : 8;
    a.q_vec = r.D % 16 == 0 && (uintptr_t)r.q % 16 == 0 && a.q_sb % per16 == 0 && a.q_sh % per16 == 0 && a.q_sl % per16 == 0;
    a.H = (int)r.H;
    a.Hkv = (int)r.Hkv;
    a.L = (int)r.L;
    a.D = (int)r.D;
    int src;
    if (r.blocks) {
        src = r.blocks->e4m3 ? kE4m3 : kInt8;
        a.k = (const char *)r.blocks->codes[0];
        a.ks = r.blocks->scales[0];
        a.kt = (const _Float16 *)r.blocks->ops[0];
        a.kts = r.blocks->op_scales[0];
        a.shift = r.blocks->N == 32 ? 5 : r.blocks->N == 64 ? 6 : 7;
        a.units = r.blocks->units;
    } else {
        src = r.k_dtype == GT_F16 ? kF16 : r.k_dtype == GT_BF16 ? kBf16 : r.k_dtype == GT_F32 ? kF32 : kQ8;
        a.k = (const char *)r.k;
        a.row_bytes = r.k_dtype == GT_Q8_0 ? r.D / 32 * 34 : r.k_dtype == GT_F32 ? r.D * 4 : r.D * 2;
        a.k_dtype = r.k_dtype;
        if (src != kQ8 && (r.D % 16 != 0 || (uintptr_t)r.k % 16 != 0)) src = kAny;
    }
    const int Dp = padded_dim(r.D), keys = 16 * (Dp == 256 ? 2 : 4) * kWaves;
    const void *kernel = r.q_dtype == GT_F16   ? kernel_src<_Float16>(src, Dp)
                         : r.q_dtype == GT_BF16 ? kernel_src<__bf16>(src, Dp)
                                                : kernel_src<float>(src, Dp);
    const int64_t rows = r.H / r.Hkv * r.L, tiles = (rows + 15) / 16, wgs = (r.max_len + keys - 1) / keys;
    // column splits: towards 512 workgroups (two a CU), of 8 columns of 16 rows at least (a wavefront's keys cost
    // about as much as four).  A float16 cache, D128 H32/8, us with the attention, without splits and with: B1 S512
    // L512 110, 32; B1 S2048 L512 150, 72; B1 S4096 L256 136, 106.  Towards 256 workgroups 33, 79, 113, towards 1024
    // 32, 81, 114; splits of 4 columns 34, 72, 106, of 16 37, 72, 106.
    int64_t splits = std::min<int64_t>(tiles / 8, 512 / std::max<int64_t>(1, wgs * r.B * r.Hkv));
    splits = std::max<int64_t>(1, splits);
    a.col_tiles = (int)tiles;
    a.span = (int)((tiles + splits - 1) / splits);
    splits = (tiles + a.span - 1) / a.span;
    gt_scratch parts;
    if (splits > 1) {
        if (!gt_scratch_alloc(parts, (size_t)(splits * r.B * r.Hkv * r.max_len) * sizeof(float), dev)) return hipErrorOutOfMemory;
        a.parts = (float *)parts.ptr();
        a.max_len = r.max_len;
    }
    void *args[] = {(void *)&a};
    hipError_t e = hipLaunchKernel(kernel, dim3((unsigned)wgs, (unsigned)(r.B * r.Hkv), (unsigned)splits), dim3(64 * kWaves), args, 0, s);
    if (e != hipSuccess || splits == 1) return e;
    hipLaunchKernelGGL(add_parts_kernel, dim3((unsigned)((r.max_len + 255) / 256), (unsigned)(r.B * r.Hkv)), dim3(256), 0, s,
                       (const float *)a.parts, (int)splits, r.max_len, r.len, r.sums, r.keep, (int)r.Hkv, r.cap);
    return hipGetLastError();
}
