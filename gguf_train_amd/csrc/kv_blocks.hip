// The 8-bit block cache (kv_blocks.h): appending tokens (quantizing the blocks that become full), moving the
// tokens that an eviction leaves together, and reading back the values that the cache stands for.
//
// Append, bound by HBM (the rows once, a byte per value back): a workgroup owns 64 tokens of one sequence and
// head (128 where a block has as many) and keeps their values in registers between the largest magnitude and
// the codes, so a row is read once.  A thread's 16 values are 16 dims of a token for K and 16 tokens of a dim for
// V, what lies together in the codes' order.  An eviction is the same with the old cache's tokens for source.
// Read, bound by HBM (mostly the values written): a workgroup stages a unit of 64 tokens' codes in LDS, from
// which each thread gathers 8 dims of a token.
//
// Measured (GPU time, B4 Hkv8 D128, float16, int8): append of 4096 tokens 21 us, 4.8 TB/s (38 before all of a thread's
// loads were issued together); eviction of 4096 to 2048 tokens 22, of which half the memory rate: V's codes come in
// single bytes; read of 1500 tokens 13.5, 2.7 TB/s; append of one token 4.5, latency.

#include "gt_internal.h"
#include "kv_blocks.h"
#include "vec_dims.h"

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
__device__ inline float finite(float x) {
    if constexpr (__is_same(T, _Float16)) return fabsf(x) < INFINITY && fabsf(x) > 65504.0f ? copysignf(65504.0f, x) : x;
    return x;
}

// Four values already divided by the scale, as codes (round to nearest even).
template <bool E4M3>
__device__ inline uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
        return (uint32_t)w;
    } else {
        // + 128 (kv_blocks.h): the rounded value + 128 is 1 .. 255, whose float32 sum with 2^23 holds it in its low byte
        auto q = [](float x) { return __float_as_uint(rintf(x) + (8388608.0f + 128.0f)) & 0xffu; };
        return q(a) | q(b) << 8 | q(c) << 16 | q(d) << 24;
    }
}
template <bool E4M3>
__device__ inline void decode4(uint32_t w, float *v) {
    if constexpr (E4M3) {
        v[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
        v[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
        v[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
        v[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)((int)(w >> (8 * j) & 0xffu) - 128);
    }
}

// One tensor (K or V) of the cache: the codes, scales, tail and the tail's operands.
struct Side {
    uint8_t *codes;
    float *scales, *tail;
    _Float16 *ops;
    float *op_scales;
};

struct AppendArgs {
    Side to[2];
    int T, Hkv, D;
    int shift;             // log2 of the tokens of a block
    int64_t units;         // of 64 tokens per sequence and head
    // rows: `T` after the pos[b] tokens held before
    const void *src[2];
    int64_t st[2][4];      // element strides (B, Hkv, T, D)
    const int32_t *pos;
    int32_t *pos_next;     // tokens held afterwards
    // eviction: the kept[b, g, 0 .. min(len[b], keep) - 1] of another cache, into an empty one
    Side from[2];
    const int32_t *len;
    const int64_t *kept;
    int keep;
};

// Where an append's tokens come from, in two steps, so that all of a thread's loads are in flight together: no branch
// around a load (a token that is not wanted is read at a place that is there), and the values afterwards.
//   Dims: 16 dims of token p from d0 on, zeros from D on;
//   Column: dim d (below the padded size; zeros from D on) of the tokens t + 16 (e / 4) + e % 4, e < 16, t the same
//   for a whole wavefront (their addresses are scalar).
template <typename T, bool VEC>
struct RowSource {
    const T *rows;
    int64_t sr, sd;
    const float *tail;
    int held, count, shift, D;
    struct Dims {
        gtvec::Dims16<T> w;
        T y[VEC ? 1 : 16];
    };
    struct Column {
        T y[16];
    };
    __device__ const T *row(int p) const { return rows + (int64_t)min(max(p - held, 0), count - 1) * sr; }
    __device__ void load(Dims &r, int p, int d0) const {
        if constexpr (VEC) {  // contiguous dims, 16-byte aligned rows, D a multiple of 16
            r.w.load(row(p) + (d0 < D ? d0 : 0));
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) r.y[e] = row(p)[(int64_t)min(d0 + e, D - 1) * sd];
        }
    }
    __device__ void values(const Dims &r, int p, int d0, float *v) const {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            float x;
            if constexpr (VEC) x = r.w.get(e);
            else x = to_f(r.y[e]);
            v[e] = (VEC ? d0 : d0 + e) < D ? x : 0.0f;
        }
        if (in_tail(p, held, shift)) {
            const float *waiting = tail + (int64_t)(p - (held >> shift << shift)) * D;
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = d0 + e < D ? waiting[d0 + e] : 0.0f;
        }
    }
    __device__ void load(Column &r, int t, int d) const {
        const int64_t at = min(d, D - 1) * sd;
#pragma unroll
        for (int e = 0; e < 16; ++e) r.y[e] = row(t + 16 * (e >> 2) + (e & 3))[at];
    }
    __device__ void values(const Column &r, int t, int d, float *v) const {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = d < D ? to_f(r.y[e]) : 0.0f;
        if (t < held) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int p = t + 16 * (e >> 2) + (e & 3);
                if (in_tail(p, held, shift)) v[e] = d < D ? tail[(int64_t)(p - (held >> shift << shift)) * D + d] : 0.0f;
            }
        }
    }
};

// Tokens of another block cache (z 0 keys, 1 values): token `first` + i of the new cache is kept[i], in LDS.  A
// token's V codes are 16 bytes apart, so that a wavefront's 64 take 16 lines of which the others hold other tokens'.
// The caches take care of that: with the units copied to LDS first, int8 D128 B4 Hkv8 4096 to 2048 tokens took 57.5
// us with the append before it, without 55.3.
template <bool E4M3>
struct KeptSource {
    const uint8_t *codes;
    const float *scales, *tail;
    const int *kept;
    int first, here, full, shift, D, Dp, z;  // here: places of kept
    bool late;  // some of the workgroup's tokens are in the old tail
    struct Dims {
        uint32_t w[4];
        float s;
    };
    struct Column {
        uint32_t q[16];
        float s[16];
    };
    __device__ void load(Dims &r, int p, int d0) const {
        const int t = kept[p - first], tc = t < full ? t : 0;  // (token 0's place is there to be read)
        if (z == 0) {
            const uint4 w = *(const uint4 *)(codes + k_at(tc, d0, Dp));
            r.w[0] = w.x, r.w[1] = w.y, r.w[2] = w.z, r.w[3] = w.w;
        } else {
            const uint8_t *q = codes + v_at(tc, d0, Dp);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r.w[j] = q[64 * j] | (uint32_t)q[64 * j + 16] << 8 | (uint32_t)q[64 * j + 32] << 16 | (uint32_t)q[64 * j + 48] << 24;
        }
        r.s = scales[tc >> shift];
    }
    __device__ void values(const Dims &r, int p, int d0, float *v) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) decode4<E4M3>(r.w[j], v + 4 * j);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= r.s;
        const int t = kept[p - first];
        if (t >= full) {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = d0 + e < D ? tail[(int64_t)(t - full) * D + d0 + e] : 0.0f;
        }
    }
    // (past the workgroup's tokens: its last)
    __device__ int token(int t, int e) const { return __builtin_amdgcn_readfirstlane(kept[min(t + 16 * (e >> 2) + (e & 3) - first, here - 1)]); }
    __device__ void load(Column &r, int t, int d) const {
        const uint32_t at = (uint32_t)((d >> 4) * 1024 + (d & 15) * 16);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int u = token(t, e), uc = u < full ? u : 0;
            r.q[e] = (codes + v_at(uc, 0, Dp))[at];
            r.s[e] = scales[uc >> shift];
        }
    }
    __device__ void values(const Column &r, int t, int d, float *v) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) decode4<E4M3>(r.q[4 * j] | r.q[4 * j + 1] << 8 | r.q[4 * j + 2] << 16 | r.q[4 * j + 3] << 24, v + 4 * j);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= r.s[e];
        if (late) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int u = token(t, e);
                if (u >= full) v[e] = d < D ? tail[(int64_t)(u - full) * D + d] : 0.0f;
            }
        }
    }
};

// NT tokens a workgroup, whole blocks of N.  `held` tokens were there, `total` are there afterwards; the workgroup
// x of a (sequence, head) takes the x-th NT tokens from those of the block in progress on, t0 the first.
template <bool E4M3, int DP, int NT, typename Source>
__device__ inline void append_blocks(const Source &src, const Side &to, int shift, int D, int z, int t0, int held, int total) {
    constexpr int ITEMS = NT * DP / 16 / kThreads, CH = DP / 16, BLOCKS = NT / 32;
    const int tid = threadIdx.x, lane = tid & 63;
    __shared__ uint32_t s_max[BLOCKS][kThreads / 64];
    // a block is written when it becomes full
    auto fills = [&](int t) { return t >> shift >= held >> shift && t >> shift < total >> shift; };
    // item i of a thread.  K: dims 16 ch .. of token t, 16 lanes next to each other the 16 tokens of a tile, whose
    // chunk is contiguous in the codes.  V: the 16 tokens 16 kb + 4g + r of dim d, contiguous in the codes as well.
    auto k_token = [&](int i) { return t0 + i / (16 * CH) * 16 + (i & 15); };
    auto k_dim = [&](int i) { return i / 16 % CH * 16; };
    // + 16 kb + r; the same for the 64 threads of a wavefront
    auto v_unit = [&](int i) { return __builtin_amdgcn_readfirstlane(t0 + i / (4 * DP) * kUnit + 4 * (i / DP % 4)); };
    float x[ITEMS][16];
    // magnitudes as their bits, whose order is theirs, NaN above infinity
    uint32_t amax[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) amax[b] = 0;
    auto magnitude = [&](float v) { return __float_as_uint(v) & 0x7fffffffu; };
    auto count = [&](int t, uint32_t most) {  // a block not to be written counts for nothing: its scale is not used
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) amax[b] = b == (t - t0) >> shift ? max(amax[b], most) : amax[b];
    };
    if (z == 0) {
        typename Source::Dims raw[ITEMS];
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) src.load(raw[it], k_token(tid + kThreads * it), k_dim(tid + kThreads * it));
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int t = k_token(tid + kThreads * it);
            src.values(raw[it], t, k_dim(tid + kThreads * it), x[it]);
            uint32_t most = 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) most = max(most, magnitude(x[it][e]));
            count(t, most);
        }
    } else {
        typename Source::Column raw[ITEMS];
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) src.load(raw[it], v_unit(tid + kThreads * it), (tid + kThreads * it) % DP);
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int t = v_unit(tid + kThreads * it);
            src.values(raw[it], t, (tid + kThreads * it) % DP, x[it]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t most = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) most = max(most, magnitude(x[it][8 * h + e]));
                count(t + 32 * h, most);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        for (int m = 32; m >= 1; m >>= 1) amax[b] = max(amax[b], (uint32_t)__shfl_xor((int)amax[b], m, 64));
        if (lane == 0) s_max[b][tid >> 6] = amax[b];
    }
    __syncthreads();
    float inv[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        const uint32_t most = max(max(s_max[b][0], s_max[b][1]), max(s_max[b][2], s_max[b][3]));
        const bool bad = most >= 0x7f800000u;
        const int e2 = bad ? 0 : scale_exponent(most, E4M3);
        // (a block with an infinity or NaN has no scale: all of it reads as NaN)
        inv[b] = bad ? NAN : __uint_as_float((uint32_t)(127 - e2) << 23);
        if (tid == 0 && b << shift < NT && fills(t0 + (b << shift)))
            to.scales[(t0 >> shift) + b] = bad ? NAN : __uint_as_float((uint32_t)(e2 + 127) << 23);
    }
    auto inv_of = [&](int t) {
        float f = 0.0f;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) f = b == (t - t0) >> shift ? inv[b] : f;
        return f;
    };
    auto encode = [&](const float *v, float f) {
        return f != f ? (E4M3 ? 0u : 0x80808080u) : encode4<E4M3>(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
    };
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
        const int i = tid + kThreads * it;
        if (z == 0) {
            const int t = k_token(i);
            if (!fills(t)) continue;
            const float f = inv_of(t);
            *(uint4 *)(to.codes + k_at(t, k_dim(i), DP)) = make_uint4(encode(x[it], f), encode(x[it] + 4, f), encode(x[it] + 8, f), encode(x[it] + 12, f));
        } else {
            const int t = v_unit(i), d = i % DP;
            uint2 *o = (uint2 *)(to.codes + v_at(t, d, DP));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!fills(t + 32 * h)) {
                    // the other block, of tokens to come, of a unit whose first is whole: the attention reads it, with
                    // weights of 0, so it must not be e4m3 NaNs
                    const int whole = total >> shift << shift;
                    if (h == 1 && t < whole && t + 32 >= whole) o[1] = make_uint2(0u, 0u);
                    continue;
                }
                const float f = inv_of(t + 32 * h);
                o[h] = make_uint2(encode(x[it] + 8 * h, f), encode(x[it] + 8 * h + 4, f));
            }
        }
    }
}

// The tokens after the last whole block, from token `from` of the cache on (those before are there): their values,
// and the operands that the attention takes them as (the row divided by its own power of two, float16 hi + lo, in
// the codes' order).  DP / 16 lanes a row, for its largest magnitude.  V's operands, 32 bytes apart, are written an element
// at a time; a second pass that wrote them 16 tokens of a dim together was slower up to 64 rows (B4 Hkv8 D128: 17 rows
// of a block of 32 6.5 against 5.6 us, 100 of a block of 128 12.6 against 14.3).  clear: the operands of tokens to come
// become zeros.
template <int DP, typename Source>
__device__ inline void append_tail(const Source &src, const Side &to, int shift, int D, int z, int from, int total, bool clear) {
    constexpr int CH = DP / 16;
    const int whole = total >> shift << shift, room = max(1 << shift, kUnit);
    const int64_t plane = (int64_t)room * DP;
    if (clear) {
        for (int i = threadIdx.x; i < (int)(plane / 4); i += kThreads) ((uint4 *)to.ops)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    }
    for (int i = threadIdx.x; i < (total - from) * CH; i += kThreads) {
        const int p = from + i / CH, t = p - whole, d0 = i % CH * 16;
        float v[16];
        typename Source::Dims raw;
        src.load(raw, p, d0);
        src.values(raw, p, d0, v);
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
        for (int m = CH / 2; m >= 1; m >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m, 64));
        const bool bad = most >= 0x7f800000u;
        const int e2 = bad || most == 0 ? -126 : min(max((int)(most >> 23) - 127, -126), 126);
        const float f = bad ? 0.0f : __uint_as_float((uint32_t)(127 - e2) << 23);
        if (d0 == 0) to.op_scales[t] = bad ? NAN : __uint_as_float((uint32_t)(127 + e2) << 23);
        float *row = to.tail + (int64_t)t * D + d0;
        if (D % 16 == 0) {
            if (d0 < D) {
#pragma unroll
                for (int e = 0; e < 4; ++e) ((float4 *)row)[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (d0 + e < D) row[e] = v[e];
        }
        typedef _Float16 half8 __attribute__((ext_vector_type(8)));
        half8 hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float y = bad ? 0.0f : v[e] * f;
            hi[e >> 3][e & 7] = (_Float16)y;
            lo[e >> 3][e & 7] = (_Float16)(y - (float)hi[e >> 3][e & 7]);
        }
        if (z == 0) {
            half8 *o = (half8 *)(to.ops + k_at(t, d0, DP));
            o[0] = hi[0], o[1] = hi[1];
            o = (half8 *)(to.ops + plane + k_at(t, d0, DP));
            o[0] = lo[0], o[1] = lo[1];
        } else {
            _Float16 *o = to.ops + v_at(t, d0, DP);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                o[16 * e] = hi[e >> 3][e & 7];
                o[plane + 16 * e] = lo[e >> 3][e & 7];
            }
        }
    }
}

template <int DP>
__device__ inline Side slice(const Side &s, const AppendArgs &a, int64_t bg) {
    Side r;
    r.codes = s.codes + bg * a.units * kUnit * DP;
    const int N = 1 << a.shift, room = max(N, kUnit);
    r.scales = s.scales + bg * (a.units * kUnit >> a.shift);
    r.tail = s.tail + bg * N * a.D;
    r.ops = s.ops + bg * 2 * room * DP;
    r.op_scales = s.op_scales + bg * room;
    return r;
}

// grid: (NT tokens each, B * Hkv, K and V)
template <typename T, bool E4M3, bool VEC, int DP, int NT>
__global__ __launch_bounds__(kThreads) void kv_blocks_append_kernel(AppendArgs a) {
    const int z = blockIdx.z;
    const int64_t bg = blockIdx.y, b = bg / a.Hkv, g = bg - b * a.Hkv;
    const int held = a.pos[b], total = held + a.T;
    if (threadIdx.x == 0 && g == 0 && z == 0 && blockIdx.x == 0) a.pos_next[b] = total;
    const int t0 = (held / NT + (int)blockIdx.x) * NT;
    const Side to = slice<DP>(a.to[z], a, bg);
    const RowSource<T, VEC> src = {(const T *)a.src[z] + b * a.st[z][0] + g * a.st[z][1], a.st[z][2], a.st[z][3], to.tail,
                                   held, a.T, a.shift, a.D};
    // (a decode step that fills no block has none to look at, nor has a workgroup past the whole blocks: the grid is of
    // the sequence that takes most, and another may be at the end of its room)
    if (held >> a.shift != total >> a.shift && t0 < total >> a.shift << a.shift) append_blocks<E4M3, DP, NT>(src, to, a.shift, a.D, z, t0, held, total);
    // The new tail: by the workgroup of its tokens, which often has no whole block, or, where there is an old one, by the
    // one that has read it.  (A workgroup for it alone: B4 Hkv8 D128, 2048 tokens 13.8 against 12.0 us, 2001 14.0, 14.9.)
    const int from = max(held, total >> a.shift << a.shift), old = held & ((1 << a.shift) - 1);
    if (from == total || (int)blockIdx.x != (old ? 0 : from / NT - held / NT)) return;
    __syncthreads();
    append_tail<DP>(src, to, a.shift, a.D, z, from, total, false);
}

template <bool E4M3, int DP, int NT>
__global__ __launch_bounds__(kThreads) void kv_blocks_evict_kernel(AppendArgs a) {
    __shared__ int s_kept[NT];
    const int z = blockIdx.z;
    const int64_t bg = blockIdx.y, b = bg / a.Hkv;
    const int total = min(a.len[b], a.keep), t0 = (int)blockIdx.x * NT, full = a.len[b] >> a.shift << a.shift;
    if (t0 >= total && (int)blockIdx.x > 0) return;  // (an empty sequence: its operands are cleared)
    bool late = false;
    for (int i = threadIdx.x; i < NT; i += kThreads) {  // (places past the last token: token 0, not used)
        const int t = t0 + i < total ? (int)a.kept[bg * a.keep + t0 + i] : 0;
        s_kept[i] = t;
        late = late || t >= full;
    }
    late = __syncthreads_or(late);
    const Side from = slice<DP>(a.from[z], a, bg), to = slice<DP>(a.to[z], a, bg);
    const int whole = total >> a.shift << a.shift;
    const bool last = total - t0 <= NT;  // the tail's tokens are among the last workgroup's, or there are none
    const KeptSource<E4M3> src = {from.codes, from.scales, from.tail, s_kept, t0, NT, full, a.shift, a.D, DP, z, late};
    if (t0 < whole) append_blocks<E4M3, DP, NT>(src, to, a.shift, a.D, z, t0, 0, total);
    if (last) append_tail<DP>(src, to, a.shift, a.D, z, whole, total, true);
}

struct ReadArgs {
    const uint8_t *codes[2];
    const float *scales[2], *tail[2];
    void *out[2];            // dense (B, Hkv, rows, D)
    const int32_t *len;      // tokens held per sequence
    int rows, Hkv, shift, D, Dp;
    int64_t units;
};

// grid: (units of 64 rows, B * Hkv, K and V); rows past what is held are zero
template <typename TO, bool E4M3>
__global__ __launch_bounds__(kThreads) void kv_blocks_read_kernel(ReadArgs a) {
    // (K: a chunk of 16 dims at a pitch of 64 more bytes a tile, V: 16 dims at one of 16 more a unit, so that the lanes
    // of a row, 8 dims each, read from different banks)
    constexpr int KP = 256 + 64, VP = 1024 + 16;
    __shared__ __attribute__((aligned(16))) uint8_t raw[kMaxDim / 16 * 4 * KP];
    const int z = blockIdx.z, D = a.D, Dp = a.Dp, tid = threadIdx.x;
    const int64_t bg = blockIdx.y, b = bg / a.Hkv;
    const int r0 = blockIdx.x * kUnit, held = a.len[b], full = held >> a.shift << a.shift;
    const uint8_t *codes = a.codes[z] + bg * a.units * kUnit * Dp;
    const float *scales = a.scales[z] + bg * (a.units * kUnit >> a.shift);
    const float *tail = a.tail[z] + (bg << a.shift) * D;
    TO *out = (TO *)a.out[z] + bg * (int64_t)a.rows * D;
    if (r0 < full) {
        for (int i = tid; i < kUnit * Dp / 16; i += kThreads)
            *(uint4 *)(raw + (z == 0 ? i / 16 * KP + i % 16 * 16 : i / 64 * VP + i % 64 * 16)) = *(const uint4 *)(codes + (int64_t)r0 * Dp + 16 * i);
    }
    __syncthreads();
    const int groups = Dp / 8, n = min(kUnit, a.rows - r0);
    for (int i = tid; i < n * groups; i += kThreads) {
        const int r = i / groups, d0 = i % groups * 8;
        if (d0 >= D) continue;
        const int t = r0 + r;
        float v[8];
        if (t >= held) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        } else if (t >= full) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = d0 + e < D ? finite<TO>(tail[(int64_t)(t - full) * D + d0 + e]) : 0.0f;
        } else {
            uint32_t w[2];
            if (z == 0) {
                const uint2 q = *(const uint2 *)(raw + ((r >> 4) * (Dp / 16) + (d0 >> 4)) * KP + (r & 15) * 16 + (d0 & 15));
                w[0] = q.x;
                w[1] = q.y;
            } else {
                const uint8_t *p = raw + (d0 >> 4) * VP + v_at(r, d0 & 15, 16);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    w[j] = p[64 * j] | (uint32_t)p[64 * j + 16] << 8 | (uint32_t)p[64 * j + 32] << 16 | (uint32_t)p[64 * j + 48] << 24;
            }
            const float s = scales[t >> a.shift];
            if (!E4M3 && s < 128.0f) {
                // (byte - 128) s in one step: the product and the difference are exact
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = fmaf((float)(w[e >> 2] >> (8 * (e & 3)) & 0xffu), s, -128.0f * s);
            } else {
                decode4<E4M3>(w[0], v);
                decode4<E4M3>(w[1], v + 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= s;
                if (s >= 128.0f) {  // (448 s passes float16's largest)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = finite<TO>(v[e]);
                }
            }
        }
        TO *o = out + (int64_t)(r0 + r) * D + d0;
        if (D % 8 == 0) {
            struct alignas(sizeof(TO) * 8 < 16 ? sizeof(TO) * 8 : 16) P {
                TO e[8];
            } p;
#pragma unroll
            for (int e = 0; e < 8; ++e) p.e[e] = (TO)v[e];
            *(P *)o = p;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (d0 + e < D) o[e] = (TO)v[e];
        }
    }
}

// The kernel for head sizes padded to Dp and blocks of N.
template <typename T, bool E4M3, bool VEC>
const void *append_kernel(int Dp, int N) {
#define GT_A(DP) (N == 128 ? (const void *)kv_blocks_append_kernel<T, E4M3, VEC, DP, 128> : (const void *)kv_blocks_append_kernel<T, E4M3, VEC, DP, 64>)
    return Dp == 64 ? GT_A(64) : Dp == 128 ? GT_A(128) : GT_A(256);
#undef GT_A
}
template <typename T>
const void *append_kernel(bool e4m3, bool vec, int Dp, int N) {
    if (e4m3) return vec ? append_kernel<T, true, true>(Dp, N) : append_kernel<T, true, false>(Dp, N);
    return vec ? append_kernel<T, false, true>(Dp, N) : append_kernel<T, false, false>(Dp, N);
}
template <bool E4M3>
const void *evict_kernel(int Dp, int N) {
#define GT_E(DP) (N == 128 ? (const void *)kv_blocks_evict_kernel<E4M3, DP, 128> : (const void *)kv_blocks_evict_kernel<E4M3, DP, 64>)
    return Dp == 64 ? GT_E(64) : Dp == 128 ? GT_E(128) : GT_E(256);
#undef GT_E
}

int block_shift(int N) { return N == 32 ? 5 : N == 64 ? 6 : 7; }

void fill_sides(Side *s, const gt_kv_blocks &c) {
    for (int z = 0; z < 2; ++z) s[z] = {(uint8_t *)c.codes[z], c.scales[z], c.tail[z], (_Float16 *)c.ops[z], c.op_scales[z]};
}

hipError_t launch(const void *kernel, AppendArgs &a, int64_t groups, int64_t bg, hipStream_t s) {
    if (bg > 65535 || groups > 0x7fffffff) return hipErrorInvalidConfiguration;
    void *args[] = {(void *)&a};
    return hipLaunchKernel(kernel, dim3((unsigned)std::max<int64_t>(groups, 1), (unsigned)bg, 2), dim3(kThreads), args, 0, s);
}

template <typename TO>
hipError_t launch_read(const ReadArgs &a, bool e4m3, dim3 grid, hipStream_t s) {
    if (e4m3) hipLaunchKernelGGL((kv_blocks_read_kernel<TO, true>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((kv_blocks_read_kernel<TO, false>), grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t gt_launch_kv_blocks_append(const gt_kv_blocks &c, const void *const *src, int src_dtype,
                                      const int64_t *const *strides, const int32_t *pos, int32_t *pos_next, int64_t T,
                                      int64_t groups, hipStream_t s) {
    AppendArgs a{};
    bool vec = c.D % 16 == 0;
    const int64_t es = src_dtype == GT_F32 ? 4 : 2;
    for (int z = 0; z < 2; ++z) {
        a.src[z] = src[z];
        for (int i = 0; i < 4; ++i) a.st[z][i] = strides[z][i];
        vec = vec && strides[z][3] == 1 && (uintptr_t)src[z] % 16 == 0;
        for (int i = 0; i < 3; ++i) vec = vec && strides[z][i] * es % 16 == 0;
    }
    fill_sides(a.to, c);
    a.pos = pos;
    a.pos_next = pos_next;
    a.T = (int)T;
    a.Hkv = (int)c.Hkv;
    a.shift = block_shift(c.N);
    a.D = (int)c.D;
    a.units = c.units;
    const void *kernel = src_dtype == GT_F32   ? append_kernel<float>(c.e4m3, vec, c.Dp, c.N)
                         : src_dtype == GT_F16 ? append_kernel<_Float16>(c.e4m3, vec, c.Dp, c.N)
                                               : append_kernel<__bf16>(c.e4m3, vec, c.Dp, c.N);
    return launch(kernel, a, groups, c.B * c.Hkv, s);
}

hipError_t gt_launch_kv_blocks_evict(const gt_kv_blocks &from, const gt_kv_blocks &to, const int32_t *len, const int64_t *kept,
                                     int64_t keep, hipStream_t s) {
    AppendArgs a{};
    fill_sides(a.to, to);
    fill_sides(a.from, from);
    a.len = len;
    a.kept = kept;
    a.keep = (int)keep;
    a.Hkv = (int)from.Hkv;
    a.shift = block_shift(from.N);
    a.D = (int)from.D;
    a.units = from.units;
    const int64_t nt = std::max(from.N, kUnit);
    return launch(from.e4m3 ? evict_kernel<true>(from.Dp, from.N) : evict_kernel<false>(from.Dp, from.N), a, (keep + nt - 1) / nt,
                  from.B * from.Hkv, s);
}

hipError_t gt_launch_kv_blocks_read(const gt_kv_blocks &c, const int32_t *len, int64_t rows, void *k, void *v, int dtype,
                                    hipStream_t s) {
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
    a.rows = (int)rows;
    a.Hkv = (int)c.Hkv;
    a.shift = block_shift(c.N);
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
