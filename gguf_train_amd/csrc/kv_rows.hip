// Rows of the KV cache that move or are read: choosing the tokens that stay when others are evicted, moving
// their rows together, and reading a float or Q8_0 cache back as values.
//
// Choosing (kv_select_kernel): per sequence and kv head, the `recent` last tokens and the `keep - recent`
// others of the largest weights, the lowest index of equal ones, in order.  A workgroup finds the smallest
// weight that stays by radix selection, 8 bits of the order-preserving integer form of the floats a pass, and then
// gives those that stay their places in order, from ballots and a scan of their counts.  Up to kSelectCached tokens
// a thread keeps its weights in registers and one scan serves them all, more are read again from the caches, 1024
// tokens a scan.  Bound: latency, the passes' barriers and counting (LDS atomics), not the 4 bytes a token.  Integer
// counts alone decide, so the result does not depend on timing.  B4 Hkv8, half of 4096 tokens: 11.4 us (12.7 with a
// scan for every 1024 tokens); an append of 8192 tokens and an eviction of half 75.0 us against 84.6 with the weights
// read again in each pass.
//
// Moving, HBM-bound: the rows that change place go to scratch memory and from there to their new places, two
// launches; writing them in place would have workgroups overwrite rows that others have yet to read.  (16 threads a
// row, 16 bytes each where the rows are aligned.)

#include "gt_internal.h"

#include <algorithm>

namespace {

constexpr int kSelectThreads = 1024, kSelectKeys = 8;  // keys a thread keeps
constexpr int kSelectCached = kSelectThreads * kSelectKeys;

// Unsigned integers in the order of the floats: -0 as +0, every NaN above all others.
__device__ inline uint32_t order_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelectArgs {
    const float *w;
    int64_t wb, wg, ws;  // element strides of the weights
    const int32_t *len;
    int32_t *next;       // the lengths afterwards
    int32_t *evicted;    // tokens evicted so far, or null (none are)
    int64_t *kept;       // (B, Hkv, keep)
    int Hkv, keep, recent;
};

// CACHED: no sequence has more than kSelectCached tokens.
template <bool CACHED>
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(SelectArgs a) {
    constexpr int WAVES = kSelectThreads / 64, COPIES = 4;
    __shared__ uint32_t s_hist[COPIES][256];
    __shared__ uint32_t s_bin, s_need;
    __shared__ int s_above[WAVES], s_equal[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t bg = blockIdx.x, b = bg / a.Hkv, g = bg - b * a.Hkv;
    const int n = a.len[b];
    int64_t *kept = a.kept + bg * a.keep;
    if (g == 0 && tid == 0) {
        a.next[b] = min(n, a.keep);
        if (n > a.keep) a.evicted[b] += n - a.keep;
    }
    if (n <= a.keep) {
        for (int i = tid; i < a.keep; i += kSelectThreads) kept[i] = i < n ? i : -1;
        return;
    }
    const float *w = a.w + b * a.wb + g * a.wg;
    const int others = n - a.recent, m = a.keep - a.recent;  // 0 <= m < others
    for (int i = tid; i < a.recent; i += kSelectThreads) kept[m + i] = others + i;
    if (m == 0) return;
    uint32_t keys[CACHED ? kSelectKeys : 1];
    if constexpr (CACHED) {
        float x[kSelectKeys];
#pragma unroll
        for (int c = 0; c < kSelectKeys; ++c) x[c] = w[min(tid + c * kSelectThreads, others - 1) * a.ws];
#pragma unroll
        for (int c = 0; c < kSelectKeys; ++c) keys[c] = order_of(x[c]);
    }
    // visit(key) for every token of this thread
    auto each = [&](auto &&visit) {
        if constexpr (CACHED) {
#pragma unroll
            for (int c = 0; c < kSelectKeys; ++c)
                if (tid + c * kSelectThreads < others) visit(keys[c]);
        } else {
            for (int i = tid; i < others; i += kSelectThreads) visit(order_of(w[i * a.ws]));
        }
    };
    uint32_t prefix = 0, mask = 0, need = (uint32_t)m;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < COPIES * 256; i += kSelectThreads) (&s_hist[0][0])[i] = 0;
        __syncthreads();
        each([&](uint32_t k) {
            if ((k & mask) == prefix) atomicAdd(&s_hist[wv % COPIES][(k >> shift) & 255], 1u);
        });
        __syncthreads();
        if (wv == 0) {
            // bins 255 - 4 lane downwards; the bin in which the count from the top reaches `need`
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int bin = 255 - 4 * lane - j;
                c[j] = s_hist[0][bin] + s_hist[1][bin] + s_hist[2][bin] + s_hist[3][bin];
                sum += c[j];
            }
            uint32_t upto = sum;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(upto, o, 64);
                if (lane >= o) upto += y;
            }
            uint32_t before = upto - sum;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (before < need && before + c[j] >= need) {
                    s_bin = 255 - 4 * lane - j;
                    s_need = need - before;
                }
                before += c[j];
            }
        }
        __syncthreads();
        prefix |= s_bin << shift;
        mask |= 255u << shift;
        need = s_need;
    }
    // tokens above the border all stay, and the first `need` of those on it
    int above = 0, equal = 0;  // of the tokens before this chunk
    auto chunk = [&](int i, uint32_t k) {
        const bool up = i < others && k > prefix, eq = i < others && k == prefix;
        const uint64_t bu = __ballot(up), be = __ballot(eq);
        if (lane == 0) {
            s_above[wv] = __popcll(bu);
            s_equal[wv] = __popcll(be);
        }
        __syncthreads();
        int pu = above, pe = equal;
        for (int v = 0; v < WAVES; ++v) {
            if (v < wv) {
                pu += s_above[v];
                pe += s_equal[v];
            }
            above += s_above[v];
            equal += s_equal[v];
        }
        const uint64_t lower = (1ull << lane) - 1;
        pu += __popcll(bu & lower);
        pe += __popcll(be & lower);
        if (up || (eq && pe < (int)need)) kept[pu + min(pe, (int)need)] = i;
        __syncthreads();
    };
    if constexpr (CACHED) {
        // counts of every 64 tokens: above the border in the low half, on it in the high half (each below 2^16)
        __shared__ uint32_t s_count[kSelectKeys * WAVES];
        static_assert(kSelectKeys * WAVES == 128, "two counts a lane");
        uint64_t bu[kSelectKeys], be[kSelectKeys];
#pragma unroll
        for (int c = 0; c < kSelectKeys; ++c) {
            const bool there = tid + c * kSelectThreads < others;
            bu[c] = __ballot(there && keys[c] > prefix);
            be[c] = __ballot(there && keys[c] == prefix);
            if (lane == 0) s_count[c * WAVES + wv] = (uint32_t)__popcll(bu[c]) | (uint32_t)__popcll(be[c]) << 16;
        }
        __syncthreads();
        if (wv == 0) {
            const uint32_t x0 = s_count[2 * lane], x1 = s_count[2 * lane + 1];
            uint32_t upto = x0 + x1;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(upto, o, 64);
                if (lane >= o) upto += y;
            }
            s_count[2 * lane] = upto - x1 - x0;
            s_count[2 * lane + 1] = upto - x1;
        }
        __syncthreads();
        const uint64_t lower = (1ull << lane) - 1;
#pragma unroll
        for (int c = 0; c < kSelectKeys; ++c) {
            const uint32_t before = s_count[c * WAVES + wv];
            const int pu = (int)(before & 0xffffu) + __popcll(bu[c] & lower), pe = (int)(before >> 16) + __popcll(be[c] & lower);
            const bool up = bu[c] >> lane & 1, eq = be[c] >> lane & 1;
            if (up || (eq && pe < (int)need)) kept[pu + min(pe, (int)need)] = tid + c * kSelectThreads;
        }
    } else {
        for (int i0 = 0; i0 < others; i0 += kSelectThreads) {
            const int i = i0 + tid;
            chunk(i, i < others ? order_of(w[i * a.ws]) : 0u);
        }
    }
}

struct MoveArgs {
    char *rows[3];        // (B, Hkv, cap) rows
    char *temp[3];        // (B, Hkv, keep) rows
    int64_t row_bytes[3];
    int piece[3];         // bytes a thread moves: 16, 8, 4 or 2
    const int64_t *kept;
    const int32_t *len;
    int Hkv, keep, zeroed;  // zeroed: the tensor (float32, 4-byte rows) whose places left behind become zero, or -1
    int64_t cap;
};

template <typename P>
__device__ inline void move_pieces(char *dst, const char *src, int64_t nbytes) {
    for (int64_t i = (int64_t)(threadIdx.x & 15) * sizeof(P); i < nbytes; i += 16 * sizeof(P)) *(P *)(dst + i) = *(const P *)(src + i);
}

// grid: (16 rows a workgroup, B * Hkv, tensors); 16 threads a row.  BACK: from the scratch rows into place, and
// the accumulated weights of the places left behind to zero.
template <bool BACK>
__global__ __launch_bounds__(256) void kv_move_kernel(MoveArgs a) {
    const int z = blockIdx.z;
    const int64_t bg = blockIdx.y, b = bg / a.Hkv;
    const int n = a.len[b];
    if (n <= a.keep) return;
    const int64_t j = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int64_t rb = a.row_bytes[z];
    if (j >= a.keep) {
        if (BACK && z == a.zeroed && j < n && (threadIdx.x & 15) == 0) *(float *)(a.rows[z] + (bg * a.cap + j) * 4) = 0.0f;
        return;
    }
    const int64_t from = a.kept[bg * a.keep + j];
    if (from == j) return;
    char *t = a.temp[z] + (bg * a.keep + j) * rb;
    char *dst = BACK ? a.rows[z] + (bg * a.cap + j) * rb : t;
    const char *src = BACK ? t : a.rows[z] + (bg * a.cap + from) * rb;
    switch (a.piece[z]) {
        case 16: move_pieces<uint4>(dst, src, rb); break;
        case 8: move_pieces<uint64_t>(dst, src, rb); break;
        case 4: move_pieces<uint32_t>(dst, src, rb); break;
        default: move_pieces<uint16_t>(dst, src, rb); break;
    }
}

template <int DT>
__device__ inline float cached_value(const char *row, int d) {
    if constexpr (DT == GT_F32) return ((const float *)row)[d];
    else if constexpr (DT == GT_F16) return (float)((const _Float16 *)row)[d];
    else if constexpr (DT == GT_BF16) return (float)((const __bf16 *)row)[d];
    else {
        const uint8_t *blk = (const uint8_t *)row + (d >> 5) * 34;
        return (float)*(const _Float16 *)blk * (float)*(const int8_t *)(blk + 2 + (d & 31));
    }
}

template <int DT, typename TO>
__global__ void kv_rows_read_kernel(const char *k, const char *v, const int32_t *len, TO *ko, TO *vo, int Hkv, int rows, int D,
                                    int64_t cap, int64_t row_bytes, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int64_t row = i / D, bg = row / rows;
    const int d = (int)(i - row * D), t = (int)(row - bg * rows);
    const char *src = (blockIdx.y ? v : k) + (bg * cap + t) * row_bytes;
    (blockIdx.y ? vo : ko)[i] = t < len[bg / Hkv] ? (TO)cached_value<DT>(src, d) : (TO)0.0f;
}

template <int DT>
hipError_t launch_rows_read(const void *k, const void *v, const int32_t *len, void *ko, void *vo, int out, int64_t B, int64_t Hkv,
                            int64_t rows, int64_t D, int64_t cap, int64_t rb, hipStream_t s) {
    const int64_t n = B * Hkv * rows * D, blocks = (n + 255) / 256;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)blocks, 2);
    switch (out) {
        case GT_F32:
            hipLaunchKernelGGL((kv_rows_read_kernel<DT, float>), grid, dim3(256), 0, s, (const char *)k, (const char *)v, len,
                               (float *)ko, (float *)vo, (int)Hkv, (int)rows, (int)D, cap, rb, n);
            break;
        case GT_F16:
            hipLaunchKernelGGL((kv_rows_read_kernel<DT, _Float16>), grid, dim3(256), 0, s, (const char *)k, (const char *)v, len,
                               (_Float16 *)ko, (_Float16 *)vo, (int)Hkv, (int)rows, (int)D, cap, rb, n);
            break;
        case GT_BF16:
            hipLaunchKernelGGL((kv_rows_read_kernel<DT, __bf16>), grid, dim3(256), 0, s, (const char *)k, (const char *)v, len,
                               (__bf16 *)ko, (__bf16 *)vo, (int)Hkv, (int)rows, (int)D, cap, rb, n);
            break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t gt_launch_kv_select(const float *w, const int64_t *strides, const int32_t *len, int32_t *next, int32_t *evicted, int64_t *kept,
                               int64_t B, int64_t Hkv, int64_t max_len, int64_t keep, int64_t recent, hipStream_t s) {
    SelectArgs a{w, strides[0], strides[1], strides[2], len, next, evicted, kept, (int)Hkv, (int)keep, (int)recent};
    if (B * Hkv > 0x7fffffff) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)(B * Hkv));
    if (max_len <= kSelectCached) hipLaunchKernelGGL(kv_select_kernel<true>, grid, dim3(kSelectThreads), 0, s, a);
    else hipLaunchKernelGGL(kv_select_kernel<false>, grid, dim3(kSelectThreads), 0, s, a);
    return hipGetLastError();
}

hipError_t gt_launch_kv_move(const gt_kv_moved *t, int count, int zeroed, const int64_t *kept, const int32_t *len, int64_t B, int64_t Hkv,
                             int64_t keep, int64_t max_len, int64_t cap, hipStream_t s) {
    if (count <= 0) return hipSuccess;
    if (count > 3 || B * Hkv > 65535) return hipErrorInvalidConfiguration;
    MoveArgs a{};
    for (int z = 0; z < count; ++z) {
        a.rows[z] = (char *)t[z].rows;
        a.temp[z] = (char *)t[z].temp;
        a.row_bytes[z] = t[z].row_bytes;
        int p = 16;
        while (p > 2 && (t[z].row_bytes % p || (uintptr_t)t[z].rows % p || (uintptr_t)t[z].temp % p)) p /= 2;
        a.piece[z] = p;
    }
    a.kept = kept;
    a.len = len;
    a.Hkv = (int)Hkv;
    a.keep = (int)keep;
    a.zeroed = zeroed;
    a.cap = cap;
    const unsigned out = (unsigned)((keep + 15) / 16), back = (unsigned)((std::max(keep, max_len) + 15) / 16);
    hipLaunchKernelGGL((kv_move_kernel<false>), dim3(out, (unsigned)(B * Hkv), (unsigned)count), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((kv_move_kernel<true>), dim3(back, (unsigned)(B * Hkv), (unsigned)count), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t gt_launch_kv_rows_read(const void *k, const void *v, int dtype, const int32_t *len, void *ko, void *vo, int out_dtype,
                                  int64_t B, int64_t Hkv, int64_t rows, int64_t D, int64_t cap, hipStream_t s) {
    if (B * Hkv * rows * D <= 0) return hipSuccess;
    switch (dtype) {
        case GT_F32: return launch_rows_read<GT_F32>(k, v, len, ko, vo, out_dtype, B, Hkv, rows, D, cap, D * 4, s);
        case GT_F16: return launch_rows_read<GT_F16>(k, v, len, ko, vo, out_dtype, B, Hkv, rows, D, cap, D * 2, s);
        case GT_BF16: return launch_rows_read<GT_BF16>(k, v, len, ko, vo, out_dtype, B, Hkv, rows, D, cap, D * 2, s);
        case GT_Q8_0: return launch_rows_read<GT_Q8_0>(k, v, len, ko, vo, out_dtype, B, Hkv, rows, D, cap, D / 32 * 34, s);
        default: return hipErrorInvalidValue;
    }
}
