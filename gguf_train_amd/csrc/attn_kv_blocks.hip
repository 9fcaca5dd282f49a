// Launches of the attention over the 8-bit block cache (attn_kv_blocks.h).

#include "attn_kv_blocks.h"

#include <cmath>
#include <string>

namespace {

using namespace gtkvb;

const void *kernel_of(int q_dtype, int Dp, bool e4m3, int waves) {
    switch (q_dtype) {
        case GT_F16: return attn_kernel_f16(Dp, e4m3, waves);
        case GT_BF16: return attn_kernel_bf16(Dp, e4m3, waves);
        case GT_F32: return attn_kernel_f32(Dp, e4m3, waves);
        default: return nullptr;
    }
}

// Workgroups of `kernel` the device runs at once.
int64_t resident_groups(const void *kernel, int waves) {
    static std::mutex mu;
    static std::map<std::pair<int, const void *>, int64_t> known;
    int dev = 0;
    (void)hipGetDevice(&dev);
    std::lock_guard<std::mutex> lock(mu);
    auto it = known.find({dev, kernel});
    if (it != known.end()) return it->second;
    int cus = 0, per = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, 64 * waves, 0) != hipSuccess || per <= 0) per = 1;
    return known[{dev, kernel}] = (int64_t)cus * per;
}

}  // namespace

// Whether this attention serves the call, or the values are read back and the attention over rows of values does.
// Its work grows with the rows, and fills the GPU whatever their number, as the sequence is split; the other path
// costs the reading back and runs faster per row, once it has rows enough.  Measured (int8, float16 queries, us, this
// against the other): D128 B8 Hkv8 S4096 128 rows 60 against 110, 256 rows (1024 groups) 120 against 112, 512 rows
// 205 against 118; B16 Hkv8 S2048 128 rows 78 against 96, 256 rows 118 against 101; B1 Hkv8 S4096 1024 rows (512
// groups) 57 against 90, 2048 rows 100 against 91; B4 Hkv8 S512 256 rows 13.7 against 21.7, 1024 rows 37 against 24;
// B1 Hkv2 S16384 4096 rows (512 groups) 169 against 302.  float32 queries and more than 128 dims have no such fast
// path (D128 B16 Hkv8 S2048 64 rows float32 39 against 567, D256 B8 Hkv8 S4096 512 rows 487 against 49550).
bool gt_kv_blocks_attn_supported(const gt_kv_blocks &c, int64_t H, int64_t L, int q_dtype) {
    const int64_t rows = H / c.Hkv * L, groups = c.B * c.Hkv * ((rows + kColumns - 1) / kColumns);
    const bool better = rows <= 128 || groups <= 512 || q_dtype == GT_F32 || c.Dp > 128;
    return (q_dtype == GT_F16 || q_dtype == GT_BF16 || q_dtype == GT_F32) && better && c.B * H * L < (1LL << 31);
}

hipError_t gt_launch_kv_blocks_attn(const gt_kv_blocks &c, const gt_kv_blocks_attn &r, int dev, hipStream_t s, std::string &note) {
    AttnArgs a{};
    a.q = r.q;
    a.q_sb = r.q_strides[0];
    a.q_sh = r.q_strides[1];
    a.q_sl = r.q_strides[2];
    a.o = r.o;
    a.lse = r.lse;
    a.k = (const uint8_t *)c.codes[0];
    a.v = (const uint8_t *)c.codes[1];
    a.ks = c.scales[0];
    a.vs = c.scales[1];
    a.kt = (const _Float16 *)c.ops[0];
    a.vt = (const _Float16 *)c.ops[1];
    a.kts = c.op_scales[0];
    a.vts = c.op_scales[1];
    a.len = r.len;
    a.scale = r.scale;
    a.causal = r.causal;
    const int64_t per16 = r.q_dtype == GT_F32 ? 4 : 8;
    a.q_vec = c.D % 16 == 0 && (uintptr_t)r.q % 16 == 0 && a.q_sb % per16 == 0 && a.q_sh % per16 == 0 && a.q_sl % per16 == 0;
    a.B = (int)c.B;
    a.H = (int)r.H;
    a.Hkv = (int)c.Hkv;
    a.L = (int)r.L;
    a.D = (int)c.D;
    a.shift = c.N == 32 ? 5 : c.N == 64 ? 6 : 7;
    a.units = c.units;
    const int64_t rows = r.H / c.Hkv * r.L, groups = (rows + kColumns - 1) / kColumns;
    // splits: a workgroup's wavefronts take a unit each per step
    const int64_t units = (r.max_len / c.N * c.N + kUnit - 1) / kUnit;
    const int64_t grid = c.B * c.Hkv * groups;
    if (grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    const void *kernel = nullptr;
    int64_t per = 0;
    int n = 0;
    auto split = [&](int waves) {
        kernel = kernel_of(r.q_dtype, c.Dp, c.e4m3, waves);
        if (!kernel) return;
        const int64_t steps = std::max<int64_t>(1, (units + waves - 1) / waves);
        n = decode_split_count(grid, steps, resident_groups(kernel, waves), std::min<int64_t>(64, steps));
        per = (steps + n - 1) / n;
        n = (int)((steps + per - 1) / per);
    };
    // Workgroups of four wavefronts where they need no splits; otherwise of eight, which leave half the partials to
    // join or none.  (int8, float16, D128 Hkv8 G4, us with four and eight: B4 S4096 32 tokens 31.5, 27.0; B4 S1024
    // 32 tokens 16.4, 11.8; B8 S4096 5 tokens 25.9, 21.9; B4 S16384 one token 29.1, 25.9; B1 S4096 one token 10.6,
    // 11.3; without splits B64 S512 one token 13.8, 20.4; B8 S777 32 tokens 17.8, 24.3.)
    int waves = 4;
    split(waves);
    if (n > 1 && c.Dp <= 128) split(waves = 8);
    if (!kernel) return hipErrorInvalidValue;
    gt_decode_ws ws{};
    if (n > 1) {
        const size_t out_rows = (size_t)(c.B * r.H * r.L) * (size_t)n;
        if (gt_decode_workspace(dev, s, grid, out_rows * (size_t)(c.Dp + 2) * sizeof(float), ws)) {
            a.counters = ws.counters;
            a.part_o = (float *)ws.parts;
            a.part_ml = a.part_o + out_rows * (size_t)c.Dp;
        } else {
            n = 1;  // (no workspace for this stream, or a batch that fills the GPU without splits)
            per = (units + waves - 1) / waves;
        }
    }
    a.nsplit = n;
    a.span = (int)(per * waves);
    note = std::string("decode ") + (c.e4m3 ? "e4m3" : "int8") + " blocks of " + std::to_string(c.N) + " D=" + std::to_string(c.D) +
           " rows=" + std::to_string(rows) + " splits=" + std::to_string(n) +
           " units=" + std::to_string(grid);
    void *args[] = {(void *)&a};
    const size_t lds = (size_t)attn_lds_floats((int)std::min<int64_t>(rows, kColumns), c.Dp, n, waves) * sizeof(float);
    return hipLaunchKernel(kernel, dim3((unsigned)grid, (unsigned)n), dim3((unsigned)(64 * waves)), args, lds, s);
}
