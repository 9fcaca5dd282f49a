// attn_kv_blocks.h for float32 queries.
#include "attn_kv_blocks.h"

const void *gtkvb::attn_kernel_f32(int Dp, bool e4m3, int waves) { return attn_kernel<float>(Dp, e4m3, waves); }
