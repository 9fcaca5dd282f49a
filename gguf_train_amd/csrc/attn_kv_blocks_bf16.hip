// attn_kv_blocks.h for bfloat16 queries.
#include "attn_kv_blocks.h"

const void *gtkvb::attn_kernel_bf16(int Dp, bool e4m3, int waves) { return attn_kernel<__bf16>(Dp, e4m3, waves); }
