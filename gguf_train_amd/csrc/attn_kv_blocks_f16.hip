// attn_kv_blocks.h for float16 queries.
#include "attn_kv_blocks.h"

const void *gtkvb::attn_kernel_f16(int Dp, bool e4m3, int waves) { return attn_kernel<_Float16>(Dp, e4m3, waves); }
