// The fast decode (decode_wg.h) over rows that attend through a window with sinks.
#include "decode_wg.h"

namespace ckv {

hipError_t launch_window_fast(hipStream_t s, const pool_view& p, const meta_view& m,
                              uint32_t layer, const void* q, uint32_t q_heads, float scale_log2,
                              void* out, const void* k_in, const void* v_in, const void* gate,
                              int cu_count, split_scratch split, const rope_table* rope,
                              uint32_t rotary)
{
    return launch_width<true>(p.head_dim, q_heads / p.kv_heads, s, p, m, layer, q, q_heads,
                              scale_log2, out, p.dtype, k_in, v_in, gate, cu_count, split, rope,
                              rotary);
}

} // namespace ckv
