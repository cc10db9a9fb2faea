// The fast decode (decode_wg.h) over rows that attend through a window with sinks.
//
// Bound by HBM once the rows fill the GPU, by the chain of a launch before. Measured on
// MI355X, bf16, new rows appended in the launch: 48 rows of 900 to 12,000 tokens, 8 kv
// and 16 q heads of 128, behind 1,024 tokens and 4 sinks, 39.5 us, 5.1 TB/s (one wave
// for each chunk of tokens and kv head, then a merge, took 334); 24 gated rows of 2 kv
// and 8 q heads of 256 behind 2,048 and 16 sinks 27.9 us, 3.2 TB/s (493); 4 rows of 60
// to 1,900 tokens behind 512 6.6 us (82.6).
#include "decode_wg.h"

namespace ckv {

uint32_t decode_window_waves(uint32_t head_dim, uint32_t group, int dtype, uint32_t units,
                             int cu_count, uint32_t mean_pages, uint32_t split_pages)
{
    return window_waves(head_dim, group, dtype, units, cu_count, mean_pages, split_pages);
}

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
