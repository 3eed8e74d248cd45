// The C++ calls on the paged cache, with the default arguments they rely on (compiled, not run).
#include "kernels.hpp"

void step(half* q, half* k, half* v, half* out, const half* bias, const half* norm, int32_t* selected, int8_t* bounds,
          float* steps, float* lse, void* ws, const double* turns, int32_t* table, hipStream_t s) {
    const qwen::PagedCache cache{reinterpret_cast<uint16_t*>(k), reinterpret_cast<uint16_t*>(v), 0, 16, 64,
                                 qwen::NUM_KV_HEADS, qwen::HEAD_DIM};
    const qwen::PagedBatch batch{table, nullptr, table, 4, 4, 8};
    const qwen::Rope rope{turns, 128, 0, 1.0f};
    qwen::launch_qkv_norm_rope_paged_append(q, q, k, v, bias, bias, bias, norm, norm, &rope, cache, batch, s);
    qwen::launch_qkv_norm_rope_paged_append(q, out, k, v, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, cache,
                                            batch, s, 12, 2048, 2048, 1e-5f);
    qwen::launch_attention_gqa_paged_decode(q, cache, batch, ws, out, s);
    qwen::launch_attention_gqa_paged_prefill(q, cache, batch, ws, out, s, 12, 4096, lse);
    qwen::launch_paged_key_bounds(cache, batch, bounds, steps, s);
    qwen::launch_paged_select(q, cache, batch, bounds, steps, selected, ws, s);
    qwen::launch_attention_gqa_paged_sparse(q, cache, batch, selected, ws, out, s, 12, 32, lse);
}
