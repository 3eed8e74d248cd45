// Compiles the calls a host program makes of the 4-bit cache and log probability
// launchers, with their default arguments (compile-only; see tests/test_kv4_routes.py).
#include "kernels.hpp"

using namespace qwen;

void session(const half* q, half* q_out, const half* k, const half* v, const half* qb, const half* kb, const half* vb,
             uint8_t* kc, uint8_t* vc, void* ws, half* attn, const DeviceControlBlock* ctl, int32_t* evicted,
             float* weights, float* lse, int32_t* kept, int8_t* q8, float* scale, int32_t* sum8, hipStream_t s) {
    launch_qkv_bias_rope_kv4_append(q, q_out, k, v, qb, kb, vb, kc, vc, ctl, evicted, 7, s);
    launch_attention_gqa_prefill_kv4(q_out, kc, vc, attn, ctl, evicted, 7, s);
    launch_attention_gqa_prefill_kv4(q_out, kc, vc, attn, ctl, nullptr, 7, s, 12, 2, 128, 4096, 1536, weights, weights, lse);
    size_t bytes = 0;
    if (qe_kv4_decode_workspace_bytes(NUM_Q_HEADS, MAX_SEQ_LEN, 1, &bytes) != QE_OK) return;
    launch_attention_gqa_flash_decode_kv4(q_out, kc, vc, ws, attn, ctl, evicted, s);
    launch_attention_gqa_flash_decode_kv4(q_out, kc, vc, ws, attn, ctl, evicted, s, 12, 2, 128, 4096, q8, scale, sum8, weights, weights);
    launch_kv4_evict(kc, vc, weights, evicted, kc, vc, weights, evicted, kept, ctl, 2048, 4, 512, s);
    launch_kv4_unpack(kc, vc, attn, attn, 0, 2048, s);
}

void score(const half* logits, const int32_t* ids, float* lp, float* entropy, float* top, int32_t* top_ids, void* ws,
           hipStream_t s) {
    launch_token_logprobs(logits, ids, lp, entropy, nullptr, nullptr, ws, 9, s);
    launch_token_logprobs(logits, ids, lp, nullptr, top, top_ids, ws, 9, s, VOCAB_SIZE, VOCAB_SIZE, 20);
    launch_token_logprobs(logits, nullptr, nullptr, entropy, nullptr, nullptr, ws, 1, s, 1000);
}
