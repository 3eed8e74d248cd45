// What the C++ wrapper hands to the C entry point as the width of a row of outputs
// of 4-bit prefill attention (see tests/test_kv4_mirror.py).  The entry point here
// only records it: nothing is launched and no library is linked.
#include <cstdio>

#include "kernels.hpp"

namespace {
int seen = -1;
}

extern "C" int qe_launch_attention_gqa_prefill_kv4(const uint16_t*, const uint8_t*, const uint8_t*, uint16_t*,
                                                   const qe_device_control_block*, const int32_t*, int, hipStream_t, int,
                                                   int, int, int, int hidden_size, const float*, float*, float*) {
    seen = hidden_size;
    return QE_OK;
}
extern "C" const char* qe_last_error() { return ""; }

int main() {
    auto call = [&](auto... rest) {
        qwen::launch_attention_gqa_prefill_kv4(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 7, nullptr, rest...);
        std::printf("%d ", seen);
    };
    call();                           // the default model: rows of 12 heads behind each other
    call(6, 2);                       // fewer heads, rows behind each other too
    call(28, 4);
    call(6, 2, 128, 4096, 768);
    call(6, 2, 128, 4096, 1536);      // given: wider rows
    call(6, 2, 128, 4096, 512);       // given: for the entry point to refuse
    return 0;
}
