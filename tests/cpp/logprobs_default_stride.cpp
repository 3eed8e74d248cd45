// What the C++ wrapper hands to the C entry point as the row stride of log
// probability calls (see tests/test_kv4_mirror.py).  The entry point here only
// records it: nothing is launched and no library is linked.
#include <cstdio>

#include "kernels.hpp"

namespace {
long long seen = -1;
}

extern "C" int qe_launch_token_logprobs(const uint16_t*, const int32_t*, float*, float*, float*, int32_t*, void*, int, int,
                                        long long row_stride, int, hipStream_t) {
    seen = row_stride;
    return QE_OK;
}
extern "C" const char* qe_last_error() { return ""; }

int main() {
    const half* x = nullptr;
    const int32_t* ids = nullptr;
    float* out = nullptr;
    auto call = [&](auto... rest) {
        qwen::launch_token_logprobs(x, ids, out, out, nullptr, nullptr, nullptr, 2, nullptr, rest...);
        std::printf("%lld ", seen);
    };
    call();               // the default vocabulary, rows behind each other
    call(1000);           // a smaller one, rows behind each other too
    call(1000, 1000LL);
    call(1000, 1024LL);
    call(1000, 999LL);    // given: for the entry point to refuse
    call(1000, -5LL);
    call(200000);
    return 0;
}
