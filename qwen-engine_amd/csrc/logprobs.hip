// Log probabilities of given tokens, entropy and the most likely alternatives of
// rows of fp16 logits, in one pass over the logits.
//
// With m = max x, S = sum exp(x - m), T = sum exp(x - m) (x - m):
//   log p(i) = x_i - m - log S,  entropy = log S - T / S.
// A row is cut into segments of 8192 logits, a block each, whose logits stay in
// registers; the segments' (m, S, T) and their k largest (logit, index) meet in a
// second kernel, a block a row.  Sums and statistics in fp32.
//
// Order of the alternatives: larger logit first, equal logits (-0 and +0 too) by
// the lower index, NaN never.  -inf has probability 0; a row of nothing else gives
// -inf for every token and entropy 0; a row with a NaN or +inf gives NaN.
#include <algorithm>

#include "qe_common.hpp"

namespace qe {
namespace {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr int kLpSegment = 8192;                      // logits of a block: 32 a thread
constexpr int kLpChunks = kLpSegment / (8 * kLpThreads);  // 16-byte chunks of a thread
constexpr int kLpMaxTop = 32;
constexpr float kLpLog2e = 1.4426950408889634f;

// Segments of a row: the first starts at a 16-byte boundary, up to 7 logits before the row.
__host__ __device__ __forceinline__ int lp_segments(int vocab) { return (vocab + 7 + kLpSegment - 1) / kLpSegment; }
// Words that one segment leaves: m, S, T, and its keys.
__host__ __device__ __forceinline__ int lp_words(int top) { return 3 + top; }

// fp16 bits as whole numbers of the same order; NaN is 0, below -inf (0x03FF).
__device__ __forceinline__ uint32_t lp_order(uint16_t b) {
    if ((b & 0x7FFFu) > 0x7C00u) return 0;
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? static_cast<uint16_t>(~b) : static_cast<uint16_t>(b | 0x8000u);
}
__device__ __forceinline__ float lp_logit(uint32_t order) {
    return h2f(static_cast<uint16_t>(order & 0x8000u ? order & 0x7FFFu : ~order));
}

// Bitonic network over the 64 lanes: lane 0 ends with the largest.
template <class T>
__device__ __forceinline__ T lp_exchange(T v, int lane, int j, bool down) {
    const T o = __shfl_xor(v, j);
    const bool larger = ((lane & j) == 0) == down;
    return larger ? (o > v ? o : v) : (o < v ? o : v);
}
template <class T>
__device__ __forceinline__ T lp_sort(T v, int lane) {
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) v = lp_exchange(v, lane, j, (lane & k) == 0);
    return v;
}
// The 64 largest of two sorted sets.
template <class T>
__device__ __forceinline__ T lp_merge(T a, T b, int lane) {
    const T o = __shfl_xor(b, 63);
    T v = a > o ? a : o;
#pragma unroll
    for (int j = 32; j > 0; j >>= 1) v = lp_exchange(v, lane, j, true);
    return v;
}

__global__ __launch_bounds__(kLpThreads) void token_logprobs_segment_kernel(const uint16_t* __restrict__ logits,
                                                                            uint32_t* __restrict__ parts, int vocab,
                                                                            long long row_stride, int segments,
                                                                            int top) {
    __shared__ uint32_t s_key[kLpWaves][kLpSegment / kLpWaves];
    __shared__ float s_st[kLpWaves][3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long row = blockIdx.x / segments;
    const int seg = static_cast<int>(blockIdx.x % segments);
    const uint16_t* x = logits + row * row_stride;
    const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) >> 1);  // logits past a 16-byte boundary
    const int seg0 = seg * kLpSegment - skew;
    uint16_t v[kLpChunks][8];
    uint32_t in = 0;  // which of the thread's logits belong to the row
#pragma unroll
    for (int c = 0; c < kLpChunks; ++c) {
        const int i0 = seg0 + (c * kLpThreads + tid) * 8;
        if (i0 >= 0 && i0 + 8 <= vocab) {
            const u32x4 raw = *reinterpret_cast<const u32x4*>(x + i0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = raw[e];
                v[c][2 * e] = static_cast<uint16_t>(w);
                v[c][2 * e + 1] = static_cast<uint16_t>(w >> 16);
            }
            in |= 0xFFu << (8 * c);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool ok = i0 + e >= 0 && i0 + e < vocab;
                v[c][e] = ok ? x[i0 + e] : 0xFC00u;  // -inf
                in |= static_cast<uint32_t>(ok) << (8 * c + e);
            }
        }
    }
    float mine = -INFINITY;
#pragma unroll
    for (int c = 0; c < kLpChunks; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) mine = fmaxf(mine, h2f(v[c][e]));
    const float m = qwen::seg_max<64>(mine);
    const float ref = m == -INFINITY ? 0.0f : m;
    float S = 0.0f, T = 0.0f;
#pragma unroll
    for (int c = 0; c < kLpChunks; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = h2f(v[c][e]) - ref;
            const float p = __builtin_amdgcn_exp2f(d * kLpLog2e);
            S += p;
            T = __builtin_fmaf(p, fmaxf(d, -1e4f), T);  // p is 0 there, and d may be -inf
        }
    S = qwen::seg_sum<64>(S);
    T = qwen::seg_sum<64>(T);
    if (lane == 0) {
        s_st[wave][0] = m;
        s_st[wave][1] = S;
        s_st[wave][2] = T;
    }
    uint32_t* out = parts + (row * segments + seg) * lp_words(top);
    if (top > 0) {
        // the top-th largest of the lanes' maxima: at least `top` logits reach it, few do
        const float cut = __shfl(lp_sort(mine, lane), top - 1);
        int n = 0;
#pragma unroll
        for (int c = 0; c < kLpChunks; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool take = h2f(v[c][e]) >= cut && ((in >> (8 * c + e)) & 1u);
                const uint64_t b = __builtin_amdgcn_ballot_w64(take);
                if (b == 0) continue;
                // index within the segment, the lower the larger
                if (take)
                    s_key[wave][n + __popcll(b & ((1ull << lane) - 1))] =
                        (lp_order(v[c][e]) << 16) | (0xFFFFu - ((c * kLpThreads + tid) * 8 + e));
                n += __popcll(b);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave reads what its lanes wrote
        uint32_t best = 0;
        for (int i = 0; i < n; i += 64) {
            const uint32_t k = lp_sort(i + lane < n ? s_key[wave][i + lane] : 0u, lane);
            best = i == 0 ? k : lp_merge(best, k, lane);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane < top) s_key[wave][lane] = best;
    }
    __syncthreads();
    if (wave != 0) return;
    float mg = s_st[0][0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) mg = fmaxf(mg, s_st[w][0]);
    float Sg = 0.0f, Tg = 0.0f;
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) {
        const float d = s_st[w][0] == mg ? 0.0f : fmaxf(s_st[w][0] - mg, -1e4f);
        const float f = __builtin_amdgcn_exp2f(d * kLpLog2e);
        Sg += f * s_st[w][1];
        Tg += f * (s_st[w][2] + d * s_st[w][1]);
    }
    if (lane == 0) {
        out[0] = __builtin_bit_cast(uint32_t, mg);
        out[1] = __builtin_bit_cast(uint32_t, Sg);
        out[2] = __builtin_bit_cast(uint32_t, Tg);
    }
    if (top > 0) {
        uint32_t best = lane < top ? s_key[0][lane] : 0u;
        for (int w = 1; w < kLpWaves; ++w) best = lp_merge(best, lane < top ? s_key[w][lane] : 0u, lane);
        if (lane < top) out[3 + lane] = best;
    }
}

__global__ __launch_bounds__(kLpThreads) void token_logprobs_row_kernel(
    const uint16_t* __restrict__ logits, const uint32_t* __restrict__ parts, const int32_t* __restrict__ ids,
    float* __restrict__ out_logprob, float* __restrict__ out_entropy, float* __restrict__ top_logprob,
    int32_t* __restrict__ top_ids, int vocab, long long row_stride, int segments, int top) {
    __shared__ float s_st[kLpWaves][3];
    __shared__ unsigned long long s_key[kLpWaves][kLpMaxTop];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long row = blockIdx.x;
    const uint16_t* x = logits + row * row_stride;
    const int words = lp_words(top);
    const uint32_t* part = parts + row * segments * words;
    float m = -INFINITY, S = 0.0f, T = 0.0f;
    for (int s = tid; s < segments; s += kLpThreads) {
        const float ms = __builtin_bit_cast(float, part[s * words]), Ss = __builtin_bit_cast(float, part[s * words + 1]),
                    Ts = __builtin_bit_cast(float, part[s * words + 2]);
        const float mn = fmaxf(m, ms);
        const float da = m == mn ? 0.0f : fmaxf(m - mn, -1e4f), db = ms == mn ? 0.0f : fmaxf(ms - mn, -1e4f);
        const float fa = __builtin_amdgcn_exp2f(da * kLpLog2e), fb = __builtin_amdgcn_exp2f(db * kLpLog2e);
        T = fa * (T + da * S) + fb * (Ts + db * Ss);
        S = fa * S + fb * Ss;
        m = mn;
    }
    const float mw = qwen::seg_max<64>(m);
    {
        const float d = m == mw ? 0.0f : fmaxf(m - mw, -1e4f), f = __builtin_amdgcn_exp2f(d * kLpLog2e);
        T = qwen::seg_sum<64>(f * (T + d * S));
        S = qwen::seg_sum<64>(f * S);
    }
    if (lane == 0) {
        s_st[wave][0] = mw;
        s_st[wave][1] = S;
        s_st[wave][2] = T;
    }
    if (top > 0) {
        const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) >> 1);
        unsigned long long best = 0;
        const int n = segments * top;
        for (int i0 = 64 * wave; i0 < n; i0 += kLpThreads) {
            const int i = i0 + lane;
            unsigned long long k = 0;
            if (i < n) {
                const int s = i / top;
                const uint32_t key = part[s * words + 3 + (i - s * top)];
                const uint32_t at = s * kLpSegment - skew + (0xFFFFu - (key & 0xFFFFu));
                if (key != 0) k = (static_cast<unsigned long long>(key >> 16) << 32) | (0xFFFFFFFFu - at);
            }
            best = lp_merge(best, lp_sort(k, lane), lane);
        }
        if (lane < top) s_key[wave][lane] = best;
    }
    __syncthreads();
    if (wave != 0) return;
    float mg = s_st[0][0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) mg = fmaxf(mg, s_st[w][0]);
    S = T = 0.0f;
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) {
        const float d = s_st[w][0] == mg ? 0.0f : fmaxf(s_st[w][0] - mg, -1e4f);
        const float f = __builtin_amdgcn_exp2f(d * kLpLog2e);
        S += f * s_st[w][1];
        T += f * (s_st[w][2] + d * s_st[w][1]);
    }
    const bool nothing = S == 0.0f;  // every logit is -inf
    const float log_s = logf(S);
    auto logprob = [&](float logit) { return nothing ? -INFINITY : logit - mg - log_s; };
    if (lane == 0) {
        if (out_logprob != nullptr) {
            const int id = ids[row];
            out_logprob[row] = id >= 0 && id < vocab ? logprob(h2f(x[id])) : 0.0f;
        }
        if (out_entropy != nullptr) out_entropy[row] = nothing ? 0.0f : log_s - T / S;
    }
    if (top > 0) {
        unsigned long long best = lane < top ? s_key[0][lane] : 0ull;
        for (int w = 1; w < kLpWaves; ++w) best = lp_merge(best, lane < top ? s_key[w][lane] : 0ull, lane);
        if (lane < top) {
            const bool none = best == 0;
            if (top_ids != nullptr)
                top_ids[row * top + lane] = none ? -1 : static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
            if (top_logprob != nullptr)
                top_logprob[row * top + lane] =
                    none ? __builtin_nanf("") : logprob(lp_logit(static_cast<uint32_t>(best >> 32)));
        }
    }
}

}  // namespace
}  // namespace qe

using namespace qe;

extern "C" int qe_token_logprobs_workspace_bytes(int num_rows, int vocab_size, int top_k, size_t* bytes) {
    const char* what = "token_logprobs_workspace_bytes";
    QE_REQUIRE(bytes != nullptr, "%s: NULL pointer", what);
    QE_REQUIRE(num_rows >= 0 && vocab_size > 0 && vocab_size <= INT32_MAX - kLpSegment && top_k >= 0 && top_k <= kLpMaxTop,
               "%s: num_rows=%d vocab_size=%d top_k=%d", what, num_rows, vocab_size, top_k);
    *bytes = static_cast<size_t>(num_rows) * lp_segments(vocab_size) * lp_words(top_k) * sizeof(uint32_t);
    return QE_OK;
}

extern "C" int qe_launch_token_logprobs(const uint16_t* logits, const int32_t* token_ids, float* out_logprob,
                                        float* out_entropy, float* out_top_logprob, int32_t* out_top_ids,
                                        void* workspace, int num_rows, int vocab_size, long long row_stride, int top_k,
                                        hipStream_t stream) {
    const char* what = "token_logprobs";
    QE_REQUIRE(logits && workspace, "%s: NULL pointer", what);
    QE_REQUIRE((token_ids == nullptr) == (out_logprob == nullptr), "%s: token_ids and out_logprob are given together",
               what);
    QE_REQUIRE(vocab_size > 0 && vocab_size <= INT32_MAX - kLpSegment, "%s: vocab_size=%d", what, vocab_size);
    QE_REQUIRE(row_stride >= vocab_size || num_rows <= 1, "%s: row_stride=%lld < vocab_size=%d", what, row_stride,
               vocab_size);
    QE_REQUIRE(top_k >= 0 && top_k <= kLpMaxTop && top_k <= vocab_size, "%s: top_k=%d (0..%d, at most vocab_size)", what,
               top_k, kLpMaxTop);
    QE_REQUIRE((out_top_logprob == nullptr && out_top_ids == nullptr) || top_k > 0, "%s: top outputs with top_k=0", what);
    QE_REQUIRE(top_k == 0 || out_top_logprob || out_top_ids, "%s: top_k=%d without an output", what, top_k);
    QE_REQUIRE(aligned(logits, 2) && aligned(workspace, 4), "%s: alignment", what);
    if (num_rows <= 0) return QE_OK;
    const int segments = lp_segments(vocab_size);
    QE_REQUIRE(static_cast<long long>(num_rows) * segments <= INT32_MAX, "%s: num_rows=%d", what, num_rows);
    uint32_t* parts = static_cast<uint32_t*>(workspace);
    token_logprobs_segment_kernel<<<num_rows * segments, kLpThreads, 0, stream>>>(logits, parts, vocab_size, row_stride,
                                                                                  segments, top_k);
    token_logprobs_row_kernel<<<num_rows, kLpThreads, 0, stream>>>(logits, parts, token_ids, out_logprob, out_entropy,
                                                                   out_top_logprob, out_top_ids, vocab_size, row_stride,
                                                                   segments, top_k);
    return check_launch(what);
}
