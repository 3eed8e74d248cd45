// Log probabilities of given tokens, entropy and the most likely alternatives of
// rows of fp16 logits, in one pass over the logits.
//
// With m = max x, S = sum exp(x - m), T = sum exp(x - m) (x - m):
//   log p(i) = x_i - m - log S,  entropy = log S - T / S.
// A row is cut into segments of 8192 or 32768 logits, a block each, whose logits stay in
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
constexpr int kLpMaxTop = 32;
constexpr float kLpLog2e = 1.4426950408889634f, kLpLn2 = 0.6931471805599453f;
// 16-byte chunks of a thread of the segment kernel: with many rows 16 (segments of
// 32768 logits), so that the selection of the alternatives, the same work for a
// segment of any length, is seldom; with few 4 (8192), so that a row is spread over the chip.
constexpr int kLpFew = 4, kLpMany = 16;
constexpr int lp_segment(int chunks) { return 8 * kLpThreads * chunks; }
// Vocabularies, at most: a row's last segment, which begins before index vocab + 7, ends within 31 bits.
constexpr int kLpMaxVocab = INT32_MAX - 7 - lp_segment(kLpMany);

// Candidates of a wave in LDS.
constexpr int kLpCandidates = 1024;

// Segments of a row: the first starts at a 16-byte boundary, up to 7 logits before the row.
__host__ __device__ __forceinline__ int lp_segments(int vocab, int chunks) {
    return (vocab + 7 + lp_segment(chunks) - 1) / lp_segment(chunks);
}
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

// The value of lane ^ J, by DPP within 16 lanes and lane swaps above.
template <int J>
__device__ __forceinline__ uint32_t lp_partner(uint32_t v) {
    const int x = static_cast<int>(v);
    if constexpr (J == 1) return static_cast<uint32_t>(qwen::dpp_i32<0xB1>(x));
    if constexpr (J == 2) return static_cast<uint32_t>(qwen::dpp_i32<0x4E>(x));
    if constexpr (J == 4) return static_cast<uint32_t>(qwen::dpp_i32<0x1B>(qwen::dpp_i32<0x141>(x)));  // ^7, ^3
    if constexpr (J == 8) return static_cast<uint32_t>(qwen::dpp_i32<0x128>(x));                       // row_ror 8
    if constexpr (J == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        const uint32_t a = r[0], b = r[1];
        return (threadIdx.x & 16) ? a : b;
    }
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t a = r[0], b = r[1];
    return (threadIdx.x & 32) ? a : b;
}
template <int J>
__device__ __forceinline__ unsigned long long lp_partner(unsigned long long v) {
    return static_cast<unsigned long long>(lp_partner<J>(static_cast<uint32_t>(v))) |
           (static_cast<unsigned long long>(lp_partner<J>(static_cast<uint32_t>(v >> 32))) << 32);
}

// Bitonic network over the 64 lanes: lane 0 ends with the largest.
template <int J, class T>
__device__ __forceinline__ T lp_exchange(T v, bool larger) {
    const T o = lp_partner<J>(v);
    return larger ? (o > v ? o : v) : (o < v ? o : v);
}
// The steps from J down, where `down` says whether the block of lanes sorts downwards.
template <int J, class T>
__device__ __forceinline__ T lp_steps(T v, int lane, bool down) {
    v = lp_exchange<J>(v, ((lane & J) == 0) == down);
    if constexpr (J > 1) return lp_steps<J / 2>(v, lane, down);
    else return v;
}
template <class T>
__device__ __forceinline__ T lp_sort(T v, int lane) {
    v = lp_steps<1>(v, lane, (lane & 2) == 0);
    v = lp_steps<2>(v, lane, (lane & 4) == 0);
    v = lp_steps<4>(v, lane, (lane & 8) == 0);
    v = lp_steps<8>(v, lane, (lane & 16) == 0);
    v = lp_steps<16>(v, lane, (lane & 32) == 0);
    return lp_steps<32>(v, lane, true);
}
// The 64 largest of two sorted sets.
template <class T>
__device__ __forceinline__ T lp_merge(T a, T b, int lane) {
    const T o = __shfl_xor(b, 63);
    return lp_steps<32>(a > o ? a : o, lane, true);
}

// One segment.  exp(x - m) is 2^(x L - m L), L = log2 e, in one fused multiply-add
// with c = m L rounded; what the rounding leaves, r = m L - c, is the same for every
// logit of the wave and comes off at the end: S = 2^-r S', T = ln 2 (T' - r S') 2^-r.
// Per logit that is a conversion, the multiply-add, the exponential, two sums, a clamp
// (-inf times 0) and a comparison, 6.5 vector instructions, and with long segments as many
// again that a wave has whatever its logits are (filling with -inf, the row's edges, the
// alternatives' cut and sorts): 12.7 counted, beside the memory.  1024 rows of 151936 with
// five alternatives 61 us (311 MB, 5.1 TB/s; a plain read takes 47), one row 6.2.
template <int CHUNKS>
__global__ __launch_bounds__(kLpThreads, 4) void token_logprobs_segment_kernel(const uint16_t* __restrict__ logits,
                                                                               float* __restrict__ stats,
                                                                               uint32_t* __restrict__ keys, int vocab,
                                                                               long long row_stride, int segments,
                                                                               int top) {
    constexpr int kSegment = lp_segment(CHUNKS);
    static_assert(kSegment <= 0x10000, "an index is 16 bits of a key");
    __shared__ uint32_t s_key[kLpWaves][kLpCandidates];
    __shared__ float s_st[kLpWaves][3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long row = blockIdx.x / segments;
    const int seg = static_cast<int>(blockIdx.x % segments);
    const uint16_t* x = logits + row * row_stride;
    const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) >> 1);  // logits past a 16-byte boundary
    const int seg0 = seg * kSegment - skew;
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    uint32_t v[CHUNKS][4];
    uint32_t part = 0;  // chunks that lie only partly in the row, or behind it
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int i0 = seg0 + (c * kLpThreads + tid) * 8;
        if (i0 >= 0 && i0 + 8 <= vocab) {
            const u32x4 raw = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x + i0));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] = raw[e];
        } else {
            part |= 1u << c;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] = 0xFC00FC00u;  // -inf
        }
    }
    if (__builtin_amdgcn_ballot_w64(part != 0) != 0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int i0 = seg0 + (c * kLpThreads + tid) * 8;
            if (!((part >> c) & 1) || i0 + 8 <= 0 || i0 >= vocab) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i0 + e >= 0 && i0 + e < vocab)
                    v[c][e >> 1] = e & 1 ? (v[c][e >> 1] & 0xFFFFu) | (static_cast<uint32_t>(x[i0 + e]) << 16)
                                         : (v[c][e >> 1] & 0xFFFF0000u) | x[i0 + e];
        }
    }
    auto at = [&](int c, int e) { return h2f(static_cast<uint16_t>(e & 1 ? v[c][e >> 1] >> 16 : v[c][e >> 1])); };
    f16x2 most = {(_Float16)-INFINITY, (_Float16)-INFINITY};
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = v[c][e];
            most = __builtin_elementwise_max(most, __builtin_bit_cast(f16x2, w));  // a NaN is passed over
        }
    const float mine = fmaxf(static_cast<float>(most.x), static_cast<float>(most.y));
    const float m = qwen::seg_max<64>(mine);
    const float ref = m == -INFINITY ? 0.0f : m;
    const float c0 = ref * kLpLog2e, rest = __builtin_fmaf(ref, kLpLog2e, -c0);
    float S = 0.0f, T = 0.0f, S1 = 0.0f, T1 = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float t0 = __builtin_fmaf(at(c, e), kLpLog2e, -c0), t1 = __builtin_fmaf(at(c, e + 1), kLpLog2e, -c0);
            const float p0 = __builtin_amdgcn_exp2f(t0), p1 = __builtin_amdgcn_exp2f(t1);
            S += p0;
            S1 += p1;
            T = __builtin_fmaf(p0, fmaxf(t0, -1e4f), T);  // p is 0 there, and t may be -inf
            T1 = __builtin_fmaf(p1, fmaxf(t1, -1e4f), T1);
        }
    S = qwen::seg_sum<64>(S + S1);
    T = qwen::seg_sum<64>(T + T1);
    if (lane == 0) {
        const float f = __builtin_amdgcn_exp2f(-rest);
        s_st[wave][0] = m;
        s_st[wave][1] = f * S;
        s_st[wave][2] = f * kLpLn2 * (T - rest * S);
    }
    if (top > 0) {
        // The top-th largest of the lanes' maxima: at least `top` logits reach it, few
        // do.  They are collected as bits and index, and sorted 64 at a time.
        float cut = lp_logit(__shfl(lp_sort(lp_order(__builtin_bit_cast(uint16_t, static_cast<_Float16>(mine))), lane), top - 1));
        int n = 0;
        uint32_t best = 0;
        // Index within the segment, the lower the larger.
        auto collect = [&](bool take, uint32_t bits, int i) __attribute__((always_inline)) {
            const uint64_t b = __builtin_amdgcn_ballot_w64(take);
            if (b == 0) return;
            const int slot = n + static_cast<int>(__builtin_amdgcn_mbcnt_hi(
                                     static_cast<uint32_t>(b >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(b), 0u)));
            if (take) s_key[wave][slot] = (bits << 16) | (0xFFFFu - i);
            n += __popcll(b);
        };
        // The last n - from of them, at most 64, into the best so far.
        auto sort_last = [&](int from) __attribute__((always_inline)) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave reads what its lanes wrote
            uint32_t k = 0;
            if (from + lane < n) {
                k = s_key[wave][from + lane];
                const int i = seg0 + static_cast<int>(0xFFFFu - (k & 0xFFFFu));
                // what stands for logits outside the row is -inf, and reaches a cut of -inf
                k = i >= 0 && i < vocab ? (lp_order(static_cast<uint16_t>(k >> 16)) << 16) | (k & 0xFFFFu) : 0u;
            }
            best = lp_merge(best, lp_sort(k, lane), lane);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            n = from;
        };
        bool fits = true;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            bool any = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) any |= at(c, e) >= cut;
            if (!fits || __builtin_amdgcn_ballot_w64(any) == 0) continue;
            fits = n <= kLpCandidates - 8 * 64;
            if (!fits) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                collect(at(c, e) >= cut, e & 1 ? v[c][e >> 1] >> 16 : v[c][e >> 1] & 0xFFFFu, (c * kLpThreads + tid) * 8 + e);
        }
        if (!fits) {
            // Hundreds of equal logits: again, from memory, sorting on the way.  What
            // comes after a sort has to beat the top-th of it, being later in the row.
            n = 0;
            for (int c = 0; c < CHUNKS; ++c) {
                const int i = (c * kLpThreads + tid) * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int j = seg0 + i + e;
                    const bool in = j >= 0 && j < vocab;
                    const uint16_t bits = in ? x[j] : 0x7E00u;
                    collect(in && h2f(bits) >= cut, bits, i + e);
                }
                if (n >= 64) {
                    while (n >= 64) sort_last(n - 64);
                    cut = lp_logit((__shfl(best, top - 1) >> 16) + 1);
                }
            }
        }
        while (n > 0) sort_last(max(n - 64, 0));
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
        float* out = stats + (row * segments + seg) * 3;
        out[0] = mg;
        out[1] = Sg;
        out[2] = Tg;
    }
    if (top > 0) {
        uint32_t best = lane < top ? s_key[0][lane] : 0u;
        for (int w = 1; w < kLpWaves; ++w) best = lp_merge(best, lane < top ? s_key[w][lane] : 0u, lane);
        if (lane < top) keys[(row * segments + seg) * top + lane] = best;
    }
}

// A row's segments together.  Of 64 keys, the segments' best, the top-th largest
// is a bound for the alternatives; the keys that reach it, usually few more than asked
// for, are ordered at once.  Latency only: one row 4.2 us, 1024 rows 5.0.
__global__ __launch_bounds__(kLpThreads) void token_logprobs_row_kernel(
    const uint16_t* __restrict__ logits, const float* __restrict__ stats, const uint32_t* __restrict__ keys,
    const int32_t* __restrict__ ids,
    float* __restrict__ out_logprob, float* __restrict__ out_entropy, float* __restrict__ top_logprob,
    int32_t* __restrict__ top_ids, int vocab, long long row_stride, int segments, int segment, int top) {
    __shared__ float s_st[kLpWaves][3];
    __shared__ unsigned long long s_key[kLpWaves][kLpMaxTop];
    __shared__ unsigned long long s_list[64];
    __shared__ int s_n;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long row = blockIdx.x;
    const uint16_t* x = logits + row * row_stride;
    const float* part = stats + row * segments * 3;
    const int n = segments * top;
    const uint32_t* row_keys = keys + row * n;
    const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) >> 1);
    // key i of the row as (order, index)
    auto whole = [&](uint32_t k, int i) {
        const uint32_t at = (i / top) * segment - skew + (0xFFFFu - (k & 0xFFFFu));
        return k != 0 ? (static_cast<unsigned long long>(k >> 16) << 32) | (0xFFFFFFFFu - at) : 0ull;
    };
    constexpr int EARLY = 4;  // keys of a thread, requested with the sums
    uint32_t early[EARLY];
    if (top > 0) {
#pragma unroll
        for (int i = 0; i < EARLY; ++i) early[i] = row_keys[min(tid + kLpThreads * i, n - 1)];
    }
    const int id = out_logprob != nullptr ? ids[row] : -1;
    if (tid == 0) s_n = 0;
    float m = -INFINITY, S = 0.0f, T = 0.0f;
    // the best keys of every segment, best first, 64 in all (with more segments: of 64 groups)
    uint32_t front = 0;
    if (top > 0) {
        if (segments <= 64) {
            const int rank = lane / segments;
            if (rank < top) front = row_keys[(lane - rank * segments) * top + rank];
        } else {
            for (int s = lane; s < segments; s += 64) front = max(front, row_keys[s * top]);
        }
    }
    for (int s = tid; s < segments; s += kLpThreads) {
        const float ms = part[3 * s], Ss = part[3 * s + 1], Ts = part[3 * s + 2];
        const float mn = fmaxf(m, ms);
        const float da = m == mn ? 0.0f : fmaxf(m - mn, -1e4f), db = ms == mn ? 0.0f : fmaxf(ms - mn, -1e4f);
        const float fa = __builtin_amdgcn_exp2f(da * kLpLog2e), fb = __builtin_amdgcn_exp2f(db * kLpLog2e);
        T = fa * (T + da * S) + fb * (Ts + db * Ss);
        S = fa * S + fb * Ss;
        m = mn;
    }
    const bool has_id = id >= 0 && id < vocab;
    const uint16_t x_id = x[has_id ? id : 0];  // not waited for until the end
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
    bool few = true;
    if (top > 0) {
        const uint32_t cut = __shfl(lp_sort(front, lane), top - 1) >> 16;
        __syncthreads();  // s_n
#pragma unroll
        for (int i = 0; i < EARLY; ++i)
            if (tid + kLpThreads * i < n && early[i] != 0 && (early[i] >> 16) >= cut) {
                const int slot = atomicAdd(&s_n, 1);
                if (slot < 64) s_list[slot] = whole(early[i], tid + kLpThreads * i);
            }
        __syncthreads();
        few = s_n <= 64 && n <= EARLY * kLpThreads;
        if (!few) {  // long rows, or many equal logits: every key, 64 at a time
            unsigned long long best = 0;
            for (int i0 = 64 * wave; i0 < n; i0 += kLpThreads) {
                const int i = i0 + lane;
                best = lp_merge(best, lp_sort(i < n ? whole(row_keys[i], i) : 0ull, lane), lane);
            }
            if (lane < top) s_key[wave][lane] = best;
        }
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
        if (out_logprob != nullptr) out_logprob[row] = has_id ? logprob(h2f(x_id)) : 0.0f;
        if (out_entropy != nullptr) out_entropy[row] = nothing ? 0.0f : log_s - T / S;
    }
    if (top > 0) {
        unsigned long long best = 0;
        int rank = lane;
        if (few) {
            // a lane's place is the number of larger keys: a short loop, where a sort
            // is 21 steps of straight code that has to be fetched first
            best = lane < s_n ? s_list[lane] : 0ull;
            const int count = __builtin_amdgcn_readfirstlane(s_n);
            if (lane < count) rank = 0;
            for (int j = 0; j < count; ++j) {
                const unsigned long long o =
                    (static_cast<unsigned long long>(__builtin_amdgcn_readlane(static_cast<int>(best >> 32), j)) << 32) |
                    static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(best), j));
                rank += lane < count && o > best;
            }
        } else {
            best = lane < top ? s_key[0][lane] : 0ull;
            for (int w = 1; w < kLpWaves; ++w) best = lp_merge(best, lane < top ? s_key[w][lane] : 0ull, lane);
        }
        if (rank < top) {
            const bool none = best == 0;
            if (top_ids != nullptr)
                top_ids[row * top + rank] = none ? -1 : static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
            if (top_logprob != nullptr)
                top_logprob[row * top + rank] =
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
    QE_REQUIRE(num_rows >= 0 && vocab_size > 0 && vocab_size <= kLpMaxVocab && top_k >= 0 && top_k <= kLpMaxTop,
               "%s: num_rows=%d vocab_size=%d top_k=%d", what, num_rows, vocab_size, top_k);
    *bytes = static_cast<size_t>(num_rows) * lp_segments(vocab_size, kLpFew) * lp_words(top_k) * sizeof(uint32_t);
    return QE_OK;
}

extern "C" int qe_launch_token_logprobs(const uint16_t* logits, const int32_t* token_ids, float* out_logprob,
                                        float* out_entropy, float* out_top_logprob, int32_t* out_top_ids,
                                        void* workspace, int num_rows, int vocab_size, long long row_stride, int top_k,
                                        hipStream_t stream) {
    const char* what = "token_logprobs";
    QE_REQUIRE(vocab_size > 0 && vocab_size <= kLpMaxVocab, "%s: vocab_size=%d", what, vocab_size);
    QE_REQUIRE(row_stride >= vocab_size || num_rows <= 1, "%s: row_stride=%lld < vocab_size=%d", what, row_stride,
               vocab_size);
    QE_REQUIRE(top_k >= 0 && top_k <= kLpMaxTop && top_k <= vocab_size, "%s: top_k=%d (0..%d, at most vocab_size)", what,
               top_k, kLpMaxTop);
    if (num_rows <= 0) return QE_OK;  // buffers of no rows may be NULL
    QE_REQUIRE(logits && workspace, "%s: NULL pointer", what);
    QE_REQUIRE((token_ids == nullptr) == (out_logprob == nullptr), "%s: token_ids and out_logprob are given together",
               what);
    QE_REQUIRE((out_top_logprob == nullptr && out_top_ids == nullptr) || top_k > 0, "%s: top outputs with top_k=0", what);
    QE_REQUIRE(top_k == 0 || out_top_logprob || out_top_ids, "%s: top_k=%d without an output", what, top_k);
    QE_REQUIRE(aligned(logits, 2) && aligned(workspace, 4), "%s: alignment", what);
    // many: enough rows for two blocks of long segments on every CU
    const bool many = static_cast<long long>(num_rows) * lp_segments(vocab_size, kLpMany) >= 2LL * cu_count();
    const int chunks = many ? kLpMany : kLpFew, segments = lp_segments(vocab_size, chunks);
    QE_REQUIRE(static_cast<long long>(num_rows) * segments <= INT32_MAX, "%s: num_rows=%d", what, num_rows);
    float* stats = static_cast<float*>(workspace);
    uint32_t* keys = reinterpret_cast<uint32_t*>(stats + static_cast<size_t>(num_rows) * segments * 3);
    if (many)
        token_logprobs_segment_kernel<kLpMany><<<num_rows * segments, kLpThreads, 0, stream>>>(
            logits, stats, keys, vocab_size, row_stride, segments, top_k);
    else
        token_logprobs_segment_kernel<kLpFew><<<num_rows * segments, kLpThreads, 0, stream>>>(
            logits, stats, keys, vocab_size, row_stride, segments, top_k);
    token_logprobs_row_kernel<<<num_rows, kLpThreads, 0, stream>>>(logits, stats, keys, token_ids, out_logprob,
                                                                   out_entropy, out_top_logprob, out_top_ids,
                                                                   vocab_size, row_stride, segments,
                                                                   lp_segment(chunks), top_k);
    return check_launch(what);
}
