// 4-bit key/value cache (layout: kv4_common.hpp): append of new tokens, reading
// rows back as fp16, and eviction of the rows with the least attention.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv4_common.hpp"

namespace qe {
namespace {

// ---- append ------------------------------------------------------------------
// x = q, k, v + bias in fp32, q and k rotated (NeoX pairs i, i + rot / 2 by
// the angle pos * theta^(-2 i / rot)), q rounded once to fp16, k and v straight
// to 4 bits: per 32 elements low = fp16(min), scale = fp16((max - low) / 15) (one
// fp16 less where 15 scale + low would round to infinity), nibble =
// clamp(rint((x - low) / scale), 0, 15); a scale of 0 gives nibbles 0.
//
// Angles: position times frequency in 64 bits, reduced to [-pi, pi] there, then
// sine and cosine in fp32.  In fp32 the angle of position 100000 is off by
// up to 4e-3.
//
// grid (tokens, ceil((nq + nkv) / 16)), 256 threads: 16 lanes a head, 8 elements a
// lane, so a group of 32 is a quad of lanes; the first rot / 2 threads make the
// token's sines and cosines.  The partner of a rotation is read from memory a
// second time (it is in the cache) instead of being exchanged.
// Latency: one token 3.1 us (a launch alone 1.7, then the loads, the sines and the
// quantization behind each other; with the row's place loaded after the rotation and
// plain divisions 3.5), 1000 tokens 5.1 (12 q heads, 2 kv heads: 7.5 MB).
__global__ __launch_bounds__(256) void qkv_bias_rope_kv4_append_kernel(
    const uint16_t* q, uint16_t* q_out, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
    const uint16_t* __restrict__ qb, const uint16_t* __restrict__ kb, const uint16_t* __restrict__ vb,
    uint8_t* __restrict__ kc, uint8_t* __restrict__ vc, const qe_device_control_block* ctl, const int32_t* evicted,
    int nq, int nkv, int max_seq, int rot, double log2_step) {
#pragma clang fp contract(off)
    __shared__ float s_sin[kKv4Dim / 2], s_cos[kKv4Dim / 2];
    const int t = blockIdx.x, j = threadIdx.x & 15;
    const int head = blockIdx.y * 16 + (threadIdx.x >> 4);
    const int half = rot / 2;
    const bool live = head < nq + nkv, is_k = head >= nq;
    const int hk = is_k ? head - nq : 0;
    // own 8 elements, their rotation partners, and v's
    const bool turned = 8 * j < rot;
    const int pd = turned ? (8 * j < half ? 8 * j + half : 8 * j - half) : 8 * j;
    float x[8], y[8], w[8];
    if (live) {
        const uint16_t* src = is_k ? k + (static_cast<size_t>(t) * nkv + hk) * kKv4Dim
                                   : q + (static_cast<size_t>(t) * nq + head) * kKv4Dim;
        const uint16_t* bias = is_k ? (kb ? kb + hk * kKv4Dim : nullptr) : (qb ? qb + head * kKv4Dim : nullptr);
        auto load8 = [](const uint16_t* p, const uint16_t* b, int d, float (&o)[8]) {
            const f16x8 a = *reinterpret_cast<const f16x8*>(p + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = static_cast<float>(a[e]);
            if (b != nullptr) {
                const f16x8 c = *reinterpret_cast<const f16x8*>(b + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] += static_cast<float>(c[e]);
            }
        };
        load8(src, bias, 8 * j, x);
        load8(src, bias, pd, y);
        if (is_k) load8(v + (static_cast<size_t>(t) * nkv + hk) * kKv4Dim, vb ? vb + hk * kKv4Dim : nullptr, 8 * j, w);
    }
    const long long row = static_cast<long long>(kv4_row(ctl, evicted, hk)) + t;
    if (static_cast<int>(threadIdx.x) < half) {
        const int i = threadIdx.x;
        const double pos = static_cast<double>((ctl != nullptr ? ctl->seq_pos : 0)) + t;
        const double a = pos * exp2(-log2_step * i);
        constexpr double kTwoPi = 6.283185307179586476925;
        const float r = static_cast<float>(a - kTwoPi * rint(a * (1.0 / kTwoPi)));
        float sn, cs;
        sincosf(r, &sn, &cs);
        s_sin[i] = sn;
        s_cos[i] = cs;
    }
    // also: the partners of q are read before q_out, which may be q, is written
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (!live) return;
    if (turned) {
        const bool first = 8 * j < half;
        const int i0 = first ? 8 * j : 8 * j - half;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float sn = s_sin[i0 + e], cs = s_cos[i0 + e];
            x[e] = first ? x[e] * cs - y[e] * sn : x[e] * cs + y[e] * sn;
        }
    }
    if (!is_k) {
        f16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = static_cast<_Float16>(x[e]);
        *reinterpret_cast<f16x8*>(q_out + (static_cast<size_t>(t) * nq + head) * kKv4Dim + 8 * j) = o;
        return;
    }
    if (row >= max_seq) return;  // no room: not stored
    // a value that rounds to no finite fp16, anywhere in the 16 lanes of the head
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) bad |= !(fabsf(x[e]) < 65520.0f) || !(fabsf(w[e]) < 65520.0f);
    const uint64_t mine = 0xFFFFull << (threadIdx.x & 48);
    bad = (__builtin_amdgcn_ballot_w64(bad) & mine) != 0;
    auto store = [&](const float (&z)[8], uint8_t* cache, uint32_t bad_param) {
        float lo = z[0], hi = z[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) {
            lo = fminf(lo, z[e]);
            hi = fmaxf(hi, z[e]);
        }
        lo = -qwen::seg_max<4>(-lo);
        hi = qwen::seg_max<4>(hi);
        const uint16_t lo16 = f2h(lo);
        const float low = h2f(lo16);
        uint16_t sc16 = f2h((hi - low) / 15.0f);
        // a scale rounded up must not take the largest value past 65504: one step less
        // takes 15 of its units off, more than the at most 7.5 that it rounded up
        if (__builtin_fmaf(15.0f, h2f(sc16), low) >= 65520.0f) --sc16;
        const float scale = h2f(sc16), r = 1.0f / scale;
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // (z - low) / scale, correctly rounded: the quotient from the rounded reciprocal
            // and one step with its remainder, exact in a fused multiply-add
            const float d = z[e] - low, q0 = d * r;
            const float n = fminf(fmaxf(rintf(__builtin_fmaf(__builtin_fmaf(-q0, scale, d), r, q0)), 0.0f), 15.0f);
            const uint32_t u = scale > 0.0f ? static_cast<uint32_t>(n) : 0u;
            word |= u << (16 * (e & 1) + 4 * (e >> 1));
        }
        uint32_t param = static_cast<uint32_t>(sc16) | (static_cast<uint32_t>(lo16) << 16);
        if (bad) {
            word = 0;
            param = bad_param;
        }
        uint8_t* dst = cache + (static_cast<size_t>(hk) * max_seq + row) * kKv4Row;
        *reinterpret_cast<uint32_t*>(dst + 4 * j) = word;
        if ((j & 3) == 0) *reinterpret_cast<uint32_t*>(dst + kKv4Params + j) = param;
    };
    store(x, kc, 0x7E007E00u);
    store(w, vc, 0u);
}

// ---- rows as fp16 --------------------------------------------------------------
// A lane per word: 4 bytes and the group's pair in, 16 bytes out.  blockIdx.z: K, V.
// Bound by its stores: 8000 rows x 8 heads of K and V, 43 MB, 7.9 us, 5.4 TB/s.
__global__ __launch_bounds__(256) void kv4_unpack_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                         uint16_t* __restrict__ ok, uint16_t* __restrict__ ov,
                                                         int row0, int rows, int max_seq) {
    const uint8_t* cache = blockIdx.z == 0 ? kc : vc;
    uint16_t* out = blockIdx.z == 0 ? ok : ov;
    if (cache == nullptr) return;
    const int h = blockIdx.y, w = threadIdx.x & 15;
    const long long r = static_cast<long long>(blockIdx.x) * 16 + (threadIdx.x >> 4);
    if (r >= rows) return;
    const uint8_t* src = cache + (static_cast<size_t>(h) * max_seq + row0 + r) * kKv4Row;
    const f16x8 x = kv4_expand_word(*reinterpret_cast<const uint32_t*>(src + 4 * w),
                                    *reinterpret_cast<const uint32_t*>(src + kKv4Params + (w & ~3)));
    *reinterpret_cast<f16x8*>(out + (static_cast<size_t>(h) * rows + r) * kKv4Dim + 8 * w) = x;
}

// ---- eviction ------------------------------------------------------------------
// Weights as whole numbers of the same order: NaN (1) below everything, -0 as +0.
// 0 and kEvictSafe are left over: no row, and a row that stays whatever its weight.
constexpr uint32_t kEvictSafe = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t evict_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return w != w ? 1u : u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        x += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value,
                                                               decltype(rows)::value, 0xF, false));
    };
    using std::integral_constant;
    add(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // row_shr 1, 2, 4, 8
    add(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
    add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // lane 15 of a row to the next row
    add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});  // lane 31 to rows 2 and 3
    return x;
}

// What a head has before an eviction.
struct EvictHead {
    int pos, gone, row, n, m;  // position, rows gone, row of the position, rows in use, rows that stay
};
__device__ __forceinline__ EvictHead evict_head(const int32_t* evicted, const qe_device_control_block* ctl, int h, int keep,
                                                int max_seq) {
    EvictHead e;
    e.pos = ctl != nullptr ? ctl->seq_pos : 0;
    e.gone = evicted != nullptr ? evicted[h] : 0;
    e.row = max(e.pos - e.gone, 0);
    e.n = min(e.row, max_seq);
    e.m = min(e.n, keep);
    return e;
}
// The weights behind the kept rows start over, and so does the count of evicted rows.
// By all threads of the one block that does it, behind a barrier that all have
// passed since they read `evicted` (it may be out_evicted).
__device__ __forceinline__ void evict_finish(float* out_weights, int32_t* out_evicted, const EvictHead& e, int h,
                                             int max_seq) {
    const size_t base = static_cast<size_t>(h) * max_seq;
    for (int i = e.m + threadIdx.x; i < e.n; i += blockDim.x) out_weights[base + i] = 0.0f;
    // the next position's row is m: positions that found the cache full count as gone too
    if (threadIdx.x == 0) out_evicted[h] = e.row == 0 ? e.gone : e.pos - e.m;
}

// Rows kept of one kv head, a block each.  The first `sinks` and the last
// `recent` rows count as larger than every weight, so what stays are the `keep`
// largest keys, equal ones by the lowest index: radix selection of the keep-th
// largest, then one ordered pass that writes the kept indices.
// Up to 32768 rows the keys are read from memory once and stay in LDS; more rows are
// read again in every pass, eight loads a lane ahead (60000 rows, copy included, 40 to 48 us; with
// four loads and their wait at a time 81).  A wave owns a run of rows, a multiple of 256
// so that a lane can take four keys with one LDS read wherever their order does not
// matter.  Digits of 11, 11 and 10 bits: the first holds the sign, the exponent and two
// bits of the mantissa, so that weights of like size still spread over the bins and
// lanes seldom meet in one; the third is looked at only where some, not all, of
// the keys with the same first 22 bits stay.  One CU a head, its vector units busy a
// little over half the time, then waits, barriers and LDS: 4096 rows take 6.0 us (2
// heads), 32000 17.7 (8 heads); with the loads waited for before the first count and always
// three digits 7.3 and 21, with digits of 8 bits, four rounds over memory and a branch for
// every key 10.3 and 53.
constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;
constexpr int kEvictCached = 32768;  // keys in LDS
constexpr int kEvictBins = 2048;

// Rows of a wave's run for n rows.
__host__ __device__ __forceinline__ int evict_run(int n) {
    return ((n + kEvictWaves - 1) / kEvictWaves + 255) & ~255;
}

__global__ __launch_bounds__(kEvictThreads) void kv4_evict_select_kernel(const float* __restrict__ weights,
                                                                         const int32_t* evicted,
                                                                         const qe_device_control_block* ctl,
                                                                         int32_t* __restrict__ kept, int keep,
                                                                         int sinks, int recent, int max_seq,
                                                                         float* apart_weights, int32_t* apart_evicted) {
    constexpr int W = kEvictWaves;
    extern __shared__ uint32_t s_key[];  // W evict_run(max_seq), at most kEvictCached
    __shared__ __align__(16) uint32_t s_hist[3 * kEvictBins];  // the first digit counts in the first two
    __shared__ uint32_t s_wave[W];
    __shared__ uint32_t s_pick[3];  // digit, keys above it, keys of it
    __shared__ int2 s_cnt[W];
    const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const EvictHead head = evict_head(evicted, ctl, h, keep, max_seq);
    const int n = head.n;
    int32_t* out = kept + static_cast<size_t>(h) * keep;
    // moved apart, nothing here is read again, and the head's end can be written here
    auto finish = [&]() __attribute__((always_inline)) {
        if (apart_weights != nullptr) evict_finish(apart_weights, apart_evicted, head, h, max_seq);
    };
    if (n <= keep) {
        for (int i = tid; i < keep; i += kEvictThreads) out[i] = i < n ? i : -1;
        __syncthreads();
        finish();
        return;
    }
    const float* w = weights + static_cast<size_t>(h) * max_seq;
    const int lo = sinks, hi = n - recent;
    auto key_of = [&](int i, float x) { return i >= n ? 0u : i < lo || i >= hi ? kEvictSafe : evict_key(x); };
    const int per = evict_run(n);
    const bool cached = W * per <= kEvictCached;
    const int r0 = wave * per, r1 = min(r0 + per, n);
    // f(keys of rows i0 + 64 u + lane, i0) for all of the wave's, from memory: eight loads
    // at a time, the next eight requested before these are used.  No load is behind a branch
    // of its own, and none is copied: the compiler would wait for all at the first use.
    float even[8], odd[8];
    auto fetch = [&](int b0, float (&x)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = w[min(b0 + 64 * u + lane, n - 1)];
    };
    auto each_read = [&](auto f) __attribute__((always_inline)) {
        auto use = [&](int b0, const float (&x)[8]) __attribute__((always_inline)) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int i0 = b0 + 256 * v;
                if (i0 >= r1) break;  // the next wave's
                uint32_t k[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) k[u] = evict_key(x[4 * v + u]);
                if (i0 < lo || i0 + 256 > hi) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) k[u] = key_of(i0 + 64 * u + lane, x[4 * v + u]);
                }
                f(k, i0);
            }
        };
        for (int b0 = r0; b0 < r1; b0 += 1024) {  // `even` is requested
            if (b0 + 512 < r1) {
                fetch(b0 + 512, odd);
                use(b0, even);
                fetch(b0 + 1024, even);
                use(b0 + 512, odd);
            } else {
                use(b0, even);
            }
        }
    };
    fetch(r0, even);
    for (int i = tid; i < 3 * kEvictBins; i += kEvictThreads) s_hist[i] = 0;
    // a barrier for LDS alone: the loads stay in flight
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // The first digit, lanes of odd and even number apart; rows that stay anyway are
    // many and in one place: counted together, not one by one.
    auto count_first = [&](uint32_t k) __attribute__((always_inline)) {
        if (k + 1u > 1u) atomicAdd(&s_hist[(lane & 1) * kEvictBins + (k >> 21)], 1u);
    };
    if (tid == 0) atomicAdd(&s_hist[kEvictBins - 1], static_cast<uint32_t>(sinks + recent));
    each_read([&](const uint32_t(&k)[4], int i0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (cached) s_key[i0 + 64 * u + lane] = k[u];
            count_first(k[u]);
        }
    });
    // f(four keys) for all of the wave's, in any order
    auto each = [&](auto f) __attribute__((always_inline)) {
        if (!cached) {
            fetch(r0, even);
            each_read(f);
            return;
        }
        for (int i0 = r0; i0 < r1; i0 += 256) {
            const u32x4 k = *reinterpret_cast<const u32x4*>(s_key + i0 + 4 * lane);
            const uint32_t k4[4] = {k[0], k[1], k[2], k[3]};
            f(k4, i0);
        }
    };
    uint32_t prefix = 0, need = keep;  // digits found so far, keys still to take at or below them
    auto round = [&](auto number) __attribute__((always_inline)) {
        constexpr int R = decltype(number)::value, shift = R == 0 ? 21 : R == 1 ? 10 : 0, bits = R == 2 ? 10 : 11;
        if constexpr (R > 0)
            each([&](const uint32_t(&k)[4], int) {
                bool is[4], any = false;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    is[u] = (k[u] >> ((shift + bits) & 31)) == prefix;
                    any |= is[u];
                }
                if (__builtin_amdgcn_ballot_w64(any) == 0) return;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (is[u]) atomicAdd(&s_hist[R * kEvictBins + ((k[u] >> shift) & ((1u << bits) - 1u))], 1u);
            });
        __syncthreads();
        // thread t holds bins 2047 - 2 t and 2046 - 2 t; the digit where the count from above reaches `need`
        uint2* bins = reinterpret_cast<uint2*>(&s_hist[R * kEvictBins + kEvictBins - 2 - 2 * tid]);
        uint2 b = *bins;
        if (R == 0) {
            const uint2 odd = bins[kEvictBins / 2];
            b = make_uint2(b.x + odd.x, b.y + odd.y);
            bins[kEvictBins / 2] = make_uint2(0, 0);  // the next digit's
        }
        const uint32_t incl = wave_scan(b.x + b.y);
        if (lane == 63) s_wave[wave] = incl;
        __syncthreads();
        uint32_t above = incl - b.x - b.y;
#pragma unroll
        for (int v = 0; v < W; ++v) {
            const uint32_t x = s_wave[v];
            above += v < wave ? x : 0u;
        }
        if (above < need && above + b.x + b.y >= need) {
            const bool first = above + b.y >= need;
            s_pick[0] = kEvictBins - 1 - 2 * tid - (first ? 0 : 1);
            s_pick[1] = above + (first ? 0 : b.y);
            s_pick[2] = first ? b.y : b.x;
        }
        __syncthreads();
        prefix = (prefix << bits) | s_pick[0];
        need -= s_pick[1];
    };
    round(std::integral_constant<int, 0>{});
    round(std::integral_constant<int, 1>{});
    uint32_t cut;  // keys above it stay, and the first `need` equal to it
    if (prefix != 0 && s_pick[2] == need) {  // all that begin like this, often one: the last digit does not matter
        cut = (prefix << 10) - 1;
        need = 0;
    } else {
        __syncthreads();  // s_pick is read
        round(std::integral_constant<int, 2>{});
        cut = prefix;
    }
    int sure_n = 0, tie_n = 0;
    each([&](const uint32_t(&k)[4], int) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            sure_n += __popcll(__builtin_amdgcn_ballot_w64(k[u] > cut));
            tie_n += __popcll(__builtin_amdgcn_ballot_w64(k[u] == cut));
        }
    });
    if (lane == 0) s_cnt[wave] = make_int2(sure_n, tie_n);
    __syncthreads();
    int at = 0, ties = 0;
#pragma unroll
    for (int v = 0; v < W; ++v) {
        const int2 x = s_cnt[v];
        at += v < wave ? x.x : 0;
        ties += v < wave ? x.y : 0;
    }
    const int wanted = static_cast<int>(need);
    at = __builtin_amdgcn_readfirstlane(at + min(ties, wanted));
    ties = __builtin_amdgcn_readfirstlane(ties);
    auto write = [&](const uint32_t(&k)[4], int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            uint64_t take = __builtin_amdgcn_ballot_w64(k[u] > cut);
            const uint64_t tb = __builtin_amdgcn_ballot_w64(k[u] == cut);
            if (tb != 0) {
                const bool t = k[u] == cut && ties + __popcll(tb & ((1ull << lane) - 1)) < wanted;
                take |= __builtin_amdgcn_ballot_w64(t);
                ties += __popcll(tb);
            }
            if ((take >> lane) & 1)
                out[at + static_cast<int>(__builtin_amdgcn_mbcnt_hi(
                             static_cast<uint32_t>(take >> 32),
                             __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(take), 0u)))] = i0 + 64 * u + lane;
            at += __popcll(take);
        }
    };
    if (cached) {
        for (int i0 = r0; i0 < r1; i0 += 256) {
            uint32_t k[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) k[u] = s_key[i0 + 64 * u + lane];
            write(k, i0);
        }
    } else {
        fetch(r0, even);
        each_read(write);
    }
    finish();
}

struct EvictMove {
    const uint8_t* kc;
    const uint8_t* vc;
    const float* weights;
    const int32_t* evicted;
    uint8_t* out_k;
    uint8_t* out_v;
    float* out_weights;
    int32_t* out_evicted;
    const int32_t* kept;
    const qe_device_control_block* ctl;
    int keep, max_seq;
};

// The kept rows to the front, in their order, into memory apart from the caches:
// a lane per 16-byte piece, 5 pieces a row, K (blockIdx.z 0, with the weights) and V (1).
// One round of loads behind the list: 8000 rows x 8 heads (21 MB both ways) 6.9 us, 3.0 TB/s.
constexpr int kCopyRows = 51;  // rows of a block of 256 threads
__global__ __launch_bounds__(256) void kv4_evict_copy_kernel(EvictMove p) {
    const int h = blockIdx.y, tid = threadIdx.x;
    const int32_t* list = p.kept + static_cast<size_t>(h) * p.keep;
    const size_t base = static_cast<size_t>(h) * p.max_seq;
    const int r0 = blockIdx.x * kCopyRows, r = r0 + tid / 5, piece = tid % 5;
    if (tid < 5 * kCopyRows && r < p.keep) {
        const int from = list[r];
        if (from >= 0) {
            const uint8_t* src = (blockIdx.z == 0 ? p.kc : p.vc) + (base + from) * kKv4Row + 16 * piece;
            uint8_t* dst = (blockIdx.z == 0 ? p.out_k : p.out_v) + (base + r) * kKv4Row + 16 * piece;
            *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(src);
        }
    }
    if (blockIdx.z == 0 && tid < kCopyRows && r0 + tid < p.keep) {
        const int from = list[r0 + tid];
        if (from >= 0) p.out_weights[base + r0 + tid] = p.weights[base + from];
    }
}

// The same in place: row i comes from kept[i] >= i, a block takes all rows of a
// head's K or V pieces 0..2 or 3..4, or its weights, in runs from the front, and
// within a run every load is done before the first store; later runs read behind
// everything stored so far, and nobody else touches the block's pieces.  Rows in front of
// the first one that left stay where they are.  PIECES of STRIDE values T a row, U
// a thread and run: few runs, since each waits for memory twice.  Five blocks a head, so
// bound by a CU's loads: 8000 rows x 8 heads 20 us, three times the copy apart, which needs
// a second cache.
template <class T, int PIECES, int STRIDE, int U>
__device__ __forceinline__ void move_rows(T* data, const int32_t* kept, int keep) {
    const uint32_t all = static_cast<uint32_t>(keep) * PIECES;
    for (uint32_t i0 = 0; i0 < all; i0 += kEvictThreads * U) {
        T v[U];
        bool moves[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = i0 + u * kEvictThreads + threadIdx.x, row = i / PIECES, piece = i - row * PIECES;
            const int from = i < all ? kept[row] : -1;
            moves[u] = from > static_cast<int>(row);
            if (moves[u]) v[u] = data[static_cast<size_t>(from) * STRIDE + piece];
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = i0 + u * kEvictThreads + threadIdx.x, row = i / PIECES, piece = i - row * PIECES;
            if (moves[u]) data[static_cast<size_t>(row) * STRIDE + piece] = v[u];
        }
    }
}

__global__ __launch_bounds__(kEvictThreads) void kv4_evict_move_kernel(EvictMove p) {
    const int h = blockIdx.y;
    const int32_t* list = p.kept + static_cast<size_t>(h) * p.keep;
    const size_t base = static_cast<size_t>(h) * p.max_seq;
    u32x4* rows = reinterpret_cast<u32x4*>((blockIdx.x < 2 ? p.out_k : p.out_v) + base * kKv4Row);
    if (blockIdx.x < 4) {
        if (blockIdx.x % 2 == 0) move_rows<u32x4, 3, 5, 12>(rows, list, p.keep);
        else move_rows<u32x4, 2, 5, 12>(rows + 3, list, p.keep);
        return;
    }
    const EvictHead head = evict_head(p.evicted, p.ctl, h, p.keep, p.max_seq);
    move_rows<float, 1, 1, 8>(p.out_weights + base, list, p.keep);
    evict_finish(p.out_weights, p.out_evicted, head, h, p.max_seq);
}

struct Span {
    const void* at;
    size_t bytes;
};
inline bool apart(const Span& a, const Span& b) { return qe::apart(a.at, a.bytes, b.at, b.bytes); }

}  // namespace
}  // namespace qe

using namespace qe;

extern "C" int qe_launch_qkv_bias_rope_kv4_append(const uint16_t* q, uint16_t* q_out, const uint16_t* k,
                                                  const uint16_t* v, const uint16_t* q_bias, const uint16_t* k_bias,
                                                  const uint16_t* v_bias, uint8_t* layer_k_cache,
                                                  uint8_t* layer_v_cache, const qe_device_control_block* d_control,
                                                  const int32_t* d_evicted, int num_tokens, hipStream_t stream,
                                                  int num_q_heads, int num_kv_heads, int head_dim, int max_seq_len,
                                                  int rotary_dim, float rope_theta) {
    const char* what = "qkv_bias_rope_kv4_append";
    QE_REQUIRE(q && q_out && k && v, "%s: NULL pointer", what);
    QE_TRY(kv4_check(what, layer_k_cache, layer_v_cache, num_kv_heads, head_dim, max_seq_len));
    QE_REQUIRE(num_q_heads > 0, "%s: num_q_heads=%d", what, num_q_heads);
    const int rot = rotary_dim == 0 ? head_dim : rotary_dim;
    QE_REQUIRE(rot > 0 && rot <= head_dim && rot % 16 == 0, "%s: rotary_dim=%d (a multiple of 16 up to 128)", what,
               rotary_dim);
    QE_REQUIRE(rope_theta > 0.0f && std::isfinite(rope_theta), "%s: rope_theta=%g", what, rope_theta);
    QE_REQUIRE(aligned(q, 16) && aligned(q_out, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_bias, 16) &&
                   aligned(k_bias, 16) && aligned(v_bias, 16),
               "%s: q, k, v and the biases must be 16-byte aligned", what);
    if (num_tokens <= 0) return QE_OK;
    // Blocks do not wait for each other: q_out may be q, and otherwise what is written meets nothing.
    const size_t head = kKv4Dim * 2, q_row = num_q_heads * head, kv_row = num_kv_heads * head;
    const size_t cache = static_cast<size_t>(num_kv_heads) * max_seq_len * kKv4Row;
    const Span in[] = {{q, num_tokens * q_row},       {k, num_tokens * kv_row},       {v, num_tokens * kv_row},
                       {q_bias, q_bias ? q_row : 0},  {k_bias, k_bias ? kv_row : 0},  {v_bias, v_bias ? kv_row : 0},
                       {d_evicted, d_evicted ? num_kv_heads * sizeof(int32_t) : 0}};
    const Span out[] = {{q_out, num_tokens * q_row}, {layer_k_cache, cache}, {layer_v_cache, cache}};
    bool clear = apart(out[0], out[1]) && apart(out[0], out[2]) && apart(out[1], out[2]);
    for (const Span& o : out)
        for (const Span& i : in) clear &= apart(i, o) || (&o == out && &i == in && q == q_out);
    QE_REQUIRE(clear, "%s: q_out or a cache overlaps another buffer", what);
    const long long heads = static_cast<long long>(num_q_heads) + num_kv_heads;
    QE_REQUIRE(heads <= 65535 * 16, "%s: %lld heads", what, heads);
    const dim3 grid(num_tokens, static_cast<unsigned>((heads + 15) / 16));
    qkv_bias_rope_kv4_append_kernel<<<grid, 256, 0, stream>>>(
        q, q_out, k, v, q_bias, k_bias, v_bias, layer_k_cache, layer_v_cache, d_control, d_evicted, num_q_heads,
        num_kv_heads, max_seq_len, rot, std::log2(static_cast<double>(rope_theta)) / (rot / 2));
    return check_launch(what);
}

extern "C" int qe_launch_kv4_unpack(const uint8_t* layer_k_cache, const uint8_t* layer_v_cache, uint16_t* out_k,
                                    uint16_t* out_v, int first_row, int num_rows, hipStream_t stream,
                                    int num_kv_heads, int head_dim, int max_seq_len) {
    const char* what = "kv4_unpack";
    QE_REQUIRE((layer_k_cache == nullptr) == (out_k == nullptr) && (layer_v_cache == nullptr) == (out_v == nullptr) &&
                   (out_k || out_v),
               "%s: a cache and its output are given together", what);
    const uint8_t* any = layer_k_cache ? layer_k_cache : layer_v_cache;
    QE_TRY(kv4_check(what, layer_k_cache ? layer_k_cache : any, layer_v_cache ? layer_v_cache : any, num_kv_heads,
                     head_dim, max_seq_len));
    QE_REQUIRE(aligned(out_k, 16) && aligned(out_v, 16), "%s: the outputs must be 16-byte aligned", what);
    QE_REQUIRE(num_kv_heads <= 65535, "%s: num_kv_heads=%d", what, num_kv_heads);
    if (num_rows <= 0) return QE_OK;
    QE_REQUIRE(first_row >= 0 && first_row <= max_seq_len - num_rows, "%s: rows %d..%lld of %d", what, first_row,
               static_cast<long long>(first_row) + num_rows - 1, max_seq_len);
    const size_t cache = static_cast<size_t>(num_kv_heads) * max_seq_len * kKv4Row;
    const size_t rows = static_cast<size_t>(num_kv_heads) * num_rows * kKv4Dim * 2;
    const Span in[] = {{layer_k_cache, layer_k_cache ? cache : 0}, {layer_v_cache, layer_v_cache ? cache : 0}};
    const Span out[] = {{out_k, out_k ? rows : 0}, {out_v, out_v ? rows : 0}};
    bool clear = apart(out[0], out[1]);
    for (const Span& x : out)
        for (const Span& i : in) clear &= apart(i, x);
    QE_REQUIRE(clear, "%s: an output overlaps another buffer", what);
    const dim3 grid((static_cast<unsigned>(num_rows) + 15) / 16, num_kv_heads, 2);
    kv4_unpack_kernel<<<grid, 256, 0, stream>>>(layer_k_cache, layer_v_cache, out_k, out_v, first_row, num_rows,
                                                max_seq_len);
    return check_launch(what);
}

extern "C" int qe_launch_kv4_evict(const uint8_t* layer_k_cache, const uint8_t* layer_v_cache,
                                   const float* key_weights, const int32_t* d_evicted, uint8_t* out_k_cache,
                                   uint8_t* out_v_cache, float* out_key_weights, int32_t* out_evicted,
                                   int32_t* kept_rows, const qe_device_control_block* d_control, int keep, int sinks,
                                   int recent, hipStream_t stream, int num_kv_heads, int head_dim, int max_seq_len) {
    const char* what = "kv4_evict";
    QE_TRY(kv4_check(what, layer_k_cache, layer_v_cache, num_kv_heads, head_dim, max_seq_len));
    QE_TRY(kv4_check(what, out_k_cache, out_v_cache, num_kv_heads, head_dim, max_seq_len));
    QE_REQUIRE(key_weights && out_key_weights && out_evicted && kept_rows && d_control, "%s: NULL pointer", what);
    QE_REQUIRE(max_seq_len <= (1 << 28), "%s: max_seq_len=%d", what, max_seq_len);
    QE_REQUIRE(keep > 0 && keep <= max_seq_len, "%s: keep=%d of %d rows", what, keep, max_seq_len);
    QE_REQUIRE(sinks >= 0 && recent >= 0 && sinks <= keep && recent <= keep - sinks,
               "%s: sinks=%d and recent=%d do not fit in keep=%d", what, sinks, recent, keep);
    QE_REQUIRE(num_kv_heads <= 65535, "%s: num_kv_heads=%d", what, num_kv_heads);
    QE_REQUIRE(aligned(key_weights, 4) && aligned(out_key_weights, 4) && aligned(kept_rows, 4), "%s: alignment", what);
    const size_t rows = static_cast<size_t>(num_kv_heads) * max_seq_len;
    const bool in_place = layer_k_cache == out_k_cache;
    QE_REQUIRE(in_place == (layer_v_cache == out_v_cache) && in_place == (key_weights == out_key_weights),
               "%s: K, V and weights are all in place or all apart", what);
    // Blocks do not wait for each other: an output may be its own input, and otherwise meets nothing.
    const size_t counts = num_kv_heads * sizeof(int32_t);
    const Span in[] = {{layer_k_cache, rows * kKv4Row}, {layer_v_cache, rows * kKv4Row}, {key_weights, rows * sizeof(float)},
                       {d_evicted, d_evicted ? counts : 0}};
    const Span out[] = {{out_k_cache, rows * kKv4Row}, {out_v_cache, rows * kKv4Row}, {out_key_weights, rows * sizeof(float)},
                        {out_evicted, counts}, {kept_rows, static_cast<size_t>(num_kv_heads) * keep * sizeof(int32_t)}};
    bool clear = true;
    for (int o = 0; o < 5; ++o) {
        for (int i = 0; i < 4; ++i) clear &= apart(in[i], out[o]) || (i == o && in[i].at == out[o].at);
        for (int u = 0; u < o; ++u) clear &= apart(out[u], out[o]);
    }
    QE_REQUIRE(clear, "%s: an output overlaps another, or an input without being it", what);
    const size_t lds = std::min(kEvictWaves * evict_run(max_seq_len), kEvictCached) * sizeof(uint32_t);
    kv4_evict_select_kernel<<<num_kv_heads, kEvictThreads, lds, stream>>>(key_weights, d_evicted, d_control, kept_rows,
                                                                          keep, sinks, recent, max_seq_len,
                                                                          in_place ? nullptr : out_key_weights, out_evicted);
    const EvictMove p{layer_k_cache, layer_v_cache, key_weights, d_evicted, out_k_cache, out_v_cache, out_key_weights,
                      out_evicted, kept_rows, d_control, keep, max_seq_len};
    if (in_place)
        kv4_evict_move_kernel<<<dim3(5, num_kv_heads), kEvictThreads, 0, stream>>>(p);
    else
        kv4_evict_copy_kernel<<<dim3((keep + kCopyRows - 1) / kCopyRows, num_kv_heads, 2), 256, 0, stream>>>(p);
    return check_launch(what);
}
