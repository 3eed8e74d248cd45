// Attention over the 4-bit key/value cache (layout: kv4_common.hpp): one token
// (flash decode) and the rows of a chunk (causal prefill), each with the weights
// that its rows give to the cache rows, added up per kv head, when asked for.
//
// Rows of the cache come from positions less those evicted (kv4_row); a token at
// row r sees rows 0..r.  q [T][q heads][128] fp16, head dimension 128.
#include <algorithm>
#include <type_traits>

#include "attn_common.hpp"
#include "kv4_common.hpp"
#include "lds_dma.hpp"

namespace qe {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kScoreScale = kLog2e * 0.08838834764831845f;  // log2(e) / sqrt(128)
// How far a row's maximum grows before its reference value follows: the
// probabilities then reach 2^8, and their relative precision in fp16 is the same.
constexpr float kReferenceLag = 8.0f;
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The largest value over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_over_quarters(float x) {
    x = fmaxf(x, qwen::swz_xor16_f32(x));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_quarters(float x) {
    x += qwen::swz_xor16_f32(x);
    return x + __shfl_xor(x, 32);
}

// ---- one token -------------------------------------------------------------------
// Split over the cache rows: a block takes a run of rows of one kv head for up to
// 16 of its q heads, a wave 32 rows at a time, with its own running maximum,
// sum and output; the waves meet in LDS, the blocks in the second kernel.
// v_mfma_f32_16x16x32_f16 with the q heads as the columns:
//   S (16 rows x 16 heads) = K . Q^T: lane l holds cache row l % 16 and, of the
//   k order, dims 32 (l / 16) + 8 kk..: its four MFMAs take the four words of
//   one 16-byte chunk, i.e. one quantization group;
//   the result has lane l = head l % 16 holding rows 4 (l / 16) + i;
//   O^T (16 dims x 16 heads) += V^T . P^T over 32 rows: P^T is the lane's own
//   eight probabilities; V^T wants eight rows of one dim in a lane, and MFMA dt
//   takes dim 8 (l % 16) + dt, so a lane reads word l % 16 of its eight rows.
//   Two rows' words joined half by half (v_perm) expand to (row, row + 1)
//   pairs of one dim with the rows' own scales: no transposition through LDS.
// The whole group of q heads shares one expansion of K and V.
// A run is short where the cache is short (a block's start and end cost 2 us, a tile
// of 32 rows 0.15), and there are at most 128: the merge reads them all.  12 q heads
// on 2 kv heads, with the merge's 3 to 4 us behind it: 300 rows 4.3 us, 16001 with the
// scores kept 5.1, 131000 12.1 (42 MB, 3.5 TB/s; a plain read of as much takes 7.6).
// Short caches wait for the launch and one round of loads.  At 131000 rows a wave has two
// tiles: its vector instructions (24 for each MFMA) fill 57 % of the cycles, the matrix
// cores 9 %, and the rest is the start, the two waits for loads, the meeting in LDS and
// the end.  Neither more rows in flight nor 8 waves for 16 changed it.
// Probabilities are rounded to fp16 for the product with V, their sum l is not (the
// fp16 flash decode keeps both in fp32): 2^-11 of each, as prefill does, and below what a
// nibble leaves of V.
constexpr int kKd4MaxSplits = 128;   // runs of a kv head, at most
constexpr int kKd4MinRun = 128;      // rows of a run, at least: 32 for each of four waves
constexpr int kKd4MaxGroup = 64;     // q heads of a kv head
constexpr int kKd4ManyWaves = 16;    // of a block where runs may be longer (waves without rows do nothing)
// rows of a cache, at most: the last run ends up to 32 kKd4MaxSplits rows behind it, a wave's next tile 32 kKd4ManyWaves
constexpr int kKd4MaxRows = INT32_MAX - 8191;

// rows of a run for `ctx` rows over at most `splits` runs
__host__ __device__ __forceinline__ int kd4_run(int ctx, int splits) {
    const int per = (ctx + splits - 1) / splits;
    return per > kKd4MinRun ? (per + 31) & ~31 : kKd4MinRun;
}

struct Decode4Params {
    const uint16_t* q;
    const uint8_t* kc;
    const uint8_t* vc;
    const qe_device_control_block* ctl;
    const int32_t* evicted;
    float* part_o;   // [q head][split][128], relative to the run's reference value
    float* part_ml;  // [q head][split][2] (reference value in the exp2 domain, sum)
    float* scores;   // [q head][score_stride] before the scale, with key weights only
    uint16_t* out;
    int8_t* q8;
    float* q_scale;
    int32_t* q_sum8;
    const float* w_in;
    float* w_out;
    int nq, nkv, group, head_blocks, max_seq, splits, waves, score_stride;
};

// cache rows the token sees (one that found the cache full sees all of it)
__device__ __forceinline__ int kd4_context(const Decode4Params& p, int kvh) {
    return min(kv4_row(p.ctl, p.evicted, kvh), p.max_seq - 1) + 1;
}

struct Kd4Tile {
    u32x4 k[2];          // chunk l / 16 of rows l % 16 and 16 + l % 16
    uint32_t kp[2];      // its (scale, low)
    uint32_t v[8], vp[8];  // word l % 16 of the lane's eight rows, its group's (scale, low)
};

template <bool WEIGHTS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 4) void kv4_decode_kernel(Decode4Params p) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n = lane & 15, h = lane >> 4;
    const int kvh = blockIdx.x % p.nkv;
    const int hb = (blockIdx.x / p.nkv) % p.head_blocks, split = blockIdx.x / (p.nkv * p.head_blocks);
    const int heads = min(16, p.group - 16 * hb), qh0 = kvh * p.group + 16 * hb;
    const int ctx = kd4_context(p, kvh);
    const int run = kd4_run(ctx, p.splits);
    const int t0 = split * run, t1 = min(t0 + run, ctx);
    if (t0 >= t1) return;

    const size_t head_base = static_cast<size_t>(kvh) * p.max_seq * kKv4Row;
    const uint8_t* kh = p.kc + head_base;
    const uint8_t* vh = p.vc + head_base;
    // Rows r0.. of the wave up to `end`; the lane's places in a tile are four
    // offsets, and rows from `end` on read as zeros.
    const uint32_t ko = n * kKv4Row + 16 * h, kpo = n * kKv4Row + kKv4Params + 4 * h;
    const uint32_t vo = 4 * h * kKv4Row + 4 * n, vpo = 4 * h * kKv4Row + kKv4Params + 4 * (n >> 2);
    auto load = [&](int r0, int end, Kd4Tile& t) __attribute__((always_inline)) {
        const auto k = kv4_rows(kh + static_cast<size_t>(r0) * kKv4Row, min(end - r0, 32));
        const auto v = kv4_rows(vh + static_cast<size_t>(r0) * kKv4Row, min(end - r0, 32));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            t.k[i] = kv4_load4(k, ko + 16 * i * kKv4Row);
            t.kp[i] = kv4_load(k, kpo + 16 * i * kKv4Row);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            t.v[i] = kv4_load(v, vo + (16 * (i >> 2) + (i & 3)) * kKv4Row);
            t.vp[i] = kv4_load(v, vpo + (16 * (i >> 2) + (i & 3)) * kKv4Row);
        }
    };
    f16x8 qf[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        qf[kk] = f16x8{};
        if (n < heads)
            qf[kk] = *reinterpret_cast<const f16x8*>(p.q + static_cast<size_t>(qh0 + n) * kKv4Dim + 32 * h + 8 * kk);
    }
    f32x4 acc[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) acc[dt] = f32x4{};
    float m = -INFINITY, l = 0.0f;
    auto use = [&](int r0, const Kd4Tile& t) __attribute__((always_inline)) {
        float s[8];  // before the scale, which the exponent's multiply-add brings in
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x4 c = {};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                const uint32_t w = t.k[i][kk];
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv4_expand_word(w, t.kp[i]), qf[kk], c, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * i + e] = c[e];
            if constexpr (WEIGHTS) {
                if (n < heads)  // the row of scores is padded to whole tiles
                    *reinterpret_cast<float4*>(p.scores + static_cast<size_t>(qh0 + n) * p.score_stride + r0 + 16 * i +
                                               4 * h) = make_float4(c[0], c[1], c[2], c[3]);
            }
        }
        if (r0 + 31 >= t1) {  // uniform
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = r0 + 16 * (e >> 2) + 4 * h + (e & 3) < t1 ? s[e] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e]);
        mx = max_over_quarters(mx) * kScoreScale;
        // the reference value follows the maximum once it has grown by more than 8
        const bool grow = mx > m + kReferenceLag;
        if (__builtin_amdgcn_ballot_w64(grow) != 0) {
            const float alpha = grow ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
            m = grow ? mx : m;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) acc[dt] *= alpha;
        }
        const float neg = m == -INFINITY ? 0.0f : -m;
        u32x4 pw;
        float ps[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f32x2 x = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e], kScoreScale, neg)),
                             __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e + 1], kScoreScale, neg))};
            ps[0] += x.x;
            ps[1] += x.y;
            pw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
        }
        l += ps[0] + ps[1];
        const f16x8 pf = __builtin_bit_cast(f16x8, pw);
        // V^T: pairs of rows, all eight dims of the lane's word
        uint32_t vf[8][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = t.v[2 * j], b = t.v[2 * j + 1], pa = t.vp[2 * j], pb = t.vp[2 * j + 1];
            const f16x2 sc = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(pb, pa, 0x05040100u));
            const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(pb, pa, 0x07060302u));
            f16x2 even[4], odd[4];
            kv4_expand(__builtin_amdgcn_perm(b, a, 0x05040100u), sc, lo, even);
            kv4_expand(__builtin_amdgcn_perm(b, a, 0x07060302u), sc, lo, odd);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                vf[2 * e][j] = __builtin_bit_cast(uint32_t, even[e]);
                vf[2 * e + 1][j] = __builtin_bit_cast(uint32_t, odd[e]);
            }
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            const u32x4 a = {vf[dt][0], vf[dt][1], vf[dt][2], vf[dt][3]};
            acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), pf, acc[dt], 0, 0, 0);
        }
    };
    // One copy of the code in a loop, and the other waves to cover its loads: with the
    // next rows in flight from a second copy it was no faster (a launch runs it a
    // few times, and has to fetch it first).
    Kd4Tile tile;
    for (int r0 = t0 + 32 * wave; r0 < t1; r0 += 32 * WAVES) {
        load(r0, t1, tile);
        use(r0, tile);
    }
    l = sum_over_quarters(l);
    // the waves meet: common maximum, then outputs
    __shared__ float s_m[WAVES][16], s_l[WAVES][16];
    extern __shared__ __align__(16) float s_o[];  // [wave][head][128 + 4]
    constexpr int kRow = kKv4Dim + 4;
    const int active = min(WAVES, (t1 - t0 + 31) / 32);  // waves that have rows
    if (wave < active) {
        if (h == 0) {
            s_m[wave][n] = m;
            s_l[wave][n] = l;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // dims 8 (4 h + i) + dt
            if (n >= heads) break;
            float* o = &s_o[(wave * heads + n) * kRow + 8 * (4 * h + i)];
            *reinterpret_cast<float4*>(o) = make_float4(acc[0][i], acc[1][i], acc[2][i], acc[3][i]);
            *reinterpret_cast<float4*>(o + 4) = make_float4(acc[4][i], acc[5][i], acc[6][i], acc[7][i]);
        }
    }
    __syncthreads();
    for (int u = threadIdx.x; u < heads * 32; u += 64 * WAVES) {
        const int head = u >> 5, d = 4 * (u & 31);
        float mg = s_m[0][head];
        for (int w = 1; w < active; ++w) mg = fmaxf(mg, s_m[w][head]);
        float lg = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int w = 0; w < active; ++w) {
            const float mw = s_m[w][head];
            const float f = mw == mg ? 1.0f : __builtin_amdgcn_exp2f(mw - mg);
            const float4 x = *reinterpret_cast<const float4*>(&s_o[(w * heads + head) * kRow + d]);
            lg += f * s_l[w][head];
            o.x += f * x.x;
            o.y += f * x.y;
            o.z += f * x.z;
            o.w += f * x.w;
        }
        const size_t at = static_cast<size_t>(qh0 + head) * p.splits + split;
        *reinterpret_cast<float4*>(p.part_o + at * kKv4Dim + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(mg, lg);
    }
}

// Weight of every run of one head and the head's sum, by one wave: w = exp2(m - M),
// L = sum w l.  A NaN sum (a NaN score) makes L NaN.
struct Kd4RunSums {
    float2 x[kKd4MaxSplits / 64];
};
__device__ __forceinline__ Kd4RunSums kd4_run_sums(const float* ml, int splits, int lane) {
    Kd4RunSums r;
#pragma unroll
    for (int i = 0; i < kKd4MaxSplits / 64; ++i)
        r.x[i] = *reinterpret_cast<const float2*>(ml + 2 * min(lane + 64 * i, splits - 1));
    return r;
}
__device__ __forceinline__ void kd4_run_weights(Kd4RunSums& r, int live, int lane, float (&w)[kKd4MaxSplits / 64],
                                                float& M, float& L) {
    float2(&x)[kKd4MaxSplits / 64] = r.x;
    M = -INFINITY;
#pragma unroll
    for (int i = 0; i < kKd4MaxSplits / 64; ++i) {
        if (lane + 64 * i >= live) x[i] = make_float2(-INFINITY, 0.0f);
        M = fmaxf(M, x[i].x);
    }
    M = qwen::seg_max<64>(M);
    L = 0.0f;
#pragma unroll
    for (int i = 0; i < kKd4MaxSplits / 64; ++i) {
        w[i] = x[i].x == M ? 1.0f : __builtin_amdgcn_exp2f(x[i].x - M);
        if (lane + 64 * i >= live) w[i] = 0.0f;
        L += w[i] * x[i].y;
    }
    L = qwen::seg_sum<64>(L);
}

// Blocks 0..nq-1: one q head each, its runs merged (32 lanes x 4 dims, 16 groups
// of runs), rounded once to fp16, and the Q8_1 of it when asked for.  The blocks
// behind them, with key weights: 512 rows of one kv head, the sum over its q
// heads of exp2(score - M) / L added to the weight so far; the newest row
// starts at its own sum.  A launch and two rounds of loads: 3.0 us with 3 runs,
// 3.8 with 128, 4.2 with the weights of 16001 rows.
constexpr int kKd4MergeThreads = 512;
template <bool WEIGHTS>
__global__ __launch_bounds__(kKd4MergeThreads) void kv4_decode_merge_kernel(Decode4Params p) {
    constexpr int G = kKd4MergeThreads / 32, PER = kKd4MaxSplits / G;
    __shared__ __align__(16) float s_o[G][kKv4Dim];
    __shared__ float s_w[kKd4MaxSplits];
    __shared__ float s_M[kKd4MaxGroup], s_inv[kKd4MaxGroup];
    __shared__ float s_max[kKd4MergeThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (WEIGHTS && static_cast<int>(blockIdx.x) >= p.nq) {
        const int b = blockIdx.x - p.nq, kvh = b % p.nkv;
        const int row = (b / p.nkv) * kKd4MergeThreads + tid;
        const int ctx = kd4_context(p, kvh);
        if (row - tid >= ctx) return;
        const int run = kd4_run(ctx, p.splits), live = (ctx + run - 1) / run;
        for (int g = wave; g < p.group; g += kKd4MergeThreads / 64) {
            float w[kKd4MaxSplits / 64], M, L;
            Kd4RunSums sums = kd4_run_sums(p.part_ml + static_cast<size_t>(kvh * p.group + g) * p.splits * 2, p.splits, lane);
            kd4_run_weights(sums, live, lane, w, M, L);
            if (lane == 0) {
                s_M[g] = M == -INFINITY ? 0.0f : M;
                s_inv[g] = 1.0f / L;
            }
        }
        __syncthreads();
        if (row >= ctx) return;
        const size_t at = static_cast<size_t>(kvh) * p.max_seq + row;
        float sum = 0.0f;
        for (int g = 0; g < p.group; ++g)
            sum += __builtin_amdgcn_exp2f(__builtin_fmaf(p.scores[static_cast<size_t>(kvh * p.group + g) * p.score_stride + row],
                                                         kScoreScale, -s_M[g])) * s_inv[g];
        p.w_out[at] = (p.w_in != nullptr && row < kv4_row(p.ctl, p.evicted, kvh) ? p.w_in[at] : 0.0f) + sum;
        return;
    }
    const int qh = blockIdx.x, kvh = qh / p.group;
    const int d = 4 * (tid & 31), g = tid >> 5;
    const float* po = p.part_o + static_cast<size_t>(qh) * p.splits * kKv4Dim;
    float4 x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)  // requested before the context is known; runs without rows are never used
        if (g + G * i < p.splits) x[i] = *reinterpret_cast<const float4*>(po + static_cast<size_t>(g + G * i) * kKv4Dim + d);
    Kd4RunSums sums;
    if (wave == 0) sums = kd4_run_sums(p.part_ml + static_cast<size_t>(qh) * p.splits * 2, p.splits, lane);
    const int ctx = kd4_context(p, kvh);
    const int run = kd4_run(ctx, p.splits), live = (ctx + run - 1) / run;
    if (wave == 0) {
        float w[kKd4MaxSplits / 64], M, L;
        kd4_run_weights(sums, live, lane, w, M, L);
        const float inv = 1.0f / L;
#pragma unroll
        for (int i = 0; i < kKd4MaxSplits / 64; ++i) s_w[lane + 64 * i] = w[i] * inv;
    }
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (g + G * i >= live) break;
        const float w = s_w[g + G * i];
        o.x += w * x[i].x;
        o.y += w * x[i].y;
        o.z += w * x[i].z;
        o.w += w * x[i].w;
    }
    *reinterpret_cast<float4*>(&s_o[g][d]) = o;
    __syncthreads();
    float acc = 0.0f;
    if (tid < kKv4Dim) {
#pragma unroll
        for (int i = 0; i < G; ++i) acc += s_o[i][tid];
        p.out[static_cast<size_t>(qh) * kKv4Dim + tid] = f2h(acc);
    }
    if (p.q8 == nullptr) return;
    // Q8_1 of the head (one group of 128), as the fp16 flash decode writes it
    const float mx = qwen::seg_max<64>(fabsf(acc));
    if (lane == 0) s_max[wave] = mx;
    __syncthreads();
    if (tid >= kKv4Dim) return;
    const float dd = flash_q8_scale(fmaxf(s_max[0], s_max[1]));
    if (tid == 0 && p.q_scale != nullptr) p.q_scale[qh] = dd;
    const int v = flash_q8_value(acc, dd);
    p.q8[static_cast<size_t>(qh) * kKv4Dim + tid] = static_cast<int8_t>(v);
    int s8 = -8 * v;
    s8 += qwen::dpp_i32<0xB1>(s8);
    s8 += qwen::dpp_i32<0x4E>(s8);
    s8 += qwen::dpp_i32<0x141>(s8);
    if ((tid & 7) == 0 && p.q_sum8 != nullptr) p.q_sum8[qh * (kKv4Dim / 8) + (tid >> 3)] = s8;
}

// ---- the rows of a chunk -------------------------------------------------------------
// Query rows r = token r / group, head kvh * group + r % group; a block takes
// 32 WAVES consecutive rows of one kv head, 32 a wave, and walks its run of
// key tiles (64 cache rows).  Both products are v_mfma_f32_32x32x16_f16 with the
// rows as columns, as in the fp16 prefill: S^T = K . Q^T, a row's maximum and sum
// in its own lane and lane ^ 32; O^T += V^T . P^T with P^T the lane's own.
// A tile is expanded once per block, into LDS as fp16: a thread takes 16-byte chunk
// g (one quantization group) of one row and writes four 16-byte chunks, 4 g + i,
// stored at chunk ^ swz(row).  16 lanes hold 16 rows of one g, so they touch 16
// different bank groups, like the readers (16 rows of one chunk for K; 4 rows x 4
// chunks through ds_read_b64_tr_b16 for V); a store moves 128 bytes a cycle, so the
// rows are numbered for 8 lanes to touch 8 groups that differ mod 8 as well (rows in
// order: 8 more cycles a store, 1 % of the kernel).
// The raw 20 bytes of the tile after the next are in registers a whole step
// before they are expanded; a split's first two tiles are requested at once, and four
// waves with no more than two take them from there (17 tokens at 1200: 12.9 -> 10.4 us in
// all, a third of it the coalesced partials below).
// 2048 tokens at 14000 (12 q heads, 2 kv heads) take 224 us with the merge, 0.84 PFLOP/s of
// the 1.5 to 1.6 that a large product reaches.  Two things bound them.  Splits are whole
// per row block: 96 row blocks make 192 blocks of one per CU, and a quarter of the CUs has
// none.  On the others MFMAs are busy 54 %, beside the vector instructions between them
// (6.5 for each MFMA, one of them an exponential at a quarter of the rate), which overlap in
// part; without the exponentials or without the expansion they would take a tenth less,
// without the barrier 3 %.  Slower: 64 rows a wave (by 15 %: the scores move through the
// accumulation registers), the block's halves half a step apart (by 24 %: the
// probabilities that cross the barrier do not fit the registers).
// Registers: all 256, and scratch where a wave ends with two tiles: with four waves 70
// values (216 bytes a lane), with eight 2, stored and read back once; the steps have none.
// Probabilities are rounded to fp16 for the product with V, their sum is not.
constexpr int kP4Keys = 64;
constexpr int kP4TileBytes = kP4Keys * kKv4Dim * 2;
// Tiles of a split, at least, and of the splits beyond the eighth, whose merge costs
// more: still 2 where a row is merged by several groups, else 8.  (us, 12 q heads, 2 kv
// heads: 17 tokens at 1200 10.7 with 2, 12.5 with 3 or 4; 509 at 0 14.9 with 2, 17.5 with
// 3; 300 at 2000 22.5 with 2 and then 8, 25.3 with 2 and then 4.)
constexpr int kP4MinTiles = 2, kP4FarTiles = 8, kP4FarTilesMany = 2;
constexpr int kP4MaxSplits = 64;
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct Prefill4Params {
    const uint16_t* q;
    const uint8_t* kc;
    const uint8_t* vc;
    uint16_t* out;
    const qe_device_control_block* ctl;
    const int32_t* evicted;
    float* part_o;   // [split][kv head][32 rows] unnormalized, 16 bytes of [4 dt + g][h][row]: dims 32 dt + 8 g + 4 h
    float* part_ml;  // [split][kv head][row][2] (reference value, sum)
    float* lse;      // [token][q head] natural log, or NULL
    const float* w_in;
    float* w_out;
    float* part_w;   // [split of the q rows][kv head][max_seq]
    int T, nq, nkv, group, max_seq, out_stride, splits, row_blocks, block_rows, far_tiles, weight_splits;
};

__device__ __forceinline__ int p4_live_splits(const Prefill4Params& p, int tiles) {
    return max(1, min(p.splits, max(min(tiles / kP4MinTiles, 8), tiles / p.far_tiles)));
}
// key tiles of row block rb (the rows of the cache that its last row sees)
__device__ __forceinline__ int p4_tiles(const Prefill4Params& p, int rb, int base) {
    const int last = min((rb + 1) * p.block_rows, p.T * p.group) - 1;
    const int len = min(base, p.max_seq) + last / p.group + 1;
    return (min(len, p.max_seq) + kP4Keys - 1) / kP4Keys;
}

// Where the partials of row r's 32 rows begin, in float4: a wave's stores of them are
// 1 KB each, and the readers take 8 rows of a piece, 128 bytes.
__device__ __forceinline__ size_t p4_part(const Prefill4Params& p, int split, int kvh, int r) {
    return ((static_cast<size_t>(split) * p.nkv + kvh) * ((p.T * p.group + 31) / 32) + (r >> 5)) * 1024;
}

__device__ __forceinline__ float xor32_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                    false, false);
    const uint32_t a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

template <int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void kv4_prefill_kernel(Prefill4Params p) {
    // K buffers 0 and 1, V buffers 0 and 1; aligned for reads that turn address bits 5 to 7
    __shared__ __align__(256) char smem[4 * kP4TileBytes];
    constexpr int UNITS = 8 / WAVES;  // (K or V) chunks a thread expands for a tile: 512 in all
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int fr = lane & 31, h = lane >> 5;
    const int rb = p.row_blocks - 1 - static_cast<int>(blockIdx.x) % p.row_blocks;  // longest rows first
    const int cb = static_cast<int>(blockIdx.x) / p.row_blocks;
    const int kvh = cb % p.nkv, split = cb / p.nkv;
    const int rows = p.T * p.group;
    const int base = min(kv4_row(p.ctl, p.evicted, kvh), p.max_seq);
    const int nt_all = p4_tiles(p, rb, base);
    const int live = p4_live_splits(p, nt_all);
    if (split >= live) return;
    const int it0 = static_cast<int>((static_cast<long long>(split) * nt_all) / live);
    const int it1 = static_cast<int>((static_cast<long long>(split + 1) * nt_all) / live);
    const int r = rb * (32 * WAVES) + wave * 32 + fr;
    const int rc = min(r, rows - 1);
    const int qi = rc / p.group, qh = kvh * p.group + rc % p.group;
    const int lim = min(min(base + qi, p.max_seq - 1), it1 * kP4Keys - 1);  // last cache row this row takes here
    const int wave_lim = __builtin_amdgcn_readlane(lim, 0);
    const int wave_last = __builtin_amdgcn_readlane(lim, 31);
    const int key_max = min(base + p.T, p.max_seq) - 1;  // the last cache row that holds anything

    u32x4 qf[8];
    {
        const uint16_t* qr = p.q + (static_cast<size_t>(qi) * p.nq + qh) * kKv4Dim + 8 * h;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) qf[kk] = *reinterpret_cast<const u32x4*>(qr + 16 * kk);
    }
    // staging: unit u = chunk g of row srow, K units first; with 8 waves, waves
    // 0..3 expand K and 4..7 V, with 4 every thread does one of each
    const int su = threadIdx.x & 255, sg = (su >> 4) & 3;
    const int srow = ((su & 1) | ((su & 6) << 1) | ((su & 8) >> 2)) + 16 * (su >> 6);
    const size_t hb = static_cast<size_t>(kvh) * p.max_seq * kKv4Row;
    const uint8_t* src[UNITS];
    char* dst[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const bool is_v = UNITS == 2 ? u == 1 : wave >= 4;
        src[u] = (is_v ? p.vc : p.kc) + hb;
        dst[u] = smem + (is_v ? 2 : 0) * kP4TileBytes + srow * 256;
    }
    const int sswz = ((srow & 3) << 2) | ((srow >> 2) & 3);
    struct Raw {
        u32x4 w[UNITS];
        uint32_t p[UNITS];
    } raw;
    // tile tk for the K units, tv for the V units
    auto fetch = [&](Raw& raw, int tk, int tv) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const bool is_v = UNITS == 2 ? u == 1 : wave >= 4;
            const uint8_t* row = src[u] + static_cast<size_t>(min((is_v ? tv : tk) * kP4Keys + srow, key_max)) * kKv4Row;
            raw.w[u] = *reinterpret_cast<const u32x4*>(row + 16 * sg);
            raw.p[u] = *reinterpret_cast<const uint32_t*>(row + kKv4Params + 4 * sg);
        }
    };
    // word i of a unit
    auto expand_word = [&](const Raw& raw, int u, int i, int kbuf, int vbuf) __attribute__((always_inline)) {
        const bool is_v = UNITS == 2 ? u == 1 : wave >= 4;
        const uint32_t w = raw.w[u][i];
        *reinterpret_cast<f16x8*>(dst[u] + (is_v ? vbuf : kbuf) * kP4TileBytes + 16 * ((4 * sg + i) ^ sswz)) =
            kv4_expand_word(w, raw.p[u]);
    };
    auto expand = [&](const Raw& raw, int kbuf, int vbuf) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) expand_word(raw, u, i, kbuf, vbuf);
    };
    auto tile_barrier = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) void*)smem));
    // LDS addresses: K chunk 2 kk + h of row fr; V^T reads (dt: 32 dims, u: rows + 8)
    uint32_t k0 = lds0 + fr * 256 + 16 * (h ^ (((fr & 3) << 2) | ((fr >> 2) & 3)));
    uint32_t va[4][2];
    {
        const int s16 = lane & 15, b16 = (lane >> 4) & 1;
        const uint32_t v0 = lds0 + 2 * kP4TileBytes + (4 * h + (s16 >> 2)) * 256 +
                            16 * ((2 * b16 + ((s16 & 3) >> 1)) ^ (((s16 >> 2) << 2) | h)) + 8 * (s16 & 1);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
            va[dt][0] = v0 ^ (64 * dt);
            va[dt][1] = (v0 ^ (64 * dt) ^ 32) + 8 * 256;
        }
    }
    // K operand of MFMA i of a tile: 32-row half i % 2, dims 16 (i / 2); V^T
    // operand: 16-row quarter i / 4, dims 32 (i % 4)
    auto read_k = [&](int buf, int i) __attribute__((always_inline)) {
        typedef const __attribute__((address_space(3))) f16x8* lptr;
        return *reinterpret_cast<lptr>((k0 ^ (32 * (i >> 1))) + buf * kP4TileBytes + (i & 1) * 32 * 256);
    };
    auto read_v = [&](int buf, int i) __attribute__((always_inline)) {
        typedef __attribute__((address_space(3))) s16x4* lptr;
        const uint32_t off = buf * kP4TileBytes + (i >> 2) * 16 * 256;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lptr>(va[i & 3][0] + off));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lptr>(va[i & 3][1] + off));
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    f32x16 acc[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) acc[dt] = f32x16{};
    float mref = -INFINITY, lsum = 0.0f;
    auto mask = [&](int t, f32x16 (&sc)[2]) __attribute__((always_inline)) {
        if ((t + 1) * kP4Keys - 1 > wave_lim) {  // wave-uniform
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int key = t * kP4Keys + 32 * j + 8 * (v >> 2) + 4 * h + (v & 3);
                    sc[j][v] = key <= lim ? sc[j][v] : -INFINITY;
                }
        }
    };
    auto renew_ref = [&](float mx) __attribute__((always_inline)) {
        const bool grow = mx > mref + kReferenceLag;
        if (__builtin_amdgcn_ballot_w64(grow) != 0) {
            const float alpha = grow ? __builtin_amdgcn_exp2f(mref - mx) : 1.0f;
            mref = grow ? mx : mref;
            lsum *= alpha;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[dt][v] *= alpha;
        }
    };
    auto row_max = [&](const f32x16 (&sc)[2]) __attribute__((always_inline)) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[j][v]);
        return xor32_max(mx) * kScoreScale;
    };
    // probabilities 2 i and 2 i + 1 of a tile's scores (32-row half i / 8), packed
    auto probs = [&](const f32x16 (&sc)[2], int i, float neg, float (&ps)[2]) __attribute__((always_inline)) {
        const int j = i >> 3, v = 2 * (i & 7);
        const f32x2 e = {__builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][v], kScoreScale, neg)),
                         __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][v + 1], kScoreScale, neg))};
        ps[0] += e.x;
        ps[1] += e.y;
        uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(e, f16x2));
        asm volatile("" : "+v"(w), "+v"(ps[0]), "+v"(ps[1]));  // here, not past the mask's branch
        return w;
    };
    constexpr int AHEAD = 3;  // operand reads in flight before their MFMA
    // Scores of the K tile in `buf`; beside them, when EXP, the probabilities of
    // the scores `cur`, each MFMA fenced together with its share of the vector work.
    auto scores = [&](auto exp_too, int buf, f32x16 (&sc)[2], const f32x16 (&cur)[2],
                      uint32_t (&pw)[2][8]) __attribute__((always_inline)) {
        const float neg = mref == -INFINITY ? 0.0f : -mref;  // masked scores give exp2(-inf) = 0
        float ps[2] = {0.0f, 0.0f};
        // (four waves: the eight turned addresses are made anew, kept ones are spilled; 500 rows at 15000 71 against 74 us)
        if constexpr (WAVES == 4) asm volatile("" : "+v"(k0));
        f16x8 kf[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) kf[i] = read_k(buf, i);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i % AHEAD], __builtin_bit_cast(f16x8, qf[i >> 1]),
                                                               i < 2 ? f32x16{} : sc[i & 1], 0, 0, 0);
            if (i + AHEAD < 16) kf[i % AHEAD] = read_k(buf, i + AHEAD);
            if constexpr (decltype(exp_too)::value) pw[i >> 3][i & 7] = probs(cur, i, neg, ps);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (decltype(exp_too)::value) lsum += ps[0] + ps[1];
    };
    // O^T += V^T . P^T; beside it, when MORE, the (scaled) row maximum of nxt, and
    // the tiles in registers go to LDS, K to buffer buf and V to the other
    auto add_pv = [&](auto more, const uint32_t (&pw)[2][8], int buf,
                      const f32x16 (&nxt)[2]) __attribute__((always_inline)) {
        f16x8 vf[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) vf[i] = read_v(buf, i);
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int j = i >> 3, ks = (i >> 2) & 1, dt = i & 3;
            const u32x4 pf = {pw[j][4 * ks], pw[j][4 * ks + 1], pw[j][4 * ks + 2], pw[j][4 * ks + 3]};
            acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i % AHEAD], __builtin_bit_cast(f16x8, pf), acc[dt], 0, 0, 0);
            if (i + AHEAD < 16) vf[i % AHEAD] = read_v(buf, i + AHEAD);
            if constexpr (decltype(more)::value) {
                mx = fmaxf(fmaxf(mx, nxt[j][2 * (i & 7)]), nxt[j][2 * (i & 7) + 1]);
                if (UNITS == 2 && (i & 1) == 0) expand_word(raw, i >> 3, (i >> 1) & 3, buf, buf ^ 1);
                if (UNITS == 1 && (i & 3) == 0) expand_word(raw, 0, i >> 2, buf, buf ^ 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        return decltype(more)::value ? xor32_max(mx) * kScoreScale : 0.0f;
    };
    typedef std::true_type yes;
    typedef std::false_type no;
    // What a step does for everyone: K of the tile after next and V of the next
    // go to LDS (b: parity of tile t), the raw bytes behind them are requested.
    auto stage = [&](int t, int b) __attribute__((always_inline)) {
        expand(raw, b, b ^ 1);
        fetch(raw, t + 3, t + 2);
    };
    // Tile t's scores are in cur: the scores of the next tile beside the
    // probabilities of t, then V of t beside the next tile's maximum.
    auto step = [&](int t, int b, f32x16 (&cur)[2], f32x16 (&nxt)[2]) __attribute__((always_inline)) {
        uint32_t pw[2][8];
        scores(yes{}, b ^ 1, nxt, cur, pw);
        mask(t + 1, nxt);
        const float mx = add_pv(yes{}, pw, b, nxt);
        fetch(raw, t + 3, t + 2);
        renew_ref(mx);
        tile_barrier();
    };
    auto finish = [&](int b, f32x16 (&cur)[2]) __attribute__((always_inline)) {
        uint32_t pw[2][8];
        const float neg = mref == -INFINITY ? 0.0f : -mref;
        float ps[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; ++i) pw[i >> 3][i & 7] = probs(cur, i, neg, ps);
        lsum += ps[0] + ps[1];
        add_pv(no{}, pw, b, cur);
    };
    auto run = [&]() __attribute__((always_inline)) {
        const int n = it1 - it0;
        int t = it0;
        // two tiles are requested before the first is waited for
        Raw first;
        fetch(first, t, t);
        fetch(raw, t + 1, t + 1);
        expand(first, 0, 0);
        // K of the second tile now; V of it comes with the first step, which
        // expands what is in registers: K of the third, V of the second
        if constexpr (UNITS == 2) {
            expand(raw, 1, 1);
        } else {
            if (wave < 4) expand(raw, 1, 1);
        }
        // tiles past the wave's last key are not multiplied
        const int mine = wave_last < t * kP4Keys ? 0 : min(n, wave_last / kP4Keys - t + 1);
        f32x16 s0[2], s1[2];
        uint32_t none[2][8];
        if (UNITS == 2 && n <= 2) {  // all there: nothing left to overlap with
            tile_barrier();
#pragma unroll 1
            for (int i = 0; i < mine; ++i) {
                scores(no{}, i, s0, s1, none);
                mask(t + i, s0);
                renew_ref(row_max(s0));
                finish(i, s0);
            }
            return;
        }
        fetch(raw, t + 2, t + 1);
        tile_barrier();
        scores(no{}, 0, s0, s1, none);
        mask(t, s0);
        renew_ref(row_max(s0));
        tile_barrier();  // K buffer 0 is read
        int left = mine;
        for (; left > 2; left -= 2) {
            step(t, 0, s0, s1);
            step(t + 1, 1, s1, s0);
            t += 2;
        }
        if (left == 2) {
            // (one after the other: a step here costs registers that the loop needs)
            scores(no{}, 1, s1, s0, none);
            mask(t + 1, s1);
            finish(0, s0);
            stage(t, 0);
            tile_barrier();
            renew_ref(row_max(s1));
            finish(1, s1);
        } else if (left == 1) {
            finish(0, s0);
        }
        for (int i = max(mine - 1, 0); i < n - 1; ++i) {  // the tiles of the other waves
            stage(it0 + i, i & 1);
            tile_barrier();
        }
    };
    if (it0 < it1) run();
    lsum += __shfl_xor(lsum, 32);
    if (r >= rows) return;
    if (live == 1) {
        const float inv = 1.0f / lsum;  // (0 only where every score is -inf: NaN)
        uint16_t* o = p.out + static_cast<size_t>(qi) * p.out_stride + qh * kKv4Dim;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {  // dims 32dt + 8g + 4h .. +3
                const uint32_t w0 = static_cast<uint32_t>(f2h(acc[dt][4 * g] * inv)) |
                                    (static_cast<uint32_t>(f2h(acc[dt][4 * g + 1] * inv)) << 16);
                const uint32_t w1 = static_cast<uint32_t>(f2h(acc[dt][4 * g + 2] * inv)) |
                                    (static_cast<uint32_t>(f2h(acc[dt][4 * g + 3] * inv)) << 16);
                *reinterpret_cast<uint2*>(o + 32 * dt + 8 * g + 4 * h) = make_uint2(w0, w1);
            }
        if (p.lse != nullptr && h == 0)
            p.lse[static_cast<size_t>(qi) * p.nq + qh] = (mref == -INFINITY ? 0.0f : mref) * kLn2 + logf(lsum);
        return;
    }
    const size_t prow = (static_cast<size_t>(split) * p.nkv + kvh) * rows + r;
    if (h == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * prow) = make_float2(mref, lsum);
    float4* po = reinterpret_cast<float4*>(p.part_o) + p4_part(p, split, kvh, r) + lane;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            po[64 * (4 * dt + g)] = make_float4(acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]);
}

// Merges the splits of eight rows of one kv head: a thread per row and 4 dims, rows
// first, so that 8 lanes read 128 bytes; GROUPS groups of 256 threads, a group takes
// every GROUPS-th split and LDS adds the groups up in their order.  One group; four
// for few rows with more than 8 splits, where what counts is how many rounds of loads
// a row waits for.  The rows' weights of the splits come first, a half wave a row.
// Rows whose block had one split are already written.  Bound by the partials: 12000
// rows in 5 splits 7.7 us (31 MB), 204 rows in 9 splits 3.3 (a launch alone 1.7).
constexpr int kP4MergeMany = 4;
template <int GROUPS>
__global__ __launch_bounds__(256 * GROUPS) void kv4_prefill_merge_kernel(Prefill4Params p) {
    static_assert(kP4MaxSplits <= 64, "two splits a lane");
    __shared__ __align__(16) float4 s_o[GROUPS][256];
    __shared__ float s_w[8][kP4MaxSplits], s_inv[8];
    const int rows = p.T * p.group, blocks = (rows + 7) / 8;
    const int kvh = static_cast<int>(blockIdx.x) / blocks, r0 = 8 * (static_cast<int>(blockIdx.x) % blocks);
    const int base = min(kv4_row(p.ctl, p.evicted, kvh), p.max_seq);
    const int live = p4_live_splits(p, p4_tiles(p, r0 / p.block_rows, base));
    if (live == 1) return;
    const int tid = threadIdx.x & 255, g = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int c = tid >> 3, r = min(r0 + (tid & 7), rows - 1);
    constexpr int B = 8;
    const float4* po = reinterpret_cast<const float4*>(p.part_o) + p4_part(p, 0, kvh, r) + 32 * c + (r & 31);
    const size_t stride = p4_part(p, 1, 0, 0);
    float4 v[B];
    auto request = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (s0 + GROUPS * b < live) v[b] = po[(s0 + GROUPS * b) * stride];  // wave-uniform
    };
    request(g);
    if (g == 0) {
        const int row = tid >> 5, lane = tid & 31;
        const int rr = min(r0 + row, rows - 1);
        float2 ml[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int s = lane + 32 * k;
            ml[k] = make_float2(-INFINITY, 0.0f);
            if (s < live)
                ml[k] = *reinterpret_cast<const float2*>(p.part_ml + 2 * ((static_cast<size_t>(s) * p.nkv + kvh) * rows + rr));
        }
        const float m = qwen::seg_max<32>(fmaxf(ml[0].x, ml[1].x));
        // (a split whose scores are all NaN has no maximum and a NaN sum, which the products below keep)
        float w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            w[k] = ml[k].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[k].x - m);
            s_w[row][lane + 32 * k] = w[k];
        }
        const float l = qwen::seg_sum<32>(w[0] * ml[0].y + w[1] * ml[1].y);
        if (lane == 0) {
            s_inv[row] = 1.0f / l;
            if (p.lse != nullptr && r0 + row < rows)
                p.lse[static_cast<size_t>(rr / p.group) * p.nq + kvh * p.group + rr % p.group] =
                    (m == -INFINITY ? 0.0f : m) * kLn2 + logf(l);
        }
    }
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = g; s0 < live; s0 += GROUPS * B) {
        if (s0 > g) request(s0);
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int s = s0 + GROUPS * b;
            if (s >= live) break;
            const float ws = s_w[tid & 7][s];
            o.x += ws * v[b].x;
            o.y += ws * v[b].y;
            o.z += ws * v[b].z;
            o.w += ws * v[b].w;
        }
    }
    if constexpr (GROUPS > 1) {
        s_o[g][tid] = o;
        __syncthreads();
        if (g != 0) return;
#pragma unroll
        for (int k = 1; k < GROUPS; ++k) {
            const float4 x = s_o[k][tid];
            o.x += x.x;
            o.y += x.y;
            o.z += x.z;
            o.w += x.w;
        }
    }
    if (r0 + (tid & 7) >= rows) return;
    const float inv = s_inv[tid & 7];
    const int qi = r / p.group, qh = kvh * p.group + r % p.group;
    uint16_t* dst = p.out + static_cast<size_t>(qi) * p.out_stride + qh * kKv4Dim + 4 * c;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(static_cast<uint32_t>(f2h(o.x * inv)) | (static_cast<uint32_t>(f2h(o.y * inv)) << 16),
                   static_cast<uint32_t>(f2h(o.z * inv)) | (static_cast<uint32_t>(f2h(o.w * inv)) << 16));
}

// Column sums of the probabilities: what the rows of the chunk give to 64 cache
// rows of one kv head.  S^T = K . Q^T again, p = exp(s - lse) with the row's final log
// sum.  Four waves hold the first 32 K rows in registers, expanded once, four the
// other 32; a tile of q rows, the whole tokens that 128 rows hold (so that a lane's
// places in a tile are always the same), comes to LDS by DMA, whole rows of 256 bytes,
// while the one before is used, and wave w takes its rows 32 (w % 4).. for its K
// rows.  A lane keeps 16 sums; lanes, then waves, then the splits of the q rows add
// up in one order.  The log sum's rounding, 2^-24 of it, is in every weight of its row.
// Bound by the exponentials and what little is around them (MFMAs busy 29 %).  1000 rows on 2900..3900 positions (12 q heads, 2 kv heads): 50 us with
// operands read from memory, 32 bytes of 32 rows at a time (their addresses alone), 29
// with 32 K rows a block and a q tile for each wave, 22 and 5 for the splits' merge now.
constexpr int kW4Keys = 64, kW4Rows = 128;
constexpr int kW4Buffer = kW4Rows * 256 + kW4Rows * 4;  // q rows, their log sums
constexpr int kW4MaxSplits = 4;
__global__ __launch_bounds__(512, 4) void kv4_prefill_weights_kernel(Prefill4Params p) {
    __shared__ __align__(256) char smem[2 * kW4Buffer];  // as in the prefill
    __shared__ float s_sum[8][32];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int fr = lane & 31, h = lane >> 5, rw = wave & 3, kg = wave >> 2;
    const int kvh = blockIdx.x % p.nkv, rest = blockIdx.x / p.nkv;
    const int split = rest % p.weight_splits, t = rest / p.weight_splits;
    const int base = min(kv4_row(p.ctl, p.evicted, kvh), p.max_seq);
    const int len = min(base + p.T, p.max_seq);
    if (t * kW4Keys >= len) return;
    const int key0 = t * kW4Keys + 32 * kg;
    f32x16 sum = {};
    // this split's share of the q tiles from the first token that sees a key of the block
    const int per = kW4Rows / p.group, held = per * p.group;  // tokens and rows of a tile
    const int first = max(0, min(t * kW4Keys - base, p.T - 1)) / per;
    const int tiles = (p.T + per - 1) / per - first;
    int u = first + tiles * split / p.weight_splits;
    const int u1 = first + tiles * (split + 1) / p.weight_splits;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) void*)smem));
    const uint16_t* q_head = p.q + static_cast<size_t>(kvh) * p.group * kKv4Dim;
    const float* lse_head = p.lse + static_cast<size_t>(kvh) * p.group;
    // x / group for x < 128: group <= 64, so x (group inverse - 2^16) <= 2^13 stays below 2^16
    const uint32_t inverse = 65536u / p.group + 1u;
    auto over_group = [&](int x) { return static_cast<int>((static_cast<uint32_t>(x) * inverse) >> 16); };
    // Row x of a tile: token x / group of it, q head x % group; rows past the last are
    // read as the last.  Its place counted from the tile's first q row; `tokens` are there.
    auto place = [&](int x, int tokens) __attribute__((always_inline)) {
        x = min(x, tokens * p.group - 1);
        const int token = over_group(x);
        return static_cast<uint32_t>(token * p.nq + x - token * p.group);
    };
    // Tile load i: rows 16 wave + 4 i + lane / 16, stored chunk lane % 16, i.e.
    // chunk (lane % 16) ^ swz(row) of memory.
    uint32_t q_at[4], lse_at;
    auto places = [&](int tokens) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q_at[i] = place(16 * wave + 4 * i + (lane >> 4), tokens) * (2 * kKv4Dim) +
                      16 * ((lane & 15) ^ (((lane >> 4) << 2) | i));
        lse_at = place(64 * (wave & 1) + lane, tokens);
    };
    places(per);
    auto request = [&](int tile, int buf) __attribute__((always_inline)) {
        if (p.T - tile * per < per) places(p.T - tile * per);  // the last tile, not whole
        const uint32_t dst = lds0 + buf * kW4Buffer;
        const size_t q0 = static_cast<size_t>(tile) * per * p.nq;
#pragma unroll
        for (int i = 0; i < 4; ++i) lds_load_x4(dst + 4096 * wave + 1024 * i, q_head + q0 * kKv4Dim, q_at[i]);
        if (wave < kW4Rows / 64) lds_load_dword(dst + kW4Rows * 256 + 256 * wave, lse_head + q0 + lse_at);
    };
    const int mine = 32 * rw + fr, my_token = over_group(min(mine, held - 1));  // the lane's row of a tile
    const uint32_t qa = lds0 + mine * 256 + 16 * (h ^ (((fr & 3) << 2) | ((fr >> 2) & 3)));
    if (u < u1) request(u, 0);
    f16x8 kf[8];
    {
        const uint8_t* row = p.kc + (static_cast<size_t>(kvh) * p.max_seq + min(key0 + fr, len - 1)) * kKv4Row;
        u32x4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const u32x4*>(row + 16 * i);
        const u32x4 par = *reinterpret_cast<const u32x4*>(row + kKv4Params);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {  // word 2 kk + h: dims 16 kk + 8 h..
            const uint32_t even = w[kk >> 1][2 * (kk & 1)], odd = w[kk >> 1][2 * (kk & 1) + 1], pr = par[kk >> 1];
            kf[kk] = kv4_expand_word(h ? odd : even, pr);
        }
    }
    for (int buf = 0; u < u1; ++u, buf ^= 1) {
        typedef const __attribute__((address_space(3))) f16x8* lptr;
        typedef const __attribute__((address_space(3))) float* lfptr;
        // the tile is there for every wave, and the other buffer is read by all
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (u + 1 < u1) request(u + 1, buf ^ 1);
        f32x16 sc = {};
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                kf[kk], *reinterpret_cast<lptr>((qa ^ (32 * kk)) + buf * kW4Buffer), sc, 0, 0, 0);
        const float lse = *reinterpret_cast<lfptr>(lds0 + buf * kW4Buffer + kW4Rows * 256 + 4 * mine);
        const int token = u * per + my_token;
        // a row that is not there counts nothing (it stands for another, whose score is as finite)
        const float neg = mine < held && token < p.T ? -lse * kLog2e : -INFINITY;
        // every row of the tile sees every key (limits grow with the rows)
        if (min(base + u * per, p.max_seq - 1) >= key0 + 31) {
#pragma unroll
            for (int v = 0; v < 16; ++v) sum[v] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[v], kScoreScale, neg));
        } else {
            const int lim = min(base + token, p.max_seq - 1);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int key = key0 + 8 * (v >> 2) + 4 * h + (v & 3);
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[v], kScoreScale, neg));
                sum[v] += key <= lim ? e : 0.0f;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const float x = qwen::seg_sum<32>(sum[v]);
        if (fr == 0) s_sum[wave][8 * (v >> 2) + 4 * h + (v & 3)] = x;
    }
    __syncthreads();
    const int k = threadIdx.x, key = t * kW4Keys + k;
    if (k >= kW4Keys || key >= len) return;
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) x += s_sum[4 * (k >> 5) + w][k & 31];
    const size_t at = static_cast<size_t>(kvh) * p.max_seq + key;
    if (p.weight_splits > 1)
        p.part_w[static_cast<size_t>(split) * p.nkv * p.max_seq + at] = x;
    else
        p.w_out[at] = (p.w_in != nullptr && key < base ? p.w_in[at] : 0.0f) + x;
}

// The splits of the q rows together: a launch and a round of loads, 5 us for 2 x 4096 rows.
__global__ __launch_bounds__(256) void kv4_prefill_weights_merge_kernel(Prefill4Params p) {
    const int kvh = blockIdx.x % p.nkv, key = (blockIdx.x / p.nkv) * 256 + threadIdx.x;
    if (key >= p.max_seq) return;
    const size_t at = static_cast<size_t>(kvh) * p.max_seq + key, stride = static_cast<size_t>(p.nkv) * p.max_seq;
    float part[kW4MaxSplits];  // requested before the position is known
#pragma unroll
    for (int s = 0; s < kW4MaxSplits; ++s) part[s] = p.part_w[min(s, p.weight_splits - 1) * stride + at];
    const float was = p.w_in != nullptr ? p.w_in[at] : 0.0f;
    const int base = min(kv4_row(p.ctl, p.evicted, kvh), p.max_seq);
    if (key >= min(base + p.T, p.max_seq)) return;
    float x = 0.0f;
#pragma unroll
    for (int s = 0; s < kW4MaxSplits; ++s) x += s < p.weight_splits ? part[s] : 0.0f;
    p.w_out[at] = (key < base ? was : 0.0f) + x;
}

inline int check_heads(const char* what, int nq, int nkv) {
    QE_REQUIRE(nq > 0 && nq % nkv == 0, "%s: %d q heads over %d kv heads", what, nq, nkv);
    QE_REQUIRE(nq / nkv <= kKd4MaxGroup, "%s: %d q heads for each kv head (at most %d)", what, nq / nkv, kKd4MaxGroup);
    return QE_OK;
}

// key weights in place or apart
inline int check_weights(const char* what, const float* in, const float* out, int nkv, int max_seq) {
    QE_REQUIRE(in == nullptr || out != nullptr, "%s: key_weights_in without key_weights_out", what);
    const size_t bytes = static_cast<size_t>(nkv) * max_seq * sizeof(float);
    QE_REQUIRE(in == nullptr || in == out || apart(in, bytes, out, bytes),
               "%s: key_weights_out overlaps key_weights_in without being it", what);
    return QE_OK;
}

inline int score_stride(int max_seq) { return (max_seq + 31) / 32 * 32; }

}  // namespace
}  // namespace qe

using namespace qe;

extern "C" int qe_kv4_decode_workspace_bytes(int num_q_heads, int max_seq_len, int with_key_weights, size_t* bytes) {
    QE_REQUIRE(bytes != nullptr, "kv4_decode_workspace_bytes: NULL pointer");
    QE_REQUIRE(num_q_heads > 0 && max_seq_len > 0 && max_seq_len <= kKd4MaxRows,
               "kv4_decode_workspace_bytes: num_q_heads=%d max_seq_len=%d", num_q_heads, max_seq_len);
    size_t floats = static_cast<size_t>(num_q_heads) * kKd4MaxSplits * (kKv4Dim + 2);
    if (with_key_weights) floats += static_cast<size_t>(num_q_heads) * score_stride(max_seq_len);
    *bytes = floats * sizeof(float);
    return QE_OK;
}

extern "C" int qe_launch_attention_gqa_flash_decode_kv4(const uint16_t* q, const uint8_t* layer_k_cache,
                                                        const uint8_t* layer_v_cache, void* workspace,
                                                        uint16_t* attn_out, const qe_device_control_block* d_control,
                                                        const int32_t* d_evicted, hipStream_t stream,
                                                        int num_q_heads, int num_kv_heads, int head_dim,
                                                        int max_seq_len, int8_t* out_q8, float* out_scale,
                                                        int32_t* out_sum8, const float* key_weights_in,
                                                        float* key_weights_out) {
    const char* what = "attention_gqa_flash_decode_kv4";
    QE_REQUIRE(q && workspace && attn_out, "%s: NULL pointer", what);
    QE_TRY(kv4_check(what, layer_k_cache, layer_v_cache, num_kv_heads, head_dim, max_seq_len));
    QE_TRY(check_heads(what, num_q_heads, num_kv_heads));
    QE_REQUIRE(max_seq_len <= kKd4MaxRows, "%s: max_seq_len=%d", what, max_seq_len);
    QE_REQUIRE(aligned(q, 16) && aligned(workspace, 16), "%s: q and the workspace must be 16-byte aligned", what);
    QE_TRY(check_weights(what, key_weights_in, key_weights_out, num_kv_heads, max_seq_len));
    Decode4Params p{};
    p.q = q;
    p.kc = layer_k_cache;
    p.vc = layer_v_cache;
    p.ctl = d_control;
    p.evicted = d_evicted;
    p.out = attn_out;
    p.q8 = out_q8;
    p.q_scale = out_scale;
    p.q_sum8 = out_sum8;
    p.w_in = key_weights_in;
    p.w_out = key_weights_out;
    p.nq = num_q_heads;
    p.nkv = num_kv_heads;
    p.group = num_q_heads / num_kv_heads;
    p.head_blocks = (p.group + 15) / 16;
    p.max_seq = max_seq_len;
    p.score_stride = score_stride(max_seq_len);
    // Two blocks per CU, and no more runs than the cache can fill.
    const long long units = static_cast<long long>(num_kv_heads) * p.head_blocks;
    p.splits = static_cast<int>(std::max(8LL, std::min<long long>(kKd4MaxSplits, 2LL * cu_count() / units)));
    p.waves = max_seq_len > static_cast<long long>(kKd4MinRun) * p.splits ? kKd4ManyWaves : 4;
    p.splits = std::min(p.splits, (max_seq_len - 1) / kKd4MinRun + 1);
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + static_cast<size_t>(num_q_heads) * kKd4MaxSplits * kKv4Dim;
    p.scores = p.part_ml + static_cast<size_t>(num_q_heads) * kKd4MaxSplits * 2;
    const long long blocks = units * p.splits;
    const long long weight_blocks =
        static_cast<long long>(num_kv_heads) * ((static_cast<long long>(max_seq_len) + kKd4MergeThreads - 1) / kKd4MergeThreads);
    QE_REQUIRE(blocks <= INT32_MAX && weight_blocks + num_q_heads <= INT32_MAX, "%s: too many heads", what);
    const unsigned grid = static_cast<unsigned>(blocks), threads = 64 * p.waves;
    const size_t lds = static_cast<size_t>(p.waves) * std::min(16, p.group) * (kKv4Dim + 4) * sizeof(float);
    if (key_weights_out != nullptr) {
        if (p.waves == 4) kv4_decode_kernel<true, 4><<<grid, threads, lds, stream>>>(p);
        else kv4_decode_kernel<true, kKd4ManyWaves><<<grid, threads, lds, stream>>>(p);
        kv4_decode_merge_kernel<true><<<static_cast<unsigned>(num_q_heads + weight_blocks), kKd4MergeThreads, 0, stream>>>(p);
    } else {
        if (p.waves == 4) kv4_decode_kernel<false, 4><<<grid, threads, lds, stream>>>(p);
        else kv4_decode_kernel<false, kKd4ManyWaves><<<grid, threads, lds, stream>>>(p);
        kv4_decode_merge_kernel<false><<<static_cast<unsigned>(num_q_heads), kKd4MergeThreads, 0, stream>>>(p);
    }
    return check_launch(what);
}

extern "C" int qe_launch_attention_gqa_prefill_kv4(const uint16_t* q, const uint8_t* layer_k_cache,
                                                   const uint8_t* layer_v_cache, uint16_t* attn_out,
                                                   const qe_device_control_block* d_control, const int32_t* d_evicted,
                                                   int num_tokens, hipStream_t stream, int num_q_heads,
                                                   int num_kv_heads, int head_dim, int max_seq_len, int hidden_size,
                                                   const float* key_weights_in, float* key_weights_out,
                                                   float* row_lse) {
    const char* what = "attention_gqa_prefill_kv4";
    QE_REQUIRE(q && attn_out, "%s: NULL pointer", what);
    QE_TRY(kv4_check(what, layer_k_cache, layer_v_cache, num_kv_heads, head_dim, max_seq_len));
    QE_TRY(check_heads(what, num_q_heads, num_kv_heads));
    QE_REQUIRE(hidden_size >= static_cast<long long>(num_q_heads) * head_dim && hidden_size % 4 == 0, "%s: hidden_size=%d", what,
               hidden_size);
    QE_TRY(check_weights(what, key_weights_in, key_weights_out, num_kv_heads, max_seq_len));
    QE_REQUIRE(key_weights_out == nullptr || row_lse != nullptr, "%s: key weights need row_lse", what);
    QE_REQUIRE(aligned(q, 16) && aligned(attn_out, 8), "%s: q must be 16-byte and attn_out 8-byte aligned", what);
    if (num_tokens <= 0) return QE_OK;
    // a block writes its rows while others read theirs, and the weights' kernel reads q after that
    const size_t q_row = static_cast<size_t>(num_q_heads) * kKv4Dim * 2;
    QE_REQUIRE((key_weights_out == nullptr && q == attn_out && (hidden_size == num_q_heads * kKv4Dim || num_tokens == 1)) ||
                   apart(q, num_tokens * q_row, attn_out, (num_tokens - 1) * static_cast<size_t>(hidden_size) * 2 + q_row),
               "%s: attn_out overlaps q", what);
    Prefill4Params p{};
    p.q = q;
    p.kc = layer_k_cache;
    p.vc = layer_v_cache;
    p.out = attn_out;
    p.ctl = d_control;
    p.evicted = d_evicted;
    p.lse = row_lse;
    p.w_in = key_weights_in;
    p.w_out = key_weights_out;
    p.T = num_tokens;
    p.nq = num_q_heads;
    p.nkv = num_kv_heads;
    p.group = num_q_heads / num_kv_heads;
    p.max_seq = max_seq_len;
    p.out_stride = hidden_size;
    const long long rows = static_cast<long long>(num_tokens) * p.group;
    QE_REQUIRE(rows <= (1 << 29) && max_seq_len <= (1 << 29), "%s: num_tokens=%d max_seq_len=%d", what, num_tokens,
               max_seq_len);
    // the weights' kernel counts a tile of q rows in 32 bits of bytes
    QE_REQUIRE(key_weights_out == nullptr ||
                   static_cast<long long>(kW4Rows / p.group) * num_q_heads * kKv4Dim * 2 <= (1LL << 32),
               "%s: num_q_heads=%d with key weights", what, num_q_heads);
    // Eight waves and one block per CU expand a tile for 256 rows; four waves for
    // 128, two blocks per CU, where there are few row blocks: their splits are shorter and
    // fewer rows idle.  (12 q heads, 2 kv heads, all in us: 40 tokens at 1200 13.1 against
    // 11.1, 509 at 0 17.4 against 14.0; 600 at 1000 25.7 against 27.0, 1000 at 2900 41.5
    // against 45.1, 1024 at 15000 117 against 129.)
    const int waves = (rows + 255) / 256 * num_kv_heads >= 28 ? 8 : 4;
    p.block_rows = 32 * waves;
    p.row_blocks = static_cast<int>((rows + p.block_rows - 1) / p.block_rows);
    const long long blocks = static_cast<long long>(p.row_blocks) * num_kv_heads;
    // Key splits as far as the chip has room for their blocks, the stream's
    // workspace for their partials, and the cache has tiles.
    const int cus = cu_count();
    const WorkspaceLease lease(stream);  // until every kernel is enqueued
    const StreamWorkspace ws = lease.ws;
    const long long part_rows = (rows + 31) / 32 * 32 * num_kv_heads;  // outputs of one split, whole waves
    const long long part = part_rows * kKv4Dim + rows * num_kv_heads * 2;  // floats of one split
    // (few rows: a block for every CU; twice as many cost more in the merge, us in all: 60
    // tokens at 8000 24.0 against 21.2, at 30000 35.0 against 32.0, 17 at 1200 10.5 both)
    const bool few_rows = rows * num_kv_heads <= 2048;
    const long long slots = waves == 4 && !few_rows ? 2LL * cus : cus;
    p.far_tiles = few_rows ? kP4FarTilesMany : kP4FarTiles;
    p.splits = 1;
    if (ws.ptr != nullptr && max_seq_len >= 16 * kP4Keys)
        p.splits = static_cast<int>(std::max(1LL, std::min({static_cast<long long>(kP4MaxSplits), slots / blocks,
                                                            static_cast<long long>(ws.floats) / part,
                                                            static_cast<long long>(max_seq_len) / (kP4Keys * kP4MinTiles)})));
    // A graph may be replayed on any stream and after the workspace is gone: a recorded launch touches none.
    if (p.splits > 1 && capturing(stream)) p.splits = 1;
    QE_REQUIRE(blocks * p.splits <= INT32_MAX, "%s: num_tokens=%d", what, num_tokens);
    p.part_o = ws.ptr;
    p.part_ml = ws.ptr + p.splits * part_rows * kKv4Dim;
    const unsigned grid = static_cast<unsigned>(blocks * p.splits);
    if (waves == 4) kv4_prefill_kernel<4><<<grid, 256, 0, stream>>>(p);
    else kv4_prefill_kernel<8><<<grid, 512, 0, stream>>>(p);
    const unsigned merge_grid = static_cast<unsigned>((rows + 7) / 8 * num_kv_heads);
    if (p.splits > 8 && few_rows) kv4_prefill_merge_kernel<kP4MergeMany><<<merge_grid, 256 * kP4MergeMany, 0, stream>>>(p);
    else if (p.splits > 1) kv4_prefill_merge_kernel<1><<<merge_grid, 256, 0, stream>>>(p);
    if (key_weights_out != nullptr) {
        // The q rows are shared by several blocks where there are many, if their sums find
        // room in the workspace (the attention's partials there are merged by now).  (300
        // tokens at 2000 33.0 against 37.8 us in all with two or three; at 16000 in a cache
        // of 32768, where there are blocks enough, 84 against 78.)
        const long long sums = static_cast<long long>(num_kv_heads) * max_seq_len;
        const long long key_blocks = (static_cast<long long>(max_seq_len) + kW4Keys - 1) / kW4Keys * num_kv_heads;
        p.weight_splits = static_cast<int>(
            std::max(1LL, std::min<long long>(kW4MaxSplits, rows / (key_blocks > 2LL * cus ? 1024 : 512))));
        if (p.weight_splits > 1 && (ws.ptr == nullptr || static_cast<long long>(ws.floats) < sums * p.weight_splits || capturing(stream)))
            p.weight_splits = 1;
        p.part_w = ws.ptr;
        QE_REQUIRE(key_blocks * p.weight_splits <= INT32_MAX, "%s: max_seq_len=%d", what, max_seq_len);
        kv4_prefill_weights_kernel<<<static_cast<unsigned>(key_blocks * p.weight_splits), 512, 0, stream>>>(p);
        if (p.weight_splits > 1)
            kv4_prefill_weights_merge_kernel<<<static_cast<unsigned>((static_cast<long long>(max_seq_len) + 255) / 256 * num_kv_heads),
                                               256, 0, stream>>>(p);
    }
    return check_launch(what);
}
