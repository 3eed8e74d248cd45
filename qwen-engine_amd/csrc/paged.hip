// Paged key/value cache: rotary tables, append of the tokens of many sequences,
// the pages' bounds and the selection of blocks by them.
#include <algorithm>
#include <cmath>

#include "paged_common.hpp"

namespace qe {
namespace {

// sum over the 16 lanes of a DPP row, the same in all of them
__device__ __forceinline__ float row16_sum(float x) {
    auto add = [&](auto ctrl) __attribute__((always_inline)) {
        x += __builtin_bit_cast(float, qwen::dpp_i32<decltype(ctrl)::value>(__builtin_bit_cast(int, x)));
    };
    add(std::integral_constant<int, 0xB1>{});
    add(std::integral_constant<int, 0x4E>{});
    add(std::integral_constant<int, 0x141>{});
    add(std::integral_constant<int, 0x140>{});
    return x;
}

// ---- append ------------------------------------------------------------------
// x + bias; times weight / sqrt(mean(x^2) + eps) where the head has a norm; pairs
// turned by position * turns[i]: (x0 c - x1 s, x0 s + x1 c), c and s times the
// rotation's factor; one rounding to fp16.  q to q_out, k and v to the row of
// their position's page.
//
// Angles: position times turns in 64 bits, less the whole turns there, then sine
// and cosine of what is left in fp32.
//
// grid (rows, ceil((nq + nkv) / 16)), 256 threads: 16 lanes a head, 8 elements a
// lane (the lanes of a k head do its v too); the first wave finds the row's sequence and
// makes its sines and cosines, while what the others asked for comes in.  Partners of a rotation in
// halves are exchanged between lanes.  One row 3 us, of which the launch is 1.7.  6150 rows of 12 q and
// 2 kv heads (50 MB) 13.2 us, 3.8 TB/s, bound by instructions: 227 vector instructions a wave, issued 97 % of
// the time (14.5 us at 295, with IEEE square root and division and partners read and normed a second time).
struct AppendParams {
    PagedView c;
    uint16_t* kp;
    uint16_t* vp;
    const uint16_t* q;
    uint16_t* q_out;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t *qb, *kb, *vb, *qn, *kn;
    const double* turns;
    long long q_stride, kv_stride;
    int nq, rot, interleaved;
    float scale, eps;
};

__device__ __forceinline__ f16x8 eight(const uint16_t* p) { return *reinterpret_cast<const f16x8*>(p); }
__device__ __forceinline__ void widen(const f16x8& a, float (&o)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<float>(a[e]);
}
// x += b, x *= r * g: where there are some
__device__ __forceinline__ void add8(bool some, const f16x8& b, float (&x)[8]) {
    if (!some) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += static_cast<float>(b[e]);
}
__device__ __forceinline__ void scale8(bool some, const f16x8& g, float r, float (&x)[8]) {
    if (!some) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= r * static_cast<float>(g[e]);
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&x)[8]) {
    f16x8 a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = static_cast<_Float16>(x[e]);
    *reinterpret_cast<f16x8*>(p) = a;
}

__global__ __launch_bounds__(256) void qkv_norm_rope_paged_append_kernel(AppendParams p) {
    __shared__ float s_sin[kPgDim / 2], s_cos[kPgDim / 2];
    __shared__ int2 s_place;  // the row's sequence and position
    const int t = blockIdx.x, j = threadIdx.x & 15, d = 8 * j, half = p.rot / 2;
    const int head = blockIdx.y * 16 + (threadIdx.x >> 4);
    const bool there = head < p.nq + p.c.nkv;  // whole rows of 16 lanes
    const bool is_k = head >= p.nq;
    const int h = is_k ? head - p.nq : head;
    const uint16_t* bias = is_k ? p.kb : p.qb;
    const uint16_t* norm = is_k ? p.kn : p.qn;
    // all that a row's place in memory gives is asked for before its place in the batch is known
    f16x8 x8, v8, bx, bv, gx;
    if (there) {
        const uint16_t* src = (is_k ? p.k + t * p.kv_stride : p.q + t * p.q_stride) + h * kPgDim;
        x8 = eight(src + d);
        if (is_k) {
            v8 = eight(p.v + t * p.kv_stride + h * kPgDim + d);
            if (p.vb != nullptr) bv = eight(p.vb + h * kPgDim + d);
        }
        if (bias != nullptr) bx = eight(bias + h * kPgDim + d);
        if (norm != nullptr) gx = eight(norm + d);
    }
    if (threadIdx.x < 64) {  // one wave for all
        const double turns = static_cast<int>(threadIdx.x) < half ? p.turns[threadIdx.x] : 0.0;
        int found = paged_seq_of_row(p.c, t), at = 0;
        if (found >= 0) {
            const PagedSeq s = paged_seq(p.c, found);
            if (t < s.first || t >= s.first + s.n) found = -1;
            at = s.ctx + t - s.first;
        }
        if (found >= 0 && static_cast<int>(threadIdx.x) < half) {
            const double a = static_cast<double>(at) * turns;
            float sn, cs;
            sincospif(2.0f * static_cast<float>(a - rint(a)), &sn, &cs);
            s_sin[threadIdx.x] = sn * p.scale;
            s_cos[threadIdx.x] = cs * p.scale;
        }
        if (threadIdx.x == 0) s_place = make_int2(found, at);
    }
    __syncthreads();
    const int seq = __builtin_amdgcn_readfirstlane(s_place.x), pos = __builtin_amdgcn_readfirstlane(s_place.y);
    if (seq < 0) return;
    const int page = is_k && there ? paged_page(p.c, seq, pos >> p.c.shift) : -1;
    if (!there) return;
    float x[8];
    widen(x8, x);
    add8(bias != nullptr, bx, x);
    float r = 1.0f;
    if (norm != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
        r = __builtin_amdgcn_rsqf(row16_sum(ss) * (1.0f / kPgDim) + p.eps);  // off by 2^-23 at most
    }
    scale8(norm != nullptr, gx, r, x);
    if (d < p.rot) {
        float o[8];
        if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float sn = s_sin[(d + e) / 2], cs = s_cos[(d + e) / 2];
                o[e] = x[e] * cs - x[e + 1] * sn;
                o[e + 1] = x[e] * sn + x[e + 1] * cs;
            }
        } else {
            // the partner's lane is of the same head and turns too
            const bool low = d < half;
            const int pd = low ? d + half : d - half, from = (threadIdx.x & 48) | pd / 8;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __shfl(x[e], from);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = (low ? d : pd) + e;
                o[e] = low ? x[e] * s_cos[i] - y[e] * s_sin[i] : y[e] * s_sin[i] + x[e] * s_cos[i];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = o[e];
    }
    if (!is_k) {
        store8(p.q_out + (static_cast<size_t>(t) * p.nq + h) * kPgDim + d, x);
        return;
    }
    if (page < 0) return;
    float w[8];
    widen(v8, w);
    add8(p.vb != nullptr, bv, w);
    // an element that fp16 cannot hold poisons the token's K row in place of its V row
    bool fits = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) fits = fits && fabsf(w[e]) < 65520.0f;
    const uint64_t spoilt = __builtin_amdgcn_ballot_w64(!fits);
    if ((spoilt >> (threadIdx.x & 48) & 0xFFFF) != 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf(""), w[e] = 0.0f;
    }
    const size_t at = static_cast<size_t>(page) * p.c.page_stride +
                      ((static_cast<size_t>(h) << p.c.shift) + (pos & (p.c.page_size() - 1))) * kPgDim + d;
    store8(p.kp + at, x);
    store8(p.vp + at, w);
}

// ---- bounds of pages -----------------------------------------------------------
// For each page that a sequence's new tokens reach, and each kv head, over the page's rows in
// use: m = max |k|, high = ceil(127 max / m), low = floor(127 min / m) for each of the 128
// dims (bytes 0..127 and 128..255 of a row of bounds), m beside them.  127 x / m in fp32:
// 127 x is exact, and x and m have 11 bits, so a quotient that is no whole number is farther
// from one than its rounding: the bytes are those of exact arithmetic.  A page with an infinity or
// NaN has m = inf and bytes of 0.
//
// grid (rows, kv heads), 256 threads: a block works where its row is the first of its page or of its
// sequence; 16 lanes a row of keys, 16 rows at once, up to four rounds of them requested together.  Bound by
// latency: the row's sequence, its page, the keys, the meeting in LDS behind each other, 3.4 us for one row and 4.7 for 200.
__global__ __launch_bounds__(256) void paged_key_bounds_kernel(PagedView c, int8_t* bounds, float* step) {
    __shared__ __align__(16) uint16_t s_high[4][kPgDim], s_low[4][kPgDim];
    __shared__ uint32_t s_odd[4];
    const int t = blockIdx.x, h = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int seq = paged_seq_of_row(c, t);
    if (seq < 0) return;
    const PagedSeq s = paged_seq(c, seq);
    if (t < s.first || t >= s.first + s.n) return;
    const int pos = s.ctx + t - s.first;
    if (t != s.first && (pos & (c.page_size() - 1)) != 0) return;
    const int block = pos >> c.shift, page = paged_page(c, seq, block);
    if (page < 0) return;
    // rows of the page in use once all new tokens are there (ctx + n is below 2^31)
    const int live = min(c.page_size(), s.ctx + s.n - (block << c.shift));
    const int j = lane & 15, row0 = threadIdx.x >> 4;
    const uint16_t* k = c.k + static_cast<long long>(page) * c.page_stride + (static_cast<long long>(h) << c.shift) * kPgDim + 8 * j;
    f16x8 high, low;
    uint32_t odd = 0;  // exponent of all ones somewhere
#pragma unroll
    for (int e = 0; e < 8; ++e) high[e] = static_cast<_Float16>(-65504.0f), low[e] = static_cast<_Float16>(65504.0f);
    for (int r0 = 0; r0 < live; r0 += 64) {
        u32x4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)  // (a row behind the last: the last again)
            w[i] = *reinterpret_cast<const u32x4*>(k + static_cast<size_t>(min(r0 + 16 * i + row0, live - 1)) * kPgDim);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x8 x = __builtin_bit_cast(f16x8, w[i]);
            high = __builtin_elementwise_max(high, x);
            low = __builtin_elementwise_min(low, x);
#pragma unroll
            for (int d = 0; d < 4; ++d)
                odd |= static_cast<uint32_t>((w[i][d] & 0x7C00u) == 0x7C00u || (w[i][d] & 0x7C000000u) == 0x7C000000u);
        }
    }
    // over the four rows of the wave, then over the waves
#pragma unroll
    for (int d = 16; d < 64; d *= 2) {
        u32x4 a = __builtin_bit_cast(u32x4, high), b = __builtin_bit_cast(u32x4, low);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = __shfl_xor(a[i], d);
            b[i] = __shfl_xor(b[i], d);
        }
        high = __builtin_elementwise_max(high, __builtin_bit_cast(f16x8, a));
        low = __builtin_elementwise_min(low, __builtin_bit_cast(f16x8, b));
    }
    const bool spoilt_here = __builtin_amdgcn_ballot_w64(odd != 0) != 0;
    if (lane < 16) {
        *reinterpret_cast<f16x8*>(&s_high[wave][8 * j]) = high;
        *reinterpret_cast<f16x8*>(&s_low[wave][8 * j]) = low;
        if (lane == 0) s_odd[wave] = spoilt_here;
    }
    __syncthreads();
    if (threadIdx.x >= 16) return;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        high = __builtin_elementwise_max(high, *reinterpret_cast<const f16x8*>(&s_high[w][8 * j]));
        low = __builtin_elementwise_min(low, *reinterpret_cast<const f16x8*>(&s_low[w][8 * j]));
    }
    const bool spoilt = (s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3]) != 0;
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fmaxf(fabsf(static_cast<float>(high[e])), fabsf(static_cast<float>(low[e]))));
    m = qwen::seg_max_nonneg<16>(m);
    const float div = m > 0.0f ? m : 1.0f;
    uint32_t bytes[4] = {0, 0, 0, 0};
    if (!spoilt) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int a = static_cast<int>(ceilf(127.0f * static_cast<float>(high[e]) / div));
            const int b = static_cast<int>(floorf(127.0f * static_cast<float>(low[e]) / div));
            bytes[e >> 2] |= static_cast<uint32_t>(a & 0xFF) << (8 * (e & 3));
            bytes[2 + (e >> 2)] |= static_cast<uint32_t>(b & 0xFF) << (8 * (e & 3));
        }
    }
    const size_t at = static_cast<size_t>(page) * c.nkv + h;
    *reinterpret_cast<uint2*>(bounds + at * 2 * kPgDim + 8 * j) = make_uint2(bytes[0], bytes[1]);
    *reinterpret_cast<uint2*>(bounds + at * 2 * kPgDim + kPgDim + 8 * j) = make_uint2(bytes[2], bytes[3]);
    if (j == 0) step[at] = spoilt ? INFINITY : m;
}

// ---- selection of blocks ---------------------------------------------------------
// score(row, kv head, block) = m_b * max over the q heads h of m_h * sum_d max(n_d high_d, n_d low_d),
// n = rint(127 q / m_h), m_h = max |q| (a head with an infinity or NaN counts as zeros): the
// largest value that a key within the block's bounds can give any of the heads.  The sums are
// whole numbers below 2^21, then there are two products rounded to fp32 each: every program that
// follows the definition orders the blocks alike.  max(n high, n low) is n high for n > 0, else n
// low: a product over 256 bytes with the positive and the negative parts of n, on
// v_mfma_i32_16x16x64_i8 with 16 blocks as rows and 16 (q row, head) as columns.
struct SelectParams {
    PagedView c;
    const uint16_t* q;
    const int8_t* bounds;
    const float* step;
    uint32_t* keys;  // [row][kv head][max_pages]: scores as whole numbers of the same order
    int32_t* selected;
    int nq, group, rows_per_tile, rows_per_run, chunks, num_selected, sinks, recent;
};
constexpr uint32_t kForced = 0xFFFFFFFFu, kSpoilt = 0xFFFFFFFEu;  // above every score
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// grid (runs of rows * chunks of 64 blocks, kv heads), 256 threads: a wave 16 blocks, whose bounds stay in
// registers for the rows of the run that are of one sequence.  Rows are taken as many at a time as 16
// columns hold; more than 16 q heads take several runs of columns.  The block quantizes q once, 16
// threads a column (every wave for itself, and the bounds read again for every 16 columns, 200 rows on
// 1563 blocks took 39 us; so it is 17.3: vector instructions 72 % of the time, of which the divisions of q take
// 2.5 us; one row on 2047 blocks 4.5).
__global__ __launch_bounds__(256) void paged_score_kernel(SelectParams p) {
    __shared__ float s_t[4][16][17];
    __shared__ __align__(16) int8_t s_q[16][2 * kPgDim + 16];  // positive and negative parts of each column (and 16 bytes, for the banks)
    __shared__ float s_m[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int run = blockIdx.x / p.chunks, chunk = blockIdx.x - run * p.chunks, h = blockIdx.y;
    const int r_end = min((run + 1) * p.rows_per_run, p.c.rows);
    const int b = (chunk * 4 + wave) * 16 + c, cols = min(p.group, 16);  // the lane's block
    int loaded = -1, page = -1;  // the sequence whose bounds are in a
    i32x4 a[4];
    float m_b = 0.0f;
    for (int r = run * p.rows_per_run; r < r_end;) {
        const int seq = paged_seq_of_row(p.c, r);
        if (seq < 0) {
            ++r;
            continue;
        }
        const PagedSeq s = paged_seq(p.c, seq);
        if (r < s.first || r >= s.first + s.n) {
            ++r;
            continue;
        }
        for (const int seq_end = min(r_end, s.first + s.n); r < seq_end;) {
            const int n = min(p.rows_per_tile, seq_end - r), pos = s.ctx + r - s.first;
            const int b_end = min(((pos + n - 1) >> p.c.shift) + 1, p.c.max_pages);
            if (chunk * 64 < b_end) {  // (the same for the whole block)
                if (seq != loaded) page = paged_page(p.c, seq, b);
                // lane (c, g) of the result: block c, rows g, g + 4, ... of the tile
                float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                for (int hb = 0; hb < p.group; hb += 16) {
                    {
                        const int col = threadIdx.x >> 4, j = threadIdx.x & 15;
                        const int col_row = min(col / cols, n - 1), col_head = min(hb + col % cols, p.group - 1);
                        const f16x8 x = *reinterpret_cast<const f16x8*>(
                            p.q + (static_cast<size_t>(r + col_row) * p.nq + h * p.group + col_head) * kPgDim + 8 * j);
                        if (seq != loaded) {  // asked for behind q
                            loaded = seq;
                            const size_t at = static_cast<size_t>(max(page, 0)) * p.c.nkv + h;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                a[kk] = *reinterpret_cast<const i32x4*>(p.bounds + at * 2 * kPgDim + 64 * kk + 16 * g);
                            m_b = p.step[at];
                        }
                        float m = 0.0f;
                        bool odd = false;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float v = fabsf(static_cast<float>(x[e]));
                            odd = odd || !(v < INFINITY);
                            m = fmaxf(m, v);
                        }
                        m = qwen::seg_max_nonneg<16>(odd ? INFINITY : m);
                        const bool none = !(m > 0.0f && m < INFINITY);
                        uint32_t up[2] = {0, 0}, down[2] = {0, 0};
                        if (!none) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const int y = static_cast<int>(rintf(127.0f * static_cast<float>(x[e]) / m));
                                up[e >> 2] |= static_cast<uint32_t>(max(y, 0)) << (8 * (e & 3));
                                down[e >> 2] |= static_cast<uint32_t>(min(y, 0) & 0xFF) << (8 * (e & 3));
                            }
                        }
                        __syncthreads();  // the last columns are read
                        *reinterpret_cast<uint2*>(&s_q[col][8 * j]) = make_uint2(up[0], up[1]);
                        *reinterpret_cast<uint2*>(&s_q[col][kPgDim + 8 * j]) = make_uint2(down[0], down[1]);
                        if (j == 0) s_m[col] = none ? 0.0f : m;
                        __syncthreads();
                    }
                    const float m_h = s_m[c];
                    i32x4 dot = {0, 0, 0, 0};
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[kk], *reinterpret_cast<const i32x4*>(&s_q[c][64 * kk + 16 * g]),
                                                                    dot, 0, 0, 0);
                    __builtin_amdgcn_wave_barrier();  // the last columns' values are read
#pragma unroll
                    for (int k = 0; k < 4; ++k) s_t[wave][4 * g + k][c] = static_cast<float>(dot[k]) * m_h;
                    __builtin_amdgcn_wave_barrier();
                    const int heads = min(cols, p.group - hb);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int row = g + 4 * k;
                        if (row >= n) break;
                        for (int e = 0; e < heads; ++e) best[k] = fmaxf(best[k], s_t[wave][c][row * cols + e]);
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = g + 4 * k, own = (pos + row) >> p.c.shift;
                    if (row >= n || b > own || b >= p.c.max_pages) continue;
                    const uint32_t u = __builtin_bit_cast(uint32_t, best[k] * m_b + 0.0f);  // (no -0)
                    uint32_t key = u >> 31 ? ~u : u | 0x80000000u;
                    if (m_b == INFINITY) key = kSpoilt;
                    if (b < p.sinks || b > own - p.recent) key = kForced;
                    if (page < 0) key = 0;
                    p.keys[(static_cast<size_t>(r + row) * p.c.nkv + h) * p.c.max_pages + b] = key;
                }
            }
            r += n;
        }
    }
}

// Sum over the threads of a block up to and without each; `all` gets the sum.  Two barriers.
template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int& all, int* s_part) {
    const int wave = threadIdx.x >> 6, y = wave_scan(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s_part[wave] = y;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        before += w < wave ? s_part[w] : 0;
        all += s_part[w];
    }
    return before + y - x;
}

// Which row and kv head a block of the selection has, and how many blocks it chooses from; false: none.
__device__ __forceinline__ bool select_range(const SelectParams& p, int& n) {
    const int row = blockIdx.x / p.c.nkv;
    const int seq = paged_seq_of_row(p.c, row);
    if (seq < 0) return false;
    const PagedSeq s = paged_seq(p.c, seq);
    if (row < s.first || row >= s.first + s.n) return false;
    n = min(((s.ctx + row - s.first) >> p.c.shift) + 1, p.c.max_pages);
    return true;
}

// The num_selected largest keys of a (row, kv head), equal ones the lower block first, as ascending
// blocks and -1 behind.  A block each, KEYS keys a thread in registers: the last key that is in is
// found by two bits at once, from the highest in which the scores differ, until as many keys as wanted
// are left above: three counts by ballots, and one barrier, each time.  (A count of digits in LDS, as
// below, took 12.8 us for the 2048 keys of 131000 positions: scores have few different first digits,
// so the lanes met at the same counters.  So it is 8.0, the 400 lists of 1563 keys 10.)
template <int THREADS, int KEYS>
__global__ __launch_bounds__(THREADS) void paged_select_kernel(SelectParams p) {
    constexpr int kWaves = THREADS / 64;
    __shared__ int s_part[kWaves];
    __shared__ int4 s_count[2][kWaves];
    __shared__ uint2 s_bits[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int n;
    if (!select_range(p, n)) return;
    const uint32_t* keys = p.keys + static_cast<size_t>(blockIdx.x) * p.c.max_pages;
    int32_t* out = p.selected + static_cast<size_t>(blockIdx.x) * p.num_selected;
    // each thread a stretch of blocks, so that they come out in order
    const int per = (n + THREADS - 1) / THREADS, i0 = tid * per;
    uint32_t k[KEYS];
#pragma unroll
    for (int j = 0; j < KEYS; ++j) k[j] = j < per && i0 + j < n ? keys[i0 + j] : 0u;
    int turn = 0;
    // keys of at least a, b and c each; one barrier
    auto count = [&](uint32_t a, uint32_t b, uint32_t c) __attribute__((always_inline)) {
        int3 mine = make_int3(0, 0, 0);
#pragma unroll
        for (int j = 0; j < KEYS; ++j)
            if (j < per) {
                mine.x += __popcll(__builtin_amdgcn_ballot_w64(k[j] >= a));
                mine.y += __popcll(__builtin_amdgcn_ballot_w64(k[j] >= b));
                mine.z += __popcll(__builtin_amdgcn_ballot_w64(k[j] >= c));
            }
        if (lane == 0) s_count[turn][wave] = make_int4(mine.x, mine.y, mine.z, 0);
        __syncthreads();
        int3 all = make_int3(0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int4 x = s_count[turn][w];
            all.x += x.x;
            all.y += x.y;
            all.z += x.z;
        }
        turn ^= 1;
        return all;
    };
    // bits that are set in some score and in every one
    uint32_t some = 0, every = ~0u;
#pragma unroll
    for (int j = 0; j < KEYS; ++j)
        if (k[j] != 0 && k[j] < kSpoilt) some |= k[j], every &= k[j];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) some |= __shfl_xor(some, d), every &= __shfl_xor(every, d);
    if (lane == 0) s_bits[wave] = make_uint2(some, every);
    const int3 kinds = count(1u, kSpoilt, kForced);  // (its barrier is that of s_bits too)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) some |= s_bits[w].x, every &= s_bits[w].y;
    const int there = kinds.x, need = min(p.num_selected, there);
    uint32_t limit = 1;     // keys of at least this are in, but of those equal to it
    int equal = INT32_MAX;  // only so many
    if (need < there) {
        if (need <= kinds.z) {
            limit = kForced;
            equal = need;
        } else if (need <= kinds.y) {
            limit = kSpoilt;
            equal = need - kinds.z;
        } else {
            const uint32_t differ = some & ~every;
            int bit = differ == 0 ? -2 : (31 - __clz(differ)) & ~1;  // the lower of the two looked at
            limit = bit < 0 ? every : every & ~((4u << bit) - 1u);   // what all scores begin with
            bool exact = false;
            for (; bit >= 0 && !exact; bit -= 2) {
                const uint32_t one = 1u << bit;
                const int3 c = count(limit + one, limit + 2 * one, limit + 3 * one);
                const int got = c.z >= need ? c.z : c.y >= need ? c.y : c.x >= need ? c.x : 0;
                limit += c.z >= need ? 3 * one : c.y >= need ? 2 * one : c.x >= need ? one : 0;
                exact = got == need;
            }
            if (!exact) equal = need - count(limit + 1, ~0u, ~0u).x;
        }
    }
    int above = 0, same = 0;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
        above += k[j] > limit;
        same += k[j] == limit;
    }
    int all;
    const int both = block_scan<THREADS>(above << 16 | same, all, s_part);  // (neither passes 2^15)
    int same_before = both & 0xFFFF;
    int at = (both >> 16) + min(same_before, equal);
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
        if (k[j] > limit || (k[j] == limit && same_before < equal)) out[at++] = i0 + j;
        same_before += k[j] == limit;
    }
    for (int i = need + tid; i < p.num_selected; i += THREADS) out[i] = -1;
}

// The same for longer lists: digit by digit (8 bits, counts in LDS), the keys read again for each.
__global__ __launch_bounds__(1024) void paged_select_long_kernel(SelectParams p) {
    constexpr int kThreads = 1024;
    __shared__ int s_count[256], s_part[kThreads / 64], s_found[2];
    const int tid = threadIdx.x;
    int n;
    if (!select_range(p, n)) return;
    const uint32_t* keys = p.keys + static_cast<size_t>(blockIdx.x) * p.c.max_pages;
    int32_t* out = p.selected + static_cast<size_t>(blockIdx.x) * p.num_selected;
    int mine = 0;
    for (int i = tid; i < n; i += kThreads) mine += keys[i] != 0;
    int there;
    block_scan<kThreads>(mine, there, s_part);
    const int need = min(p.num_selected, there);
    uint32_t limit = 1;  // keys above it are in, and the first `equal` of those equal to it
    int equal = INT32_MAX;
    if (need < there) {
        equal = need;
        limit = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s_count[tid] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t k = keys[i];
                if ((k & mask) == limit) atomicAdd(&s_count[(k >> shift) & 255], 1);
            }
            __syncthreads();
            const int digit = 255 - tid, here = tid < 256 ? s_count[digit & 255] : 0;  // from the largest down
            int all;
            const int above = block_scan<kThreads>(here, all, s_part);
            if (tid < 256 && above < equal && equal <= above + here) s_found[0] = digit, s_found[1] = above;
            __syncthreads();
            limit |= static_cast<uint32_t>(s_found[0]) << shift;
            equal -= s_found[1];
        }
    }
    const int per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    int above = 0, same = 0;
    for (int i = i0; i < i1; ++i) {
        above += keys[i] > limit;
        same += keys[i] == limit;
    }
    int all;
    const int above_before = block_scan<kThreads>(above, all, s_part);
    int same_before = block_scan<kThreads>(same, all, s_part);
    int at = above_before + min(same_before, equal);
    for (int i = i0; i < i1; ++i) {
        const uint32_t k = keys[i];
        if (k > limit || (k == limit && same_before < equal)) out[at++] = i;
        same_before += k == limit;
    }
    for (int i = need + tid; i < p.num_selected; i += kThreads) out[i] = -1;
}

}  // namespace
}  // namespace qe

using namespace qe;

extern "C" int qe_rope_turns(double* turns, float* scale, int rotary_dim, double theta, int kind, double factor,
                             double original_positions, double low_turns, double high_turns) {
    QE_REQUIRE(turns && scale, "rope_turns: NULL pointer");
    QE_REQUIRE(rotary_dim > 0 && rotary_dim <= kPgDim && rotary_dim % 16 == 0,
               "rope_turns: rotary_dim=%d (a multiple of 16 up to 128)", rotary_dim);
    QE_REQUIRE(theta > 1.0 && std::isfinite(theta), "rope_turns: theta=%g", theta);
    QE_REQUIRE(kind >= QE_ROPE_PLAIN && kind <= QE_ROPE_BANDS, "rope_turns: kind=%d", kind);
    if (kind != QE_ROPE_PLAIN) QE_REQUIRE(factor >= 1.0 && std::isfinite(factor), "rope_turns: factor=%g", factor);
    if (kind >= QE_ROPE_RAMP) {
        QE_REQUIRE(original_positions > 0.0 && std::isfinite(original_positions), "rope_turns: original_positions=%g",
                   original_positions);
        QE_REQUIRE(low_turns > 0.0 && high_turns > low_turns && std::isfinite(high_turns),
                   "rope_turns: low_turns=%g high_turns=%g", low_turns, high_turns);
    }
    constexpr double kTwoPi = 6.283185307179586476925286766559;
    // the pair, as a real number, that turns n times within the trained length
    auto pair_of = [&](double n) { return rotary_dim * std::log(original_positions / (n * kTwoPi)) / (2.0 * std::log(theta)); };
    double first = 0.0, last = 0.0;
    if (kind == QE_ROPE_RAMP) {
        first = std::max(std::floor(pair_of(high_turns)), 0.0);
        last = std::min(std::ceil(pair_of(low_turns)), rotary_dim - 1.0);
    }
    for (int i = 0; i < rotary_dim / 2; ++i) {
        const double f = std::pow(theta, -2.0 * i / rotary_dim) / kTwoPi;
        double r = 0.0;  // share of the slowed frequency
        if (kind == QE_ROPE_LINEAR) r = 1.0;
        if (kind == QE_ROPE_RAMP) r = (i - first) / std::max(last - first, 0.001);
        if (kind == QE_ROPE_BANDS) r = (high_turns - original_positions * f) / (high_turns - low_turns);
        r = std::min(std::max(r, 0.0), 1.0);
        turns[i] = kind == QE_ROPE_PLAIN ? f : (1.0 - r) * f + r * (f / factor);
    }
    *scale = kind == QE_ROPE_RAMP ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
    clear_error();
    return QE_OK;
}

extern "C" int qe_launch_qkv_norm_rope_paged_append(const uint16_t* q, uint16_t* q_out, const uint16_t* k,
                                                    const uint16_t* v, const uint16_t* q_bias, const uint16_t* k_bias,
                                                    const uint16_t* v_bias, const uint16_t* q_norm,
                                                    const uint16_t* k_norm, const qe_rope* rope,
                                                    const qe_paged_cache* cache, const qe_paged_batch* batch,
                                                    hipStream_t stream, int num_q_heads, long long q_stride,
                                                    long long kv_stride, float norm_eps) {
    const char* what = "qkv_norm_rope_paged_append";
    AppendParams p{};
    QE_TRY(paged_check(what, cache, batch, &p.c));
    QE_TRY(paged_check_heads(what, cache, num_q_heads));
    const long long q_row = static_cast<long long>(num_q_heads) * kPgDim;
    const long long kv_row = static_cast<long long>(cache->num_kv_heads) * kPgDim;
    if (q_stride == 0) q_stride = q_row;
    if (kv_stride == 0) kv_stride = kv_row;
    QE_REQUIRE(q_stride >= q_row && q_stride % 8 == 0 && q_stride <= (1LL << 32), "%s: q_stride=%lld", what, q_stride);
    QE_REQUIRE(kv_stride >= kv_row && kv_stride % 8 == 0 && kv_stride <= (1LL << 32), "%s: kv_stride=%lld", what, kv_stride);
    if (rope != nullptr) {
        QE_REQUIRE(rope->turns != nullptr && aligned(rope->turns, 8), "%s: the rotation's turns", what);
        QE_REQUIRE(rope->rotary_dim > 0 && rope->rotary_dim <= kPgDim && rope->rotary_dim % 16 == 0,
                   "%s: rotary_dim=%d (a multiple of 16 up to 128)", what, rope->rotary_dim);
        QE_REQUIRE(std::isfinite(rope->scale), "%s: rotation scale", what);
    }
    QE_REQUIRE(norm_eps >= 0.0f && std::isfinite(norm_eps), "%s: norm_eps=%g", what, norm_eps);
    if (batch->num_tokens == 0 || batch->num_seqs == 0) return QE_OK;
    QE_REQUIRE(q && q_out && k && v, "%s: NULL pointer", what);
    for (const uint16_t* a : {q, static_cast<const uint16_t*>(q_out), k, v, q_bias, k_bias, v_bias, q_norm, k_norm})
        QE_REQUIRE(aligned(a, 16), "%s: the buffers must be 16-byte aligned", what);
    QE_REQUIRE(q_out != q || q_stride == q_row, "%s: q_out over q with q_stride=%lld", what, q_stride);
    const size_t n = batch->num_tokens;
    const int in_place = q_out == q ? 2 : 0;
    const PagedSpan spans[] = {{q_out, 2 * n * q_row, "q_out", in_place},
                               paged_k_span(cache),
                               paged_v_span(cache),
                               {q, 2 * ((n - 1) * q_stride + q_row), "q", in_place},
                               {k, 2 * ((n - 1) * kv_stride + kv_row), "k"},
                               {v, 2 * ((n - 1) * kv_stride + kv_row), "v"},
                               {q_bias, 2 * static_cast<size_t>(q_row), "q_bias"},
                               {k_bias, 2 * static_cast<size_t>(kv_row), "k_bias"},
                               {v_bias, 2 * static_cast<size_t>(kv_row), "v_bias"},
                               {q_norm, 2 * kPgDim, "q_norm"},
                               {k_norm, 2 * kPgDim, "k_norm"},
                               {rope != nullptr ? rope->turns : nullptr, rope != nullptr ? 4 * static_cast<size_t>(rope->rotary_dim) : 0,
                                "the rotation's turns"},
                               paged_table_span(batch),
                               paged_starts_span(batch),
                               paged_context_span(batch)};
    QE_TRY(paged_check_pools(what, cache));
    QE_TRY(paged_check_apart(what, spans, 3));
    p.kp = cache->k;
    p.vp = cache->v;
    p.q = q;
    p.q_out = q_out;
    p.k = k;
    p.v = v;
    p.qb = q_bias;
    p.kb = k_bias;
    p.vb = v_bias;
    p.qn = q_norm;
    p.kn = k_norm;
    p.q_stride = q_stride;
    p.kv_stride = kv_stride;
    p.nq = num_q_heads;
    if (rope != nullptr) {
        p.turns = rope->turns;
        p.rot = rope->rotary_dim;
        p.interleaved = rope->interleaved != 0;
        p.scale = rope->scale;
    }
    p.eps = norm_eps;
    const dim3 grid(batch->num_tokens, (num_q_heads + cache->num_kv_heads + 15) / 16);
    qkv_norm_rope_paged_append_kernel<<<grid, 256, 0, stream>>>(p);
    return check_launch(what);
}

extern "C" int qe_launch_paged_key_bounds(const qe_paged_cache* cache, const qe_paged_batch* batch, int8_t* bounds,
                                          float* bound_steps, hipStream_t stream) {
    const char* what = "paged_key_bounds";
    PagedView c;
    QE_TRY(paged_check(what, cache, batch, &c));
    if (batch->num_tokens == 0 || batch->num_seqs == 0) return QE_OK;
    QE_REQUIRE(bounds && bound_steps, "%s: NULL pointer", what);
    QE_REQUIRE(aligned(bounds, 16) && aligned(bound_steps, 4), "%s: bounds must be 16-byte aligned", what);
    const size_t n = static_cast<size_t>(cache->num_pages) * cache->num_kv_heads;
    const PagedSpan spans[] = {{bounds, 2 * kPgDim * n, "bounds"}, {bound_steps, 4 * n, "bound_steps"}, paged_k_span(cache),
                               paged_v_span(cache), paged_table_span(batch), paged_starts_span(batch),
                               paged_context_span(batch)};
    QE_TRY(paged_check_apart(what, spans, 2));
    paged_key_bounds_kernel<<<dim3(batch->num_tokens, cache->num_kv_heads), 256, 0, stream>>>(c, bounds, bound_steps);
    return check_launch(what);
}

namespace {
// a key for each (row, kv head, block)
bool select_workspace(long long num_tokens, long long num_kv_heads, long long max_pages, size_t* bytes) {
    const long long lists = num_tokens * num_kv_heads;  // at most 2^34
    if (max_pages > 0 && lists > (1LL << 40) / max_pages) return false;
    *bytes = static_cast<size_t>(4 * lists * max_pages);
    return true;
}
}  // namespace

extern "C" int qe_paged_select_workspace_bytes(int num_tokens, int num_kv_heads, int max_pages, size_t* bytes) {
    QE_REQUIRE(bytes, "paged_select_workspace_bytes: NULL pointer");
    QE_REQUIRE(num_tokens >= 0 && num_tokens < (1 << 24) && num_kv_heads > 0 && num_kv_heads <= 1024 && max_pages > 0 &&
                   select_workspace(num_tokens, num_kv_heads, max_pages, bytes),
               "paged_select_workspace_bytes: num_tokens=%d num_kv_heads=%d max_pages=%d", num_tokens, num_kv_heads,
               max_pages);
    clear_error();
    return QE_OK;
}

extern "C" int qe_launch_paged_select(const uint16_t* q, const qe_paged_cache* cache, const qe_paged_batch* batch,
                                      const int8_t* bounds, const float* bound_steps, int32_t* selected, void* workspace,
                                      hipStream_t stream, int num_q_heads, int num_selected, int sinks, int recent) {
    const char* what = "paged_select";
    SelectParams p{};
    QE_TRY(paged_check(what, cache, batch, &p.c));
    QE_TRY(paged_check_heads(what, cache, num_q_heads));
    QE_REQUIRE(num_selected > 0 && num_selected <= (1 << 20), "%s: num_selected=%d", what, num_selected);
    QE_REQUIRE(sinks >= 0 && recent >= 0 && static_cast<long long>(sinks) + recent <= num_selected,
               "%s: %d first and %d last blocks do not fit num_selected=%d", what, sinks, recent, num_selected);
    if (batch->num_tokens == 0 || batch->num_seqs == 0) return QE_OK;
    QE_REQUIRE(q && bounds && bound_steps && selected && workspace, "%s: NULL pointer", what);
    QE_REQUIRE(aligned(q, 16) && aligned(bounds, 16) && aligned(bound_steps, 4) && aligned(selected, 4) && aligned(workspace, 4),
               "%s: q and bounds must be 16-byte aligned", what);
    const int nkv = cache->num_kv_heads;
    const long long n = batch->num_tokens;
    p.group = num_q_heads / nkv;
    p.rows_per_tile = batch->query_start == nullptr ? 1 : std::max(1, 16 / p.group);
    const long long tiles = (n + p.rows_per_tile - 1) / p.rows_per_tile;
    p.chunks = (batch->max_pages + 63) / 64;
    // several tiles a block where that leaves four blocks a CU
    const long long tiles_per_run = std::max(1LL, std::min(8LL, tiles * p.chunks * nkv / 1024));
    const long long runs = (tiles + tiles_per_run - 1) / tiles_per_run;
    p.rows_per_run = static_cast<int>(p.rows_per_tile * tiles_per_run);
    size_t bytes = 0;
    // (a launch has fewer than 2^32 threads)
    QE_REQUIRE(select_workspace(n, nkv, batch->max_pages, &bytes) && runs * p.chunks < (1 << 24) && n * nkv < (1 << 22),
               "%s: num_tokens=%d max_pages=%d", what, batch->num_tokens, batch->max_pages);
    const size_t pages = static_cast<size_t>(cache->num_pages) * nkv;
    const PagedSpan spans[] = {{selected, 4 * static_cast<size_t>(n) * nkv * num_selected, "selected"},
                               {workspace, bytes, "the workspace"},
                               {q, 2 * static_cast<size_t>(n) * num_q_heads * kPgDim, "q"},
                               {bounds, 2 * kPgDim * pages, "bounds"},
                               {bound_steps, 4 * pages, "bound_steps"},
                               paged_k_span(cache),
                               paged_v_span(cache),
                               paged_table_span(batch),
                               paged_starts_span(batch),
                               paged_context_span(batch)};
    QE_TRY(paged_check_apart(what, spans, 2));
    p.q = q;
    p.bounds = bounds;
    p.step = bound_steps;
    p.keys = static_cast<uint32_t*>(workspace);
    p.selected = selected;
    p.nq = num_q_heads;
    p.num_selected = num_selected;
    p.sinks = sinks;
    p.recent = recent;
    paged_score_kernel<<<dim3(static_cast<unsigned>(runs * p.chunks), nkv), 256, 0, stream>>>(p);
    const unsigned lists = static_cast<unsigned>(n * nkv);
    if (batch->max_pages <= 256 * 8)
        paged_select_kernel<256, 8><<<lists, 256, 0, stream>>>(p);
    else if (batch->max_pages <= 512 * 8)
        paged_select_kernel<512, 8><<<lists, 512, 0, stream>>>(p);
    else if (batch->max_pages <= 1024 * 16)
        paged_select_kernel<1024, 16><<<lists, 1024, 0, stream>>>(p);
    else
        paged_select_long_kernel<<<lists, 1024, 0, stream>>>(p);
    return check_launch(what);
}
