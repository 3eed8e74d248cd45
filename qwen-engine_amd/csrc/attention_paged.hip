// Attention over the paged key/value cache: single tokens, selected blocks, and
// chunks of many sequences.
#include <algorithm>
#include <type_traits>

#include "lds_dma.hpp"
#include "paged_common.hpp"

namespace qe {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kPgScale = 1.4426950408889634f * 0.08838834764831845f;  // log2(e) / sqrt(128)
constexpr float kPgLowest = -3.4e38f;  // the maximum of keys whose every score is -inf: a sum of 0, so NaN
// A row's reference value (what its scores are lowered by before the exponential) lies kPgRoom below
// its running maximum (in chunks rounded down to a whole number), and is renewed only when the maximum
// has grown by more than kPgLag.  So the largest weight is between 2^7 and 2^15, as high as fp16 goes: weights down to
// 2^-21 of it are normal numbers there and keep their relative precision, smaller ones are off by 2^-32 of it.
// (Beside weights of 1 those of 2^-16 had 8 bits left and those of 2^-25 none, which a key far above
// many others, as long texts have it, makes visible: 4 % of the others' sum at 2^-20.6.)
constexpr float kPgRoom = 7.0f, kPgLag = 8.0f;

// ---- shares of the work ------------------------------------------------------
// The lengths are on the device, so the division of the work is made there.  A
// segment is one row tile of one kv head of one sequence (or row): a list of key
// tiles, none of whose parts depend on another's.  All segments behind each other,
// each as long as its weight (about its number of key tiles), form a line, which is
// cut into equal shares, one for each block of the launch: every block has the same
// work whatever the lengths, and a segment that is cut leaves partial results (row
// maximum, sum and unnormalized outputs), which a second kernel merges.  A block has
// at most two cut segments: the one that its share begins in (slot 0) and the one
// that it ends in (slot 1).  Tile t of a segment of n tiles and weight w belongs to the
// place t * w / n of its stretch; the bits of a row depend on the lengths of the whole
// batch and on the launch's sizes, through where the cuts fall, and on nothing else.
//
// Where there are few segments for the blocks (at most one for four), every segment is
// given whole shares, so that no block has two: a second one costs as much again as a
// short share (17 rows on 1200 positions: 20 us of a launch instead of 13).
//
// Weights are whole numbers whose sum is below 2^30: the launcher says by how many
// bits they have to be shortened (kernels: `coarse`).
struct SegmentCut {  // of the block that has a segment's beginning but not its end
    int at, share, weight;            // where the segment begins; the length of a share
    int tiles, item, head, row_tile;
    int rows;  // of the segment; 0: there is no such segment
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Tiles of a segment that lie before place x of the line.  (In fp32: it rises with x, and everyone
// who asks gets the same.)
__device__ __forceinline__ int tiles_before(int x, int at, int weight, int tiles) {
    if (x <= at) return 0;
    if (x >= at + weight) return tiles;
    return min(tiles, static_cast<int>(static_cast<float>(x - at) * (static_cast<float>(tiles) / static_cast<float>(weight))));
}

// One sequence on the line: `heads` times row tiles whose weights are first + (i + 1 << step)
// (step < 0: first), but at most `most`.
struct SeqWork {
    int first, step, most;
    int row_tiles, heads;

    __device__ __forceinline__ int before(int i) const {  // weight of the first i row tiles
        if (step < 0) return i * min(first, most);
        const int m = min(i, max(0, most - first) >> step);
        return m * first + ((m * (m + 1) / 2) << step) + (i - m) * most;
    }
    __device__ __forceinline__ int weight(int i) const { return min(most, step < 0 ? first : first + ((i + 1) << step)); }
    __device__ __forceinline__ int segments() const { return heads * row_tiles; }
    // every row tile with the weight of the last, rounded up to whole shares
    __device__ __forceinline__ void fill_shares(int share) {
        first = most = (weight(row_tiles - 1) + share - 1) / share * share;
        step = -1;
    }
};

// 64 sequences of the batch, one a lane.
struct SeqChunk {
    int base, first, n, ctx;
    __device__ __forceinline__ void read(const PagedView& c, int at) {
        base = at;
        const int s = at + (threadIdx.x & 63);
        PagedSeq q{0, 0, 0};
        if (s < c.seqs) q = paged_seq(c, s);
        first = q.first;
        n = q.n;
        ctx = q.ctx;
    }
    __device__ __forceinline__ PagedSeq lane() const { return PagedSeq{first, n, ctx}; }
    __device__ __forceinline__ PagedSeq seq(const PagedView& c, int s) {  // s: the same in all lanes
        if (s < base || s >= base + 64) read(c, s);
        const int k = s - base;
        return PagedSeq{__builtin_amdgcn_readlane(first, k), __builtin_amdgcn_readlane(n, k), __builtin_amdgcn_readlane(ctx, k)};
    }
};

// Runs body(item, its sequence, head, row tile, first tile, end tile, slot) for each piece of a segment
// in this block's share, by all waves of the block alike; then cut(the cut that its last
// segment makes).  slot: -1 for a whole segment, else where its partials go.  work(sequence):
// the SeqWork of one of the batch's sequences; tiles(sequence, row tile): its key tiles; rows(sequence,
// head, row tile): its rows.
// LISTED: there is only one item, whose work is work({}).
template <bool LISTED, class Work, class Tiles, class Rows, class Body, class Cut>
__device__ __forceinline__ void for_share(const PagedView& c, int block, int blocks, int least_share, Work work,
                                          Tiles tiles, Rows rows, Body body, Cut cut) {
    // the whole line, then the sequence in which the share begins
    SeqChunk chunk{};
    const int seqs = LISTED ? 1 : c.seqs;
    int total = 0, segments = 0, level = 0, s = 0, at = 0, w = 0;  // level: were every row tile as heavy as its sequence's last
    auto sum = [&](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(wave_scan(x), 63); };
    if constexpr (LISTED) {
        const SeqWork q = work(PagedSeq{0, 1, 0});
        segments = q.segments();
        total = level = segments * q.first;
    } else {
        for (int s0 = 0; s0 < seqs; s0 += 64) {
            chunk.read(c, s0);
            const SeqWork q = work(chunk.lane());
            w = wave_scan(q.heads * q.before(q.row_tiles));
            total += __builtin_amdgcn_readlane(w, 63);
            segments += sum(q.segments());
            level += sum(q.row_tiles > 0 ? q.segments() * q.weight(q.row_tiles - 1) : 0);
        }
    }
    const bool few = segments <= blocks / 4;
    const int share = few ? max(least_share, (level + blocks - segments - 1) / (blocks - segments))
                          : max(least_share, (total + blocks - 1) / blocks);
    auto work_of = [&](const PagedSeq& q) __attribute__((always_inline)) {
        SeqWork x = work(q);
        if (few && x.row_tiles > 0) x.fill_shares(share);
        return x;
    };
    auto all_of = [&](const PagedSeq& q) __attribute__((always_inline)) {
        const SeqWork x = work_of(q);
        return x.row_tiles > 0 ? x.heads * x.before(x.row_tiles) : 0;
    };
    if (few) {
        total = 0;
        if constexpr (LISTED) {
            total = all_of(PagedSeq{0, 1, 0});
        } else {
            for (int s0 = 0; s0 < seqs; s0 += 64) {
                if (seqs > 64) chunk.read(c, s0);
                w = wave_scan(all_of(chunk.lane()));
                total += __builtin_amdgcn_readlane(w, 63);
            }
        }
    }
    const int x0 = min(total, share * block), x1 = min(total, x0 + share);
    SegmentCut last{};
    if (x0 >= x1) {
        cut(last);
        return;
    }
    if constexpr (!LISTED) {
        for (int s0 = 0; s0 < seqs; s0 += 64) {
            if (seqs > 64) {
                chunk.read(c, s0);
                w = wave_scan(all_of(chunk.lane()));
            }
            const int all = __builtin_amdgcn_readlane(w, 63);
            if (x0 < at + all) {
                const int k = __popcll(__builtin_amdgcn_ballot_w64(at + w <= x0));  // sequences before
                s = s0 + k;
                if (k > 0) at += __builtin_amdgcn_readlane(w, k - 1);
                break;
            }
            at += all;
        }
    }
    PagedSeq seq = LISTED ? PagedSeq{0, 1, 0} : chunk.seq(c, s);
    SeqWork q = work_of(seq);
    int head, rt;
    {
        const int one = q.before(q.row_tiles);
        head = static_cast<int>(static_cast<uint32_t>(x0 - at) / static_cast<uint32_t>(one));
        at += one * head;
        int lo = 0, hi = q.row_tiles;  // before(lo) <= x0 - at < before(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (q.before(mid) <= x0 - at) lo = mid; else hi = mid;
        }
        rt = lo;
        at += q.before(rt);
    }
    head = uniform(head);
    rt = uniform(rt);
    at = uniform(at);
    while (true) {
        const int weight = q.weight(rt);
        const int n = uniform(tiles(seq, rt));
        const int t0 = uniform(tiles_before(x0, at, weight, n)), t1 = uniform(tiles_before(x1, at, weight, n));
        const bool whole = t0 == 0 && t1 == n;
        if (whole ? n > 0 || x0 <= at : t0 < t1) body(s, seq, head, rt, t0, t1, whole ? -1 : t0 == 0 ? 1 : 0);
        if (t0 == 0 && t1 > 0 && t1 < n) last = SegmentCut{at, share, weight, n, s, head, rt, rows(seq, head, rt)};
        at += weight;
        if (at >= x1) break;
        if (++rt == q.row_tiles) {
            rt = 0;
            if (++head == q.heads) {
                head = 0;
                do {
                    if (++s >= seqs) return cut(last);  // (only where query_start decreases)
                    seq = chunk.seq(c, s);
                    q = work_of(seq);
                } while (q.row_tiles == 0);
            }
        }
    }
    cut(last);
}

// ---- partial results and their merge ------------------------------------------
// Workspace of a launch of `blocks` blocks and segments of ROWS rows: the cuts, then a
// (reference value, sum) for each block, slot and row, then 128 unnormalized outputs.
struct Partials {
    SegmentCut* cuts;
    float2* ml;
    float* o;
};
template <int ROWS>
__host__ __device__ __forceinline__ Partials partials(void* ws, int blocks) {
    char* at = static_cast<char*>(ws);
    Partials p;
    p.cuts = reinterpret_cast<SegmentCut*>(at);
    at += (sizeof(SegmentCut) * blocks + 255) / 256 * 256;
    p.ml = reinterpret_cast<float2*>(at);
    p.o = reinterpret_cast<float*>(at + sizeof(float2) * 2 * blocks * ROWS);
    return p;
}
template <int ROWS>
constexpr size_t partials_bytes(int blocks) {
    return (sizeof(SegmentCut) * blocks + 255) / 256 * 256 +
           static_cast<size_t>(2) * blocks * ROWS * (sizeof(float2) + kPgDim * sizeof(float));
}

// Where the rows of a segment are: row r of it is q row first + (r0 + r) / per_row (in the
// order of q rows and, within one, of the group's heads) and head head0 + (r0 + r) % per_row.
struct RowMap {
    int first, r0, per_row, head0;
    __device__ __forceinline__ int row(int r) const { return first + (r0 + r) / per_row; }
    __device__ __forceinline__ int head(int r) const { return head0 + (r0 + r) % per_row; }
};

// A merged row: o / sum, and the logarithm of the sum.  No key at all: zeros and -inf.
__device__ __forceinline__ float row_inverse(float m, float l) { return m == -INFINITY ? 0.0f : 1.0f / l; }
__device__ __forceinline__ float row_log_sum(float m, float l) {
    return m == -INFINITY ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}
// What a part with reference value m counts against the common one.
__device__ __forceinline__ float part_weight(float m, float common) {
    return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - common);
}
__device__ __forceinline__ float xor32_max(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float xor16_max(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
    return make_uint2(static_cast<uint32_t>(f2h(a)) | static_cast<uint32_t>(f2h(b)) << 16,
                      static_cast<uint32_t>(f2h(c)) | static_cast<uint32_t>(f2h(d)) << 16);
}

// Merges the parts of the segments that were cut.  An item is THREADS / 32 / GROUPS rows of one cut
// segment, GROUPS times 32 lanes a row (4 dims each): the groups take every GROUPS-th part, eight
// partial outputs requested at once.  Every block counts the cuts and takes its share of the items.
constexpr int kMergeCuts = 512;  // cuts of a launch, at most
template <int ROWS, int GROUPS, int THREADS, class Map>
__device__ __forceinline__ void merge_parts(void* ws, int blocks, uint16_t* out, float* lse, int nq, Map map) {
    constexpr int kRows = THREADS / 32 / GROUPS;  // rows of an item
    constexpr int kParts = GROUPS > 1 ? 512 : 32;  // weights kept at once
    constexpr int kWaves = THREADS / 64;
    __shared__ float s_w[kRows][kParts], s_l[kRows][kParts];
    __shared__ float s_red[THREADS / 32];
    __shared__ float4 s_o[GROUPS > 1 ? THREADS / 32 : 1][32];
    __shared__ int s_first[kMergeCuts + 1];  // the items before those of each cut
    __shared__ short s_cut[kMergeCuts];      // its block
    __shared__ int2 s_count[kWaves];
    __shared__ int s_found;
    const Partials p = partials<ROWS>(ws, blocks);
    const int tid = threadIdx.x, grp = tid >> 5, lane = tid & 31;
    // the blocks with a cut, in their order
    int cuts = 0, items = 0;
    for (int b0 = 0; b0 < blocks; b0 += THREADS) {
        const int b = b0 + tid;
        const int mine = b < blocks ? (p.cuts[b].rows + kRows - 1) / kRows : 0;
        const uint64_t live = __builtin_amdgcn_ballot_w64(mine != 0);
        const int upto = wave_scan(mine);
        if ((tid & 63) == 63) s_count[tid >> 6] = make_int2(__popcll(live), upto);
        __syncthreads();
        int at = cuts + __popcll(live & ((1ull << (tid & 63)) - 1)), first = items + upto - mine;
        for (int w = 0; w < kWaves; ++w) {
            at += w < (tid >> 6) ? s_count[w].x : 0;
            first += w < (tid >> 6) ? s_count[w].y : 0;
            cuts += s_count[w].x;
            items += s_count[w].y;
        }
        if (mine != 0) s_cut[at] = static_cast<short>(b), s_first[at] = first;
        __syncthreads();
    }
    if (tid == 0) s_first[cuts] = items;
    __syncthreads();
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        for (int k = tid; k < cuts; k += THREADS)
            if (s_first[k] <= item && item < s_first[k + 1]) s_found = k;
        __syncthreads();
        const int b = s_cut[s_found], r_first = (item - s_first[s_found]) * kRows;
        const SegmentCut c = p.cuts[b];
        const RowMap rows = map(c);
        const int live = c.rows;
        const int parts = (c.at + c.weight - 1) / c.share - b + 1;  // blocks that share the segment
        const int row_in = grp / GROUPS, part_in = grp % GROUPS, r = r_first + row_in;
        auto slot = [&](int i) { return static_cast<size_t>(2 * (b + i) + (i == 0 ? 1 : 0)) * ROWS; };
        auto holds = [&](int i) {  // block b + i has tiles of the segment
            const int x = (b + i) * c.share;
            return tiles_before(x, c.at, c.weight, c.tiles) < tiles_before(x + c.share, c.at, c.weight, c.tiles);
        };
        // the common reference value of each row
        constexpr int kPer = THREADS / kRows;  // threads of a row
        const int vi = tid % kPer;
        float m = -INFINITY;
        for (int i = vi; i < parts; i += kPer) {
            float2 v = make_float2(-INFINITY, 0.0f);
            if (r < live && holds(i)) v = p.ml[slot(i) + r];
            if (i < kParts) s_w[row_in][i] = v.x, s_l[row_in][i] = v.y;
            m = fmaxf(m, v.x);
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
        if (lane == 0) s_red[grp] = m;
        __syncthreads();
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) m = fmaxf(m, s_red[row_in * GROUPS + g]);
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < live) {
            constexpr int B = 8;
            for (int i0 = part_in; i0 < parts; i0 += GROUPS * B) {
                float mi[B], li[B];
                float4 v[B];
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    const int i = i0 + k * GROUPS;
                    mi[k] = -INFINITY;
                    if (i < kParts) {
                        if (i < parts) mi[k] = s_w[row_in][i], li[k] = s_l[row_in][i];
                    } else if (i < parts && holds(i)) {
                        const float2 ml = p.ml[slot(i) + r];
                        mi[k] = ml.x, li[k] = ml.y;
                    }
                    if (mi[k] != -INFINITY) v[k] = *reinterpret_cast<const float4*>(p.o + (slot(i) + r) * kPgDim + 4 * lane);
                }
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    if (mi[k] == -INFINITY) continue;
                    const float w = part_weight(mi[k], m);
                    l += w * li[k];
                    o.x += w * v[k].x;
                    o.y += w * v[k].y;
                    o.z += w * v[k].z;
                    o.w += w * v[k].w;
                }
            }
        }
        if constexpr (GROUPS > 1) {
            __syncthreads();  // s_red is read
            s_o[grp][lane] = o;
            if (lane == 0) s_red[grp] = l;
            __syncthreads();
            l = 0.0f;
            o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (part_in == 0)
                for (int g = 0; g < GROUPS; ++g) {
                    const float4 v = s_o[grp + g][lane];
                    l += s_red[grp + g];
                    o.x += v.x;
                    o.y += v.y;
                    o.z += v.z;
                    o.w += v.w;
                }
        }
        if (r < live && part_in == 0) {
            const float inv = row_inverse(m, l);
            const size_t at = static_cast<size_t>(rows.row(r)) * nq + rows.head(r);
            *reinterpret_cast<uint2*>(out + at * kPgDim + 4 * lane) = pack4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            if (lse != nullptr && lane == 0) lse[at] = row_log_sum(m, l);
        }
        __syncthreads();  // the next item writes s_w, s_red and s_o
    }
}

// ---- single tokens and selected blocks -----------------------------------------
// o = softmax(q K^T / sqrt(128)) V for one token: its q heads of one kv head, 16 at a
// time, are the columns of v_mfma_f32_16x16x32_f16; a tile is 32 keys, a wave's own.
//   S^T (16 keys x 16 heads) = K . Q^T: lane l (c = l % 16, g = l / 16) gives K row m = c and Q^T
//   column c, dims 32 kk + 8 g .. + 7, and receives S of head c and m = 4 g + r;
//   O^T (16 dims x 16 heads) += V^T . P^T: lane l gives eight keys of dim c and of head c.  The
//   order of the keys within the product is free: P^T uses what the lane holds of S, m = 4 g + r of
//   both halves of the tile, so row m of half u stands for key 16 u + 4 r + g, and then V^T's
//   eight keys of a lane are those of its own eight 16-byte loads (load i: key 4 i + g, dims 8 c .. 8 c + 7):
//   product j takes element j of each, put together by v_perm, and belongs to dims 8 c + j.
// So K and V go from memory to registers to the matrix cores with no trip through LDS, and a
// lane ends with dims 32 g .. 32 g + 31 of head c.  The softmax weights go into the product with V
// as two fp16 numbers each (2^-22): the second product costs nothing beside the loads, and with one (2^-11) the
// error of a single token's output came to 1.4 to 1.6 times that of fp32 weights.  Scores, sums and outputs are fp32.
//
// Bound by memory: K and V are read once, 512 bytes a key and kv head.  The next tile's K is
// requested as soon as this one's is in the matrix cores, and its V as soon as that is: 16 KB in
// flight a wave, 128 KB a CU.  A block a CU with 8 waves: with two of 4 waves the runs take as long, but
// have twice the parts, and the merge takes 0.5 to 4 us more.  V goes past the caches (48 sequences 51 us, else 55;
// 131000 keys 24, else 28), but not where other tokens may have selected the same blocks.
// 48 sequences (286000 keys, 293 MB): 51 us, 5.7 TB/s, and 5.6 for the merge; one of
// 131000 (134 MB): 24 (5.6 TB/s) and 6.  2.2 us of either are the division of the work.
constexpr int kDecWaves = 8;     // waves of a block
constexpr int kDecBlocks = 256;  // of a launch: one a CU
constexpr int kDecKeys = 32;     // keys of a tile
constexpr int kDecRows = 16;     // rows of a segment
constexpr int kDecOver = 4;      // what starting a segment costs, in tiles

struct DecodeParams {
    PagedView c;
    const uint16_t* q;
    const int32_t* selected;  // [row][kv head][num_selected]
    uint16_t* out;
    float* lse;
    void* ws;
    int nq, group, window, num_selected, coarse;
};

// The keys of a token, in tiles of 32: of the whole context or window (tile t: positions 32 t ..),
// or of the list of selected blocks (tile t: entries from 32 t / page size on).
struct DecodeRange {
    int pos, lo, lim, first_tile, tiles;
};
template <bool SPARSE>
__device__ __forceinline__ DecodeRange decode_range(const DecodeParams& p, const PagedSeq& s, int row) {
    DecodeRange r;
    r.pos = s.ctx + row - s.first;
    r.lim = min(r.pos, p.c.capacity() - 1);
    r.lo = !SPARSE && p.window > 0 ? max(0, r.pos - p.window + 1) : 0;
    if (SPARSE) {
        r.first_tile = 0;
        r.tiles = static_cast<int>(((static_cast<long long>(p.num_selected) << p.c.shift) + kDecKeys - 1) / kDecKeys);
    } else {
        r.first_tile = r.lo / kDecKeys;
        r.tiles = r.lim < r.lo ? 0 : r.lim / kDecKeys - r.first_tile + 1;
    }
    return r;
}

// Where the waves of a block meet: each row's reference value and sum, and its outputs.
template <int WAVES>
struct TokenShared {
    float m[WAVES][kDecRows], l[WAVES][kDecRows];
    __align__(16) float o[WAVES][kDecRows][kPgDim + 4];
};

// Up to 16 rows (lane (c, g): row c, with keys lo .. lim) of a kv head against tiles first .. end - 1 of a
// sequence's keys, or of its list of blocks, the waves of the block a run each; store(row, dim, four
// outputs, reference value, sum) for every row < live and every fourth dim.  KEEP: rows of V are read by others too.
template <bool SPARSE, bool KEEP, int WAVES, class Store>
__device__ __forceinline__ void token_rows(const PagedView& p, int seq, int h, const int32_t* list, int num_selected, int first,
                                           int end, const f16x8 (&qf)[4], int lo, int lim, int live,
                                           TokenShared<WAVES>& shared, Store store) {
    const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const int c = lane & 15, g = lane >> 4;
    const ptrdiff_t v_minus_k = reinterpret_cast<const char*>(p.v) - reinterpret_cast<const char*>(p.k);
    // rows in the order of positions: the keys that all see, and those that any does
    const int lo_all = __builtin_amdgcn_readlane(lo, live - 1), lo_any = __builtin_amdgcn_readlane(lo, 0);
    const int lim_all = __builtin_amdgcn_readlane(lim, 0), lim_any = __builtin_amdgcn_readlane(lim, live - 1);
    // this wave's run of tiles
    const int a = first + static_cast<int>(static_cast<long long>(end - first) * wave / WAVES);
    const int e = first + static_cast<int>(static_cast<long long>(end - first) * (wave + 1) / WAVES);
    // 64 entries of the list or of the table from `base` on, one a lane: page and block number
    int base = 0, page_l = -1, block_l = 0;
    auto refill = [&](int entry) __attribute__((always_inline)) {
        base = entry;
        block_l = entry + lane;
        if constexpr (SPARSE) block_l = block_l < num_selected ? list[block_l] : -1;
        page_l = block_l >= 0 && block_l < p.max_pages && (block_l << p.shift) <= lim_any ? paged_page(p, seq, block_l) : -1;
    };
    struct Tile {
        const char* k[2];  // of the first key of each half
        int pos[2];        // its position
        bool there[2];     // it has a page
    };
    auto tile_at = [&](int t) __attribute__((always_inline)) {
        Tile x;
        const int per_page = p.shift - 5;  // log2 of the tiles of a page, -1 for two pages a tile
        const int entry = per_page >= 0 ? t >> per_page : 2 * t;
        const int span = per_page >= 0 ? 1 : 2;
        if (entry + span > base + 64) refill(entry);
        const int in_page = per_page >= 0 ? (t & ((1 << per_page) - 1)) * kDecKeys : 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int at = entry - base + (span == 2 ? u : 0);
            const int page = __builtin_amdgcn_readlane(page_l, at);
            const int row0 = in_page + (span == 2 ? 0 : 16 * u);
            x.there[u] = page >= 0;
            x.pos[u] = (__builtin_amdgcn_readlane(block_l, at) << p.shift) + row0;
            x.k[u] = reinterpret_cast<const char*>(p.k + static_cast<long long>(max(page, 0)) * p.page_stride +
                                                   ((static_cast<long long>(h) << p.shift) + row0) * kPgDim);
        }
        return x;
    };
    const uint32_t k_off = static_cast<uint32_t>((4 * (c & 3) + (c >> 2)) * kPgDim * 2 + 16 * g);
    const uint32_t v_off = static_cast<uint32_t>(g * kPgDim * 2 + 16 * c);
    u32x4 kf[8], vf[8];
    auto request_k = [&](const Tile& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) kf[i] = *reinterpret_cast<const u32x4*>(x.k[i >> 2] + (k_off + 64 * (i & 3)));
    };
    auto request_v = [&](const Tile& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const u32x4* v = reinterpret_cast<const u32x4*>(x.k[i >> 2] + v_minus_k + (v_off + 4 * (i & 3) * kPgDim * 2));
            vf[i] = KEEP ? *v : __builtin_nontemporal_load(v);
        }
    };
    f32x4 acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = f32x4{};
    float mref = -INFINITY, lsum = 0.0f;
    bool any = false;
    Tile cur{};
    if (a < e) {
        const int entry = p.shift >= 5 ? a >> (p.shift - 5) : 2 * a;
        refill(entry);
        cur = tile_at(a);
        request_k(cur);
        request_v(cur);
    }
    for (int t = a; t < e; ++t) {
        f32x4 sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            sc[u] = f32x4{};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, kf[4 * u + kk]), qf[kk], sc[u],
                                                               0, 0, 0);
        }
        Tile nxt = cur;
        if (t + 1 < e) {
            nxt = tile_at(t + 1);
            request_k(nxt);
        }
        // keys out of sight (and rows that are none): the weights are 0, but what lies in the rows may be anything
        const bool plain = cur.there[0] && cur.there[1] && cur.pos[0] >= lo_all && cur.pos[0] + 15 <= lim_all &&
                           cur.pos[1] >= lo_all && cur.pos[1] + 15 <= lim_all;
        if (plain) {
            any = true;
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = cur.pos[u] + 4 * r + g;
                    const bool seen = cur.there[u] && key >= lo && key <= lim;
                    any = any || seen;
                    sc[u][r] = seen ? sc[u][r] : -INFINITY;
                }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = cur.pos[i >> 2] + 4 * (i & 3) + g;
                const bool seen = cur.there[i >> 2] && key >= lo_any && key <= lim_any;
#pragma unroll
                for (int d = 0; d < 4; ++d) vf[i][d] = seen ? vf[i][d] : 0u;
            }
        }
        float mx = sc[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i >> 2][i & 3]);
        mx = xor32_max(xor16_max(mx)) * kPgScale;
        const bool grow = mx > mref + (kPgRoom + kPgLag);
        if (__builtin_amdgcn_ballot_w64(grow) != 0) {
            const float to = grow ? mx - kPgRoom : mref;
            const float alpha = grow ? __builtin_amdgcn_exp2f(mref - to) : 1.0f;
            mref = to;
            lsum *= alpha;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[j][r] *= alpha;
        }
        const float neg = mref == -INFINITY ? 0.0f : -mref;  // masked scores give exp2(-inf) = 0
        f16x8 pf, rest;  // a weight in two parts
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 2][i & 3], kPgScale, neg));
            lsum += w;
            pf[i] = static_cast<_Float16>(w);
            rest[i] = static_cast<_Float16>(w - static_cast<float>(pf[i]));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t take = j & 1 ? 0x07060302u : 0x05040100u;
            u32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_perm(vf[2 * i + 1][j >> 1], vf[2 * i][j >> 1], take);
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), pf, acc[j], 0, 0, 0);
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), rest, acc[j], 0, 0, 0);
        }
        if (t + 1 < e) request_v(nxt);
        cur = nxt;
    }
    // the waves meet: each row's common reference value, then the sum of the rescaled outputs
    lsum += __shfl_xor(lsum, 16);
    lsum += __shfl_xor(lsum, 32);
    // the row has had a key (all lanes ask: one that leaves early would answer the others with 0)
    int some = any;
    some |= __shfl_xor(some, 16);
    some |= __shfl_xor(some, 32);
    if (some != 0) mref = fmaxf(mref, kPgLowest);
    if (g == 0) shared.m[wave][c] = mref, shared.l[wave][c] = lsum;
    __syncthreads();
    {
        float m = shared.m[0][c];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) m = fmaxf(m, shared.m[w][c]);
        const float f = part_weight(mref, m);
        float* o = &shared.o[wave][c][32 * g];
#pragma unroll
        for (int i = 0; i < 8; ++i)  // dims 32 g + 4 i .. + 3: r = i / 2, j = 4 (i % 2) ..
            *reinterpret_cast<float4*>(o + 4 * i) =
                make_float4(acc[4 * (i & 1)][i >> 1] * f, acc[4 * (i & 1) + 1][i >> 1] * f, acc[4 * (i & 1) + 2][i >> 1] * f,
                            acc[4 * (i & 1) + 3][i >> 1] * f);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < live * (kPgDim / 4); i += 64 * WAVES) {
        const int r = i / (kPgDim / 4), d = 4 * (i % (kPgDim / 4));
        float m = shared.m[0][r], l = 0.0f;
        for (int w = 1; w < WAVES; ++w) m = fmaxf(m, shared.m[w][r]);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < WAVES; ++w) {
            l += shared.m[w][r] == -INFINITY ? 0.0f : shared.l[w][r] * part_weight(shared.m[w][r], m);
            const float4 x = *reinterpret_cast<const float4*>(&shared.o[w][r][d]);
            o.x += x.x;
            o.y += x.y;
            o.z += x.z;
            o.w += x.w;
        }
        store(r, d, o, m, l);
    }
    __syncthreads();  // the next segment writes shared.m
}

// The sequence of a row of a list; -1: the row is of none.
__device__ __forceinline__ int seq_of_listed_row(const PagedView& p, int row, PagedSeq& s) {
    const int seq = uniform(paged_seq_of_row(p, row));
    if (seq < 0) return -1;
    s = paged_seq(p, seq);
    return row < s.first || row >= s.first + s.n ? -1 : seq;
}

// Tiles t0 .. t1 - 1 of a segment, into the output (at < 0) or into the partials from row `at` on.
template <bool SPARSE, int WAVES>
__device__ __forceinline__ void token_segment(const DecodeParams& p, const PagedSeq& s, int seq, int row, int h, int rt, int t0,
                                              int t1, long long at, const Partials& part, TokenShared<WAVES>& shared) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const DecodeRange range = decode_range<SPARSE>(p, s, row);
    const int live = min(kDecRows, p.group - rt * kDecRows);
    const int head0 = h * p.group + rt * kDecRows;
    f16x8 qf[4];
    const uint16_t* q = p.q + (static_cast<size_t>(row) * p.nq + head0 + min(c, live - 1)) * kPgDim + 8 * g;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[kk] = *reinterpret_cast<const f16x8*>(q + 32 * kk);
    const int* list = SPARSE ? p.selected + (static_cast<size_t>(row) * p.c.nkv + h) * p.num_selected : nullptr;
    token_rows<SPARSE, SPARSE, WAVES>(
        p.c, seq, h, list, p.num_selected, range.first_tile + t0, range.first_tile + t1, qf, uniform(range.lo), uniform(range.lim),
        live, shared, [&](int r, int d, float4 o, float m, float l) __attribute__((always_inline)) {
            if (at < 0) {
                const float inv = row_inverse(m, l);
                const size_t to = static_cast<size_t>(row) * p.nq + head0 + r;
                *reinterpret_cast<uint2*>(p.out + to * kPgDim + d) = pack4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
                if (p.lse != nullptr && d == 0) p.lse[to] = row_log_sum(m, l);
            } else {
                *reinterpret_cast<float4*>(part.o + (at + r) * kPgDim + d) = o;
                if (d == 0) part.ml[at + r] = make_float2(m, l);
            }
        });
}

// A block for each segment, and nothing to merge: where no row has more than kShortKeys keys, or where there
// are kManySegments and none is far longer than the others (lists are all alike; single tokens of up to twice
// as many keys).  Blocks of 4 waves, three of them a CU.  (us, with the merge, shares against this: 1 token on
// 300 keys 13.0 and 7.2, on 1000 14.8 and 12.8, on 2000 15.3 and 21.8; 200 on 1 to 2000 53.6 and 39.5; 400 lists of
// 2048 keys 84 and 72, 200 of 4096 82 and 65, 128 of 4096 54 and 64.  With 8 waves a block: 7.8, 14.1, ... 75.)
constexpr int kShortWaves = 4, kShortKeys = 1024, kManySegments = 192;
template <bool SPARSE>
__global__ __launch_bounds__(64 * kShortWaves, 3) void paged_short_kernel(DecodeParams p) {
    __shared__ TokenShared<kShortWaves> shared;
    const int row_tiles = (p.group + kDecRows - 1) / kDecRows;
    const int of_row = p.c.nkv * row_tiles, row = blockIdx.x / of_row, h = (blockIdx.x - row * of_row) / row_tiles;
    PagedSeq s;
    int seq = row;
    if constexpr (SPARSE) {
        seq = seq_of_listed_row(p.c, row, s);
        if (seq < 0) return;
    } else {
        s = paged_seq(p.c, seq);
        if (s.n == 0) return;
    }
    token_segment<SPARSE>(p, s, seq, row, h, blockIdx.x % row_tiles, 0, decode_range<SPARSE>(p, s, row).tiles, -1, Partials{}, shared);
}

template <bool SPARSE>
__global__ __launch_bounds__(64 * kDecWaves, 2) void paged_decode_kernel(DecodeParams p) {
    __shared__ TokenShared<kDecWaves> shared;
    const Partials part = partials<kDecRows>(p.ws, kDecBlocks);
    const int row_tiles = (p.group + kDecRows - 1) / kDecRows;

    // On the line: each sequence has its token's heads; or one sequence has those of all rows, the heads of
    // a row behind each other (all alike: which rows have a token is seen when their turn comes).
    auto work = [&](const PagedSeq& s) __attribute__((always_inline)) {
        SeqWork w{0, -1, 0, s.n > 0 ? row_tiles : 0, SPARSE ? p.c.rows * p.c.nkv : p.c.nkv};
        w.first = w.most = (decode_range<SPARSE>(p, s, s.first).tiles >> p.coarse) + kDecOver;
        return w;
    };
    auto tiles = [&](const PagedSeq& s, int) __attribute__((always_inline)) { return decode_range<SPARSE>(p, s, s.first).tiles; };

    auto body = [&](int item, PagedSeq s, int head, int rt, int t0, int t1, int slot) __attribute__((always_inline)) {
        const int row = SPARSE ? head / p.c.nkv : s.first, h = SPARSE ? head - row * p.c.nkv : head;
        const int seq = SPARSE ? seq_of_listed_row(p.c, row, s) : item;
        if (SPARSE && seq < 0) return;  // not written
        token_segment<SPARSE>(p, s, seq, row, h, rt, t0, t1, slot < 0 ? -1 : static_cast<long long>(2 * blockIdx.x + slot) * kDecRows,
                              part, shared);
    };
    auto rows = [&](const PagedSeq&, int head, int rt) __attribute__((always_inline)) {
        if constexpr (SPARSE) {
            PagedSeq s;
            if (seq_of_listed_row(p.c, head / p.c.nkv, s) < 0) return 0;
        }
        return min(kDecRows, p.group - rt * kDecRows);
    };
    for_share<SPARSE>(p.c, blockIdx.x, kDecBlocks, (kDecWaves >> p.coarse) + kDecOver, work, tiles, rows, body, [&](SegmentCut cut) {
        if (threadIdx.x == 0) part.cuts[blockIdx.x] = cut;
    });
}

template <bool SPARSE, int GROUPS, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_decode_merge_kernel(DecodeParams p) {
    static_assert(kDecBlocks <= kMergeCuts, "a cut for each block");
    merge_parts<kDecRows, GROUPS, THREADS>(p.ws, kDecBlocks, p.out, p.lse, p.nq, [&](const SegmentCut& c) {
        const int row = SPARSE ? c.head / p.c.nkv : paged_seq(p.c, c.item).first, h = SPARSE ? c.head - row * p.c.nkv : c.head;
        return RowMap{row, 0, kDecRows, h * p.group + c.row_tile * kDecRows};
    });
}

// ---- chunks -----------------------------------------------------------------------
// Causal attention of the rows of many sequences.  The q heads of a kv head and a
// sequence's new tokens form one list of rows, row r = token r / group, head kvh *
// group + r % group; a segment is 32 of them for each wave of a block, whatever the group.  The
// waves share the keys in LDS, in halves of 32, filled from the pages by DMA.
// v_mfma_f32_32x32x16_f16 with the rows as columns:
//   S^T (32 keys x 32 rows) = K . Q^T: lane l holds key l % 32 and row l % 32, dims 8 (l / 32) +
//   16 kk; Q stays in registers; the result has lane l = row l % 32 with the keys
//   8 (v / 4) + 4 (l / 32) + v % 4, so a row's maximum and sum are in-lane and one swap;
//   O^T (128 dims x 32 rows) += V^T . P^T: P^T is the lane's own weights as fp16, V^T comes
//   out of the row-major tile by ds_read_b64_tr_b16.
// A tile row is 256 bytes, its 16-byte chunk c stored at c ^ swz(key), so that the reads
// of K (16 keys, one chunk) and of V (4 keys x 4 chunks a half wave) meet no bank twice.
// Rows that no one may see (behind the sequence's end, before every window, of missing
// pages) are filled from a row of zeros: their weights are 0, and what lies there may be
// anything.
//
// Bound by the matrix cores where rows are many (4 * 128 operations a row and key): a wave's
// stage is 16 MFMAs (32 cycles each) and the scores of half t + 1, the weights of half t and the outputs
// of half t - 1, which do not depend on each other and share the issue slots MFMA by MFMA.
// Between two barriers lie 4 such stages, and a CU holds one block of 8 waves with a ring of 8 halves of
// K and V (128 KB): a segment of 256 rows reads each key once, and the waves drift apart and fill each
// other's gaps.  Rows that are few for their sequences (num_tokens * group < 512 num_seqs) take two
// blocks of 4 waves a CU, with 2 stages and rings of 4 halves: segments of 128 rows, half the waste on short
// ones, and one block starts while the other works.  2048 tokens at 14000, 12 heads over 2: 214 to 220 us (880
// TF) before the chip lowers its clock and 225 to 269 after, with 4 waves a tenth more; a mixed batch of
// 43 sequences: 56 to 60 us, with 8 waves a fifth more; 17 tokens at 1200: 14.9 us, with 8 waves 15.
//
// All eight forms take every vector register of a wave or nearly; those with FEW spill 14 to 17 of them, offsets of the
// fill by rows: it reloads each before its load, and the wait for that is a wait for all loads before.  So halves
// with rows that no one may see (at every sequence's start and end) cost several latencies, not one.
//
// The weights are rounded to fp16 for the product with V (2^-11, as in this library's other
// attention of chunks): a second product, as for single tokens, would be half as many MFMAs again.
// Outputs are divided by the sum of the rounded weights, so that the roundings of a row's largest ones cancel (a
// lone key gives its V; the mixed batch's error 2.6e-4 instead of 2.9e-4; 4 % of the long chunk's time); log
// sums are of the weights themselves.
//
// A sequence with up to 16 rows of a kv head (single tokens beside the chunks, drafts) is attended as in
// the section above, each wave on keys of its own: a tile of 128 rows would be mostly empty.  It counts half
// on the line (when it was chosen, the mixed batch: 54 us so, 59 where such rows fill tiles; 66 where they count whole, 67
// where a quarter).
constexpr int kPfKeys = 64;           // keys of a tile: what shares are cut between
constexpr int kPfHalf = 32;           // keys of a stage
constexpr int kPfHalfBytes = kPfHalf * kPgDim * 2;
constexpr int kPfOver = 4 * kPfKeys;  // what a segment costs beside its keys, in keys
constexpr int kLeastTiles = 2;        // of a share
constexpr long long kMergeBlocks = 1024;
// Blocks of WAVES waves, 32 rows each; a CU holds eight waves.
template <int WAVES>
struct PrefillShape {
    static constexpr int rows = 32 * WAVES;          // rows of a segment
    static constexpr int blocks = 256 * 8 / WAVES;   // of a launch
    static constexpr int period = WAVES / 2;         // stages between barriers
    static constexpr int ring = 2 * period;          // halves of K, and of V, in LDS
};

__device__ __align__(256) const uint16_t g_zero_row[kPgDim] = {};

struct PrefillParams {
    PagedView c;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    void* ws;
    int nq, group, window, coarse;
};

struct PrefillRange {
    int r0, rows;           // first row of the segment, rows of the sequence
    int first_tile, tiles;  // key tiles that its rows see
    int low;                // the first key that one of them sees
};
template <int WAVES>
__device__ __forceinline__ PrefillRange prefill_range(const PrefillParams& p, const PagedSeq& s, int rt) {
    constexpr int kRows = PrefillShape<WAVES>::rows;
    PrefillRange r;
    r.r0 = rt * kRows;
    r.rows = s.n * p.group;
    const int first = s.ctx + r.r0 / p.group;
    const int last = min(s.ctx + (min(r.r0 + kRows, r.rows) - 1) / p.group, p.c.capacity() - 1);
    r.low = p.window > 0 ? max(0, first - p.window + 1) : 0;
    r.first_tile = r.low / kPfKeys;
    r.tiles = last < r.low ? 0 : last / kPfKeys - r.first_tile + 1;
    return r;
}

// Weight of so many keys for a token's group: shortened as the launch says, 1 to 2^29.
__device__ __forceinline__ int weight_of(const PrefillParams& p, int keys) {
    const long long w = static_cast<long long>(p.group) * (static_cast<long long>(keys) + kPfOver) >> p.coarse;
    return static_cast<int>(max(1LL, min(w, 1LL << 29)));
}

// ONE: pages of 32 tokens and more (a half tile lies in one page).  FEW: sequences of few rows may be there (a
// kernel that knows of none starts 3 us sooner: 17 tokens at 1200 14 us instead of 17).
template <bool ONE, int WAVES, bool FEW>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_prefill_kernel(PrefillParams p) {
    typedef PrefillShape<WAVES> Shape;
    constexpr int kRows = Shape::rows, kBlocks = Shape::blocks, P = Shape::period, R = Shape::ring;
    __shared__ __align__(256) char smem[2 * R * kPfHalfBytes];  // the last R halves of K, of V
    static_assert(sizeof(TokenShared<WAVES>) <= sizeof(smem), "segments of few rows meet there");
    const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const int fr = lane & 31, h = lane >> 5;
    // blocks of one XCD take neighbouring shares: they read the same pages
    const int block = static_cast<int>(blockIdx.x & 7) * (kBlocks / 8) + static_cast<int>(blockIdx.x >> 3);
    const Partials part = partials<kRows>(p.ws, kBlocks);
    constexpr int NP = ONE ? 1 : 2;             // pages of a half tile, at most

    // Every tile requested so far is in LDS, for every wave, and what was read before is read: the reads' own
    // wait too, for nothing else holds the products that need them before the barrier.
    auto tile_barrier = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

    auto work = [&](const PagedSeq& s) __attribute__((always_inline)) {
        // weights: keys times group, as if the rows were cut between tokens
        const int g = p.group;
        constexpr int kStep = WAVES == 8 ? 8 : 7;
        static_assert(1 << kStep == kRows, "the weight of a row tile's own tokens");
        SeqWork w{weight_of(p, s.ctx), max(kStep - p.coarse, -1), weight_of(p, p.c.capacity()), (s.n * g + kRows - 1) / kRows, p.c.nkv};
        if (p.window > 0) w.most = min(w.most, weight_of(p, min(p.window, p.c.capacity()) + kRows / g + kPfKeys));
        if (FEW && s.n * g <= kDecRows) {  // half: as measured
            w.first = (w.first + 1) / 2;
            w.most = (w.most + 1) / 2;
        }
        return w;
    };
    auto tiles = [&](const PagedSeq& s, int rt) __attribute__((always_inline)) { return prefill_range<WAVES>(p, s, rt).tiles; };

    auto body = [&](int seq, const PagedSeq& s, int kvh, int rt, int t0, int t1, int slot) __attribute__((always_inline)) {
        const PrefillRange range = prefill_range<WAVES>(p, s, rt);
        const int rows = uniform(range.rows), first_tile = uniform(range.first_tile), low = uniform(range.low);
        const int it0 = first_tile + t0, it1 = first_tile + t1;
        if (FEW && rows <= kDecRows) {  // as single tokens are attended: each wave keys of its own, no rows to share them
            const int c = lane & 15, rc = min(c, rows - 1), qi = rc / p.group, qh = kvh * p.group + rc - qi * p.group;
            const int pos = s.ctx + qi, lim = min(pos, p.c.capacity() - 1), lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
            const uint16_t* q = p.q + (static_cast<size_t>(s.first + qi) * p.nq + qh) * kPgDim + 8 * (lane >> 4);
            f16x8 qf[4];
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) qf[kk] = *reinterpret_cast<const f16x8*>(q + 32 * kk);
            // (the last tile's second half may lie behind the last key)
            const int end = min(2 * it1, __builtin_amdgcn_readlane(lim, rows - 1) / kPfHalf + 1);
            token_rows<false, false, WAVES>(
                p.c, seq, kvh, nullptr, 0, 2 * it0, max(end, 2 * it0), qf, lo, lim, rows, *reinterpret_cast<TokenShared<WAVES>*>(smem),
                [&](int r, int d, float4 o, float m, float l) __attribute__((always_inline)) {
                    const int token = r / p.group;
                    if (slot < 0) {
                        const float inv = row_inverse(m, l);
                        const size_t at = static_cast<size_t>(s.first + token) * p.nq + kvh * p.group + r - token * p.group;
                        *reinterpret_cast<uint2*>(p.out + at * kPgDim + d) = pack4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
                        if (p.lse != nullptr && d == 0) p.lse[at] = row_log_sum(m, l);
                    } else {
                        const size_t at = static_cast<size_t>(2 * block + slot) * kRows + r;
                        *reinterpret_cast<float4*>(part.o + at * kPgDim + d) = o;
                        if (d == 0) part.ml[at] = make_float2(m, l);
                    }
                });
            return;
        }
        const uint32_t lds0 =
            static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)smem));
        // A wave loads whole halves, by eight loads of four rows: load i its rows 4 i + lane / 16, stored chunk lane % 16,
        // i.e. chunk (lane % 16) ^ swz(row) of memory.  The first four lanes' offsets (the others are 16 rows on):
        uint32_t loff[4];  // bytes
#pragma unroll
        for (int i = 0; i < 4; ++i)
            loff[i] = static_cast<uint32_t>((4 * i + (lane >> 4)) * (2 * kPgDim) + 16 * ((lane & 15) ^ (((lane >> 4) << 2) | i)));
        // LDS addresses: K chunk 2 kk + h of key fr; V^T reads (dt: 32 dims, u: keys + 8)
        uint32_t ka[8], va[4][2];
        {
            const int swz_k = ((fr & 3) << 2) | ((fr >> 2) & 3);
            const uint32_t k0 = lds0 + fr * 256 + 16 * (h ^ swz_k);
            const int s16 = lane & 15, b16 = (lane >> 4) & 1;
            const uint32_t v0 = lds0 + (R + P) * kPfHalfBytes + (4 * h + (s16 >> 2)) * 256 +
                                16 * ((2 * b16 + ((s16 & 3) >> 1)) ^ (((s16 >> 2) << 2) | h)) + 8 * (s16 & 1);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) ka[kk] = k0 ^ (32 * kk);
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                va[dt][0] = v0 ^ (64 * dt);
                va[dt][1] = (v0 ^ (64 * dt) ^ 32) + 8 * 256;
            }
        }
        // The ring is two frames of P slots, and these addresses are of one of them: of K's first at first, of V's second.
        int k_turn = P * kPfHalfBytes, v_turn = -P * kPfHalfBytes;
        auto turn_k = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) ka[kk] += k_turn;
            k_turn = -k_turn;
        };
        auto turn_v = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) va[dt][0] += v_turn, va[dt][1] += v_turn;
            v_turn = -v_turn;
        };
        // K operand of MFMA i of the half in the frame's `slot`: dims 16 i; V^T operand: 16-key quarter i / 4, dims 32 (i % 4)
        auto read_k = [&](int slot, int i) __attribute__((always_inline)) {
            typedef const __attribute__((address_space(3))) f16x8* lptr;
            return *reinterpret_cast<lptr>(ka[i] + slot * kPfHalfBytes);
        };
        auto read_v = [&](int slot, int i) __attribute__((always_inline)) {
            typedef __attribute__((address_space(3))) s16x4* lptr;
            const uint32_t off = slot * kPfHalfBytes + (i >> 2) * 16 * 256;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lptr>(va[i & 3][0] + off));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lptr>(va[i & 3][1] + off));
            return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        const int r = rt * kRows + wave * 32 + fr;
        const int rc = min(r, rows - 1);
        const int qi = rc / p.group, qh = kvh * p.group + rc - qi * p.group;
        const int pos = s.ctx + qi;
        const bool dead = rt * kRows + wave * 32 >= rows;  // the wave has no row
        // the keys that this row takes here: lo .. lim
        const int lim = min(min(pos, p.c.capacity() - 1), it1 * kPfKeys - 1);
        const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        // tiles within these take no mask; the last key that any row of the wave takes
        const int wave_lim = __builtin_amdgcn_readlane(lim, 0), wave_lo = __builtin_amdgcn_readlane(lo, 31);
        const int wave_last = dead ? -1 : __builtin_amdgcn_readlane(lim, 31);
        const int keys = uniform(min(s.ctx + s.n, p.c.capacity()));  // of the sequence

        u32x4 qf[8];
        {
            const uint16_t* qr = p.q + (static_cast<size_t>(s.first + qi) * p.nq + qh) * kPgDim + 8 * h;
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) qf[kk] = *reinterpret_cast<const u32x4*>(qr + 16 * kk);
        }
        const int key0 = it0 * kPfKeys, halves = 2 * (it1 - it0);  // the run: halves 0 .. halves - 1
        // 64 entries of the table from `base` on, one a lane, as the distance of their page from the first
        // (-1: no page); and the next ones, on their way
        int base = 0, next_base = -1, next_l = 0, page_lo = 0, page_hi = -1;
        auto entry_of = [&](int half) __attribute__((always_inline)) {
            return (key0 + kPfHalf * min(half, halves - 1)) >> p.c.shift;
        };
        bool holes = false;  // some of the run's tiles' entries among them are no page (also behind the last key, where none is needed)
        auto request_entries = [&](int entry) __attribute__((always_inline)) {
            next_base = entry;
            next_l = p.c.table[static_cast<size_t>(seq) * p.c.max_pages + min(entry + lane, p.c.max_pages - 1)];
        };
        auto take_entries = [&]() __attribute__((always_inline)) {
            base = next_base;
            next_base = -1;
            const bool page = base + lane < p.c.max_pages && next_l >= 0 && next_l < p.c.num_pages;
            const long long far = page ? 2 * static_cast<long long>(next_l) * p.c.page_stride : -1;
            page_lo = static_cast<int>(far);
            page_hi = static_cast<int>(far >> 32);
            holes = __builtin_amdgcn_ballot_w64(!page && base + lane <= entry_of(halves - 1) + NP - 1) != 0;
        };
        auto page_at = [&](int entry) __attribute__((always_inline)) {
            const uint32_t lo = __builtin_amdgcn_readlane(page_lo, entry - base), hi = __builtin_amdgcn_readlane(page_hi, entry - base);
            return static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo);
        };
        // Halves that are filled without a look at their keys, and those that no row of the wave masks (both as
        // the first one and how many).
        const int fill0 = (max(low - key0, 0) + kPfHalf - 1) / kPfHalf;
        const int fill_n = min(halves, (keys - key0) / kPfHalf) - fill0;
        const int bare0 = (max(wave_lo - key0, 0) + kPfHalf - 1) / kPfHalf;
        const int bare_n = min(halves, (wave_lim + 1 - key0) / kPfHalf) - bare0;
        auto within = [](int x, int first, int n) __attribute__((always_inline)) { return n > 0 && static_cast<uint32_t>(x - first) < static_cast<uint32_t>(n); };
        // bytes from the first page's to this head's first row
        const long long head_at = 2 * ((static_cast<long long>(kvh) << p.c.shift) * kPgDim);
        const int in_page = p.c.page_size() - 1;
        // K or V of a half on its way into its slot; tile_barrier holds the waits.  The half before the first is
        // zeros, halves behind the last are left out.
        struct Job {
            const char* from[2];  // of its rows 0 and 16
            uint32_t dst;
            bool plain;           // every row is there
        };
        auto job_of = [&](int half, bool v) __attribute__((always_inline)) {
            Job j;
            j.dst = lds0 + ((v ? R : 0) + (half & (R - 1))) * kPfHalfBytes;
            j.plain = !holes && within(half, fill0, fill_n);
            j.from[0] = j.from[1] = nullptr;
            const int key1 = key0 + kPfHalf * half;
            const char* const pool = reinterpret_cast<const char*>(v ? p.c.v : p.c.k) + head_at;
            if (__builtin_expect(j.plain, 1)) {
                const int entry = key1 >> p.c.shift;
                j.from[0] = pool + page_at(entry) + (ONE ? (key1 & in_page) * (2 * kPgDim) : 0);
                j.from[1] = ONE ? j.from[0] + 16 * 2 * kPgDim : pool + page_at(entry + 1);
            } else if (half < halves) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int row = 4 * i + (lane >> 4), key = key1 + row;
                    const long long page = half < 0 ? -1 : page_at((key1 + (ONE ? 0 : 16 * (i / 4))) >> p.c.shift);
                    const uint32_t chunk = 16 * ((lane & 15) ^ (((lane >> 4) << 2) | (i & 3)));
                    const bool seen = page >= 0 && key >= low && key < keys;
                    lds_load_x4(j.dst + 1024 * i, seen ? pool + page + (key & in_page) * (2 * kPgDim) + chunk
                                                       : reinterpret_cast<const char*>(g_zero_row) + chunk);
                }
            }
            return j;
        };
        auto load_part = [&](const Job& j, int i) __attribute__((always_inline)) {
            if (__builtin_expect(j.plain, 1)) lds_load_x4(j.dst + 1024 * i, j.from[i >> 2], loff[i & 3]);
        };
        auto load_half = [&](int half, bool v) __attribute__((always_inline)) {
            const Job j = job_of(half, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) load_part(j, i);
        };

        f32x16 acc[4];
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) acc[dt] = f32x16{};
        float mref = -INFINITY, lsum = 0.0f, lround = 0.0f;  // the sums of the weights and of what they are rounded to
        bool any = false;                                    // the row has had a key
        auto mask = [&](int half, f32x16& sc) __attribute__((always_inline)) {
            if (__builtin_expect(!holes && within(half, bare0, bare_n), 1)) {
                any = true;
                return;
            }
            const int key1 = key0 + kPfHalf * half;
            const bool there0 = page_at(entry_of(half)) >= 0, there1 = ONE ? there0 : page_at(entry_of(half) + 1) >= 0;
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int key = key1 + 8 * (v >> 2) + 4 * h + (v & 3);
                const bool seen = key <= lim && key >= lo && (v < 8 ? there0 : there1);
                any = any || seen;
                sc[v] = seen ? sc[v] : -INFINITY;
            }
        };
        // Reference values are whole numbers (exponents of two), so what was weighed by an old one, the weights pw in
        // wait among it, is scaled without rounding (but for weights that end below 2^-21 of the largest).
        auto renew_ref = [&](float mx, uint32_t (&pw)[8]) __attribute__((always_inline)) {
            const bool grow = mx > mref + (kPgRoom + kPgLag);
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(grow) != 0, 0)) {
                const float to = grow ? floorf(mx) - kPgRoom : mref;
                const float alpha = !grow ? 1.0f : __builtin_amdgcn_exp2f(mref - to);
                mref = to;
                lsum *= alpha;
                lround *= alpha;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                    for (int v = 0; v < 16; ++v) acc[dt][v] *= alpha;
#pragma unroll
                for (int i = 0; i < 8; ++i) {  // (in fp32: a scale below 2^-24 would be 0 in fp16, a weight times it need not)
                    const f32x2 w = __builtin_convertvector(__builtin_bit_cast(f16x2, pw[i]), f32x2) * alpha;
                    pw[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(w, f16x2));
                }
            }
        };
        auto max_of = [&](const f32x16& sc, int v0, int n, float mx) __attribute__((always_inline)) {
#pragma unroll
            for (int v = v0; v < v0 + n; ++v) mx = fmaxf(mx, sc[v]);
            return mx;
        };
        // weights 2 i and 2 i + 1 of a half's scores, packed
        auto weights = [&](const f32x16& sc, int i, float neg, float (&ps)[3]) __attribute__((always_inline)) {
            const f32x2 e = {__builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * i], kPgScale, neg)),
                             __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * i + 1], kPgScale, neg))};
            ps[0] += e.x;
            ps[1] += e.y;
            const f16x2 r = __builtin_convertvector(e, f16x2), ones = {1, 1};
            ps[2] = __builtin_amdgcn_fdot2(r, ones, ps[2], false);
            uint32_t w = __builtin_bit_cast(uint32_t, r);
            asm volatile("" : "+v"(w), "+v"(ps[0]), "+v"(ps[1]), "+v"(ps[2]));  // here, not past the mask's branch
            return w;
        };
        auto times_q = [&](const f16x8& k, int i, f32x16& sc) __attribute__((always_inline)) {
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, __builtin_bit_cast(f16x8, qf[i]), i == 0 ? f32x16{} : sc, 0, 0, 0);
        };
        auto add_pv = [&](const f16x8& v, int i, const uint32_t (&pw)[8]) __attribute__((always_inline)) {
            const u32x4 pf = {pw[4 * (i >> 2)], pw[4 * (i >> 2) + 1], pw[4 * (i >> 2) + 2], pw[4 * (i >> 2) + 3]};
            acc[i & 3] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, __builtin_bit_cast(f16x8, pf), acc[i & 3], 0, 0, 0);
        };
        // Stage t: the scores of half t + 1 (nxt) and the outputs of half t - 1 (weights pp) beside the weights of
        // half t (scores cur, weights pc).  ks, vs: slots of K t + 1 and V t - 1; f: the first operands of K t + 1,
        // then those of K t + 2 in slot `then` (-1: not there yet); mx: the lane's part of the maximum of cur, then of
        // nxt; parts: the first of the four parts of `job` that the stage asks for.  Each MFMA is fenced
        // together with its share of the vector work: left alone, the scheduler puts all of the one before all of
        // the other.
        constexpr int AHEAD = 4;  // operand reads in flight before their MFMA
        f16x8 f[AHEAD];
        // In the P stages from t on K of the halves t + P + 1 .. t + 2 P and V of t + P - 1 .. t + 2 P - 2 come in, a
        // half by each wave.
        static_assert(WAVES == 2 * P, "a half of K or V for each wave");
        const bool loads_v = wave < P;
        auto job_at = [&](int t) __attribute__((always_inline)) { return job_of(t + P + (loads_v ? wave - 1 : wave - P + 1), loads_v); };
        auto first_k = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) f[i] = read_k(slot, i);
        };
        auto stage = [&](int t, int ks, int vs, int then, const Job& job, auto parts, const f32x16& cur, f32x16& nxt, uint32_t (&pc)[8], uint32_t (&pp)[8],
                         float& mx) __attribute__((always_inline)) {
            constexpr int first_part = decltype(parts)::value;
            float ps[3] = {0.0f, 0.0f, 0.0f}, neg = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                times_q(f[i % AHEAD], i, nxt);
                f[i % AHEAD] = i + AHEAD < 8 ? read_k(ks, i + AHEAD) : read_v(vs, i + AHEAD - 8);
                if (i == 1) {
                    __builtin_amdgcn_sched_barrier(0);
                    renew_ref(xor32_max(mx) * kPgScale, pp);  // (scaling is monotonic)
                    neg = mref == -INFINITY ? 0.0f : -mref;   // masked scores give exp2(-inf) = 0
                }
                if (i & 1) pc[i >> 1] = weights(cur, i >> 1, neg, ps);
                if (i == 4 && first_part + 0 < 8) load_part(job, first_part + 0);
                if (i == 7 && first_part + 1 < 8) load_part(job, first_part + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            mask(t + 1, nxt);
            mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                add_pv(f[i % AHEAD], i, pp);
                if (i + AHEAD < 8) f[i % AHEAD] = read_v(vs, i + AHEAD);
                else if (then >= 0) f[i % AHEAD] = read_k(then, i + AHEAD - 8);
                if (i & 1) pc[4 + (i >> 1)] = weights(cur, 4 + (i >> 1), neg, ps);
                if (i >= 2) mx = i < 6 ? max_of(nxt, 3 * (i - 2), 3, mx) : max_of(nxt, 12 + 2 * (i - 6), 2, mx);
                if (i == 2 && first_part + 2 < 8) load_part(job, first_part + 2);
                if (i == 5 && first_part + 3 < 8) load_part(job, first_part + 3);
                __builtin_amdgcn_sched_barrier(0);
            }
            lsum += ps[0] + ps[1];
            lround += ps[2];
        };
        // The same where the wave has no half t + 1, or none of the others.
        const int mine = wave_last < key0 ? 0 : min(halves, (wave_last - key0) / kPfHalf + 1);  // its halves
        auto last_stage = [&](int t, int ks, int vs, const f32x16& cur, f32x16& nxt, uint32_t (&pc)[8], uint32_t (&pp)[8],
                              float& mx) __attribute__((always_inline)) {
            if (t < mine) renew_ref(xor32_max(mx) * kPgScale, pp);
            if (t + 1 < mine) {
#pragma unroll
                for (int i = 0; i < 8; ++i) times_q(read_k(ks, i), i, nxt);
                mask(t + 1, nxt);
                mx = max_of(nxt, 0, 16, -INFINITY);
            }
            if (t > 0 && t - 1 < mine) {
#pragma unroll
                for (int i = 0; i < 8; ++i) add_pv(read_v(vs, i), i, pp);
            }
            if (t < mine) {
                const float neg = mref == -INFINITY ? 0.0f : -mref;
                float ps[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 8; ++i) pc[i] = weights(cur, i, neg, ps);
                lsum += ps[0] + ps[1];
                lround += ps[2];
            }
        };
        if (it0 < it1) {
            f32x16 s0, s1;
            uint32_t p0[8] = {}, p1[8] = {};
            float mx = -INFINITY;
            request_entries(entry_of(0));
            take_entries();
            if (wave == 0) load_half(0, false);
            load_half(loads_v ? wave - 1 : wave - P + 1, loads_v);
            tile_barrier();
            if (mine > 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) times_q(read_k(0, i), i, s0);
                mask(0, s0);
                mx = max_of(s0, 0, 16, -INFINITY);
            }
            tile_barrier();  // K's slot 0 is read
            // P stages from t on between two barriers.  A wave asks for the parts of its half one by one within the
            // first stages (in one go, and with an address for each part of every half, the loads held the waves up
            // for a third of the time), which leaves them time to come in.  Halves past the wave's last key are not
            // multiplied.
            auto entries = [&](int t) __attribute__((always_inline)) {
                if (__builtin_expect(next_base >= 0, 0)) take_entries();
                if (__builtin_expect(entry_of(t + 3 * P) + NP > base + 64, 0)) request_entries(entry_of(t + P + 1));  // for the next time
            };
            typedef std::integral_constant<int, 0> first;
            typedef std::integral_constant<int, 4> second;
            typedef std::integral_constant<int, 8> none;
            int t = 0;
            for (; t + P < mine; t += P) {
                entries(t);
                first_k(1);
                const Job job = job_at(t);
                if constexpr (P == 4) {
                    stage(t, 1, 3, 2, job, first{}, s0, s1, p0, p1, mx);
                    turn_v();
                    stage(t + 1, 2, 0, 3, job, second{}, s1, s0, p1, p0, mx);
                    stage(t + 2, 3, 1, -1, job, none{}, s0, s1, p0, p1, mx);
                    turn_k();  // K t + P lies in the other frame
                    first_k(0);
                    stage(t + 3, 0, 2, -1, job, none{}, s1, s0, p1, p0, mx);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) load_part(job, i);
                    stage(t, 1, 1, -1, job, second{}, s0, s1, p0, p1, mx);
                    turn_v();
                    turn_k();
                    first_k(0);
                    stage(t + 1, 0, 0, -1, job, none{}, s1, s0, p1, p0, mx);
                }
                tile_barrier();
            }
            for (; t <= halves; t += P) {
                entries(t);
                const Job job = job_at(t);
#pragma unroll
                for (int i = 0; i < 8; ++i) load_part(job, i);
#pragma unroll
                for (int j = 0; j < P; j += 2) {
                    last_stage(t + j, j + 1, j == 0 ? P - 1 : j - 1, s0, s1, p0, p1, mx);
                    if (j == 0) turn_v();
                    if (j + 1 == P - 1) turn_k();
                    last_stage(t + j + 1, j + 1 == P - 1 ? 0 : j + 2, j, s1, s0, p1, p0, mx);
                }
                tile_barrier();
            }
        }
        lsum += __shfl_xor(lsum, 32);
        lround += __shfl_xor(lround, 32);
        const int other_any = __shfl_xor(static_cast<int>(any), 32);  // (asked by all lanes)
        if (any || other_any != 0) mref = fmaxf(mref, kPgLowest);
        if (r < rows) {
            if (slot < 0) {
                const float inv = row_inverse(mref, lround);
                const size_t at = static_cast<size_t>(s.first + qi) * p.nq + qh;
                uint16_t* o = p.out + at * kPgDim;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                    for (int g = 0; g < 4; ++g)  // dims 32dt + 8g + 4h .. +3
                        *reinterpret_cast<uint2*>(o + 32 * dt + 8 * g + 4 * h) =
                            pack4(acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv, acc[dt][4 * g + 3] * inv);
                if (p.lse != nullptr && h == 0) p.lse[at] = row_log_sum(mref, lsum);
            } else {
                const size_t at = static_cast<size_t>(2 * block + slot) * kRows + wave * 32 + fr;
                if (h == 0) part.ml[at] = make_float2(mref, lsum);
                const float even = lround > 0.0f ? lsum / lround : 1.0f;  // the merge divides by sums of lsum
                float* po = part.o + at * kPgDim;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<float4*>(po + 32 * dt + 8 * g + 4 * h) =
                            make_float4(acc[dt][4 * g] * even, acc[dt][4 * g + 1] * even, acc[dt][4 * g + 2] * even, acc[dt][4 * g + 3] * even);
            }
        }
        tile_barrier();  // the tiles are read: the next segment fills them
    };
    auto rows = [&](const PagedSeq& s, int, int rt) __attribute__((always_inline)) { return min(kRows, s.n * p.group - rt * kRows); };
    for_share<false>(p.c, block, kBlocks, max(1, p.group * kLeastTiles * kPfKeys >> p.coarse), work, tiles, rows, body,
                     [&](SegmentCut cut) {
                         if (threadIdx.x == 0) part.cuts[block] = cut;
                     });
}

template <int WAVES, int GROUPS>
__global__ __launch_bounds__(256) void paged_prefill_merge_kernel(PrefillParams p) {
    typedef PrefillShape<WAVES> Shape;
    static_assert(Shape::blocks <= kMergeCuts, "a cut for each block");
    merge_parts<Shape::rows, GROUPS, 256>(p.ws, Shape::blocks, p.out, p.lse, p.nq, [&](const SegmentCut& c) {
        return RowMap{paged_seq(p.c, c.item).first, c.row_tile * Shape::rows, p.group, c.head * p.group};
    });
}

// The checks that the attention entry points share.
int check_attention(const char* what, const uint16_t* q, const qe_paged_cache* cache, const qe_paged_batch* batch,
                    uint16_t* attn_out, float* row_lse, void* workspace, size_t workspace_bytes, const int32_t* selected,
                    int num_q_heads, int num_selected) {
    QE_REQUIRE(q && attn_out && workspace, "%s: NULL pointer", what);
    QE_REQUIRE(aligned(q, 16) && aligned(attn_out, 8) && aligned(workspace, 16) && aligned(row_lse, 4) &&
                   aligned(selected, 4),
               "%s: q and the workspace must be 16-byte and attn_out 8-byte aligned", what);
    const size_t n = batch->num_tokens, q_bytes = 2 * n * num_q_heads * kPgDim;
    const PagedSpan spans[] = {{attn_out, q_bytes, "attn_out"},
                               {row_lse, 4 * n * num_q_heads, "row_lse"},
                               {workspace, workspace_bytes, "the workspace"},
                               {q, q_bytes, "q"},
                               {selected, 4 * n * cache->num_kv_heads * num_selected, "selected"},
                               paged_k_span(cache),
                               paged_v_span(cache),
                               paged_table_span(batch),
                               paged_starts_span(batch),
                               paged_context_span(batch)};
    return paged_check_apart(what, spans, 3);
}

template <bool SPARSE>
int launch_decode(const char* what, const uint16_t* q, const qe_paged_cache* cache, const qe_paged_batch* batch,
                  const int32_t* selected, uint16_t* attn_out, float* row_lse, void* workspace, hipStream_t stream,
                  int num_q_heads, int window, int num_selected) {
    DecodeParams p{};
    QE_TRY(paged_check(what, cache, batch, &p.c));
    QE_TRY(paged_check_heads(what, cache, num_q_heads));
    if (batch->num_tokens == 0 || batch->num_seqs == 0) return QE_OK;
    QE_REQUIRE(selected || !SPARSE, "%s: NULL pointer", what);
    QE_TRY(check_attention(what, q, cache, batch, attn_out, row_lse, workspace, partials_bytes<kDecRows>(kDecBlocks),
                           selected, num_q_heads, num_selected));
    p.q = q;
    p.selected = selected;
    p.out = attn_out;
    p.lse = row_lse;
    p.ws = workspace;
    p.nq = num_q_heads;
    p.group = num_q_heads / cache->num_kv_heads;
    p.window = window;
    p.num_selected = num_selected;
    const long long row_tiles = (p.group + kDecRows - 1) / kDecRows;
    const long long most = SPARSE ? static_cast<long long>(num_selected) * cache->page_size
                                  : static_cast<long long>(batch->max_pages) * cache->page_size;
    const long long segments = row_tiles * cache->num_kv_heads * batch->num_tokens;
    const long long keys = window > 0 ? std::min<long long>(window, most) : most;
    if ((keys <= kShortKeys || (segments >= kManySegments && (SPARSE || keys <= 2 * kShortKeys))) &&
        segments < (1 << 24)) {  // (a launch has fewer than 2^32 threads)
        paged_short_kernel<SPARSE><<<static_cast<unsigned>(segments), 64 * kShortWaves, 0, stream>>>(p);
        return check_launch(what);
    }
    while (segments * (((most / kDecKeys + 1) >> p.coarse) + kDecOver) >= (1 << 30)) {
        QE_REQUIRE(most / kDecKeys >> p.coarse > 0, "%s: num_tokens=%d with %d kv heads", what, batch->num_tokens,
                   cache->num_kv_heads);
        ++p.coarse;
    }
    paged_decode_kernel<SPARSE><<<kDecBlocks, 64 * kDecWaves, 0, stream>>>(p);
    // Few segments have many parts each: a block a row, 32 parts at once.  (131000 keys, 12 heads: 5.8 us, with two
    // rows a block 8.2; 48 sequences 13.1 and 5.)
    const long long cuts = std::min<long long>(segments, kDecBlocks);
    if (segments < 16)
        paged_decode_merge_kernel<SPARSE, 32, 1024><<<static_cast<unsigned>(cuts * std::min(p.group, kDecRows)), 1024, 0, stream>>>(p);
    else
        paged_decode_merge_kernel<SPARSE, 4, 256><<<static_cast<unsigned>(cuts * ((std::min(p.group, kDecRows) + 1) / 2)), 256, 0, stream>>>(p);
    return check_launch(what);
}

constexpr size_t prefill_bytes() {
    return std::max(partials_bytes<PrefillShape<4>::rows>(PrefillShape<4>::blocks),
                    partials_bytes<PrefillShape<8>::rows>(PrefillShape<8>::blocks));
}

template <int WAVES>
int launch_prefill(PrefillParams p, const qe_paged_batch* batch, const qe_paged_cache* cache, hipStream_t stream,
                   const char* what) {
    typedef PrefillShape<WAVES> Shape;
    const long long row_tiles = static_cast<long long>(batch->num_tokens) * p.group / Shape::rows + batch->num_seqs;
    const long long most = static_cast<long long>(p.group) * (static_cast<long long>(batch->max_pages) * cache->page_size + kPfOver);
    while (row_tiles * cache->num_kv_heads > ((1LL << 30) - 1) / ((most >> p.coarse) + 1)) {
        QE_REQUIRE(most >> p.coarse > 0, "%s: num_tokens=%d with %d kv heads", what, batch->num_tokens, cache->num_kv_heads);
        ++p.coarse;
    }
    const bool one = p.c.shift >= 5, few = batch->num_seqs > 1 || batch->num_tokens * p.group <= kDecRows;
    auto* kernel = one ? few ? paged_prefill_kernel<true, WAVES, true> : paged_prefill_kernel<true, WAVES, false>
                       : few ? paged_prefill_kernel<false, WAVES, true> : paged_prefill_kernel<false, WAVES, false>;
    kernel<<<Shape::blocks, 64 * WAVES, 0, stream>>>(p);
    // As many blocks as fit the chip at once: each counts the cuts again (mixed batch 12.8 us, with 512 18, with 2048 15).
    // Where four times as many are no more, and rows may have more parts than a wave asks for at once, four groups of
    // lanes share a row's (in all, us: 17 tokens at 1200 20.6 and 21.8, 64 at 100000 81 and 95; 200 at 8000, which
    // are too many, 41.5 and 39.4; 40 at 0 14.3 and 13.7).
    const long long items = std::min<long long>(row_tiles * cache->num_kv_heads, Shape::blocks) * (Shape::rows / 8);
    if (4 * items <= kMergeBlocks && static_cast<long long>(batch->max_pages) * cache->page_size > 8 * kLeastTiles * kPfKeys)
        paged_prefill_merge_kernel<WAVES, 4><<<static_cast<unsigned>(4 * items), 256, 0, stream>>>(p);
    else
        paged_prefill_merge_kernel<WAVES, 1><<<static_cast<unsigned>(std::min(items, kMergeBlocks)), 256, 0, stream>>>(p);
    return QE_OK;
}

}  // namespace
}  // namespace qe

using namespace qe;

extern "C" int qe_paged_decode_workspace_bytes(int num_tokens, int num_q_heads, int num_kv_heads, size_t* bytes) {
    QE_REQUIRE(bytes, "paged_decode_workspace_bytes: NULL pointer");
    QE_REQUIRE(num_tokens >= 0 && num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
               "paged_decode_workspace_bytes: num_tokens=%d, %d q heads over %d kv heads", num_tokens, num_q_heads,
               num_kv_heads);
    *bytes = partials_bytes<kDecRows>(kDecBlocks);
    clear_error();
    return QE_OK;
}

extern "C" int qe_launch_attention_gqa_paged_decode(const uint16_t* q, const qe_paged_cache* cache,
                                                    const qe_paged_batch* batch, void* workspace, uint16_t* attn_out,
                                                    float* row_lse, hipStream_t stream, int num_q_heads, int window) {
    const char* what = "attention_gqa_paged_decode";
    QE_REQUIRE(batch == nullptr || batch->query_start == nullptr, "%s: query_start is for chunks", what);
    QE_REQUIRE(window >= 0, "%s: window=%d", what, window);
    return launch_decode<false>(what, q, cache, batch, nullptr, attn_out, row_lse, workspace, stream, num_q_heads, window, 0);
}

extern "C" int qe_launch_attention_gqa_paged_sparse(const uint16_t* q, const qe_paged_cache* cache,
                                                    const qe_paged_batch* batch, const int32_t* selected, void* workspace,
                                                    uint16_t* attn_out, float* row_lse, hipStream_t stream,
                                                    int num_q_heads, int num_selected) {
    const char* what = "attention_gqa_paged_sparse";
    QE_REQUIRE(num_selected > 0 && num_selected <= (1 << 20), "%s: num_selected=%d", what, num_selected);
    QE_REQUIRE(!cache || !batch || static_cast<long long>(batch->num_tokens) * cache->num_kv_heads <= (1 << 30),
               "%s: num_tokens=%d", what, batch->num_tokens);
    return launch_decode<true>(what, q, cache, batch, selected, attn_out, row_lse, workspace, stream, num_q_heads, 0,
                               num_selected);
}

extern "C" int qe_paged_prefill_workspace_bytes(int num_tokens, int num_q_heads, int num_kv_heads, size_t* bytes) {
    QE_REQUIRE(bytes, "paged_prefill_workspace_bytes: NULL pointer");
    QE_REQUIRE(num_tokens >= 0 && num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
               "paged_prefill_workspace_bytes: num_tokens=%d, %d q heads over %d kv heads", num_tokens, num_q_heads,
               num_kv_heads);
    *bytes = prefill_bytes();
    clear_error();
    return QE_OK;
}

extern "C" int qe_launch_attention_gqa_paged_prefill(const uint16_t* q, const qe_paged_cache* cache,
                                                     const qe_paged_batch* batch, void* workspace, uint16_t* attn_out,
                                                     float* row_lse, hipStream_t stream, int num_q_heads, int window) {
    const char* what = "attention_gqa_paged_prefill";
    PrefillParams p{};
    QE_TRY(paged_check(what, cache, batch, &p.c));
    QE_TRY(paged_check_heads(what, cache, num_q_heads));
    QE_REQUIRE(window >= 0, "%s: window=%d", what, window);
    if (batch->num_tokens == 0 || batch->num_seqs == 0) return QE_OK;
    QE_TRY(check_attention(what, q, cache, batch, attn_out, row_lse, workspace, prefill_bytes(), nullptr,
                           num_q_heads, 0));
    p.q = q;
    p.out = attn_out;
    p.lse = row_lse;
    p.ws = workspace;
    p.nq = num_q_heads;
    p.group = num_q_heads / cache->num_kv_heads;
    p.window = window;
    // Blocks of eight waves read K and V once for 256 rows, those of four waves waste less on sequences of few rows
    // (2048 rows at 14000: 213 and 234 us; 40 single tokens and three prompts: 64 and 54).
    if (static_cast<long long>(batch->num_tokens) * p.group >= 512LL * batch->num_seqs)
        QE_TRY(launch_prefill<8>(p, batch, cache, stream, what));
    else
        QE_TRY(launch_prefill<4>(p, batch, cache, stream, what));
    return check_launch(what);
}
