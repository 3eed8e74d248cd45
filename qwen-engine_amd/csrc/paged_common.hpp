// The paged key/value cache: what a kernel needs of its descriptions, the
// sequences and rows of a batch, and the checks that its entry points share.
#pragma once

#include <algorithm>
#include <type_traits>

#include "kv4_common.hpp"

namespace qe {

constexpr int kPgDim = 128;  // head dimension

// qe_paged_cache and qe_paged_batch as kernels take them.
struct PagedView {
    const uint16_t* k;
    const uint16_t* v;
    long long page_stride;
    const int32_t* table;
    const int32_t* starts;  // NULL: a row for each sequence
    const int32_t* ctx;
    int num_pages, shift, nkv, seqs, rows, max_pages;  // a page has 1 << shift tokens

    __device__ __forceinline__ int page_size() const { return 1 << shift; }
    __device__ __forceinline__ int capacity() const { return max_pages << shift; }
};

// A sequence of the batch: rows [first, first + n), the first at position ctx.
// n = 0 where there is nothing to do.  Whatever the arrays hold, the rows are
// within the batch and the positions below 2^31.
struct PagedSeq {
    int first, n, ctx;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedView& p, int s) {
    PagedSeq q{s, 1, p.ctx[s]};
    if (p.starts != nullptr) {
        q.first = min(max(p.starts[s], 0), p.rows);
        q.n = max(min(p.starts[s + 1], p.rows) - q.first, 0);
    }
    if (q.ctx < 0) q.n = 0;
    q.ctx = min(max(q.ctx, 0), INT32_MAX - p.rows);
    return q;
}

// The sequence of a row, -1 for a row of none: the last one that starts at or
// before it.  By all lanes of a wave for one row: 64 places are looked at in one
// round of loads, so 64 sequences take one and 4096 two.
__device__ __forceinline__ int paged_seq_of_row(const PagedView& p, int row) {
    if (p.starts == nullptr) return row;
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = p.seqs;  // the answer is lo - 1 or in [lo, hi)
    while (lo < hi) {
        const int step = (hi - lo + 63) >> 6, at = lo + lane * step;
        const int below = __popcll(__builtin_amdgcn_ballot_w64(at < hi && p.starts[min(at, p.seqs - 1)] <= row));
        if (below == 0) break;
        const int found = lo + (below - 1) * step;
        hi = min(hi, found + step);
        lo = found + 1;
    }
    return lo - 1;
}

// Page of a sequence's block, -1 where it has none.
__device__ __forceinline__ int paged_page(const PagedView& p, int seq, int block) {
    if (block >= p.max_pages) return -1;
    const int at = p.table[static_cast<size_t>(seq) * p.max_pages + block];
    return at >= 0 && at < p.num_pages ? at : -1;
}

// Sum over a wave up to and with each lane, in the vector unit: 1, 2, 4 and 8 lanes on within rows
// of 16, then the rows' sums.
__device__ __forceinline__ int wave_scan(int x) {
    auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    };
    typedef std::integral_constant<int, 0xF> all;
    add(std::integral_constant<int, 0x111>{}, all{});
    add(std::integral_constant<int, 0x112>{}, all{});
    add(std::integral_constant<int, 0x114>{}, all{});
    add(std::integral_constant<int, 0x118>{}, all{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row 15's and 47's sum
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row 31's
    return x;
}

// ---- host: checks -------------------------------------------------------------
struct PagedSpan {
    const void* at;
    size_t bytes;
    const char* name;
    int kin = 0;  // two of the same kind (not 0) may share memory: they are compared elsewhere
};

inline long long paged_page_elements(const qe_paged_cache* c) {
    return static_cast<long long>(c->num_kv_heads) * c->page_size * kPgDim;
}
inline long long paged_stride(const qe_paged_cache* c) {
    return c->page_stride == 0 ? paged_page_elements(c) : c->page_stride;
}
// bytes from the first page's first to the last page's last
inline size_t paged_pool_bytes(const qe_paged_cache* c) {
    return 2 * (static_cast<size_t>(c->num_pages - 1) * paged_stride(c) + paged_page_elements(c));
}

// Checks of the descriptions and of the heads; fills the kernels' view.
inline int paged_check(const char* what, const qe_paged_cache* c, const qe_paged_batch* b, PagedView* out) {
    QE_REQUIRE(c && b, "%s: NULL cache or batch", what);
    // (a batch of no sequences has empty arrays)
    QE_REQUIRE(c->k && c->v && (b->num_seqs == 0 || (b->block_table && b->context_len)),
               "%s: NULL pointer in the cache or the batch", what);
    QE_REQUIRE(c->head_dim == kPgDim, "%s: head_dim=%d (only 128 is built)", what, c->head_dim);
    QE_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128 ||
                   c->page_size == 256,
               "%s: page_size=%d (16, 32, 64, 128 or 256)", what, c->page_size);
    QE_REQUIRE(c->num_pages > 0 && c->num_kv_heads > 0 && c->num_kv_heads <= 1024, "%s: num_pages=%d num_kv_heads=%d",
               what, c->num_pages, c->num_kv_heads);
    QE_REQUIRE(paged_stride(c) >= paged_page_elements(c) && paged_stride(c) % 8 == 0 &&
                   paged_stride(c) <= (1LL << 40),
               "%s: page_stride=%lld (at least %lld, a multiple of 8)", what, c->page_stride, paged_page_elements(c));
    QE_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), "%s: the pages must be 16-byte aligned", what);
    QE_REQUIRE(b->num_seqs >= 0 && b->num_tokens >= 0 && b->max_pages > 0, "%s: num_seqs=%d num_tokens=%d max_pages=%d",
               what, b->num_seqs, b->num_tokens, b->max_pages);
    QE_REQUIRE(b->num_tokens < (1 << 24) && b->num_seqs < (1 << 24), "%s: num_tokens=%d num_seqs=%d (below 2^24)",
               what, b->num_tokens, b->num_seqs);
    QE_REQUIRE(static_cast<long long>(b->max_pages) * c->page_size <= (1LL << 30),
               "%s: max_pages=%d pages of %d tokens (2^30 positions at most)", what, b->max_pages, c->page_size);
    QE_REQUIRE(b->query_start != nullptr || b->num_tokens == b->num_seqs,
               "%s: num_tokens=%d for %d sequences without query_start", what, b->num_tokens, b->num_seqs);
    QE_REQUIRE(aligned(b->block_table, 4) && aligned(b->context_len, 4) && aligned(b->query_start, 4),
               "%s: the batch's arrays must be 4-byte aligned", what);
    int shift = 4;
    while ((1 << shift) < c->page_size) ++shift;
    *out = PagedView{c->k, c->v, paged_stride(c), b->block_table, b->query_start, b->context_len,
                     c->num_pages, shift, c->num_kv_heads, b->num_seqs, b->num_tokens, b->max_pages};
    return QE_OK;
}

inline int paged_check_heads(const char* what, const qe_paged_cache* c, int num_q_heads) {
    QE_REQUIRE(num_q_heads > 0 && num_q_heads % c->num_kv_heads == 0 && num_q_heads / c->num_kv_heads <= 64,
               "%s: %d q heads over %d kv heads (at most 64 each)", what, num_q_heads, c->num_kv_heads);
    return QE_OK;
}

// What a launch writes (the first `written` spans, NULL ones skipped) shares no
// memory with anything else it is given.
template <int N>
int paged_check_apart(const char* what, const PagedSpan (&spans)[N], int written) {
    for (int i = 0; i < written; ++i)
        for (int j = 0; j < N; ++j)
            if ((j >= written || j > i) && spans[i].at && spans[j].at && spans[i].bytes && spans[j].bytes &&
                (spans[i].kin == 0 || spans[i].kin != spans[j].kin))
                QE_REQUIRE(apart(spans[i].at, spans[i].bytes, spans[j].at, spans[j].bytes), "%s: %s overlaps %s", what,
                           spans[i].name, spans[j].name);
    return QE_OK;
}
inline PagedSpan paged_k_span(const qe_paged_cache* c) { return {c->k, paged_pool_bytes(c), "the K pages", 1}; }
inline PagedSpan paged_v_span(const qe_paged_cache* c) { return {c->v, paged_pool_bytes(c), "the V pages", 1}; }
// K and V pages: two pools, or taking turns in one.
inline int paged_check_pools(const char* what, const qe_paged_cache* c) {
    if (apart(c->k, paged_pool_bytes(c), c->v, paged_pool_bytes(c))) return QE_OK;
    const long long page = 2 * paged_page_elements(c), stride = 2 * paged_stride(c);
    const long long off = static_cast<long long>(reinterpret_cast<uintptr_t>(c->v) - reinterpret_cast<uintptr_t>(c->k));
    const long long turn = ((off % stride) + stride) % stride;
    QE_REQUIRE(turn >= page && turn <= stride - page, "%s: the K pages overlap the V pages", what);
    return QE_OK;
}
inline PagedSpan paged_table_span(const qe_paged_batch* b) {
    return {b->block_table, 4 * static_cast<size_t>(b->num_seqs) * b->max_pages, "block_table"};
}
inline PagedSpan paged_starts_span(const qe_paged_batch* b) {
    return {b->query_start, 4 * (static_cast<size_t>(b->num_seqs) + 1), "query_start"};
}
inline PagedSpan paged_context_span(const qe_paged_batch* b) {
    return {b->context_len, 4 * static_cast<size_t>(b->num_seqs), "context_len"};
}

}  // namespace qe
