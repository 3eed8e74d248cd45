// The 4-bit key/value cache: layout of a row, its expansion to fp16, and the
// position bookkeeping that append, attention and eviction share.
//
// A row is one head's 128 values of one token in 80 bytes: sixteen 32-bit words
// of eight nibbles, then four (scale, low) pairs of fp16, one for every 32
// elements.  Element 8 w + j is the nibble of word w at bit 16 (j % 2) + 4 (j / 2):
// the two halves of a word masked with 0x000F are elements 8 w and 8 w + 1, an
// fp16 pair in element order after the bias trick below.  A nibble n stands
// for fp16(n * scale + low), one rounding.
//
// 5 bits a value, 3.2 times less than fp16.  Groups of 32 and an offset: a head's
// keys differ in level from channel to channel, and the step of a group is a
// fifteenth of its own spread.
//
// A token whose K or V holds an infinity or NaN (also one that fp16 cannot
// hold) is stored with NaN (scale, low) in its K row and zeros in its V row: who
// attends to it gets NaN, and who does not, not: its score is replaced by the
// mask, and its V row adds 0 * 0.
#pragma once

#include "qe_common.hpp"

namespace qe {

constexpr int kKv4Dim = 128;                     // head dimension
constexpr int kKv4Row = QE_KV4_ROW_BYTES;        // bytes of a row
constexpr int kKv4Params = 64;                   // byte offset of its (scale, low) pairs
static_assert(kKv4Row == kKv4Params + 16, "row layout");

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Nibble i of both halves of t, expanded with the halves' own scale and low:
// out[i] = {half 0's, half 1's}.  0x6400 | n is the fp16 1024 + n, and 0x6400 |
// n << 4 is 1024 + 16 n; both come back to n exactly, so the only rounding is the
// last operation's.
__device__ __forceinline__ void kv4_expand(uint32_t t, f16x2 scale, f16x2 low, f16x2 (&out)[4]) {
    const f16x2 b1 = {(_Float16)-1024.0f, (_Float16)-1024.0f};
    const f16x2 r16 = {(_Float16)0.0625f, (_Float16)0.0625f}, b16 = {(_Float16)-64.0f, (_Float16)-64.0f};
    // masks and bias in registers: as literals they would make the and and the or two instructions
    uint32_t even = 0x000F000Fu, odd = 0x00F000F0u, bias = 0x64006400u;
    asm("" : "+s"(even));
    asm("" : "+s"(odd));
    asm("" : "+v"(bias));
    const uint32_t t8 = t >> 8;
    const uint32_t u[4] = {(t & even) | bias, (t & odd) | bias, (t8 & even) | bias, (t8 & odd) | bias};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2 x = __builtin_bit_cast(f16x2, u[i]);
        const f16x2 n = i & 1 ? __builtin_elementwise_fma(x, r16, b16) : x + b1;
        out[i] = __builtin_elementwise_fma(n, scale, low);
    }
}

// The eight elements of one word, in order; param = scale | low << 16.
__device__ __forceinline__ f16x8 kv4_expand_word(uint32_t w, uint32_t param) {
    const uint32_t s = __builtin_amdgcn_perm(param, param, 0x01000100u);  // scale twice
    const uint32_t l = __builtin_amdgcn_perm(param, param, 0x03020302u);  // low twice
    f16x2 o[4];
    kv4_expand(w, __builtin_bit_cast(f16x2, s), __builtin_bit_cast(f16x2, l), o);
    return f16x8{o[0].x, o[0].y, o[1].x, o[1].y, o[2].x, o[2].y, o[3].x, o[3].y};
}

// `rows` rows of a cache from `first` on, for loads by byte offset: what lies
// behind them reads as zeros, whose value is 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv4_rows(const uint8_t* first, int rows) {
    // (both are the same in every lane; said again, or each load becomes a loop over lanes)
    const uintptr_t at = reinterpret_cast<uintptr_t>(first);
    const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at)));
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32)));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<uint8_t*>(lo | (hi << 32)), 0,
                                             __builtin_amdgcn_readfirstlane(max(rows, 0) * kKv4Row), 0x00027000);
}
__device__ __forceinline__ uint32_t kv4_load(__amdgpu_buffer_rsrc_t rows, uint32_t offset) {
    return __builtin_amdgcn_raw_buffer_load_b32(rows, offset, 0, 0);
}
__device__ __forceinline__ u32x4 kv4_load4(__amdgpu_buffer_rsrc_t rows, uint32_t offset) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, 0));
}

// Cache row of position seq_pos for kv head h: the positions before it, less
// those evicted; never negative (a count beyond the position is taken as all).
__device__ __forceinline__ int kv4_row(const qe_device_control_block* ctl, const int32_t* evicted, int h) {
    const int pos = ctl != nullptr ? ctl->seq_pos : 0;
    const int gone = evicted != nullptr ? evicted[h] : 0;
    return max(pos - gone, 0);
}

// two buffers share no byte
inline bool apart(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x + a_bytes <= y || y + b_bytes <= x;
}

// Checks that every entry point on the caches makes.
inline int kv4_check(const char* what, const void* kc, const void* vc, int num_kv_heads, int head_dim,
                     int max_seq_len) {
    QE_REQUIRE(kc && vc, "%s: NULL pointer", what);
    QE_REQUIRE(head_dim == kKv4Dim, "%s: head_dim=%d (only 128 is built)", what, head_dim);
    QE_REQUIRE(num_kv_heads > 0 && max_seq_len > 0, "%s: num_kv_heads=%d max_seq_len=%d", what, num_kv_heads,
               max_seq_len);
    QE_REQUIRE(aligned(kc, 16) && aligned(vc, 16), "%s: the caches must be 16-byte aligned", what);
    return QE_OK;
}

}  // namespace qe
