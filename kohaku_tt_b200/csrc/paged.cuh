// Pages of keys and values, in bf16 or 4 bits, as the append, read and attention kernels address them.
//
// bf16: rows of D values, [pages, kv heads, page size, D] with any strides.
// 4 bits: per 16 tokens of a head one block of 9 D bytes: 16 D / 2 bytes of codes, then per token D / 64 words, one for
// each group of 64 channels: (step, least value) as bf16 from the low half up. A code c is worth least + step c.
// Eight channels 8 x .. 8 x + 7 share a 32-bit word: channel e of them at nibble (e >> 1) + 4 (e & 1), so that
// (word >> 4 n) & 0x000f000f holds channels 2 n and 2 n + 1 as the two halves of a register: one shift and one
// logic operation make a pair of bf16 values 128 + c of them.
//   keys: a token's words lie together, the word of channels 32 i + 8 t .. at place t D / 32 + i: thread t of the four
//         that share a row of a matrix instruction's operand reads all of its words in one piece.
//   values: the words of channels 8 g .. (and of 64 + 8 g ..) of two neighbouring tokens lie together, for token pair
//         p at place g ^ (2 (p & 3)) (D 128) or g ^ (4 ((p >> 1) & 1)) (D 64): thread (g, t) reads both tokens' words in
//         one piece, and the 32 threads read different banks.
#pragma once
#include "common.cuh"

namespace ktt {

// Word of (token 0-15 of a block, channels 8 x ..) from the block's start.
template <int D>
__host__ __device__ __forceinline__ int key_word(int token, int x) {
    return token * (D / 8) + (x & 3) * (D / 32) + (x >> 2);
}
template <int D>
__host__ __device__ __forceinline__ int value_word(int token, int x) {
    constexpr int G = D / 64;
    const int pair = token >> 1, g = x & 7;
    const int place = g ^ (D == 128 ? 2 * (pair & 3) : 4 * ((pair >> 1) & 1));
    return (pair * 8 + place) * (2 * G) + (token & 1) * G + (x >> 3);
}
template <int D>
__host__ __device__ __forceinline__ int step_word(int token, int group) {
    return 16 * (D / 8) + token * (D / 64) + group;
}

__device__ __forceinline__ float step_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float least_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// A paged cache: byte strides; pages outside [0, pages) are no pages (append: the rows go nowhere; read and
// attention: zeros).
struct Pages {
    unsigned char* k;
    unsigned char* v;
    int64_t ks[3], vs[3];   // (page, head, row) in bytes; 4 bits: the row stride is not used
    const int32_t* table;   // [batch][table_stride]
    int64_t table_stride;
    const int32_t* lengths;
    int64_t pages;
    int page_size, cap;     // cap: keys that a sequence may have
};

__device__ __forceinline__ int cached_keys(const Pages& c, int b) {
    const int n = c.lengths[b];
    return n < 0 ? 0 : (n > c.cap ? c.cap : n);
}
// Page of key j of batch entry b, or -1.
__device__ __forceinline__ int64_t page_of(const Pages& c, int b, int j) {
    const int64_t page = c.table[b * c.table_stride + j / c.page_size];
    return page >= 0 && page < c.pages ? page : -1;
}

// Fills the cache's fields from an argument block after its checks (paged.cu); null, or why not.
const char* pages_of(Pages& c, const ktt_b200_pages& a, int d);

}  // namespace ktt
