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

// The sequence of packed row n, or -1: offsets do not decrease, sequences may be empty.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int batch, int64_t n) {
    if (n < cu[0] || n >= cu[batch]) return -1;
    int lo = 0, hi = batch - 1;   // the last b with cu[b] <= n
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= n) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// What the chunk path needs behind its dense rows (int32 words): a work counter and, from word 1, the parts that tiles are cut
// into and the keys of a part; from kHeadWords the offsets of the dense rows (batch + 1), the sequences by falling length (batch),
// and for packed queries their offsets (batch + 1), none of them outside of the rows there are.
constexpr int kHeadWords = 64;
__host__ __device__ constexpr int64_t head_words(int64_t batch) { return kHeadWords + 3 * batch + 2; }
struct ChunkHead {
    int32_t* words;         // null: no chunk
    const int32_t* cu_q;    // packed queries: their offsets as they were given
    int64_t total_q;
    int32_t* powers;        // 4 bits: keys and values in fp16, divided by powers of two (AttnParams::kv_powers); null: bf16
    int chunks;
    // With them, unless q_rows is 0: the queries in fp16 too, [row][head][D], and each row's power.
    const __nv_bfloat16* q;
    int64_t qs[3], q_rows;
    int heads, sq, q_vec;   // sq: rows of a batch entry, 0: packed
    __half* q_out;
    float* q_power;
    int tiles, most_parts, sms, d;   // what parts_of_chunk goes by; most_parts 0: no parts
    __host__ __device__ int32_t* offsets() const { return words + kHeadWords; }
    __host__ __device__ int32_t* order(int batch) const { return offsets() + batch + 1; }
    __host__ __device__ int32_t* query_offsets(int batch) const { return order(batch) + batch; }
};

// An offset of packed rows, given on the device and not checked there: inside of the `total` rows there are.
__device__ __forceinline__ int64_t row_offset(const int32_t* cu, int b, int64_t total) {
    const int64_t x = cu[b];
    return x < 0 ? 0 : (x > total ? total : x);
}

// Parts (1 to `most`) that the keys of a chunk's tiles are cut into: `tiles` of 128 rows over up to `blocks` blocks of 128 keys,
// on `sms` SMs that take an item each. In tenths of a microsecond: a block, an item's start and end, and what adding up the parts
// costs (a launch, another kernel than whole tiles may take, and rows written and read at some 4 TB/s). Measured, us a call of bf16
// pages, whole and in parts: 32 heads over 8, D 128, 64 tokens x 8,192 keys 74.0 and 34.8, 128 x 8,192 75.2 and 38.3, 256 x 4,096 45.6 and
// 38.2; 2 x 16 over 2, D 64, 200 x 4,096 37.8 and 29.0; 14 over 2, D 64, 100 x 1,024 15.4 and 17.5 (left whole).
__host__ __device__ inline int parts_of_chunk(int64_t tiles, int blocks, int sms, int d, int most) {
    const int64_t block = d == 128 ? 10 : 7, item = 25;
    int best = 1;
    int64_t least = (tiles + sms - 1) / sms * (blocks * block + item);
    for (int n = 2; n <= most; ++n) {
        const int span = (blocks + n - 1) / n;
        const int64_t cost = (tiles * n + sms - 1) / sms * (span * block + item) + 60 + n * tiles * d / 390;
        if (cost < least) {
            least = cost;
            best = n;
        }
    }
    return best;
}

// Fills the cache's fields from an argument block after its checks (paged.cu); null, or why not.
const char* pages_of(Pages& c, const ktt_b200_pages& a, int d);

}  // namespace ktt
