// Attention over a paged cache, bf16 or 4 bits: one launch for a few query rows per K / V head, split over the keys.
//
//   out_r = sum_j p_rj v_j,  p_r = softmax over the keys j that row r sees of q_r k_j scale.
//
// Bound: the reading of the pages, 4 D bytes per key and head in bf16, 9 / 8 D in 4 bits. So all query rows of a K / V head
// (its group's heads x tokens, in tiles of 8 or 16 rows) share one pass over the keys, and the keys of all (sequence,
// K / V head) pairs are laid end to end and cut into equal shares (split.cuh), as in decode.cu; where the pairs are few, a
// cluster of CTAs has a pair to itself. Partial results of a pair meet in a small second launch, or in the cluster's shared
// memory, and are added in a fixed order.
//
// A CTA's share of a pair is cut into equal runs of blocks (16 keys, which lie in one page), one to a warp; a warp has a ring of
// stages of its own, each of a few blocks. Both products have the keys or channels as the rows of their matrix instruction (m16n8k16) and the queries as its 8 columns, so that a
// group of 8 heads or fewer leaves nothing idle: S^T = K Q^T, then O^T += V^T P^T. P^T comes out of S^T's registers by
// an 8 x 8 transpose (movmatrix). The reference of the exponentials moves when a score exceeds it by 2^8.
//
// 4 bits: a code c is worth least + step c per 64 channels. Codes become bf16 128 + c by one logic operation for two (the
// pages' layout is made for it, paged.cuh) and never anything else:
//   s_j   = sum_g step_jg (q_g . (128 + c_jg)) + (least_jg - 128 step_jg) sum(q_g): one product per group of channels g
//   o_g  += (2 p_j step_jg) (8 + c_jg / 2) less 12 (2 p_j step_jg), by a product with the constant 12 whose rows are all
//           alike, and p_j (least_jg + 8 step_jg) once for all channels of the group: what is left of both sums is about the
//           middle of the codes, and neither is large beside the result. (8 + c / 2 is a code shifted into the mantissa of 8; with
//           128 + c in its place the sums would be ten times as large and lose as much to fp32.)
// 2 p_j step_jg is rounded to bf16 for the product, as p_j is over bf16 pages; all else is fp32.
#include <atomic>
#include <type_traits>

#include "kept.h"
#include "paged.cuh"
#include "split.cuh"

namespace ktt {

// paged.cu: dense rows of the cache for a chunk of a prompt, and what the forward over them goes by (ChunkHead; its first words are
// cleared, the offsets of the dense rows are 0, rows, 2 rows, ..., queries are written where there are rows of them).
int read_pages(const Pages& c, int bits, int d, int batch, int kv_heads, int rows, void* k, void* v, const int64_t (&strides)[3], const ChunkHead& head, cudaStream_t stream);

namespace {

// Partials: a CTA cuts two pairs at most, the one it starts in and the one it ends in. That one, where the pair starts in the
// CTA, has the CTA's second slot, the other its first.
__device__ __forceinline__ int slot_of(int cta, bool starts_here) { return 2 * cta + (starts_here ? 1 : 0); }

struct PagedParams {
    Pages c;
    int batch, heads;
    int kv_heads;            // of the pairs: K / V heads x row tiles
    int row_tiles, group, sq, causal;
    int page_blocks;         // blocks of 16 keys in a page
    int table_width;
    float scale_log2;
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    int64_t qs[3], os[3];
    const int32_t* cu;       // packed queries
    int64_t total_q;
    int2* pieces;            // [pairs] the first CTA of a pair, and how many have a piece of it (1: its result is written)
    float2* part_ml;         // [slots][16] maximum and sum
    float* part_o;           // [slots][16][D]
    int ranks;               // CTAs of a cluster
};

constexpr int kMaxBatch = 512;    // lengths and their prefix sums live in shared memory

// What a variant has: D, bits of the pages, NT column tiles of 8 query rows. Measured, us, 64 sequences, 16 heads over 2, D 128,
// lengths U[n / 8, n], unless it says otherwise:
//   4 bits, n 16,384, one column tile: two blocks at a time, 4 warps, 3 CTAs 53.2; one block at a time 55.7; 8 warps, 2 CTAs (128
//   registers) 56.6; 4 warps, 4 CTAs 56.0. Loads alone 39.4, products alone as long as both: the stream is bound by the
//   chains between some 390 instructions a block (0.55 issued per scheduler and cycle, no pipe over 54 %). D 64, 32 heads over 8, n 512: 4 CTAs 10.0, 3 CTAs 15.3.
//   Two column tiles, 16 x 4 tokens, n 8,192: 2 CTAs 28.7, 3 (spills) 58.
//   bf16, n 4,096: 2 stages 34.3, 3 stages 34.7, 3 CTAs 34.8 (4.8 TB/s, 73 % of a copy's rate). D 64, 32 x 14 heads over 2, n 8,192: 4 CTAs of
//   3 stages 20.9, 2 of 6 22.7, 3 of 4 25.9; 64 x 32 over 8, n 512: 11.2, 18.1, 16.6.
//   What ending a pair costs, 4 bits, n 4,096 and 16,384, for 8, 12, 24, 40 blocks: 24.5, 24.2, 23.6, 24.4 and 54.8, 54.1, 53.3, 54.4; bf16,
//   n 4,096, for 4, 8, 16, 24, 32: 34.9, 34.5, 34.1, 34.1, 34.4.
template <int D, int kBits, int NT>
struct Shape {
    static constexpr int W = 4;                                               // warps
    static constexpr int kThreads = 32 * W;
    static constexpr int kBlock = kBits == 4 ? 18 * D : 64 * D;               // bytes: 16 keys, then their values
    static constexpr int NB = kBits == 16 ? 1 : (D == 128 && NT == 1 ? 2 : 4);   // blocks of a stage
    static constexpr int PB = kBits == 4 && NT == 1 ? 2 : 1;                  // blocks that the products are of at a time
    static constexpr int kStage = NB * kBlock;
    static constexpr int NS = kBits == 4 ? 2 : NT == 1 ? (D == 64 ? 3 : 2) : (D == 64 ? 6 : 3);
    static constexpr int kRows = 8 * NT;
    static constexpr int kPairCost = kBits == 4 ? 24 : 16;                    // what ending a pair costs a CTA, in blocks
    static constexpr int kCtas = D == 64 ? (NT == 1 ? 4 : kBits == 4 ? 3 : 2) : (kBits == 4 && NT == 1 ? 3 : 2);   // per SM
    static constexpr int kRing = W * NS * kStage;
    static constexpr int kStats = (2 * W + 2) * kRows * 4 + W * 4;
    static_assert(kStage >= kRows * D * 4, "a warp leaves its result in the stage it consumed last");
    static constexpr int smem(bool cluster) {
        return kRing + kStats + (cluster ? kRows * D * 4 : (2 * kMaxBatch + 1 + 8) * 4);
    }
};

// Chunk of 16 bytes of a row of the slab where its values lie: rows 2 t and 2 t + 1 of the threads that write at
// once in different banks.
__device__ __forceinline__ int slab_chunk(int row, int chunk) {
    const int t = (row >> 1) & 3;
    return chunk ^ ((t & 1) | ((t & 2) << 1));
}

// Byte offset of (row, col) in 16 rows of D bf16 values whose 16-byte chunks are XOR-ed with the row: no two rows of an
// 8 x 8 matrix in one bank.
template <int D>
__device__ __forceinline__ int swizzled(int row, int col) {
    return (row * D + (((col >> 3) ^ (row & 7)) << 3) + (col & 7)) * 2;
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Two codes of a word as the bf16 values 128 + c.
__device__ __forceinline__ uint32_t code_pair(uint32_t word) {
    uint32_t y;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(y) : "r"(word));   // (word & mask) | 128
    return y;
}
// The i-th of four pairs of codes (nibbles i and i + 4 of a word) as 8 + c / 2: in bits 3 to 6 of the mantissa; the
// first pair by 128 + c times 1 / 2 less 56, which is exact.
template <int i>
__device__ __forceinline__ uint32_t half_code_pair(uint32_t word) {
    uint32_t y;
    if constexpr (i == 0) {
        y = code_pair(word);
        asm("fma.rn.bf16x2 %0, %0, %1, %2;" : "+r"(y) : "r"(0x3f003f00u), "r"(0xc260c260u));   // 0.5, -56
    } else {
        asm("lop3.b32 %0, %1, 0x00780078, 0x41004100, 0xea;" : "=r"(y) : "r"(word >> (4 * i - 3)));
    }
    return y;
}
constexpr uint32_t kTwelve = 0x41404140u;   // bf16 12, twice
// The reference of a column that has seen no key: below every logit.
constexpr float kNoKey = -3.0e38f;

// Rows of a sequence's queries: how many tokens, and where they start.
__device__ __forceinline__ int tokens_of(const PagedParams& p, int b, int64_t& first) {
    if (!p.cu) {
        first = 0;
        return p.sq;
    }
    const int64_t hi = row_offset(p.cu, b + 1, p.total_q);
    first = row_offset(p.cu, b, p.total_q);
    return static_cast<int>(hi < first ? 0 : hi - first);
}

// One normalised chunk of 4 columns of (pair, row of its tile).
__device__ __forceinline__ void write_row(const PagedParams& p, int b, int vh, int row_in_tile, int tile_rows, int c4, float4 sum, float ll) {
    const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);   // (a NaN stays one)
    const int hk = vh / p.row_tiles, row = (vh - hk * p.row_tiles) * tile_rows + row_in_tile;
    int64_t first;
    const int n = tokens_of(p, b, first);
    const int gi = row / n, tq = row - gi * n;
    __nv_bfloat16* to = p.out + (p.cu ? 0 : b * p.os[0]) + (hk * p.group + gi) * p.os[1] + (first + tq) * p.os[2] + c4 * 4;
    uint2 packed;
    packed.x = pack_bf16(sum.x * inv, sum.y * inv);
    packed.y = pack_bf16(sum.z * inv, sum.w * inv);
    *reinterpret_cast<uint2*>(to) = packed;
}
// Rows that a pair has in its tile.
__device__ __forceinline__ int rows_of(const PagedParams& p, int b, int vh, int tile_rows) {
    int64_t first;
    const int all = p.group * tokens_of(p, b, first);
    return max(min(all - (vh % p.row_tiles) * tile_rows, tile_rows), 0);
}

template <int D, int kBits, int NT, bool kCluster>
__global__ void __launch_bounds__((Shape<D, kBits, NT>::kThreads), (Shape<D, kBits, NT>::kCtas)) paged_kernel(const __grid_constant__ PagedParams p) {
    using S = Shape<D, kBits, NT>;
    constexpr int W = S::W, NS = S::NS, NB = S::NB, PB = S::PB, kRows = S::kRows, kThreads = S::kThreads;
    constexpr int G = D / 64, MT = D / 16, kPairCost = S::kPairCost;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * NS * S::kStage;     // this warp's
    float* sm_m = reinterpret_cast<float*>(smem + S::kRing);   // [W][kRows]
    float* sm_l = sm_m + W * kRows;
    float* fin_m = sm_l + W * kRows;   // [kRows]: kCluster, the CTA's
    float* fin_l = fin_m + kRows;
    int* slab_s = reinterpret_cast<int*>(fin_l + kRows);       // [W] where a warp left its result
    int* prefix_s = slab_s + W;        // [kMaxBatch + 1]
    int* lens_s = prefix_s + kMaxBatch + 1;
    int* misc = lens_s + kMaxBatch;
    float* part_s = reinterpret_cast<float*>(slab_s + W);      // kCluster: [kRows][D] this CTA's partial

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // The blocks that this CTA streams: `left` of them from block `tile` of a pair on, through the pairs behind it.
    struct Walk {
        Cursor c;
        int left, pos, end;   // pos .. end: this warp's blocks of the CTA's piece of the pair
    } cons;
    int upc = 0, rank = 0, ranks_used = 1;
    if constexpr (kCluster) {
        const int pair = static_cast<int>(blockIdx.x) / p.ranks;
        rank = static_cast<int>(blockIdx.x) - pair * p.ranks;
        cons.c.b = pair / p.kv_heads;
        cons.c.hk = pair - cons.c.b * p.kv_heads;
        // The sequence's row of the table comes along with its length.
        if (lane * 32 < p.table_width) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.c.table + cons.c.b * p.c.table_stride + lane * 32));
        cons.c.len = cached_keys(p.c, cons.c.b);
        cons.c.ntiles = max((cons.c.len + 15) / 16, 1);
        // A rank has a block for each warp, or more.
        const int each = max((cons.c.ntiles + p.ranks - 1) / p.ranks, W);
        cons.c.tile = min(rank * each, cons.c.ntiles);
        cons.left = min(each, cons.c.ntiles - cons.c.tile);
        ranks_used = (cons.c.ntiles + each - 1) / each;
    } else {
        scan_lengths<kThreads, kMaxBatch, 16, kPairCost>(p.batch, [&](int b) { return cached_keys(p.c, b); }, prefix_s, lens_s, misc);
        const int total = p.kv_heads * prefix_s[p.batch];
        upc = max(static_cast<int>((total + gridDim.x - 1) / gridDim.x), 2 * W);
        const int64_t from = static_cast<int64_t>(blockIdx.x) * upc;
        const int first_unit = static_cast<int>(from < total ? from : total), end_unit = min(first_unit + upc, total);
        cons.left = tiles_before<kPairCost>(p, prefix_s, end_unit) - tiles_before<kPairCost>(p, prefix_s, first_unit);
        if (cons.left <= 0) return;
        cursor_seek<kPairCost>(p, prefix_s, lens_s, cons.c, first_unit);
    }
    auto piece_of = [](const Walk& w) { return min(w.c.ntiles - w.c.tile, w.left); };
    auto enter = [&](Walk& w) {
        const int m = piece_of(w), each = m / W, more = m - each * W;
        w.pos = w.c.tile + warp * each + min(warp, more);
        w.end = w.pos + each + (warp < more ? 1 : 0);
    };
    auto leave = [&](Walk& w) {   // to the next pair
        w.left -= piece_of(w);
        if (kCluster || w.left == 0) return;
        w.c.tile = w.c.ntiles - 1;
        cursor_next<kPairCost>(p, prefix_s, lens_s, w.c);
    };
    enter(cons);
    Walk prod = cons;

    // Where this warp's next 32 blocks lie, a lane each; null: no page.
    const unsigned char *k_at = nullptr, *v_at = nullptr;
    int at = 32;
    auto issue = [&](int st, int count) {
        const Cursor& c = prod.c;
        if (at + count > 32) {   // (a batch's blocks are in one lot)
            const int block = prod.pos + lane, hk = c.hk / p.row_tiles;
            k_at = v_at = nullptr;
            if (block < prod.end && static_cast<int64_t>(block) * 16 < c.len) {
                const int entry = block / p.page_blocks, row = (block - entry * p.page_blocks) * (kBits == 16 ? 16 : 1);
                const int64_t page = p.c.table[c.b * p.c.table_stride + entry];
                if (page >= 0 && page < p.c.pages) {
                    k_at = p.c.k + page * p.c.ks[0] + hk * p.c.ks[1] + row * (kBits == 16 ? p.c.ks[2] : static_cast<int64_t>(9 * D));
                    v_at = p.c.v + page * p.c.vs[0] + hk * p.c.vs[1] + row * (kBits == 16 ? p.c.vs[2] : static_cast<int64_t>(9 * D));
                }
            }
            at = 0;
        }
        const uint32_t to = smem_u32(ring + st * S::kStage);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            if (n >= count) break;
            const unsigned char* kp = reinterpret_cast<const unsigned char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(k_at), at + n));
            const unsigned char* vp = reinterpret_cast<const unsigned char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v_at), at + n));
            const bool there = kp != nullptr;
            if (!there) kp = p.c.k, vp = p.c.v;    // (not read: zeros are written)
            if constexpr (kBits == 16) {
                constexpr int CH = D / 8, kStep = 32 / CH;
                const int left = there ? c.len - prod.pos * 16 : 0, r0 = lane / CH, ch = lane % CH;   // rows behind the last key are zeros, whatever the page holds
                const unsigned char* kr = kp + ch * 16;
                const unsigned char* vr = vp + ch * 16;
#pragma unroll
                for (int it = 0; it < 16 / kStep; ++it) {
                    const int r = it * kStep + r0;
                    const bool ok = r < left;
                    cp_async_16(to + swizzled<D>(r, ch * 8), kr + (ok ? r * p.c.ks[2] : 0), ok);
                    cp_async_16(to + 32 * D + swizzled<D>(r, ch * 8), vr + (ok ? r * p.c.vs[2] : 0), ok);
                }
            } else {
                constexpr int kPieces = 9 * D / 16;   // of 16 bytes, of keys and of values
                kp += lane * 16;
                vp += lane * 16;
#pragma unroll
                for (int it = 0; it < (kPieces + 31) / 32; ++it) {
                    if (32 * it + 32 <= kPieces || lane < kPieces - 32 * it) {
                        cp_async_16(to + n * S::kBlock + (it * 32 + lane) * 16, kp + it * 512, there);
                        cp_async_16(to + n * S::kBlock + (kPieces + it * 32 + lane) * 16, vp + it * 512, there);
                    }
                }
            }
        }
        at += count;
    };

    int up_st = 0;
    auto produce = [&]() {
        while (prod.pos == prod.end && prod.left > 0) {
            leave(prod);
            if (prod.left > 0) {
                enter(prod);
                at = 32;
            }
        }
        if (prod.left > 0) {
            const int count = min(prod.end - prod.pos, NB);
            issue(up_st, count);
            prod.pos += count;
            up_st = up_st + 1 == NS ? 0 : up_st + 1;
        }
        cp_async_commit();
    };
    if (cons.left > 0) {
#pragma unroll
        for (int s = 0; s < NS - 1; ++s) produce();
    }

    uint32_t qb[NT][MT][2];           // B operands of S^T: columns are query rows
    float qsum[NT][G][2];             // 4 bits: sums of this thread's two columns by group of channels
    // Of this warp's keys: their end, the last one that a column sees, and the last that all columns see.
    int kend = 0, lim[NT][2], whole = 0;
    float o[MT][NT][4], mid[NT][G][2], m_ref[NT][2], bar[NT][2], l_run[NT][2];   // bar: the logit that moves the reference
    float twelve[NT][G][4];           // 4 bits: 12 times the weights' sums
    const float inv_scale = 1.f / p.scale_log2;
    int st = NS - 1;                  // the stage consumed last
    while (cons.left > 0) {           // pieces of pairs
        {
            const int hk = cons.c.hk / p.row_tiles, row0 = (cons.c.hk - hk * p.row_tiles) * kRows;
            int64_t first;
            const int n = tokens_of(p, cons.c.b, first), rows = p.group * n;
            kend = min(cons.c.len, cons.end * 16);
            whole = min(p.causal ? cons.c.len - n : cons.c.len - 1, kend - 1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int r = row0 + nt * 8 + g;
                const bool ok = r < rows;
                const int gi = ok ? r / n : 0, tq = ok ? r - gi * n : 0;
                // (A row past the last reads the first and is zeroed after; without any row at all nothing is read.)
                const __nv_bfloat16* from = p.q + (p.cu ? 0 : cons.c.b * p.qs[0]) + (hk * p.group + gi) * p.qs[1] + (rows > 0 ? first + tq : 0) * p.qs[2];
                if constexpr (kBits == 16) {
#pragma unroll
                    for (int kk = 0; kk < MT; ++kk) {
                        const uint32_t lo = *reinterpret_cast<const uint32_t*>(from + kk * 16 + t * 2), hi = *reinterpret_cast<const uint32_t*>(from + kk * 16 + 8 + t * 2);
                        qb[nt][kk][0] = ok ? lo : 0u;
                        qb[nt][kk][1] = ok ? hi : 0u;
                    }
                } else {
                    // Channels 32 i + 8 t .. of a word's eight, four to a k step.
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t x = *reinterpret_cast<const uint32_t*>(from + 32 * i + 8 * t + 2 * e);
                            qb[nt][2 * i + (e >> 1)][e & 1] = ok ? x : 0u;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < G; ++w) {
                        float sum = 0.f;
#pragma unroll
                        for (int kk = 4 * w; kk < 4 * w + 4; ++kk) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qb[nt][kk][e]));
                                sum += x.x + x.y;
                            }
                        }
                        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                        qsum[nt][w][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                        qsum[nt][w][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = row0 + nt * 8 + 2 * t + e;
                    lim[nt][e] = min(p.causal ? cons.c.len - n + (c < rows ? c % n : 0) : cons.c.len - 1, kend - 1);
                    m_ref[nt][e] = kNoKey;
                    bar[nt][e] = -INFINITY;
                    l_run[nt][e] = 0.f;
#pragma unroll
                    for (int w = 0; w < G; ++w) mid[nt][w][e] = twelve[nt][w][e] = twelve[nt][w][e + 2] = 0.f;
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.f;
            }
        }
        for (; cons.pos < cons.end; cons.pos += NB) {   // batches of blocks
        st = st + 1 == NS ? 0 : st + 1;
        produce();
        cp_async_wait<NS - 1>();
        __syncwarp();
        const int count = min(cons.end - cons.pos, NB);
#pragma unroll 1
        for (int n = 0; n < count; n += PB) {
            const int j0 = (cons.pos + n) * 16;
            if (j0 >= kend) break;          // (an empty sequence)
            const bool tail = j0 + 16 * PB - 1 > whole;
            const unsigned char* stage = ring + st * S::kStage + n * S::kBlock;
            float x[PB][NT][4];             // q k: key g of columns 2 t, 2 t + 1, then key g + 8
            uint2 vstep[PB][2];             // 4 bits: (step, least) of the two keys' values
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                const unsigned char *sk = stage + i * S::kBlock, *sv = sk + S::kBlock / 2;
                if constexpr (kBits == 16) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) x[i][nt][0] = x[i][nt][1] = x[i][nt][2] = x[i][nt][3] = 0.f;
                    const uint32_t base = smem_u32(sk);
                    const int r = (lane & 7) + ((lane >> 3) & 1) * 8, c = (lane >> 4) * 8;
#pragma unroll
                    for (int kk = 0; kk < MT; ++kk) {
                        uint32_t a[4];
                        ldmatrix_x4(a, base + swizzled<D>(r, kk * 16 + c));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_bf16(x[i][nt], a, qb[nt][kk][0], qb[nt][kk][1]);
                    }
                } else {
                    uint32_t kw[2][D / 32];
                    uint2 kstep[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const unsigned char* row = sk + (g + 8 * h) * (D / 2);
                        const unsigned char* steps = sk + 8 * D + (g + 8 * h) * (D / 16);
                        const unsigned char* vsteps = sv + 8 * D + (g + 8 * h) * (D / 16);
                        if constexpr (D == 128) {
                            const uint4 w = *reinterpret_cast<const uint4*>(row + 16 * t);
                            kw[h][0] = w.x; kw[h][1] = w.y; kw[h][2] = w.z; kw[h][3] = w.w;
                            kstep[h] = *reinterpret_cast<const uint2*>(steps);
                            vstep[i][h] = *reinterpret_cast<const uint2*>(vsteps);
                        } else {
                            const uint2 w = *reinterpret_cast<const uint2*>(row + 8 * t);
                            kw[h][0] = w.x; kw[h][1] = w.y;
                            kstep[h] = make_uint2(*reinterpret_cast<const uint32_t*>(steps), 0u);
                            vstep[i][h] = make_uint2(*reinterpret_cast<const uint32_t*>(vsteps), 0u);
                        }
                    }
                    if (tail) {   // whatever is behind the last key
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (j0 + 16 * i + g + 8 * h >= kend) kstep[h] = vstep[i][h] = make_uint2(0u, 0u);
                        }
                    }
#pragma unroll
                    for (int w = 0; w < G; ++w) {
                        float acc[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
                        for (int k = 2 * w; k < 2 * w + 2; ++k) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t a[4] = {code_pair(kw[0][k] >> (8 * h)), code_pair(kw[1][k] >> (8 * h)), code_pair(kw[0][k] >> (8 * h + 4)), code_pair(kw[1][k] >> (8 * h + 4))};
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) mma_bf16(acc[nt], a, qb[nt][2 * k + h][0], qb[nt][2 * k + h][1]);
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t pair = w ? kstep[h].y : kstep[h].x;
                            const float ks = step_of(pair), kl = fmaf(-128.f, ks, least_of(pair));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const float at_zero = w ? fmaf(kl, qsum[nt][w][e], x[i][nt][2 * h + e]) : kl * qsum[nt][w][e];
                                    x[i][nt][2 * h + e] = fmaf(ks, acc[nt][2 * h + e], at_zero);
                                }
                            }
                        }
                    }
                }
            }
            if (tail) {
#pragma unroll
                for (int i = 0; i < PB; ++i) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (j0 + 16 * i + g + 8 * (e >> 1) > lim[nt][e & 1]) x[i][nt][e] = -INFINITY;
                        }
                    }
                }
            }
            bool higher = false;
#pragma unroll
            for (int i = 0; i < PB; ++i) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) higher |= x[i][nt][e] > bar[nt][e & 1];
                }
            }
            if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(x[0][nt][e], x[0][nt][e + 2]);
#pragma unroll
                        for (int i = 1; i < PB; ++i) top = fmaxf(top, fmaxf(x[i][nt][e], x[i][nt][e + 2]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        top = fmaxf(top * p.scale_log2, m_ref[nt][e]);
                        const float f = fast_exp2(m_ref[nt][e] - top);
                        m_ref[nt][e] = top;
                        bar[nt][e] = (top + 8.f) * inv_scale;
                        l_run[nt][e] *= f;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            o[mt][nt][e] *= f;
                            o[mt][nt][e + 2] *= f;
                        }
#pragma unroll
                        for (int w = 0; w < G; ++w) {
                            mid[nt][w][e] *= f;
                            twelve[nt][w][e] *= f;
                            twelve[nt][w][e + 2] *= f;
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < PB; ++i) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[i][nt][e] = fast_exp2(fmaf(x[i][nt][e], p.scale_log2, -m_ref[nt][e & 1]));
                        l_run[nt][e & 1] += x[i][nt][e];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                const unsigned char* sv = stage + i * S::kBlock + S::kBlock / 2;
                if constexpr (kBits == 16) {
                    uint32_t pb[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        pb[nt][0] = transposed(pack_bf16(x[i][nt][0], x[i][nt][1]));
                        pb[nt][1] = transposed(pack_bf16(x[i][nt][2], x[i][nt][3]));
                    }
                    const uint32_t base = smem_u32(sv);
                    const int r = (lane & 7) + (lane >> 4) * 8, c = ((lane >> 3) & 1) * 8;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        uint32_t a[4];
                        ldmatrix_x4_trans(a, base + swizzled<D>(r, mt * 16 + c));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_bf16(o[mt][nt], a, pb[nt][0], pb[nt][1]);
                    }
                } else {
                    uint32_t pb[NT][G][2];
#pragma unroll
                    for (int w = 0; w < G; ++w) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t pair = w ? vstep[i][h].y : vstep[i][h].x;
                            const float vs = 2.f * step_of(pair), vm = fmaf(4.f, vs, least_of(pair));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                pb[nt][w][h] = transposed(pack_bf16(x[i][nt][2 * h] * vs, x[i][nt][2 * h + 1] * vs));
                                mid[nt][w][0] = fmaf(x[i][nt][2 * h], vm, mid[nt][w][0]);
                                mid[nt][w][1] = fmaf(x[i][nt][2 * h + 1], vm, mid[nt][w][1]);
                            }
                        }
                    }
                    uint32_t vw[2][2][G];   // token pairs t and t + 4: even token's words, odd token's
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int pair = t + 4 * h, place = g ^ (D == 128 ? 2 * (pair & 3) : 4 * ((pair >> 1) & 1));
                        const unsigned char* from = sv + (pair * 8 + place) * (8 * G);
                        if constexpr (D == 128) {
                            const uint4 w = *reinterpret_cast<const uint4*>(from);
                            vw[h][0][0] = w.x; vw[h][0][G - 1] = w.y; vw[h][1][0] = w.z; vw[h][1][G - 1] = w.w;
                        } else {
                            const uint2 w = *reinterpret_cast<const uint2*>(from);
                            vw[h][0][0] = w.x; vw[h][1][0] = w.y;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < G; ++w) {
                        const uint32_t lo0 = __byte_perm(vw[0][0][w], vw[0][1][w], 0x5410), hi0 = __byte_perm(vw[0][0][w], vw[0][1][w], 0x7632);
                        const uint32_t lo1 = __byte_perm(vw[1][0][w], vw[1][1][w], 0x5410), hi1 = __byte_perm(vw[1][0][w], vw[1][1][w], 0x7632);
                        // Rows g and g + 8 of instruction k: channels 64 w + 8 g + 2 k and the next one.
                        auto product = [&](auto which) {
                            constexpr int k = decltype(which)::value;
                            const uint32_t a[4] = {half_code_pair<k>(lo0), half_code_pair<k>(hi0), half_code_pair<k>(lo1), half_code_pair<k>(hi1)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_bf16(o[4 * w + k][nt], a, pb[nt][w][0], pb[nt][w][1]);
                        };
                        product(std::integral_constant<int, 0>());
                        product(std::integral_constant<int, 1>());
                        product(std::integral_constant<int, 2>());
                        product(std::integral_constant<int, 3>());
                        const uint32_t a[4] = {kTwelve, kTwelve, kTwelve, kTwelve};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_bf16(twelve[nt][w], a, pb[nt][w][0], pb[nt][w][1]);
                    }
                }
            }
        }
        __syncwarp();   // all lanes are done with stage `st` before it is filled again
        }

        {
            // The warps' results to shared memory, each with its own reference, in the stage that it consumed last (nothing is
            // on its way there); then their sum in the order of the warps.
            float* slab = reinterpret_cast<float*>(ring + st * S::kStage);
            if (lane == 0) slab_s[warp] = warp * NS * S::kStage + st * S::kStage;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float l = l_run[nt][e];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
                    const int r = nt * 8 + 2 * t + e;
                    if (g == 0) {
                        sm_m[warp * kRows + r] = m_ref[nt][e];
                        sm_l[warp * kRows + r] = l;
                    }
                    if constexpr (kBits == 16) {
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int c = mt * 16 + g + 8 * h;
                                slab[r * D + slab_chunk(r, c >> 2) * 4 + (c & 3)] = o[mt][nt][e + 2 * h];
                            }
                        }
                    } else {
#pragma unroll
                        for (int w = 0; w < G; ++w) {
                            float add = mid[nt][w][e];
#pragma unroll
                            for (int off = 4; off < 32; off <<= 1) add += __shfl_xor_sync(0xffffffffu, add, off);
                            const float less = twelve[nt][w][e];   // (all rows alike)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float4 y = make_float4((o[4 * w + 2 * h][nt][e] - less) + add, (o[4 * w + 2 * h][nt][e + 2] - less) + add,
                                                             (o[4 * w + 2 * h + 1][nt][e] - less) + add, (o[4 * w + 2 * h + 1][nt][e + 2] - less) + add);
                                *reinterpret_cast<float4*>(slab + r * D + slab_chunk(r, 16 * w + 2 * g + h) * 4) = y;
                            }
                        }
                    }
                }
            }
            __syncthreads();
            // Four columns of a row, its maximum and its sum: of all warps.
            auto merged = [&](int r, int c4, float& mm, float& ll) {
                const unsigned char* from = smem + (r * D + slab_chunk(r, c4) * 4) * 4;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                mm = sm_m[r];
                ll = 0.f;
#pragma unroll
                for (int w = 1; w < W; ++w) mm = fmaxf(mm, sm_m[w * kRows + r]);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(from + slab_s[w]);
                    const float f = fast_exp2(sm_m[w * kRows + r] - mm);
                    ll = fmaf(sm_l[w * kRows + r], f, ll);
                    sum.x = fmaf(y.x, f, sum.x); sum.y = fmaf(y.y, f, sum.y);
                    sum.z = fmaf(y.z, f, sum.z); sum.w = fmaf(y.w, f, sum.w);
                }
                return sum;
            };
            const int rows = rows_of(p, cons.c.b, cons.c.hk, kRows);
            if constexpr (kCluster) {
                for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kThreads) {
                    const int r = idx / (D / 4), c4 = idx % (D / 4);
                    float mm, ll;
                    const float4 sum = merged(r, c4, mm, ll);
                    if (ranks_used == 1) {
                        write_row(p, cons.c.b, cons.c.hk, r, kRows, c4, sum, ll);
                        continue;
                    }
                    reinterpret_cast<float4*>(part_s)[idx] = sum;
                    if (c4 == 0) {
                        fin_m[r] = mm;
                        fin_l[r] = ll;
                    }
                }
                break;
            }
            const int pair = cons.c.b * p.kv_heads + cons.c.hk;
            const int t0 = p.kv_heads * prefix_s[cons.c.b] + cons.c.hk * (cons.c.ntiles + kPairCost);   // the pair's first unit
            const int c_first = t0 / upc, c_last = (t0 + cons.c.ntiles - 1) / upc;
            if (c_first == c_last) {
                for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kThreads) {
                    const int r = idx / (D / 4), c4 = idx % (D / 4);
                    float mm, ll;
                    const float4 sum = merged(r, c4, mm, ll);
                    write_row(p, cons.c.b, cons.c.hk, r, kRows, c4, sum, ll);
                }
            } else {
                const int slot = slot_of(blockIdx.x, c_first == static_cast<int>(blockIdx.x));
                for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kThreads) {
                    const int r = idx / (D / 4), c4 = idx % (D / 4);
                    float mm, ll;
                    reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(slot) * 16 + r) * D)[c4] = merged(r, c4, mm, ll);
                    if (c4 == 0) p.part_ml[slot * 16 + r] = make_float2(mm, ll);
                }
            }
            if (threadIdx.x == 0 && c_last == static_cast<int>(blockIdx.x)) p.pieces[pair] = make_int2(c_first, c_last - c_first + 1);
            __syncthreads();
        }
        leave(cons);
        if (cons.left > 0) enter(cons);
    }
    cp_async_wait<0>();
    if constexpr (kCluster) {
        if (ranks_used == 1) return;   // one rank had all of it and has written it: nobody waits for anybody
        cluster_meet();
        // Every rank adds up its share of the output, the ranks that had a tile in their order.
        const int rows = rows_of(p, cons.c.b, cons.c.hk, kRows);
        const int parts = ranks_used, all = rows * (D / 4), share = (all + p.ranks - 1) / p.ranks;
        const uint32_t at_m = smem_u32(fin_m), at_l = smem_u32(fin_l), at_o = smem_u32(part_s);
        for (int idx = rank * share + threadIdx.x; idx < min((rank + 1) * share, all); idx += kThreads) {
            const int r = idx / (D / 4), c4 = idx % (D / 4);
            float ms[8], ls[8], mm = -INFINITY, ll = 0.f;
            float4 v[8], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {   // (ranks: 8 at most)
                const int from = min(j, parts - 1);
                ms[j] = ld_cluster(in_rank(at_m + r * 4, from));
                ls[j] = ld_cluster(in_rank(at_l + r * 4, from));
                v[j] = ld_cluster4(in_rank(at_o + idx * 16, from));
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) mm = fmaxf(mm, ms[j]);
            const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j >= parts) continue;
                const float f = fast_exp2(ms[j] - base);
                ll = fmaf(ls[j], f, ll);
                sum.x = fmaf(v[j].x, f, sum.x); sum.y = fmaf(v[j].y, f, sum.y);
                sum.z = fmaf(v[j].z, f, sum.z); sum.w = fmaf(v[j].w, f, sum.w);
            }
            write_row(p, cons.c.b, cons.c.hk, r, kRows, c4, sum, ll);
        }
        cluster_meet();   // nobody's shared memory goes away while another reads it
    }
}

// The pairs that were cut: their partials, in the order of the CTAs that left them. A block has two rows of a pair; four
// threads share four columns, each with every fourth partial, eight requested at a time. (A launch of its own, which starts
// up while the stream drains: a last holder that adds them up behind a ticket keeps registers from the stream, whose
// instructions were 30 % more for it.)
template <int D>
__global__ void __launch_bounds__(2 * D) merge_kernel(const __grid_constant__ PagedParams p, int tile_rows) {
    __shared__ float4 sums[2][4][D / 4];
    __shared__ float2 stats[2][4];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int pair = blockIdx.x, r = blockIdx.y * 2 + threadIdx.z, c4 = threadIdx.x, quarter = threadIdx.y;
    const int2 piece = p.pieces[pair];
    if (piece.y <= 1) return;
    const int b = pair / p.kv_heads, vh = pair - b * p.kv_heads;
    const bool there = r < rows_of(p, b, vh, tile_rows);
    float mm = kNoKey, ll = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kAhead = 8;
    for (int c0 = quarter; there && c0 < piece.y; c0 += 4 * kAhead) {
        float2 ml[kAhead];
        float4 v[kAhead];
        float top = mm;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            ml[j] = make_float2(kNoKey, 0.f);
            v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            const int i = c0 + 4 * j;
            if (i < piece.y) {
                const int64_t at = static_cast<int64_t>(slot_of(piece.x + i, i == 0)) * 16 + r;
                ml[j] = __ldcg(&p.part_ml[at]);
                v[j] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D) + c4);
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) top = fmaxf(top, ml[j].x);
        const float f = fast_exp2(mm - top);
        mm = top;
        ll *= f;
        sum.x *= f; sum.y *= f; sum.z *= f; sum.w *= f;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const float w = fast_exp2(ml[j].x - top);
            ll = fmaf(ml[j].y, w, ll);
            sum.x = fmaf(v[j].x, w, sum.x); sum.y = fmaf(v[j].y, w, sum.y);
            sum.z = fmaf(v[j].z, w, sum.z); sum.w = fmaf(v[j].w, w, sum.w);
        }
    }
    sums[threadIdx.z][quarter][c4] = sum;
    if (c4 == 0) stats[threadIdx.z][quarter] = make_float2(mm, ll);
    __syncthreads();
    if (quarter || !there) return;
    float2 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = stats[threadIdx.z][i];
    const float top = fmaxf(fmaxf(s[0].x, s[1].x), fmaxf(s[2].x, s[3].x));
    ll = 0.f;
    sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float w = fast_exp2(s[i].x - top);
        const float4 v = sums[threadIdx.z][i][c4];
        ll = fmaf(s[i].y, w, ll);
        sum.x = fmaf(v.x, w, sum.x); sum.y = fmaf(v.y, w, sum.y);
        sum.z = fmaf(v.z, w, sum.z); sum.w = fmaf(v.w, w, sum.w);
    }
    write_row(p, b, vh, r, tile_rows, c4, sum, ll);
}

// ---- host -----------------------------------------------------------------------------------

int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? dev : -1;
}

int sm_count(int dev) {
    static std::atomic<int> known[64];
    if (dev < 0) return 148;
    const int sms = kept(known[dev], [&]() {
        int n = 0;
        return cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? n : -1;
    });
    return sms > 0 ? sms : 148;
}

template <int D, int kBits, int NT, bool kCluster>
cudaLaunchConfig_t paged_config(int ctas, int ranks, cudaStream_t stream, cudaLaunchAttribute* attr) {
    using S = Shape<D, kBits, NT>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::smem(kCluster);
    cfg.stream = stream;
    if (kCluster) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
    }
    cfg.attrs = attr;
    return cfg;
}

// Clusters of `ranks` CTAs that run at the same time on the current device; asked for once. -1: no answer now.
template <int D, int kBits, int NT>
int cluster_room(int dev, int ranks) {
    static std::atomic<int> known[64][4];   // by log2 of the ranks
    if (dev < 0) return -1;
    int log = 0;
    while ((1 << log) < ranks) ++log;
    return kept(known[dev][log], [&]() {
        auto kernel = paged_kernel<D, kBits, NT, true>;
        cudaLaunchAttribute attr[1];
        cudaLaunchConfig_t cfg = paged_config<D, kBits, NT, true>(ranks, ranks, nullptr, attr);
        int n = 0;
        if (raise_smem_limit(kernel, static_cast<int>(cfg.dynamicSmemBytes)) == cudaSuccess &&
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess) return n;
        cudaGetLastError();   // not this call's failure
        return -1;
    });
}

// Set up once per device, by the first call of whatever size: both kernels' limits and the room for clusters.
template <int D, int kBits, int NT>
int paged_set_up(int dev) {
    static std::atomic<int> done[64];
    int rc = 0;
    auto shares = [&]() { return rc = ensure_smem(paged_kernel<D, kBits, NT, false>, Shape<D, kBits, NT>::smem(false), "cudaFuncSetAttribute(paged)"); };
    if (dev < 0) return shares();
    kept(done[dev], [&]() {
        int least = shares();
        for (int ranks = 1; ranks <= 8; ranks *= 2) {
            const int room = cluster_room<D, kBits, NT>(dev, ranks);
            least = room < least ? room : least;
        }
        return least < 0 ? -1 : 0;
    });
    return rc;
}

// CTAs per pair where each has a cluster of its own; 0 where the pairs are cut into equal shares. A cluster has no lengths to
// scan and nothing to add up behind the stream, 1.5 to 3 us less; but a pair is as long as it is, and CTAs that clusters leave
// out have no share. So a rank has 1,024 keys at most, and beyond 512 as many times fewer as clusters use fewer CTAs than there are
// (less a fifth). Measured, us, clusters and shares, lengths U[n / 8, n], 16 heads over 2, bf16, D 64: 1 x 1,024 6.1 and 7.4, 1 x 4,096
// 8.1 and 8.0, 4 x 4,096 8.5 and 9.2, 4 x 8,192 11.6 and 11.1, 32 x 2,048 9.2 and 11.7, 32 x 8,192 20.7 and 25.7, 64 x 4,096 (4 ranks) 19.6 and
// 23.7; D 128: 1 x 8,192 11.8 and 9.9, 16 x 4,096 14.4 and 16.6, 64 x 2,048 21.5 and 22.6, 64 x 4,096 (2 ranks) 35.5 and 34.0; 4 bits, D 128: 1 x 1,024
// 7.3 and 8.0, 16 x 2,048 10.7 and 12.2, 16 x 8,192 19.9 and 17.7, 64 x 1,024 14.2 and 15.2, 64 x 2,048 20.1 and 18.0. Pairs that outnumber the
// CTAs follow one another, up to 2,048 keys each: 64 x 16 heads, D 64, bf16, 128, 1,024 and 2,048 keys 10.2 and 15.8, 29.0 and 32.8, 52.4 and
// 57.7; 4 bits 10.3 and 15.9, 24.4 and 28.4, 40.3 and 41.2; 64 x 12, D 128, 4 bits, 2,048 49.1 and 47.9.
template <int D, int kBits, int NT>
int paged_ranks(int64_t pairs, int cap, int ctas, int dev) {
    constexpr int kTile = 16 * Shape<D, kBits, NT>::W;
    if (pairs > ctas && cap <= 2048) return 1;
    for (int ranks = 8; ranks >= 1; ranks /= 2) {
        if (ranks > 1 && (ranks / 2) * kTile >= cap) continue;   // half as many have a block for every warp
        if (pairs * ranks > ctas || cluster_room<D, kBits, NT>(dev, ranks) < pairs) continue;
        const int64_t used = pairs * ranks, all = ctas, most = 1024ll * ranks;
        return cap <= most && (2 * cap <= most || 4 * cap * all <= 5 * most * used) ? ranks : 0;
    }
    return 0;
}

struct Parts {
    int64_t piece_bytes, ml_bytes, total;
};
Parts parts_of(int64_t pairs, int d, int ctas) {
    Parts s;
    const int64_t slots = 2 * static_cast<int64_t>(ctas);
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    s.piece_bytes = up(pairs * 8);
    s.ml_bytes = up(slots * 16 * 8);
    s.total = s.piece_bytes + s.ml_bytes + up(slots * 16 * d * 4);
    return s;
}

// Up to kFewTokens tokens of a sequence there are two ways: the pass above over a K / V head's keys for every 8 or 16 of its rows
// (heads x tokens), and the tensor path below, which makes dense rows of the keys and takes 128 tokens of one head at a time, full
// or not. Which is the shorter goes by what each costs for a K / V head and 128 keys: the pass, rows / 16 times `pass`; the tensor
// path, `dense` for the rows and `tile` for each head; and by 9 and 12 us that they take whatever the sizes. Measured, us, pass and
// tensor path, bf16, D 128: 32 heads over 8, 1 x 8,192, 24 tokens 29.9 and 33.9, 48 tokens 49.4 and 34.5; 4 x 4,096, 24 tokens 54 and 59,
// 48 tokens 96 and 60; 32 x 2,048, 24 tokens 184 and 208, 32 tokens 220 and 208; 8 x 16 heads x 4,096, 48 tokens 122 and 134, 64 tokens
// 159 and 134; D 64: 32 x 16
// heads x 1,024, 48 tokens 81 and 88, 64 tokens 96 and 89, with 4 bits 77 and 79; 14 heads over 2, 1 x 4,096, 48 tokens 16 and 19.
constexpr int kFewTokens = 64;
bool pass_pays(int bits, int d, int64_t heads, int64_t kv_heads, int64_t batch, int64_t row_tiles, int64_t blocks) {
    const double pass = d == 128 ? (bits == 16 ? 0.0075 : 0.0066) : (bits == 16 ? 0.0053 : 0.0042);
    const double tile = d == 128 ? 0.006 : 0.004, dense = d == 128 ? 0.023 : 0.015;
    const double units = static_cast<double>(batch * kv_heads) * blocks;
    return 9 + units * pass * row_tiles <= 12 + units * (tile * (heads / kv_heads) + dense);
}

// What a call will do, from its sizes alone.
struct Plan {
    bool few;
    int nt, row_tiles, slice;   // sequences of a launch
    int64_t bytes;              // of workspace
    int tiles, parts;           // chunks: tiles of 128 rows of a launch, and the most parts that their keys are cut into (0: none)
    int64_t powers_at, q_at, q_powers_at, parts_at;   // where in the workspace the keys' powers of two, fp16 queries and theirs, and parts are
};

// Tiles that are too few for the SMs are cut along their keys where that pays for the longest sequence that the table has room
// for; into how many parts then goes by the longest there is (parts_of_chunk, in read_pages), of which there may be two for every SM.
constexpr int kMostParts = 16;

int64_t rows_per_head(const ktt_b200_paged_sdpa_args* a) { return static_cast<int64_t>(a->heads / a->cache.kv_heads) * a->sq; }

// Rows that parts have a place for in a launch over `batch` sequences: sq for each, or the packed rows where those are fewer (the
// launches of a call share them, and a padded buffer has more than its sequences). Parts are at most two tiles' worth for every SM.
int64_t part_rows(const ktt_b200_paged_sdpa_args* a, int batch) {
    const int64_t rows = static_cast<int64_t>(batch) * a->sq;
    return a->cu_seqlens_q && a->total_q < rows ? a->total_q : rows;
}

// Groups of 64 keys that a sequence has powers of two for, in whole blocks of 128.
int chunks_of(const Pages& c) { return (c.cap + 127) / 128 * 2; }

Plan plan_of(const ktt_b200_paged_sdpa_args* a, const Pages& c, int sms) {
    Plan s = {};
    const int64_t rows = rows_per_head(a), hk = a->cache.kv_heads;
    s.nt = rows <= 8 ? 1 : 2;
    s.row_tiles = static_cast<int>((rows + 8 * s.nt - 1) / (8 * s.nt));
    // Units of all pairs of a launch have to fit 30 bits.
    int64_t most = (1ll << 30) / ((static_cast<int64_t>(c.cap) / 16 + 32) * hk * s.row_tiles);
    s.few = a->sq <= kFewTokens && most > 0 && pass_pays(a->cache.bits, a->d, a->heads, hk, a->batch, (rows + 15) / 16, (c.cap + 127) / 128);
    if (s.few) {
        if (most > kMaxBatch) most = kMaxBatch;
        s.slice = static_cast<int>(a->batch < most ? a->batch : most);
        s.bytes = parts_of(s.slice * hk * s.row_tiles, a->d, sms * 4).total;
        return s;
    }
    // Dense rows of some sequences at a time: 1 GB, or one sequence.
    const int64_t one = 4ll * c.cap * hk * a->d;
    most = (1ll << 30) / one;
    s.slice = static_cast<int>(most < 1 ? 1 : (most < a->batch ? most : a->batch));
    if (s.slice > kMaxBatch) s.slice = kMaxBatch;
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t rows_heads = a->cache.bits == 4 ? (a->cu_seqlens_q ? a->total_q : static_cast<int64_t>(a->batch) * a->sq) * a->heads : 0;
    s.powers_at = s.slice * one + up(head_words(kMaxBatch) * 4);
    s.q_at = s.powers_at + (a->cache.bits == 4 ? up(s.slice * hk * chunks_of(c) * 4) : 0);
    s.q_powers_at = s.q_at + up(rows_heads * a->d * 2);
    s.parts_at = s.q_powers_at + up(rows_heads * 4);
    s.bytes = s.parts_at;
    const bool packed = a->cu_seqlens_q != nullptr;
    int64_t tiles = s.slice * static_cast<int64_t>((a->sq + 127) / 128);
    if (packed && a->total_q / 128 + s.slice < tiles) tiles = a->total_q / 128 + s.slice;
    tiles *= a->heads;
    int64_t parts = 2 * sms / tiles;
    if (parts > kMostParts) parts = kMostParts;
    if (parts > 1 && parts_of_chunk(tiles, (c.cap + 127) / 128, sms, a->d, static_cast<int>(parts)) > 1) {
        s.tiles = static_cast<int>(tiles);
        s.parts = static_cast<int>(parts);
        s.bytes += parts * part_rows(a, s.slice) * a->heads * (a->d + 1) * 4;
    }
    return s;
}

template <int D, int kBits, int NT>
int run_few(PagedParams& p, cudaStream_t stream) {
    using S = Shape<D, kBits, NT>;
    const int dev = current_device();
    if (int rc = paged_set_up<D, kBits, NT>(dev)) return rc;
    const int ctas = S::kCtas * sm_count(dev);
    const int64_t pairs = static_cast<int64_t>(p.batch) * p.kv_heads;
    p.ranks = paged_ranks<D, kBits, NT>(pairs, p.c.cap, ctas, dev);
    cudaLaunchAttribute attr[2];
    auto go = [&](cudaLaunchConfig_t cfg, auto kernel, auto... args) {
        cfg.attrs = attr;
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
        return check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), "paged_sdpa launch");
    };
    if (p.ranks > 0) return go(paged_config<D, kBits, NT, true>(static_cast<int>(pairs) * p.ranks, p.ranks, stream, attr), paged_kernel<D, kBits, NT, true>, p);
    if (int rc = go(paged_config<D, kBits, NT, false>(ctas, 1, stream, attr), paged_kernel<D, kBits, NT, false>, p)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(pairs), S::kRows / 2);
    cfg.blockDim = dim3(D / 4, 4, 2);
    cfg.stream = stream;
    return go(cfg, merge_kernel<D>, p, static_cast<int>(S::kRows));
}

template <int D, int kBits>
int run_few(PagedParams& p, int nt, cudaStream_t stream) { return nt == 1 ? run_few<D, kBits, 1>(p, stream) : run_few<D, kBits, 2>(p, stream); }

const char* sdpa_refusal(const ktt_b200_paged_sdpa_args* a, Pages& c) {
    if (const char* why = pages_of(c, a->cache, a->d)) return why;
    if (a->heads < 1 || a->heads % a->cache.kv_heads) return "K / V heads must divide Q heads";
    if (a->heads > 65535 || a->batch > 65535) return "batch and heads must not exceed 65535";
    if (!(a->scale > 0.f)) return "the softmax scale must be positive";
    if (rows_per_head(a) >= (1ll << 31)) return "too many query rows";
    for (int i = 0; i < 3; ++i) {
        if (a->q_strides[i] % 2 || a->out_strides[i] % 4) return "q strides must be even and out strides multiples of 4";
    }
    if ((reinterpret_cast<uintptr_t>(a->q) & 3) || (reinterpret_cast<uintptr_t>(a->out) & 7)) return "q must be 4-byte and out 8-byte aligned";
    return nullptr;
}

// Rows of chunks whose sequence has more than one part: the parts' rows, each with its base-2 logarithm of the sum of weights,
// added up. D / 4 threads have a row of a head.
struct MergeParams {
    Pages c;
    const float* o;      // [parts][rows][heads][D]
    const float* lse;    // [parts][rows][heads]
    const int32_t* cu;   // packed
    const int32_t* parts;   // (parts, keys of a part)
    int64_t rows;        // that parts have a place for
    int stride;          // places of a sequence; 0: those of the packed rows
    int batch, heads, sq;
    __nv_bfloat16* out;
    int64_t os[3];
};
template <int D>
__global__ void __launch_bounds__(256) merge_parts_kernel(const __grid_constant__ MergeParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t n = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y, place = n / p.heads;
    if (place >= p.rows) return;
    const int h = static_cast<int>(n - place * p.heads), c4 = threadIdx.x;
    const int b = p.stride ? static_cast<int>(place / p.stride) : sequence_of(p.cu, p.batch, place);
    if (b < 0) return;
    int64_t row = place - static_cast<int64_t>(b) * p.stride;   // in the sequence, then of the operands
    if (p.cu) {
        const int64_t first = p.cu[b], n_rows = p.cu[b + 1] - first;
        if (!p.stride) row -= first;
        if (row >= n_rows || row >= p.sq) return;
        row += first;
    }
    const int span = p.parts[1], parts = (cached_keys(p.c, b) + span - 1) / span;
    if (parts <= 1) return;
    const int64_t step = p.rows * p.heads;
    float m = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kAhead = 4;
    for (int i0 = 0; i0 < parts; i0 += kAhead) {
        float l[kAhead], top = m;
        float4 v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            l[j] = -INFINITY;
            v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i0 + j < parts) {
                const int64_t at = (i0 + j) * step + n;
                l[j] = __ldcg(p.lse + at);
                v[j] = __ldcg(reinterpret_cast<const float4*>(p.o + at * D) + c4);
            }
        }
        bool seen = false;   // (a NaN is seen, though it is no maximum)
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            top = fmaxf(top, l[j]);
            seen |= !(l[j] == -INFINITY);
        }
        if (!seen) continue;
        const float base = top == -INFINITY ? 0.f : top, f = fast_exp2(m - base);
        m = top;
        sum *= f;
        acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (l[j] == -INFINITY) continue;   // (a part that the row sees nothing of has written no row)
            const float w = fast_exp2(l[j] - base);
            sum += w;
            acc.x = fmaf(v[j].x, w, acc.x); acc.y = fmaf(v[j].y, w, acc.y);
            acc.z = fmaf(v[j].z, w, acc.z); acc.w = fmaf(v[j].w, w, acc.w);
        }
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);   // (a NaN stays one)
    __nv_bfloat16* to = p.out + (p.cu ? 0 : b * p.os[0]) + h * p.os[1] + row * p.os[2] + 4 * c4;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

int merge_parts(const MergeParams& p, int d, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(static_cast<unsigned>(d / 4), static_cast<unsigned>(1024 / d));
    cfg.gridDim = dim3(static_cast<unsigned>((p.rows * p.heads + cfg.blockDim.y - 1) / cfg.blockDim.y));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, d == 64 ? merge_parts_kernel<64> : merge_parts_kernel<128>, p), "paged_sdpa merge launch");
}

// A chunk of a prompt: the rows of a K / V head are many, so the work is in the products, which the tensor kernels of the
// dense and packed forward do; the pages become dense rows for them first (2 x 2 D bytes written and read per key
// and head, against 4 D operations per key and row). Those are bf16. Over 4 bits they are fp16, and so are the queries and the weights: a
// code's worth is an 8-bit step times 4 bits and a sum, which bf16 rounds by as much as it does the weights. Powers of two, of each query row
// and of each 64 keys and values, keep all magnitudes in fp16's range. Off against float64 (root mean squares of the result): 1.7e-3, all of
// it the result's own rounding, where it was 3.3e-3 with everything in bf16; the pass, which multiplies codes by bf16 weights, 2.4e-3,
// bf16 pages 2.3e-3. 4 sequences of up to 512 tokens and 8,192 keys, 16 heads over 4, D 128: 103 us, 101 in bf16, the queries' copy 2.5 of it.
int run_many(const ktt_b200_paged_sdpa_args* a, const PagedParams& p, const Plan& plan, cudaStream_t stream) {
    const int hk = a->cache.kv_heads, d = a->d, slice = plan.slice;
    const int64_t cap = p.c.cap, half = slice * cap * hk * d;
    unsigned char* base = static_cast<unsigned char*>(a->workspace);
    __nv_bfloat16* k = reinterpret_cast<__nv_bfloat16*>(base);
    __nv_bfloat16* v = k + half;
    int32_t* words = reinterpret_cast<int32_t*>(v + half);
    for (int b0 = 0; b0 < a->batch; b0 += slice) {
        const int n = a->batch - b0 < slice ? a->batch - b0 : slice;
        Pages c = p.c;
        c.table += b0 * c.table_stride;
        c.lengths += b0;
        ktt_b200_attn_args f = {};
        f.batch = n;
        f.heads = a->heads;
        f.kv_heads = hk;
        f.sq = a->sq;
        f.sk = static_cast<int32_t>(cap);
        f.d = f.dv = d;
        f.scale = a->scale;
        f.q = p.q;
        f.k = k;
        f.v = v;
        f.out = p.out;
        f.lse_strides[2] = 1;
        // All rows of a head together, sequence after sequence: a dense call's keys, and a packed one's.
        const int64_t strides[3] = {cap * d, slice * cap * d, d};
        for (int i = 0; i < 3; ++i) {
            f.q_strides[i] = a->q_strides[i];
            f.out_strides[i] = a->out_strides[i];
            f.k_strides[i] = f.v_strides[i] = strides[i];
        }
        f.key_lengths = c.lengths;
        f.causal = a->causal ? KTT_B200_CAUSAL_KEY_END : KTT_B200_CAUSAL_NONE;
        ChunkHead head = {};
        head.words = words;
        head.total_q = a->total_q;
        head.tiles = plan.tiles;
        head.most_parts = plan.parts;
        head.sms = sm_count(current_device());
        head.d = d;
        if (a->cu_seqlens_q) {
            f.total_q = a->total_q;
            f.total_k = slice * cap;
            head.cu_q = a->cu_seqlens_q + b0;
            f.cu_seqlens_q = head.query_offsets(n);   // (the forward writes what they say)
            f.cu_seqlens_k = head.offsets();
            f.q_strides[0] = f.out_strides[0] = f.k_strides[0] = f.v_strides[0] = 0;
        } else {
            f.q = p.q + b0 * a->q_strides[0];
            f.out = p.out + b0 * a->out_strides[0];
        }
        // The kernel of one tile per CTA takes parts, an order of its tiles and operands in fp16 (unless its copies cannot address the
        // operands, or the output is not aligned for it: dense rows are bf16 then, over 4 bits too). Head dim 128 is that kernel's anyway.
        const bool several = n > 1, four = a->cache.bits == 4;
        bool wide = plan.parts > 0 || four;
        if (wide) {
            const ktt_b200_attn_args given = f;
            f.kernel = KTT_B200_KERNEL_TC5_WIDE;
            if (four) {
                f.q = base + plan.q_at + (a->cu_seqlens_q ? 0 : static_cast<int64_t>(b0) * a->sq * a->heads * d * 2);
                f.q_strides[0] = a->cu_seqlens_q ? 0 : static_cast<int64_t>(a->sq) * a->heads * d;
                f.q_strides[1] = d;
                f.q_strides[2] = static_cast<int64_t>(a->heads) * d;
            }
            wide = ktt_b200_sdpa_supported(&f) != 0;
            if (!wide) f = given;
        }
        const bool parts = wide && plan.parts > 0;
        if (!parts) head.most_parts = 0;
        ForwardParts x = {};
        x.empty = true;
        if (wide && four) {
            x.kv_powers = head.powers = reinterpret_cast<int32_t*>(base + plan.powers_at);
            x.chunks = head.chunks = chunks_of(c);
            float* q_power = reinterpret_cast<float*>(base + plan.q_powers_at);
            x.q_power = q_power + (a->cu_seqlens_q ? 0 : static_cast<int64_t>(b0) * a->sq * a->heads);
            if (b0 == 0) {   // of all launches
                head.q = static_cast<const __nv_bfloat16*>(a->q);
                head.q_rows = a->cu_seqlens_q ? a->total_q : static_cast<int64_t>(a->batch) * a->sq;
                head.heads = a->heads;
                head.sq = a->cu_seqlens_q ? 0 : a->sq;
                head.q_vec = (reinterpret_cast<uintptr_t>(a->q) & 15) == 0;
                for (int i = 0; i < 3; ++i) {
                    head.qs[i] = a->q_strides[i];
                    head.q_vec = head.q_vec && a->q_strides[i] % 8 == 0;
                }
                head.q_out = reinterpret_cast<__half*>(base + plan.q_at);
                head.q_power = q_power;
            }
        }
        // Sequences differ in length: their tiles are drawn, the longest sequence's first. (That kernel does so with a
        // counter of fewer than 256 bytes, which has to be zero before the call, and an order; the head-dim-64 kernel takes 256
        // bytes and its own order.) 4 sequences of up to 512 tokens and 8,192 keys, 16 heads over 4, D 128, dealt in the order of the
        // batch, drawn in it, and drawn by length: 121, 122 and 111 us.
        const bool drawn = parts || ((d == 128 || wide) && several);
        if (drawn) x.order = head.order(n);
        f.workspace = drawn || d == 64 ? words : nullptr;
        f.workspace_bytes = drawn ? 4 : d == 64 && !wide ? 256 : 0;
        if (int rc = read_pages(c, a->cache.bits, d, n, hk, static_cast<int>(cap), k, v, strides, head, stream)) return rc;
        MergeParams m = {};
        if (parts) {
            m.c = c;
            m.cu = f.cu_seqlens_q;
            x.part_rows = m.rows = part_rows(a, n);
            x.part_stride = m.stride = m.cu && m.rows == a->total_q ? 0 : a->sq;
            x.parts = m.parts = words + 1;
            x.most_parts = plan.parts;
            m.o = x.part_o = reinterpret_cast<float*>(base + plan.parts_at);
            m.lse = x.part_lse = x.part_o + plan.parts * m.rows * a->heads * d;
            m.batch = n;
            m.heads = a->heads;
            m.sq = a->sq;
            m.out = static_cast<__nv_bfloat16*>(f.out);
            for (int i = 0; i < 3; ++i) m.os[i] = f.out_strides[i];
        }
        if (int rc = forward_in_parts(&f, x, stream)) return rc;
        if (parts) {
            if (int rc = merge_parts(m, d, stream)) return rc;
        }
    }
    return 0;
}

}  // namespace
}  // namespace ktt

using namespace ktt;

extern "C" int64_t ktt_b200_paged_sdpa_workspace(const ktt_b200_paged_sdpa_args* a) {
    Pages c = {};
    if (!a || a->batch < 1 || a->sq < 0) {
        fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_sdpa: sizes must be positive");
        return -1;
    }
    if (const char* why = sdpa_refusal(a, c)) {
        fail(KTT_B200_ERR_UNSUPPORTED, "paged_sdpa: %s", why);
        return -1;
    }
    return a->sq == 0 ? 0 : plan_of(a, c, sm_count(current_device())).bytes;
}

extern "C" int ktt_b200_paged_sdpa(const ktt_b200_paged_sdpa_args* a, void* stream) {
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_sdpa: null arguments");
    PagedParams p = {};
    if (a->batch < 1 || a->sq < 0) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_sdpa: sizes must be positive");
    if (const char* why = sdpa_refusal(a, p.c)) {
        note_call(4);
        return fail(KTT_B200_ERR_UNSUPPORTED, "paged_sdpa: %s", why);
    }
    if (a->sq == 0) return 0;
    if (!a->cache.k || !a->cache.v || !a->cache.block_table || !a->cache.lengths || !a->q || !a->out) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_sdpa: null pointer");
    }
    if (a->q == a->out) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_sdpa: out must not overlap q");
    const Plan s = plan_of(a, p.c, sm_count(current_device()));
    if (!a->workspace || a->workspace_bytes < s.bytes) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_sdpa: workspace holds %lld bytes, %lld needed", static_cast<long long>(a->workspace_bytes), static_cast<long long>(s.bytes));
    }
    if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_sdpa: the workspace must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.out = static_cast<__nv_bfloat16*>(a->out);
    if (!s.few) return run_many(a, p, s, st);
    p.heads = a->heads;
    p.row_tiles = s.row_tiles;
    p.kv_heads = a->cache.kv_heads * s.row_tiles;
    p.group = a->heads / a->cache.kv_heads;
    p.sq = a->sq;
    p.causal = a->causal != 0;
    p.page_blocks = a->cache.page_size / 16;
    p.table_width = a->cache.table_width;
    p.scale_log2 = a->scale * kLog2e;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a->q_strides[i];
        p.os[i] = a->out_strides[i];
    }
    p.total_q = a->total_q;
    const Parts parts = parts_of(static_cast<int64_t>(s.slice) * p.kv_heads, a->d, sm_count(current_device()) * 4);
    unsigned char* base = static_cast<unsigned char*>(a->workspace);
    p.pieces = reinterpret_cast<int2*>(base);
    p.part_ml = reinterpret_cast<float2*>(base + parts.piece_bytes);
    p.part_o = reinterpret_cast<float*>(base + parts.piece_bytes + parts.ml_bytes);
    const Pages all = p.c;
    note_call(3);
    for (int b0 = 0; b0 < a->batch; b0 += s.slice) {
        p.batch = a->batch - b0 < s.slice ? a->batch - b0 : s.slice;
        p.c.table = all.table + b0 * all.table_stride;
        p.c.lengths = all.lengths + b0;
        p.cu = a->cu_seqlens_q ? a->cu_seqlens_q + b0 : nullptr;
        p.q = static_cast<const __nv_bfloat16*>(a->q) + (p.cu ? 0 : b0 * a->q_strides[0]);
        p.out = static_cast<__nv_bfloat16*>(a->out) + (p.cu ? 0 : b0 * a->out_strides[0]);
        int rc;
        if (a->cache.bits == 16) rc = a->d == 64 ? run_few<64, 16>(p, s.nt, st) : run_few<128, 16>(p, s.nt, st);
        else rc = a->d == 64 ? run_few<64, 4>(p, s.nt, st) : run_few<128, 4>(p, s.nt, st);
        if (rc) return rc;
    }
    return 0;
}
