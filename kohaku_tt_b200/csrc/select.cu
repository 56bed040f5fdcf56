// Bounds of a paged cache's keys, and the pages that a query selects by them.
//
// A page's score for query q is the largest logit that a key between its bounds could have,
//   s = sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo,   q+ = max(q, 0), q- = min(q, 0),
// so the scores of all pages are two matrix products with the queries of a K / V head's group as columns. Bound: the reading of the
// bounds, 4 D bytes a page and head (1 / P of the cache in bf16, for pages of P keys).
//
// What is selected is decided by scores in 64 bits: exact, and so of no order of summation, where the products of a head and page that are not 0
// lie within a factor of 2^30 of one another (multiples of 2^-15 of the least one's power of two, 128 of which are under 2^53 of these), else summed in one
// fixed order with a rounding of 2^-53 at each addition. The products of bf16 values are exact
// in fp32; a score is the sum of four sums of up to 4 matrix instructions each, of which every one is off by 2^-22 of the magnitudes that it
// adds up at most (two bits more than a sum of fp32 rounds by), all in all by e = 2^-19 max_h sum_d |q_hd| max |bound| (measured, over equal,
// alternating and wide-ranging values: 2^-22 of it). So the value of the last page selected lies within e of the last by fp32: pages more than
// 2 e above or below are in or out, and those between, one or a few, get their scores in 64 bits where they are not all in. Bounds whose
// least value is above the largest select some pages or others, of those there are.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "four_bits.cuh"
#include "split.cuh"

namespace ktt {

const char* bounds_of(Bounds& b, void* at, const int64_t (&strides)[3]) {
    b.at = static_cast<__nv_bfloat16*>(at);
    for (int i = 0; i < 3; ++i) {
        b.stride[i] = strides[i];
        if (strides[i] % 8) return "strides of bounds must be multiples of 16 bytes";
    }
    return reinterpret_cast<uintptr_t>(at) & 15 ? "bounds must be 16-byte aligned" : nullptr;
}
const char* bounds_of(Bounds& b, void* at, const int64_t (&strides)[3], const Pages& c, int kv_heads, int d) {
    // Rows of d values are apart where each stride, from the least on, is as far as all that lies below it. (Layouts whose parts lie between one
    // another's without touching are refused too.)
    struct Dim {
        int64_t stride, count;
    } dims[3] = {{std::abs(strides[0]), c.pages}, {std::abs(strides[1]), kv_heads}, {std::abs(strides[2]), 2}};
    std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    __int128 below = d;   // values from the first to behind the last of all smaller strides
    for (const Dim& x : dims) {
        if (x.count == 1) continue;
        if (x.stride < below) return "bounds that are written must not lie on one another";
        below += static_cast<__int128>(x.stride) * (x.count - 1);
    }
    return bounds_of(b, at, strides);
}

namespace {

// ---- bounds ------------------------------------------------------------------------------------

struct BoundsParams {
    Pages c;
    Bounds bounds;
    int batch, kv_heads;
    const int32_t* since;   // without `rows`: the keys that pages have bounds of (null: none)
    const int32_t* kept;    // only the page that a sequence is cut in: made again of the keys before kept[b] (null: not asked for)
    int64_t rows;           // > 0: keys appended behind the lengths: of each sequence, or packed
    const int32_t* cu;
    const int32_t* granted; // how many of these each sequence takes (null: all)
};

constexpr int kLotOfTokens = 16;   // packed rows that a warp looks for pages in

// A warp has a page and head: a lane eight channels of every second (D 128) or fourth row, 16 rows requested before the first is used
// (8: 37 us where it is 31). Packed rows: a warp looks at 16 of them and has the pages that begin among them, or in which a sequence's rows
// begin. Bound: bf16, the reading of the keys: 16 x up to 8,192 of 8 heads, D 128, pages of 32, 212 MB: 31.6 us, 6.7 TB/s. 4 bits: 26 us
// (38 with an address for each row), of which the reading of 59 MB is 9 and instructions, 16 to make eight values of a word and those that find the
// words, are 16 at one a cycle; 0.57 are issued, as warps wait for memory and for the pipe of packed pairs by turns.
//
// kSome: keys of an append of which some are granted, or the page that a sequence is cut in. (Told apart by null pointers alone, 1,024 keys of 4 bits
// took 2.25 us where it is 2.07.)
template <int D, int kBits, bool kPacked, bool kSome>
__global__ void __launch_bounds__(256) bounds_kernel(const __grid_constant__ BoundsParams p) {
    constexpr int kChunks = D / 8, kStep = 32 / kChunks;
    const int lane = threadIdx.x & 31, chunk = lane % kChunks, page_size = p.c.page_size;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t lot = unit >> 32 ? unit / p.kv_heads : static_cast<uint32_t>(unit) / static_cast<uint32_t>(p.kv_heads);
    const int head = static_cast<int>(unit - lot * p.kv_heads);

    // Rows begin .. end - 1 of a page, into what the page has if begin > 0.
    auto widen = [&](int b, int entry, int begin, int end) {
        const int64_t page = p.c.table[b * p.c.table_stride + entry];
        if (page < 0 || page >= p.c.pages) return;
        const unsigned char* from = p.c.k + page * p.c.ks[0] + head * p.c.ks[1];
        Edges e;
#pragma unroll
        for (int i = 0; i < Eight<__nv_bfloat16>::kPieces; ++i) {
            e.lo.raw[i] = make_uint4(0x7f807f80u, 0x7f807f80u, 0x7f807f80u, 0x7f807f80u);   // infinities
            e.hi.raw[i] = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
        }
        const bool last = lane < kChunks && begin > 0;
        Edges old;
        if (last) {
            old.lo.load(p.bounds.edge(page, head, 0) + chunk * 8);
            old.hi.load(p.bounds.edge(page, head, 1) + chunk * 8);
        }
        if constexpr (kBits == 16) {
            auto rows = [&](auto ahead, int r0) {
                constexpr int kAhead = decltype(ahead)::value;
                Eight<__nv_bfloat16> x[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int r = min(r0 + lane / kChunks + i * kStep, end - 1);   // (a row twice changes nothing)
                    x[i].load(reinterpret_cast<const __nv_bfloat16*>(from + r * p.c.ks[2]) + chunk * 8);
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) e.with(x[i], x[i]);
            };
            int r0 = begin;
            for (; r0 + 8 * kStep < end; r0 += 16 * kStep) rows(std::integral_constant<int, 16>(), r0);
            if (r0 < end) rows(std::integral_constant<int, 8>(), r0);
        } else {
            // Blocks of 16 rows, whose words lie at fixed places; of blocks that are not all there, a row that is not is the nearest that is.
            constexpr int kRows = 16 / kStep, kLot = D == 128 ? 2 : 4;
            auto rows = [&](auto blocks, int r0) {
                constexpr int kBlocks = decltype(blocks)::value;
                uint2 x[kBlocks * kRows];
                if (r0 >= begin && r0 + 16 * kBlocks <= end) {
                    const uint32_t* block = reinterpret_cast<const uint32_t*>(from + static_cast<int64_t>(r0 >> 4) * (9 * D));
                    const uint32_t *word = block + key_word<D>(lane / kChunks, chunk), *step = block + step_word<D>(lane / kChunks, chunk / 8);
#pragma unroll
                    for (int i = 0; i < kBlocks * kRows; ++i) {
                        const int at = i / kRows * (9 * D / 4), row = i % kRows * kStep;
                        x[i] = make_uint2(word[at + row * (D / 8)], step[at + row * (D / 64)]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kBlocks * kRows; ++i) {
                        const int r = min(max(r0 + lane / kChunks + i * kStep, begin), end - 1);
                        const uint32_t* block = reinterpret_cast<const uint32_t*>(from + static_cast<int64_t>(r >> 4) * (9 * D));
                        x[i] = make_uint2(block[key_word<D>(r & 15, chunk)], block[step_word<D>(r & 15, chunk / 8)]);
                    }
                }
#pragma unroll
                for (int i = 0; i < kBlocks * kRows; ++i) {
                    const Eight<__nv_bfloat16> y = of_four_bits(x[i].x, x[i].y);
                    e.with(y, y);
                }
            };
            int r0 = begin & ~15;
            for (; r0 + 16 < end; r0 += 16 * kLot) rows(std::integral_constant<int, kLot>(), r0);
            if (r0 < end) rows(std::integral_constant<int, 1>(), r0);
        }
#pragma unroll
        for (int off = kChunks; off < 32; off <<= 1) {
            Edges other;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                reinterpret_cast<uint32_t*>(other.lo.raw)[i] = __shfl_xor_sync(0xffffffffu, reinterpret_cast<uint32_t*>(e.lo.raw)[i], off);
                reinterpret_cast<uint32_t*>(other.hi.raw)[i] = __shfl_xor_sync(0xffffffffu, reinterpret_cast<uint32_t*>(e.hi.raw)[i], off);
            }
            e.with(other.lo, other.hi);
        }
        if (last) e.with(old.lo, old.hi);
        if (lane < kChunks) {
            e.lo.store(p.bounds.edge(page, head, 0) + chunk * 8);
            e.hi.store(p.bounds.edge(page, head, 1) + chunk * 8);
        }
    };

    if constexpr (kPacked) {
        const int64_t n = lot * kLotOfTokens + lane;
        int b = -1, place = 0, end = 0;
        bool leads = false;
        const bool mine = lane < kLotOfTokens && n < p.rows;
        int64_t start = 0, behind = 0;
        [[maybe_unused]] int64_t many = 0;
        int keys = 0;
        if (p.batch < 32) {   // a lane looks at a sequence, its length with it, in one trip
            const int offset = p.cu[min(lane, p.batch)], have = cached_keys(p.c, min(lane, p.batch - 1));
            [[maybe_unused]] int64_t takes = 0;
            if constexpr (kSome) takes = granted_to(p.granted, min(lane, p.batch - 1));
            // (The last that starts at or before the token, -1: none; five looks at another lane's.)
#pragma unroll
            for (int step = 16; step > 0; step >>= 1) {
                const int start_of = __shfl_sync(0xffffffffu, offset, min(b + step, 31));
                if (b + step <= p.batch && start_of <= n) b += step;
            }
            if (!mine || b >= p.batch) b = -1;
            start = __shfl_sync(0xffffffffu, offset, max(b, 0));
            behind = __shfl_sync(0xffffffffu, offset, max(b, 0) + 1);
            keys = __shfl_sync(0xffffffffu, have, max(b, 0));
            if constexpr (kSome) many = __shfl_sync(0xffffffffu, takes, max(b, 0));
        } else if (mine) {
            b = sequence_of(p.cu, p.batch, n);
            if (b >= 0) {
                start = p.cu[b];
                behind = p.cu[b + 1];
                keys = cached_keys(p.c, b);
                if constexpr (kSome) many = granted_to(p.granted, b);
            }
        }
        if constexpr (kSome) behind = min(behind, start + many);
        if (b >= 0 && n >= start && n < behind) {   // (offsets that decrease)
            const int64_t in = n - start, at = keys + in, all = at + (behind - n);
            end = static_cast<int>(all < p.c.cap ? all : p.c.cap);
            leads = at < end && (in == 0 || static_cast<uint32_t>(at) % static_cast<uint32_t>(page_size) == 0);   // (at < end: 2^30 at most)
            place = leads ? static_cast<int>(at) : 0;
        }
        uint32_t leaders = __ballot_sync(0xffffffffu, leads);
        while (leaders) {
            const int from = __ffs(leaders) - 1;
            leaders &= leaders - 1;
            const int lb = __shfl_sync(0xffffffffu, b, from), at = __shfl_sync(0xffffffffu, place, from), last = __shfl_sync(0xffffffffu, end, from);
            const int entry = at / page_size;
            widen(lb, entry, at - entry * page_size, min(last - entry * page_size, page_size));
        }
    } else {
        const int b = blockIdx.y, len = cached_keys(p.c, b);
        int begin = 0, end = len;
        if (p.rows > 0) {
            begin = len;
            int64_t rows = p.rows;
            if constexpr (kSome) rows = min(rows, granted_to(p.granted, b));
            end = static_cast<int>(len + rows < p.c.cap ? len + rows : p.c.cap);
        } else if (kSome) {
            end = min(max(p.kept[b], 0), len);
            begin = end < len ? end - end % page_size : end;
        } else if (p.since) {
            begin = min(max(p.since[b], 0), len);
        }
        const int64_t entry = begin / page_size + lot, first = entry * page_size;
        if (first >= end || begin >= end) return;
        widen(b, static_cast<int>(entry), max(begin - static_cast<int>(first), 0), min(end - static_cast<int>(first), page_size));
    }
}

// Blocks of a launch in x: 8 pages (packed rows: lots of them) and heads each.
int64_t blocks_of(const BoundsParams& p) {
    const int64_t page = p.c.page_size, all = (p.c.cap + page - 1) / page;   // pages of a sequence
    const int64_t lots = p.cu ? (p.rows + kLotOfTokens - 1) / kLotOfTokens : p.kept ? 1 : (p.rows > 0 ? std::min((p.rows + page - 2) / page + 1, all) : all);
    return (lots * p.kv_heads + 7) / 8;
}
// Of lengths that the device alone knows, more pages and heads than a launch has blocks for.
const char* too_many(const BoundsParams& p) { return blocks_of(p) >= (1ll << 31) ? "bounds of fewer than 2^34 pages and heads of a sequence" : nullptr; }

template <int D, int kBits>
int launch_bounds(const BoundsParams& p, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(blocks_of(p)), static_cast<unsigned>(p.cu ? 1 : p.batch));
    const bool some = p.granted || p.kept;
    if (p.cu && some) return launch_dependent(bounds_kernel<D, kBits, true, true>, p, grid, dim3(256), stream, "paged_bounds launch");
    if (p.cu) return launch_dependent(bounds_kernel<D, kBits, true, false>, p, grid, dim3(256), stream, "paged_bounds launch");
    if (some) return launch_dependent(bounds_kernel<D, kBits, false, true>, p, grid, dim3(256), stream, "paged_bounds launch");
    return launch_dependent(bounds_kernel<D, kBits, false, false>, p, grid, dim3(256), stream, "paged_bounds launch");
}
int launch_bounds(const BoundsParams& p, int bits, int d, cudaStream_t stream) {
    if (bits == 16) return d == 64 ? launch_bounds<64, 16>(p, stream) : launch_bounds<128, 16>(p, stream);
    return d == 64 ? launch_bounds<64, 4>(p, stream) : launch_bounds<128, 4>(p, stream);
}

// ---- scores ------------------------------------------------------------------------------------

// Division of numbers under 2^31 by one that the host knows, d: with 2^s the power of two at or above it, n / d is n ceil(2^(31 + s) / d) / 2^(31 + s),
// whole part, as the product is off by less than n / 2^(31 + s) < 1 / d. (A division of 32 bits takes some 20 dependent instructions, and a
// selection has five.)
struct Divisor {
    uint32_t by, times;
    int shift;
    explicit Divisor(int64_t d = 1) : by(static_cast<uint32_t>(d)), shift(31) {
        while ((1ll << (shift - 31)) < d) ++shift;
        times = static_cast<uint32_t>(((1ull << shift) + by - 1) / by);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return static_cast<uint32_t>(static_cast<uint64_t>(n) * times >> shift); }
    __device__ __forceinline__ uint32_t rest(uint32_t n) const { return n - (*this)(n) * by; }
};

struct SelectParams {
    Divisor by_page, by_sq, by_heads, by_ranks;   // page_size, sq, kv_heads, ranks
    const __nv_bfloat16* q;
    int64_t qs[3];
    const int32_t* cu;
    int64_t total_q;
    int64_t token0, tokens;   // of this launch, of all
    int batch, sq, kv_heads, group;
    Bounds bounds;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    int64_t pages;
    int page_size, cap;
    int top, first, last;
    int width, blocks;        // pages that the table has, and blocks of 16
    int ranks;                // CTAs of a pair
    float* scores;            // [pairs][blocks][16]; null: in shared memory
    double* exact;            // [pairs][blocks][16], of the pages that need them; null: in shared memory, where the rings were
    int32_t* chosen;
    int32_t* keys;
};

// A query token: its row of q, its sequence (-1: none), and where in it. By whole warps.
struct Token {
    const __nv_bfloat16* q;
    int b;
    int64_t place, of;   // the how-many-th of its sequence's tokens, and how many there are
};
__device__ __forceinline__ Token token_of(const SelectParams& p, int64_t t) {
    Token x;
    if (p.cu) {
        // The last sequence that starts at or before t: a warp's lanes look at 32 offsets that are evenly spaced, then between two of them.
        const int lane = threadIdx.x & 31;
        int from = 0, many = p.batch + 1;   // offsets that it is among; cu[batch] too, where t lies behind all
        while (many > 1) {
            const int step = (many + 31) / 32, i = lane * step;
            const uint32_t before = __ballot_sync(0xffffffffu, i < many && p.cu[from + min(i, many - 1)] <= t);
            if (!before) break;   // (t lies before all)
            const int at = (31 - __clz(before)) * step;
            from += at;
            many = min(step, many - at);
        }
        x.q = p.q + t * p.qs[2];
        x.b = -1;
        x.place = x.of = 0;
        if (from < p.batch && p.cu[from] <= t) {
            x.place = t - p.cu[from];
            x.of = p.cu[from + 1] - p.cu[from];
            if (x.place < x.of) x.b = from;   // (offsets that decrease)
        }
    } else {
        x.b = static_cast<int>(p.by_sq(static_cast<uint32_t>(t)));
        x.place = t - static_cast<int64_t>(x.b) * p.sq;
        x.of = p.sq;
        x.q = p.q + x.b * p.qs[0] + x.place * p.qs[2];
    }
    return x;
}
// The keys that it sees.
__device__ __forceinline__ int seen_by(const SelectParams& p, const Token& x) {
    if (x.b < 0) return 0;
    const int len = min(max(p.lengths[x.b], 0), p.cap);
    const int64_t seen = len - x.of + x.place + 1;
    return static_cast<int>(seen < 0 ? 0 : (seen < len ? seen : len));
}

constexpr int kWarps = 4;        // of a CTA
constexpr int kMaxRanks = 8;
constexpr int kBins = 128;       // that scores are counted in
constexpr int kFew = 256;        // pages between in and out that are ranked one against the others

// A warp's ring: blocks of 16 pages' bounds, a row of 4 D bytes each and 16 more, so that eight rows of a matrix lie in different banks.
template <int D>
struct Ring {
    static constexpr int kRow = 4 * D + 16;
    static constexpr int kBlock = 16 * kRow;
    static constexpr int kStages = 3;
    static constexpr int kBytes = kWarps * kStages * kBlock;
};

struct SelectShared {
    int of_warp[3][kMaxRanks * kWarps];   // by warp: the largest magnitude among the bounds, the least and the largest score (ordered)
    alignas(16) int bins[kBins];
    int sums[2][kWarps];
    int found, count, need, least, largest;
    float value;
    unsigned long long exact;
};
// Of the selection, where the ring was.
constexpr int kRanked = 32 * kWarps;     // scores that are ranked one against the others
struct SelectLater {
    float ranked[kRanked];
    double few[kFew];
    int few_at[kFew];
    int few_in[kFew];
    int bins[256];
};

// Order of floats as that of integers.
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(x);
    return i < 0 ? i ^ 0x7fffffff : i;
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i < 0 ? i ^ 0x7fffffff : i); }
__device__ __forceinline__ unsigned long long ordered(double x) {
    const unsigned long long i = __double_as_longlong(x);
    return i >> 63 ? ~i : i | 1ull << 63;
}

// Exclusive sum of x over the CTA, and that of all; warps: not in use by another sum before the next barrier.
__device__ __forceinline__ int sum_before(int x, int* warps, int& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += y;
    }
    if (lane == 31) warps[warp] = sum;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const int y = warps[w];
        before += w < warp ? y : 0;
        all += y;
    }
    return before + sum - x;
}

// Stores to shared memory of the cluster's first CTA.
__device__ __forceinline__ void to_first(uint32_t at, float x) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(x) : "memory"); }
__device__ __forceinline__ void to_first(uint32_t at, int x) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at), "r"(x) : "memory"); }

// The score of a page in 64 bits: sums of products that are exact themselves. By one warp, a lane D / 32 neighbouring channels; eight heads at a
// time, whose sums over the lanes halve the heads of a lane before its lanes.
template <int D>
__device__ __forceinline__ double exact_score(const SelectParams& p, const Token& tok, int hk, int64_t page) {
    const int lane = threadIdx.x & 31;
    constexpr int kMine = D / 32;
    if (page < 0 || page >= p.pages) return 0.0;
    auto load = [&](double (&to)[kMine], const __nv_bfloat16* from) {
        __nv_bfloat162 x[kMine / 2];
        if constexpr (kMine == 4) *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(from);
        else x[0] = *reinterpret_cast<const __nv_bfloat162*>(from);
#pragma unroll
        for (int i = 0; i < kMine / 2; ++i) {
            const float2 f = __bfloat1622float2(x[i]);
            to[2 * i] = f.x;
            to[2 * i + 1] = f.y;
        }
    };
    double lo[kMine], hi[kMine], best = -INFINITY;
    load(lo, p.bounds.edge(page, hk, 0) + lane * kMine);
    load(hi, p.bounds.edge(page, hk, 1) + lane * kMine);
    for (int h0 = 0; h0 < p.group; h0 += 8) {
        double sum[8];
#pragma unroll
        for (int h = 0; h < 8; ++h) {   // (heads past the last: it again)
            double q[kMine];
            load(q, tok.q + static_cast<int64_t>(hk * p.group + min(h0 + h, p.group - 1)) * p.qs[1] + lane * kMine);
            sum[h] = 0.0;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const double a = q[i] * lo[i], b = q[i] * hi[i];
                sum[h] += a != a || a > b ? a : b;   // (a NaN of either stays)
            }
        }
#pragma unroll
        for (int n = 4; n > 0; n /= 2) {
            const bool upper = lane & (4 * n);
#pragma unroll
            for (int h = 0; h < n; ++h) {
                const double keep = upper ? sum[h + n] : sum[h], give = upper ? sum[h] : sum[h + n];
                sum[h] = keep + __shfl_xor_sync(0xffffffffu, give, 4 * n);
            }
        }
        sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 2);
        sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 1);
        double x = sum[0] != sum[0] ? INFINITY : sum[0];
#pragma unroll
        for (int off = 16; off >= 4; off /= 2) {
            const double y = __shfl_xor_sync(0xffffffffu, x, off);
            x = y > x ? y : x;
        }
        best = x > best ? x : best;
    }
    return best + 0.0;   // (no -0)
}

// A cluster of `ranks` CTAs has a (token, K / V head): all of their warps score its pages, the first selects.
//
// Scores: the blocks of 16 pages are dealt to the warps in turn, each of which takes them through a ring of its own, two or three on their way while
// one is multiplied: pages are the rows of m16n8k16, q+ and q- of 8 heads its columns. (Bounds in registers as they come, two blocks to a warp, were
// no faster than one after the other: 16 us for 38 MB.) The products of a block are four sums, for the latency of one.
//
// Selection: the value of the k-th largest score, by counts in bins of equal width, of which the one that has it is cut again while it holds many,
// and by rank among those of the last. A thread has kItems neighbouring pages in registers (0: reads them each time), and a sum over the CTA
// places those that are in. (32 thresholds, one to a lane whose warp goes through its share of the scores, were 1,700 clocks a round of 1,024
// scores; four at a time, each by a sum over the CTA, 950 and five rounds.) kNear: scores, names and exact scores lie in shared memory, else
// scores and exact ones in the workspace.
//
// Measured: 64 x up to 16,384 keys, 16 heads over 2, D 128, pages of 16, 14.1 us, of which the reading of 40 MB is 6; 1 x up to 65,536, 32 over 8,
// pages of 64, 6.1, waits that follow one another.
template <int D, int kItems, bool kNear>
__global__ void __launch_bounds__(32 * kWarps, 2) select_kernel(const __grid_constant__ SelectParams p) {
    using R = Ring<D>;
    constexpr int K = D / 16, NS = R::kStages;   // (two blocks on their way)
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ SelectShared sm;
    SelectLater& later = *reinterpret_cast<SelectLater*>(dynamic);
    static_assert(sizeof(SelectLater) <= R::kBytes, "where the ring was");
    float* score_s = reinterpret_cast<float*>(dynamic + R::kBytes);           // kNear: [blocks][16]
    int* name_s = reinterpret_cast<int*>(score_s + p.blocks * 16);
    constexpr int threads = 32 * kWarps, warps = kWarps;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    if (tid == 0) sm.found = sm.count = 0;
    for (int i = tid; i < kBins; i += threads) sm.bins[i] = 0;
    if (p.ranks > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");   // (met before the first store to another CTA)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t pair = p.by_ranks(blockIdx.x), local = p.by_heads(pair);
    const int rank = static_cast<int>(blockIdx.x - pair * p.ranks), hk = static_cast<int>(pair - local * p.kv_heads);
    const int64_t t = p.token0 + local;   // (under 2^31)
    const Token tok = token_of(p, t);
    const int32_t* row = p.table + max(tok.b, 0) * p.table_stride;
    // Requested before the length is known: the queries of the first 8 heads, and (for the cache) the table's row.
    uint32_t up[K][2], down[K][2];
    const __nv_bfloat16* queries_at = tok.q + static_cast<int64_t>(hk * p.group + min(g, p.group - 1)) * p.qs[1] + 2 * t4;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < 2; ++i) up[k][i] = *reinterpret_cast<const uint32_t*>(queries_at + 16 * k + 8 * i);
    }
    if (warp == 0 && lane * 32 < p.blocks * 16) asm volatile("prefetch.global.L1 [%0];" ::"l"(row + min(lane * 32, p.width - 1)));
    // Blocks are dealt to all warps of the cluster in turn; the first ones' bounds are requested too (names past the length: of pages of others, or none).
    const int step = p.ranks * warps, own_block = rank * warps + warp;
    const uint32_t ring = smem_u32(dynamic + warp * NS * R::kBlock), first_scores = in_rank(smem_u32(score_s), 0), first_names = in_rank(smem_u32(name_s), 0);
    auto names_of = [&](int i, int limit) {   // of this warp's blocks i and i + 1, a lane each
        const int e = (own_block + (i + (lane >> 4)) * step) * 16 + (lane & 15);
        return e < limit ? row[e] : -1;
    };
    auto issue = [&](int i, int names) {   // a block's bounds, a page's with one instruction (D 64: two pages' with one)
        const uint32_t to = ring + (i % NS) * R::kBlock;
        constexpr int kLanes = D / 4, kPages = 32 / kLanes;   // lanes to a page
        const int at = lane % kLanes * 8, edge = at / D;
        const __nv_bfloat16* from = p.bounds.at + hk * p.bounds.stride[1] + edge * p.bounds.stride[2] + (at - edge * D);
#pragma unroll
        for (int j = 0; j < 16; j += kPages) {
            const int r = j + lane / kLanes, name = __shfl_sync(0xffffffffu, names, (i & 1) * 16 + r);
            const bool there = name >= 0 && name < p.pages;
            cp_async_16(to + r * R::kRow + at * 2, from + (there ? name : 0) * p.bounds.stride[0], there);
        }
    };
    int names = names_of(0, p.width), next = names_of(2, p.width);
    const int seen = seen_by(p, tok);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (own_block + i * step < p.blocks) issue(i, names);
        cp_async_commit();
    }
    const int count = static_cast<int>(p.by_page(static_cast<uint32_t>(seen) + p.page_size - 1)), top = p.top;
    int32_t* to = p.chosen + (t * p.kv_heads + hk) * top;
    if (rank == 0 && tid == 0) {
        const int many = min(count, top);
        p.keys[t * p.kv_heads + hk] = many > 0 ? (many - 1) * p.page_size + static_cast<int>(p.by_page.rest(static_cast<uint32_t>(seen - 1))) + 1 : 0;
    }
    if (count <= top) {   // all of them
        cp_async_wait<0>();
        for (int i = rank * threads + tid; i < top; i += threads * p.ranks) to[i] = i < count ? row[i] : -1;
        return;
    }
    float* given = kNear ? score_s : p.scores + static_cast<int64_t>(pair) * p.blocks * 16;
    const int begin = p.first, end = count - p.last, k = top - p.first - p.last;   // the k largest of [begin, end), which are more

    // ---- scores
    float norm = 0.f;        // the largest sum of magnitudes of a head's query
    {
        const int all = (count + 15) / 16, blocks = all > own_block ? (all - own_block + step - 1) / step : 0;
        // up: heads h0 .. h0 + 7 as they are; then q+ and q-, and the sums of their magnitudes.
        auto split = [&](int h0) {
            const bool there = h0 + g < p.group;
            const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const __nv_bfloat162 y = *reinterpret_cast<const __nv_bfloat162*>(&up[k][i]), u = __hmax2_nan(y, zero), v = __hmin2_nan(y, zero);
                    up[k][i] = there ? *reinterpret_cast<const uint32_t*>(&u) : 0u;
                    down[k][i] = there ? *reinterpret_cast<const uint32_t*>(&v) : 0u;
                    const float2 f = __bfloat1622float2(y);
                    sum += there ? fabsf(f.x) + fabsf(f.y) : 0.f;
                }
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            // (as an integer, which a NaN is the largest of)
            norm = __uint_as_float(__reduce_max_sync(0xffffffffu, max(__float_as_uint(sum), __float_as_uint(norm))));
        };
        auto queries = [&](int h0) {
            const __nv_bfloat16* from = tok.q + static_cast<int64_t>(hk * p.group + min(h0 + g, p.group - 1)) * p.qs[1] + 2 * t4;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < 2; ++i) up[k][i] = *reinterpret_cast<const uint32_t*>(from + 16 * k + 8 * i);
            }
            split(h0);
        };
        split(0);
        for (int h0 = 8; h0 < p.group; h0 += 8) queries(h0);   // (of all for the norm, which all warps need)
        __nv_bfloat162 largest[2], least[2];
        largest[0] = largest[1] = least[0] = least[1] = __float2bfloat162_rn(0.f);
        float lo = INFINITY, hi = -INFINITY;
        if (p.ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        for (int block = 0; block < blocks; ++block) {
            // Two ahead. Names of a pair of blocks are those of the next two once their own are on their way.
            if (block & 1) {
                if (block + 2 < blocks) issue(block + 2, names);
            } else {
                if constexpr (kNear) {
                    const int of = block + (lane >> 4);
                    if (of < blocks) to_first(first_names + ((own_block + of * step) * 16 + (lane & 15)) * 4, names);
                }
                names = next;
                if (block + 2 < blocks) issue(block + 2, names);
                next = names_of(block + 4, count);
            }
            cp_async_commit();
            cp_async_wait<2>();
            __syncwarp();
            const int behind = (own_block + block * step + 1) * 16 - count;
            if (behind > 0) {   // rows past the last page count for nothing
                for (int i = lane; i < behind * (4 * D / 16); i += 32) {
                    *reinterpret_cast<uint4*>(dynamic + (warp * NS + block % NS) * R::kBlock + (15 - i / (4 * D / 16)) * R::kRow + i % (4 * D / 16) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                __syncwarp();
            }
            const uint32_t from = ring + (block % NS) * R::kBlock + ((lane & 7) + ((lane >> 3) & 1) * 8) * R::kRow + (lane >> 4) * 16;
            float s[2] = {-INFINITY, -INFINITY};
            for (int h0 = 0; h0 < p.group; h0 += 8) {
                if (p.group > 8) queries(h0);   // (more than 8 heads: each tile's again)
                float acc[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    uint32_t lo[4], hi[4];
                    ldmatrix_x4(lo, from + k * 32);
                    ldmatrix_x4(hi, from + 2 * D + k * 32);
                    mma_bf16(acc[k & 1], hi, up[k][0], up[k][1]);
                    mma_bf16(acc[2 + (k & 1)], lo, down[k][0], down[k][1]);
                    if (h0 == 0) {   // (the largest magnitude is that of a largest or a least value)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            largest[i & 1] = __hmax2_nan(largest[i & 1], *reinterpret_cast<const __nv_bfloat162*>(&hi[i]));
                            least[i & 1] = __hmin2_nan(least[i & 1], *reinterpret_cast<const __nv_bfloat162*>(&lo[i]));
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[0][i] = (acc[0][i] + acc[1][i]) + (acc[2][i] + acc[3][i]);
                // The largest of the columns that are heads.
                const bool c0 = h0 + 2 * t4 < p.group, c1 = h0 + 2 * t4 + 1 < p.group;
                s[0] = fmaxf(s[0], fmaxf(c0 ? acc[0][0] : -INFINITY, c1 ? acc[0][1] : -INFINITY));
                s[1] = fmaxf(s[1], fmaxf(c0 ? acc[0][2] : -INFINITY, c1 ? acc[0][3] : -INFINITY));
            }
            __syncwarp();   // (all lanes are done with the stage before it is filled again)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[i] = fmaxf(s[i], __shfl_xor_sync(0xffffffffu, s[i], 1));
                s[i] = fmaxf(s[i], __shfl_xor_sync(0xffffffffu, s[i], 2));
            }
            // What is not asked about is below everything.
            const int e = (own_block + block * step) * 16 + g;
            if (e >= begin && e < end) {
                lo = fminf(lo, s[0]);
                hi = fmaxf(hi, s[0]);
            } else {
                s[0] = -INFINITY;
            }
            if (e + 8 >= begin && e + 8 < end) {
                lo = fminf(lo, s[1]);
                hi = fmaxf(hi, s[1]);
            } else {
                s[1] = -INFINITY;
            }
            if (t4 == 0) {
                if constexpr (kNear) {
                    to_first(first_scores + e * 4, s[0]);
                    to_first(first_scores + (e + 8) * 4, s[1]);
                } else {
                    given[e] = s[0];
                    given[e + 8] = s[1];
                }
            }
        }
        cp_async_wait<0>();
        const __nv_bfloat162 high = __hmax2_nan(__hmax2_nan(largest[0], largest[1]), __hneg2(__hmin2_nan(least[0], least[1])));
        const uint32_t bits = *reinterpret_cast<const uint32_t*>(&high) & 0x7fff7fffu;
        const uint32_t most = __reduce_max_sync(0xffffffffu, max(bits & 0xffffu, bits >> 16)) << 16;   // (bf16 magnitudes as integers, a NaN above all)
        const int least_score = __reduce_min_sync(0xffffffffu, ordered(lo)), largest_score = __reduce_max_sync(0xffffffffu, ordered(hi));
        if (lane < 3) {
            const uint32_t slot = in_rank(smem_u32(&sm.of_warp[lane][own_block]), 0);
            to_first(slot, lane == 0 ? static_cast<int>(most) : lane == 1 ? least_score : largest_score);
        }
    }
    if (p.ranks > 1) cluster_meet(); else __syncthreads();
    if (rank > 0) return;   // (nobody looks at its shared memory)

    // ---- the selection, by the first CTA
    const int mine = kItems ? kItems : (count + threads - 1) / threads | 1, first = tid * mine;   // (odd: neighbours in different banks)
    float held[kItems ? kItems : 1];
    int held_bin[kItems ? kItems : 1];
    if constexpr (kItems > 0) {
#pragma unroll
        for (int i = 0; i < kItems; i += 4) {
            float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (first + i < count) x = *reinterpret_cast<const float4*>(given + first + i);   // (whole blocks of 16 are written, below everything past the end)
            held[i] = x.x; held[i + 1] = x.y; held[i + 2] = x.z; held[i + 3] = x.w;
        }
    }
    auto name_of = [&](int e) { return kNear ? name_s[e] : row[e]; };
    const bool slot = lane < step;
    const float most = __int_as_float(__reduce_max_sync(0xffffffffu, slot ? sm.of_warp[0][lane] : 0)), mass = norm * most;
    float lo = from_ordered(__reduce_min_sync(0xffffffffu, slot ? sm.of_warp[1][lane] : 0x7fffffff)), hi = from_ordered(__reduce_max_sync(0xffffffffu, slot ? sm.of_warp[2][lane] : static_cast<int>(0x80000000)));
    // What the fp32 scores may be off by. (What the products could lose below fp32's least normal number is in the last terms.)
    const float off = fmaf(mass, 0x1p-19f, fmaf(norm + most, 0x1p-110f, 0x1p-110f));
    // Else, and where it is no number, all in 64 bits. (Scores past it are of bounds whose least value is above the largest.)
    const bool sure = mass < 0x1p120f && lo > -0x1p121f && hi < 0x1p121f;
    // This thread's pages and their scores, and (kItems) pages that are not asked about, whose scores are below all: f(page, score, bin).
    auto each = [&](auto f) {
        if constexpr (kItems > 0) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) f(first + i, held[i], held_bin[i]);
        } else {
            int bin = 0;
            for (int e = max(first, begin); e < min(first + mine, end); ++e) f(e, sure ? given[e] : 0.f, bin);
        }
    };
    // Of those for which pick(page, score, bin) holds: use(page). The few there are, one after another, so that a warp goes through as many as its lane
    // with the most has, not through all pages of a lane.
    auto each_of = [&](auto pick, auto use) {
        if constexpr (kItems > 0) {
#pragma unroll
            for (int i0 = 0; i0 < kItems; i0 += 32) {
                uint32_t mask = 0u;
#pragma unroll
                for (int i = i0; i < i0 + 32 && i < kItems; ++i) mask |= static_cast<uint32_t>(pick(first + i, held[i], held_bin[i])) << (i - i0);
                for (; mask; mask &= mask - 1) use(first + i0 + __ffs(mask) - 1);
            }
        } else {
            each([&](int e, float x, int& bin) {
                if (pick(e, x, bin)) use(e);
            });
        }
    };
    int need = k;
    for (int round = 0; round < 6 && sure && k > 0 && hi - lo > 4.f * off; ++round) {
        const float by = (kBins - 0.5f) / (hi - lo), low = lo, high = hi;
        if (!(by < 0x1p100f)) break;
        // (falls nowhere as x rises; -1 and below: outside)
        auto bin_of = [&](float x) { return x <= high ? static_cast<int>(floorf((x - low) * by)) : -1; };
        each([&](int, float x, int& bin) {
            bin = bin_of(x);
            if (bin >= 0) atomicAdd(&sm.bins[bin], 1);
        });
        __syncthreads();
        // Every warp for itself: lane l has 4 bins from the top, kBins - 4 (l + 1) .., and looks for the one that has the need-th.
        const int4 own4 = reinterpret_cast<const int4*>(sm.bins)[kBins / 4 - 1 - lane];
        const int own[4] = {own4.w, own4.z, own4.y, own4.x}, sum = (own[0] + own[1]) + (own[2] + own[3]);
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        int above = upto - sum, which = 0, many = own[0];
        const bool holds = above < need && upto >= need;
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            if (above + many < need) {   // (only the lane that holds it matters)
                above += many;
                many = own[i];
                which = i;
            }
        }
        const int holder = __ffs(__ballot_sync(0xffffffffu, holds)) - 1;
        const int bin = __shfl_sync(0xffffffffu, kBins - 1 - 4 * lane - which, holder);
        many = __shfl_sync(0xffffffffu, many, holder);
        need -= __shfl_sync(0xffffffffu, above, holder);
        if (many <= kRanked) {
            if (tid >= many) later.ranked[tid] = -INFINITY;
            each_of([&](int, float x, int of) { return (kItems > 0 ? of : bin_of(x)) == bin; }, [&](int e) { later.ranked[atomicAdd(&sm.found, 1)] = given[e]; });
            __syncthreads();
            // The need-th of them, equal ones in any order.
            if (tid < many) {
                const float x = later.ranked[tid];
                int better = 0;
                for (int i = 0; i < many; i += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(later.ranked + i);
                    better += (y.x > x || (y.x == x && i < tid)) + (y.y > x || (y.y == x && i + 1 < tid)) + (y.z > x || (y.z == x && i + 2 < tid)) + (y.w > x || (y.w == x && i + 3 < tid));
                }
                if (better == need - 1) sm.value = x;
            }
            __syncthreads();
            lo = hi = sm.value;
            break;
        }
        __syncthreads();   // (all have looked at the bins)
        for (int i = tid; i < kBins; i += threads) sm.bins[i] = 0;
        if (tid == 0) {
            sm.least = 0x7fffffff;
            sm.largest = static_cast<int>(0x80000000);
        }
        __syncthreads();
        each_of([&](int, float x, int of) { return (kItems > 0 ? of : bin_of(x)) == bin; }, [&](int e) {
            atomicMin(&sm.least, ordered(given[e]));
            atomicMax(&sm.largest, ordered(given[e]));
        });
        __syncthreads();
        lo = from_ordered(sm.least);
        hi = from_ordered(sm.largest);
    }
    // Pages above are in, pages below are out, those between are counted. (Where nothing is sure all are between, whatever their scores.)
    const float above = sure ? hi + 2.f * off : 1.f, below = sure ? lo - 2.f * off : 0.f;
    if constexpr (kItems > 0) {
        if (!sure) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) held[i] = first + i >= begin && first + i < end ? 0.f : -INFINITY;
        }
    }
    auto score_of = [&](int e) { return sure ? given[e] : 0.f; };
    auto surely = [&](float x) { return x > above; };
    auto doubtful = [&](float x) { return x >= below && !(x > above); };
    int in = 0, some = 0;
    if (k > 0) {
        each([&](int, float x, int&) {
            in += x > above;
            some += x >= below;
        });
        some -= in;
    }
    int at, all_in, all_some;
    if (kItems > 0) {   // (fewer than 2^15 of either)
        at = sum_before(in | some << 16, sm.sums[0], all_in);
        all_some = all_in >> 16;
        all_in &= 0xffff;
        at = (at & 0xffff) + (at >> 16);
    } else {
        at = sum_before(in, sm.sums[0], all_in);
        at += sum_before(some, sm.sums[1], all_some);
    }
    const int rest = k - all_in;   // so many of the doubtful ones are in
    for (int i = tid; i < p.first; i += threads) to[i] = name_of(i);
    for (int i = tid; i < p.last; i += threads) to[top - p.last + i] = name_of(end + i);
    to += p.first;
    if (k == 0) return;
    if (all_some == rest) {
        each_of([&](int, float x, int) { return x >= below; }, [&](int e) { to[at++] = name_of(e); });
        return;
    }
    // Some of those between are in, by their exact scores.
    double* exact = kNear ? reinterpret_cast<double*>(dynamic + sizeof(SelectLater)) : p.exact + static_cast<int64_t>(pair) * p.blocks * 16;
    unsigned long long value = 0;
    int ties = 0, ties_before = 0;
    if (all_some <= kFew) {
        each_of([&](int, float x, int) { return doubtful(x); }, [&](int e) { later.few_at[atomicAdd(&sm.count, 1)] = e; });
        __syncthreads();
        for (int i = warp; i < all_some; i += warps) {
            const double x = exact_score<D>(p, tok, hk, name_of(later.few_at[i]));
            if (lane == 0) later.few[i] = x;
        }
        __syncthreads();
        // In the order of score and place, the first `rest` are in.
        for (int i = tid; i < all_some; i += threads) {
            const double x = later.few[i];
            const int e = later.few_at[i];
            int better = 0;
            for (int j = 0; j < all_some; ++j) better += later.few[j] > x || (later.few[j] == x && later.few_at[j] < e);
            later.few_in[i] = better < rest;
        }
        __syncthreads();
    } else {
        // Many that differ by less than the error (alike, most of them): the rest-th largest of their exact scores, eight bits at a time, then
        // those above it and, of its own value, the first.
        for (int e = begin + warp; e < end; e += warps) {
            if (!doubtful(score_of(e))) continue;
            const double x = exact_score<D>(p, tok, hk, name_of(e));
            if (lane == 0) exact[e] = x;
        }
        __syncthreads();
        ties = rest;
        for (int shift = 56; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += threads) later.bins[i] = 0;
            __syncthreads();
            each_of([&](int, float x, int) { return doubtful(x); }, [&](int e) {
                const unsigned long long y = ordered(exact[e]);
                if (shift == 56 || y >> (shift + 8) == value >> (shift + 8)) atomicAdd(&later.bins[y >> shift & 255], 1);
            });
            __syncthreads();
            if (tid == 0) {
                int bin = 255, left = ties;
                while (later.bins[bin] < left) left -= later.bins[bin--];
                sm.need = left;
                sm.exact = value | static_cast<unsigned long long>(bin) << shift;
            }
            __syncthreads();
            ties = sm.need;
            value = sm.exact;
            __syncthreads();
        }
        // Of this thread's pages: those of the value itself, of which the first `ties` of all are in.
        int equal = 0, all;
        each_of([&](int, float x, int) { return doubtful(x); }, [&](int e) { equal += ordered(exact[e]) == value; });
        ties_before = sum_before(equal, sm.sums[0], all);
    }
    // Whether a doubtful page is in; asked in the order of a thread's pages.
    int equal = ties_before;
    auto among = [&](int e) {
        if (all_some <= kFew) {
            int i = 0;
            while (later.few_at[i] != e) ++i;
            return later.few_in[i] != 0;
        }
        const unsigned long long y = ordered(exact[e]);
        return y > value || (y == value && equal++ < ties);
    };
    int own = in, all;
    each_of([&](int, float x, int) { return doubtful(x); }, [&](int e) { own += among(e); });
    at = sum_before(own, sm.sums[1], all);
    equal = ties_before;
    each_of([&](int, float x, int) { return x >= below; }, [&](int e) {
        if (surely(score_of(e)) || among(e)) to[at++] = name_of(e);
    });
}

// ---- host --------------------------------------------------------------------------------------

constexpr int kMaxEntries = 1 << 18;               // pages of a sequence
constexpr int64_t kWorkspace = 256ll << 20;        // bytes of scores at a time

struct SelectPlan {
    int64_t tokens, slice;   // of all, of a launch
    int blocks;
    bool near;               // scores and names in shared memory
    int64_t exact_at, bytes;
};
// Pages whose scores, names and exact scores have room in shared memory.
template <int D>
constexpr int kNearPages = D == 128 ? 8192 : 4096;

const char* select_refusal(const ktt_b200_select_args* a) {
    if (a->d != 64 && a->d != 128) return "head dim 64 or 128";
    if (a->page_size < 16 || a->page_size % 16) return "the page size must be a multiple of 16";
    if (a->table_width < 1 || a->pages < 1 || a->kv_heads < 1) return "sizes must be positive";
    if (a->kv_heads > 4096) return "at most 4096 K / V heads";
    if (a->heads < 1 || a->heads % a->kv_heads) return "K / V heads must divide Q heads";
    if (a->heads > 65535 || a->batch > 65535) return "batch and heads must not exceed 65535";
    if (a->table_width > kMaxEntries) return "at most 262144 pages of a sequence";
    if (static_cast<int64_t>(a->table_width) * a->page_size > (1 << 30)) return "at most 2^30 keys per sequence";
    if (a->first < 0 || a->last < 1 || a->top > kMaxEntries || static_cast<int64_t>(a->first) + a->last > a->top) return "0 or more first pages, 1 or more last ones, no more than `top` together";
    for (int i = 0; i < 3; ++i) {
        if (a->q_strides[i] % 8) return "q strides must be multiples of 8";
    }
    if (reinterpret_cast<uintptr_t>(a->q) & 15) return "q must be 16-byte aligned";
    return nullptr;
}

SelectPlan plan_of(const ktt_b200_select_args* a) {
    SelectPlan s = {};
    s.tokens = a->cu_seqlens_q ? a->total_q : static_cast<int64_t>(a->batch) * a->sq;
    s.blocks = (a->table_width + 15) / 16;
    s.near = s.blocks * 16 <= (a->d == 64 ? kNearPages<64> : kNearPages<128>);
    const int64_t one = static_cast<int64_t>(a->kv_heads) * s.blocks * 16 * 12;   // scores, and exact ones
    int64_t most = s.near ? s.tokens : kWorkspace / one;
    const int64_t ctas = (1ll << 30) / (static_cast<int64_t>(a->kv_heads) * kMaxRanks);   // of a launch
    if (most > ctas) most = ctas;
    s.slice = most < 1 ? 1 : (most < s.tokens ? most : s.tokens);
    const int64_t n = s.slice * a->kv_heads * s.blocks * 16;
    s.exact_at = (n * 4 + 255) / 256 * 256;
    s.bytes = s.near ? 0 : s.exact_at + n * 8;
    return s;
}

template <int D, int kItems, bool kNear>
int launch_select(const SelectParams& p, int64_t pairs, cudaStream_t stream) {
    auto kernel = select_kernel<D, kItems, kNear>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(pairs * p.ranks));
    cfg.blockDim = dim3(32 * kWarps);
    static_assert(!kNear || sizeof(SelectLater) + kNearPages<D> * 8 <= Ring<D>::kBytes, "exact scores lie where the rings were");
    cfg.dynamicSmemBytes = Ring<D>::kBytes + (kNear ? static_cast<size_t>(p.blocks) * 128 : 0);
    cfg.stream = stream;
    if (int rc = ensure_smem(kernel, Ring<D>::kBytes + (kNear ? kNearPages<D> * 8 : 0), "cudaFuncSetAttribute(select)")) return rc;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(p.ranks);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return check_cuda(cudaLaunchKernelEx(&cfg, kernel, p), "paged_select launch");
}

template <int D>
int run_select(SelectParams& p, const SelectPlan& plan, int width, cudaStream_t stream) {
    for (int64_t t0 = 0; t0 < plan.tokens; t0 += plan.slice) {
        const int64_t n = plan.tokens - t0 < plan.slice ? plan.tokens - t0 : plan.slice, pairs = n * p.kv_heads;
        p.token0 = t0;
        // Two CTAs to an SM: as many to a pair as there is room for and blocks for all their warps. Measured with half, twice and four times the
        // CTAs, us: 64 x up to 16,384 keys, 16 heads over 2, D 128, pages of 16: 21.7, 16.1 as it is, 18.8, 25.7; 24 tokens over up to 8,192, 14 over 2, D 64,
        // pages of 16: 10.0, 9.7, 9.5, 9.5.
        p.ranks = 1;
        while (p.ranks < kMaxRanks && pairs * p.ranks * 2 <= 2 * 148 && p.ranks * kWarps < plan.blocks) p.ranks *= 2;
        p.by_ranks = Divisor(p.ranks);
        // As few scores to a thread as the table's width asks for. us for one kind and the next, 16 heads over 2 or the like: 512 pages 6.0 (4 scores) and
        // 6.4 (8); 1,024 9.6 and 12.0 (8 and 32); 2,048 10.2 and 11.6 (16 and 32); 3,184 15.4 and 18.5 (32 and 64); 8,192 21.5, read each time
        // 31.2, in the workspace 57.
        int rc;
        if (!plan.near) rc = launch_select<D, 0, false>(p, pairs, stream);
        else if (width <= 4 * 32 * kWarps) rc = launch_select<D, 4, true>(p, pairs, stream);
        else if (width <= 8 * 32 * kWarps) rc = launch_select<D, 8, true>(p, pairs, stream);
        else if (width <= 16 * 32 * kWarps) rc = launch_select<D, 16, true>(p, pairs, stream);
        else if (D == 64 || width <= 32 * 32 * kWarps) rc = launch_select<D, 32, true>(p, pairs, stream);
        else rc = launch_select<D, D == 64 ? 32 : 64, true>(p, pairs, stream);
        if (rc) return rc;
    }
    return 0;
}

}  // namespace

int keep_bounds(const Pages& c, int bits, int d, int kv_heads, const Bounds& bounds, int batch, int64_t rows, const int32_t* cu, const int32_t* granted, bool launch, cudaStream_t stream) {
    if (rows == 0) return 0;
    BoundsParams p = {};
    p.c = c;
    p.bounds = bounds;
    p.batch = batch;
    p.kv_heads = kv_heads;
    p.rows = rows;
    p.cu = cu;
    p.granted = granted;
    if (const char* why = too_many(p)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_append: %s", why);
    return launch ? launch_bounds(p, bits, d, stream) : 0;
}

}  // namespace ktt

using namespace ktt;

namespace {

// The checks of a call for bounds, and its parameters.
int fill(BoundsParams& p, const ktt_b200_bounds_args* a, const int32_t* kept) {
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_bounds: null arguments");
    if (const char* why = pages_of(p.c, a->cache, a->d)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_bounds: %s", why);
    if (a->batch < 1) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_bounds: sizes must be positive");
    if (a->batch > 65535) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_bounds: at most 65535 sequences");
    if (!a->cache.k || !a->cache.block_table || !a->cache.lengths || !a->bounds) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_bounds: null pointer");
    if (const char* why = bounds_of(p.bounds, a->bounds, a->bounds_strides, p.c, a->cache.kv_heads, a->d)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_bounds: %s", why);
    p.batch = a->batch;
    p.kv_heads = a->cache.kv_heads;
    p.since = a->since;
    p.kept = kept;
    if (const char* why = too_many(p)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_bounds: %s", why);
    return 0;
}

}  // namespace

namespace ktt {

int cut_bounds(const ktt_b200_bounds_args* a, const int32_t* kept, bool launch, cudaStream_t stream) {
    BoundsParams p = {};
    if (int rc = fill(p, a, kept)) return rc;
    return launch ? launch_bounds(p, a->cache.bits, a->d, stream) : 0;
}

}  // namespace ktt

extern "C" int ktt_b200_paged_bounds(const ktt_b200_bounds_args* a, void* stream) {
    BoundsParams p = {};
    if (int rc = fill(p, a, nullptr)) return rc;
    return launch_bounds(p, a->cache.bits, a->d, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t ktt_b200_paged_select_workspace(const ktt_b200_select_args* a) {
    if (!a || a->batch < 1 || a->sq < 0 || a->total_q < 0) {
        fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_select: sizes must be positive");
        return -1;
    }
    if (const char* why = select_refusal(a)) {
        fail(KTT_B200_ERR_UNSUPPORTED, "paged_select: %s", why);
        return -1;
    }
    const SelectPlan s = plan_of(a);
    return s.tokens == 0 ? 0 : s.bytes;
}

extern "C" int ktt_b200_paged_select(const ktt_b200_select_args* a, void* stream) {
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_select: null arguments");
    if (a->batch < 1 || a->sq < 0 || a->total_q < 0) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_select: sizes must be positive");
    if (const char* why = select_refusal(a)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_select: %s", why);
    const SelectPlan s = plan_of(a);
    if (s.tokens == 0) return 0;
    if (s.tokens >= (1ll << 31)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_select: fewer than 2^31 tokens");
    if (!a->q || !a->bounds || !a->block_table || !a->lengths || !a->chosen || !a->keys) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_select: null pointer");
    if (s.bytes && (!a->workspace || a->workspace_bytes < s.bytes)) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_select: workspace holds %lld bytes, %lld needed", static_cast<long long>(a->workspace_bytes), static_cast<long long>(s.bytes));
    }
    if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_select: the workspace must be 16-byte aligned");
    SelectParams p = {};
    if (const char* why = bounds_of(p.bounds, const_cast<void*>(a->bounds), a->bounds_strides)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_select: %s", why);
    p.by_page = Divisor(a->page_size);
    p.by_sq = Divisor(a->sq < 1 ? 1 : a->sq);
    p.by_heads = Divisor(a->kv_heads);
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    for (int i = 0; i < 3; ++i) p.qs[i] = a->q_strides[i];
    p.cu = a->cu_seqlens_q;
    p.total_q = a->total_q;
    p.tokens = s.tokens;
    p.batch = a->batch;
    p.sq = a->sq;
    p.kv_heads = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.lengths = a->lengths;
    p.pages = a->pages;
    p.page_size = a->page_size;
    p.cap = a->table_width * a->page_size;
    p.top = a->top;
    p.first = a->first;
    p.last = a->last;
    p.blocks = s.blocks;
    p.width = a->table_width;
    unsigned char* base = static_cast<unsigned char*>(a->workspace);
    if (!s.near) {
        p.scores = reinterpret_cast<float*>(base);
        p.exact = reinterpret_cast<double*>(base + s.exact_at);
    }
    p.chosen = a->chosen;
    p.keys = a->keys;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->d == 64 ? run_select<64>(p, s, a->table_width, st) : run_select<128>(p, s, a->table_width, st);
}
