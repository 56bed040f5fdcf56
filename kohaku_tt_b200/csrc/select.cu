// Bounds of a paged cache's keys, and the pages that a query selects by them.
//
// A page's score for query q is the largest logit that a key between its bounds could have,
//   s = sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo,   q+ = max(q, 0), q- = min(q, 0),
// so the scores of all pages are two matrix products with the queries of a K / V head's group as columns. Bound: the reading of the
// bounds, 4 D bytes a page and head (1 / P of the cache in bf16, for pages of P keys).
//
// What is selected is decided by the exact scores, so that it does not depend on an order of summation: the products' sums are fp32, off by
// at most e = 2^-17 max_h sum_d |q_hd| max |bound| (products of bf16 values are exact in fp32; the 2 D / 16 instructions that add up a
// score round, or cut off, by some 2^-23 of the magnitudes each, together 2^-19; measured 2^-21 at most). The value t of the last page selected
// lies within e of the last by fp32. So pages more than 2 e above or below are in or out, and those between, a few, get their scores in 64 bits.
#include <algorithm>

#include "four_bits.cuh"

namespace ktt {

const char* bounds_of(Bounds& b, void* at, const int64_t (&strides)[3]) {
    b.at = static_cast<__nv_bfloat16*>(at);
    for (int i = 0; i < 3; ++i) {
        b.stride[i] = strides[i];
        if (strides[i] % 8) return "strides of bounds must be multiples of 16 bytes";
    }
    return reinterpret_cast<uintptr_t>(at) & 15 ? "bounds must be 16-byte aligned" : nullptr;
}

namespace {

// ---- bounds ------------------------------------------------------------------------------------

struct BoundsParams {
    Pages c;
    Bounds bounds;
    int batch, kv_heads;
    const int32_t* since;   // without `rows`: the keys that pages have bounds of (null: none)
    int64_t rows;           // > 0: keys appended behind the lengths: of each sequence, or packed
    const int32_t* cu;
};

constexpr int kLotOfTokens = 16;   // packed rows that a warp looks for pages in

// A warp has a page and head: a lane eight channels of every second (D 128) or fourth row, eight rows requested before the first is used.
// Packed rows: a warp looks at 16 of them and has the pages that begin among them, or in which a sequence's rows begin.
template <int D, int kBits, bool kPacked>
__global__ void __launch_bounds__(256) bounds_kernel(const __grid_constant__ BoundsParams p) {
    constexpr int kChunks = D / 8, kStep = 32 / kChunks, kAhead = 8;
    const int lane = threadIdx.x & 31, chunk = lane % kChunks, page_size = p.c.page_size;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t lot = unit / p.kv_heads;
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
        for (int r0 = begin + lane / kChunks; r0 < end; r0 += kAhead * kStep) {
            if constexpr (kBits == 16) {
                Eight<__nv_bfloat16> x[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int r = r0 + i * kStep < end ? r0 + i * kStep : r0;   // (a row twice changes nothing)
                    x[i].load(reinterpret_cast<const __nv_bfloat16*>(from + r * p.c.ks[2]) + chunk * 8);
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) e.with(x[i], x[i]);
            } else {
                uint2 x[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int r = r0 + i * kStep < end ? r0 + i * kStep : r0;
                    const uint32_t* block = reinterpret_cast<const uint32_t*>(from + static_cast<int64_t>(r >> 4) * (9 * D));
                    x[i] = make_uint2(block[key_word<D>(r & 15, chunk)], block[step_word<D>(r & 15, chunk / 8)]);
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const Eight<__nv_bfloat16> y = of_four_bits(x[i].x, x[i].y);
                    e.with(y, y);
                }
            }
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
        if (lane < kLotOfTokens && n < p.rows) {
            b = sequence_of(p.cu, p.batch, n);
            if (b >= 0 && n >= p.cu[b]) {   // (offsets that decrease)
                const int64_t in = n - p.cu[b], at = cached_keys(p.c, b) + in, all = at + (p.cu[b + 1] - n);
                end = static_cast<int>(all < p.c.cap ? all : p.c.cap);
                leads = at < end && (in == 0 || at % page_size == 0);
                place = leads ? static_cast<int>(at) : 0;
            }
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
            end = static_cast<int>(len + p.rows < p.c.cap ? len + p.rows : p.c.cap);
        } else if (p.since) {
            begin = min(max(p.since[b], 0), len);
        }
        const int64_t entry = begin / page_size + lot, first = entry * page_size;
        if (first >= end || begin >= end) return;
        widen(b, static_cast<int>(entry), max(begin - static_cast<int>(first), 0), min(end - static_cast<int>(first), page_size));
    }
}

template <int D, int kBits>
int launch_bounds(const BoundsParams& p, cudaStream_t stream) {
    const int64_t lots = p.cu ? (p.rows + kLotOfTokens - 1) / kLotOfTokens
                              : (p.rows > 0 ? (p.rows + p.c.page_size - 2) / p.c.page_size + 1 : (static_cast<int64_t>(p.c.cap) + p.c.page_size - 1) / p.c.page_size);
    const dim3 grid(static_cast<unsigned>((lots * p.kv_heads + 7) / 8), static_cast<unsigned>(p.cu ? 1 : p.batch));
    if (p.cu) return launch_dependent(bounds_kernel<D, kBits, true>, p, grid, dim3(256), stream, "paged_bounds launch");
    return launch_dependent(bounds_kernel<D, kBits, false>, p, grid, dim3(256), stream, "paged_bounds launch");
}
int launch_bounds(const BoundsParams& p, int bits, int d, cudaStream_t stream) {
    if (bits == 16) return d == 64 ? launch_bounds<64, 16>(p, stream) : launch_bounds<128, 16>(p, stream);
    return d == 64 ? launch_bounds<64, 4>(p, stream) : launch_bounds<128, 4>(p, stream);
}

// ---- scores ------------------------------------------------------------------------------------

struct SelectParams {
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
    int blocks;               // of 16 pages, that the table has
    int lots, each;           // CTAs of a pair, and blocks of a warp of them
    float* scores;            // [pairs][blocks][16]
    float* most;              // [pairs][blocks] the largest magnitude among a block's bounds
    double* exact;            // [pairs][blocks][16]
    int32_t* chosen;
    int32_t* keys;
};

// A query token: its row of q, its sequence (-1: none), and the keys it sees.
struct Token {
    const __nv_bfloat16* q;
    int b, seen;
};
__device__ __forceinline__ Token token_of(const SelectParams& p, int64_t t) {
    Token x;
    int64_t row = t, place;
    int n;
    if (p.cu) {
        x.b = sequence_of(p.cu, p.batch, t);
        x.q = p.q + t * p.qs[2];
        if (x.b < 0) {
            x.seen = 0;
            return x;
        }
        place = t - p.cu[x.b];
        n = p.cu[x.b + 1] - p.cu[x.b];
    } else {
        x.b = static_cast<int>(t / p.sq);
        place = row = t - static_cast<int64_t>(x.b) * p.sq;
        n = p.sq;
        x.q = p.q + x.b * p.qs[0] + row * p.qs[2];
    }
    const int len = min(max(p.lengths[x.b], 0), p.cap);
    const int64_t seen = len - n + place + 1;
    x.seen = static_cast<int>(seen < 0 || place < 0 ? 0 : (seen < len ? seen : len));
    return x;
}

__device__ __forceinline__ uint32_t max_magnitude(uint32_t a, uint32_t x) {
    const uint32_t y = x & 0x7fff7fffu;
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Both bounds of 16 pages as a warp's lanes load them: lane (g, t) has pages g and g + 8, channels 32 j + 8 t .., in pieces of 16 bytes.
template <int D>
struct Sixteen {
    static constexpr int J = D / 32;
    uint4 lo[J][2], hi[J][2];
};

// A warp takes up to kEach blocks of 16 pages of a (token, K / V head), one on its way while another is multiplied. Its lanes load the bounds as
// they lie, which are the operands of m16n8k16 with the channels in that order; q+ and q- of 8 heads are its columns. Nothing goes
// through shared memory: no two warps read the same bounds. The products of a block are four sums, for the latency of one.
constexpr int kEach = 4;
template <int D>
__global__ void __launch_bounds__(128, 2) score_kernel(const __grid_constant__ SelectParams p) {
    constexpr int J = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t pair = blockIdx.x / p.lots;
    const int64_t local = pair / p.kv_heads;
    const int hk = static_cast<int>(pair - local * p.kv_heads);
    const Token tok = token_of(p, p.token0 + local);
    const int count = (tok.seen + p.page_size - 1) / p.page_size;
    if (count <= p.top) return;   // (all of them)
    const int block0 = ((static_cast<int>(blockIdx.x) - static_cast<int>(pair) * p.lots) * 4 + warp) * p.each;
    const int blocks = min(p.each, (count + 15) / 16 - block0);
    if (blocks <= 0) return;
    // The names of all its pages, two to a lane.
    int names[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int e = block0 * 16 + 32 * i + lane;
        names[i] = 32 * i < blocks * 16 && e < count ? p.table[tok.b * p.table_stride + e] : -1;
    }
    auto load = [&](Sixteen<D>& x, int block) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int from = (block & 1) * 16 + g + 8 * i;
            const int n0 = __shfl_sync(0xffffffffu, names[0], from), n1 = __shfl_sync(0xffffffffu, names[1], from), name = block & 2 ? n1 : n0;
            const bool there = name >= 0 && name < p.pages;
            const __nv_bfloat16* at = p.bounds.edge(there ? name : 0, hk, 0) + 8 * t;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                x.lo[j][i] = x.hi[j][i] = make_uint4(0u, 0u, 0u, 0u);
                if (there) {
                    x.lo[j][i] = *reinterpret_cast<const uint4*>(at + 32 * j);
                    x.hi[j][i] = *reinterpret_cast<const uint4*>(at + p.bounds.stride[2] + 32 * j);
                }
            }
        }
    };
    for (int h0 = 0; h0 < p.group; h0 += 8) {   // (more than 8 heads: the bounds come from the cache again)
        Sixteen<D> x[2];
        load(x[0], 0);
        uint32_t up[J][4], down[J][4];
        {
            const bool there = h0 + g < p.group;
            const __nv_bfloat16* from = tok.q + static_cast<int64_t>(hk * p.group + (there ? h0 + g : 0)) * p.qs[1] + 8 * t;
            const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const uint4 y4 = *reinterpret_cast<const uint4*>(from + 32 * j);
                const uint32_t w[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __nv_bfloat162 y = *reinterpret_cast<const __nv_bfloat162*>(&w[i]), u = __hmax2_nan(y, zero), v = __hmin2_nan(y, zero);
                    up[j][i] = there ? *reinterpret_cast<const uint32_t*>(&u) : 0u;
                    down[j][i] = there ? *reinterpret_cast<const uint32_t*>(&v) : 0u;
                }
            }
        }
        auto score = [&](const Sixteen<D>& x, int block) {
            float acc[4][4];
            uint32_t most[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
                most[i] = 0u;
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                auto product = [&](const uint4& x, const uint4& y, const uint32_t (&b)[4], int sum) {
                    const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
                    mma_bf16(acc[sum], a0, b[0], b[1]);
                    mma_bf16(acc[sum + 1], a1, b[2], b[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) most[i] = max_magnitude(max_magnitude(most[i], a0[i]), a1[i]);
                };
                product(x.hi[j][0], x.hi[j][1], up[j], 0);
                product(x.lo[j][0], x.lo[j][1], down[j], 2);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[0][i] = (acc[0][i] + acc[1][i]) + (acc[2][i] + acc[3][i]);
            // The largest of the columns that are heads.
            const bool c0 = h0 + 2 * t < p.group, c1 = h0 + 2 * t + 1 < p.group;
            float s[2] = {fmaxf(c0 ? acc[0][0] : -INFINITY, c1 ? acc[0][1] : -INFINITY), fmaxf(c0 ? acc[0][2] : -INFINITY, c1 ? acc[0][3] : -INFINITY)};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[i] = fmaxf(s[i], __shfl_xor_sync(0xffffffffu, s[i], 1));
                s[i] = fmaxf(s[i], __shfl_xor_sync(0xffffffffu, s[i], 2));
            }
            float* to = p.scores + (pair * p.blocks + block0 + block) * 16;
            if (t == 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (h0 > 0) s[i] = fmaxf(s[i], to[g + 8 * i]);
                    to[g + 8 * i] = s[i];
                }
            }
            if (h0 == 0) {
                uint32_t m = max_magnitude(max_magnitude(most[0], most[1]), max_magnitude(most[2], most[3]));
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) m = max_magnitude(m, __shfl_xor_sync(0xffffffffu, m, off));
                const __nv_bfloat162 m2 = *reinterpret_cast<const __nv_bfloat162*>(&m);
                if (lane == 0) p.most[pair * p.blocks + block0 + block] = __bfloat162float(__hmax_nan(__low2bfloat16(m2), __high2bfloat16(m2)));
            }
        };
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i >= blocks) break;
            if (i + 1 < blocks) load(x[(i + 1) & 1], i + 1);
            score(x[i & 1], i);
        }
    }
}

// ---- the selection -----------------------------------------------------------------------------

constexpr int kBins = 512;
constexpr int kFew = 256;        // pages between in and out that are ranked one against the others

struct SelectShared {
    int bins[kBins + kBins / 16];   // (a place more for every 16: warp 0 reads 16 to a lane)
    float warps[4][32];
    int sums[32];
    float ranked[32];
    int few_at[kFew];
    double few[kFew];
    int bin, in_bin, need, count, found, all_in, lo_bits, hi_bits;
    unsigned long long exact;
};
__device__ __forceinline__ int bin_at(int bin) { return bin + (bin >> 4); }

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
__device__ __forceinline__ float larger(float a, float b) { return a != a || a > b ? a : b; }   // (a NaN stays)

// Exclusive sum of x over the CTA, and that of all. Two barriers.
__device__ __forceinline__ int sum_before(int x, int* warps, int& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    int sum = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += y;
    }
    if (lane == 31) warps[warp] = sum;
    __syncthreads();
    const int other = lane < n ? warps[lane] : 0;
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? other : 0);
    all = __reduce_add_sync(0xffffffffu, other);
    __syncthreads();
    return before + sum - x;
}

// The exact score of a page: 64-bit sums of products that are exact themselves. By one warp.
template <int D>
__device__ __forceinline__ double exact_score(const SelectParams& p, const Token& tok, int hk, int e) {
    const int lane = threadIdx.x & 31;
    constexpr int kMine = D / 32;
    const int64_t page = p.table[tok.b * p.table_stride + e];
    if (page < 0 || page >= p.pages) return 0.0;
    double lo[kMine], hi[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        lo[i] = __bfloat162float(p.bounds.edge(page, hk, 0)[lane + 32 * i]);
        hi[i] = __bfloat162float(p.bounds.edge(page, hk, 1)[lane + 32 * i]);
    }
    double best = -INFINITY;
#pragma unroll 4
    for (int h = 0; h < p.group; ++h) {
        const __nv_bfloat16* q = tok.q + static_cast<int64_t>(hk * p.group + h) * p.qs[1];
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const double x = __bfloat162float(q[lane + 32 * i]), a = x * lo[i], b = x * hi[i];
            sum += a != a || a > b ? a : b;   // (a NaN of either stays)
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (sum != sum) sum = INFINITY;
        best = sum > best ? sum : best;
    }
    return best + 0.0;   // (no -0)
}

// One CTA for a (token, K / V head); a thread has kItems neighbouring pages, their scores and names in registers (0: as many as there are, which
// it reads again each time). The k-th largest of the scores is found by bins of equal width between the least and the largest, then by
// rank among the few of its bin. Bound: latency, some ten barriers and two trips to memory.
template <int D, int kItems>
__global__ void __launch_bounds__(1024) select_kernel(const __grid_constant__ SelectParams p) {
    __shared__ SelectShared sm;
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads / 32;
    for (int i = tid; i < kBins + kBins / 16; i += threads) sm.bins[i] = 0;
    if (tid == 0) sm.count = sm.found = sm.all_in = 0;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t pair = blockIdx.x, local = pair / p.kv_heads, t = p.token0 + local;
    const int hk = static_cast<int>(pair - local * p.kv_heads);
    const Token tok = token_of(p, t);
    const int count = (tok.seen + p.page_size - 1) / p.page_size, top = p.top;
    int32_t* to = p.chosen + (t * p.kv_heads + hk) * top;
    const int32_t* row = p.table + max(tok.b, 0) * p.table_stride;
    if (tid == 0) {
        const int many = min(count, top);
        p.keys[t * p.kv_heads + hk] = many > 0 ? (many - 1) * p.page_size + (tok.seen - 1) % p.page_size + 1 : 0;
    }
    if (count <= top) {
        for (int i = tid; i < top; i += threads) to[i] = i < count ? row[i] : -1;
        return;
    }
    const float* given = p.scores + pair * p.blocks * 16;
    const int begin = p.first, end = count - p.last, k = top - p.first - p.last;   // the k largest of [begin, end), which are more
    const int mine = kItems ? kItems : ((count + threads - 1) / threads + 3) & ~3, first = tid * mine;
    // All its pages: f(page, score, place among its own).
    float held[kItems ? kItems : 1];
    if constexpr (kItems > 0) {
#pragma unroll
        for (int i = 0; i < kItems; i += 4) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (first + i < count) x = *reinterpret_cast<const float4*>(given + first + i);   // (whole blocks of 16 are written)
            held[i] = x.x; held[i + 1] = x.y; held[i + 2] = x.z; held[i + 3] = x.w;
        }
    }
    auto each = [&](auto f) {
        if constexpr (kItems > 0) {
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                if (first + i >= begin && first + i < end) f(first + i, held[i]);
            }
        } else {
            for (int e = max(first, begin); e < min(first + mine, end); ++e) f(e, given[e]);
        }
    };
    // The least and the largest, and what the scores may be off by.
    float lo = INFINITY, hi = -INFINITY, most = 0.f, norm = 0.f;
    for (int h = warp; h < p.group; h += warps) {
        const __nv_bfloat16* q = tok.q + static_cast<int64_t>(hk * p.group + h) * p.qs[1] + lane * (D / 32);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) {
            const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(q + i));
            sum += fabsf(y.x) + fabsf(y.y);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        norm = larger(sum, norm);
    }
    for (int i = tid; i < (count + 15) / 16; i += threads) most = larger(p.most[pair * p.blocks + i], most);
    each([&](int, float x) {
        lo = fminf(lo, x);
        hi = fmaxf(hi, x);
    });
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        most = larger(most, __shfl_xor_sync(0xffffffffu, most, off));
    }
    if (lane == 0) {
        sm.warps[0][warp] = lo;
        sm.warps[1][warp] = hi;
        sm.warps[2][warp] = most;
        sm.warps[3][warp] = norm;
    }
    __syncthreads();
    lo = lane < warps ? sm.warps[0][lane] : INFINITY;
    hi = lane < warps ? sm.warps[1][lane] : -INFINITY;
    most = lane < warps ? sm.warps[2][lane] : 0.f;
    norm = lane < warps ? sm.warps[3][lane] : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        most = larger(most, __shfl_xor_sync(0xffffffffu, most, off));
        norm = larger(norm, __shfl_xor_sync(0xffffffffu, norm, off));
    }
    const float mass = norm * most;
    // (What the products could lose below fp32's least normal number is in the last terms.)
    const float off = fmaf(mass, 0x1p-17f, fmaf(norm + most, 0x1p-110f, 0x1p-110f));
    const bool sure = mass < 0x1p120f;   // else, and where it is no number: all in 64 bits
    int need = k;
    for (int round = 0; round < 4 && sure && k > 0 && hi - lo > 4.f * off; ++round) {
        const float by = (kBins - 0.5f) / (hi - lo);
        if (!(by < 0x1p100f)) break;
        auto bin_of = [&](float x) { return static_cast<int>((x - lo) * by); };   // (falls nowhere as x rises)
        each([&](int, float x) {
            if (x >= lo && x <= hi) atomicAdd(&sm.bins[bin_at(bin_of(x))], 1);
        });
        __syncthreads();
        if (warp == 0) {
            // Lane l has the 16 bins from kBins - 16 l down: those above the one that has the need-th, and it.
            int own[16], sum = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += own[i] = sm.bins[bin_at(kBins - 1 - 16 * lane - i)];
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            int above = upto - sum;
            if (above < need && upto >= need) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (above < need && above + own[i] >= need) {
                        sm.bin = kBins - 1 - 16 * lane - i;
                        sm.in_bin = own[i];
                        sm.need = need - above;
                    }
                    above += own[i];
                }
            }
            if (lane == 0) {
                sm.lo_bits = 0x7fffffff;
                sm.hi_bits = static_cast<int>(0x80000000);
            }
        }
        __syncthreads();
        const int bin = sm.bin, many = sm.in_bin;
        need = sm.need;
        if (many <= 32) {
            each([&](int, float x) {
                if (x >= lo && x <= hi && bin_of(x) == bin) sm.ranked[atomicAdd(&sm.found, 1)] = x;
            });
            __syncthreads();
            // The need-th largest of them (equal ones in any order): every warp for itself.
            const float x = lane < many ? sm.ranked[lane] : -INFINITY;
            int better = 0;
            for (int i = 0; i < many; ++i) {
                const float y = __shfl_sync(0xffffffffu, x, i);
                better += y > x || (y == x && i < lane);
            }
            const uint32_t it = __ballot_sync(0xffffffffu, lane < many && better == need - 1);
            lo = hi = __shfl_sync(0xffffffffu, x, __ffs(it) - 1);
            break;
        }
        each([&](int, float x) {
            if (x >= lo && x <= hi && bin_of(x) == bin) {
                atomicMin(&sm.lo_bits, ordered(x));
                atomicMax(&sm.hi_bits, ordered(x));
            }
        });
        for (int i = tid; i < kBins + kBins / 16; i += threads) sm.bins[i] = 0;
        __syncthreads();
        lo = from_ordered(sm.lo_bits);
        hi = from_ordered(sm.hi_bits);
        __syncthreads();
    }
    // Pages above are in, pages below are out; those between are counted, and listed while they are few.
    const float above = sure ? hi + 2.f * off : INFINITY, below = sure ? lo - 2.f * off : -INFINITY;
    auto surely = [&](float x) { return sure && x > above; };
    auto doubtful = [&](float x) { return !surely(x) && !(x < below); };
    int in = 0, some = 0;
    if (k > 0) {
        each([&](int e, float x) {
            in += surely(x);
            if (doubtful(x)) {
                ++some;
                const int at = atomicAdd(&sm.count, 1);
                if (at < kFew) sm.few_at[at] = e;
            }
        });
    }
    const int warp_in = __reduce_add_sync(0xffffffffu, in);
    if (lane == 0 && warp_in > 0) atomicAdd(&sm.all_in, warp_in);
    __syncthreads();
    const int all_some = sm.count, rest = k - sm.all_in;   // so many of the doubtful ones are in
    const bool everything = all_some == rest;
    int some_before = 0;
    double* exact = p.exact + pair * p.blocks * 16;
    unsigned long long value = 0;
    int ties = 0;
    if (k > 0 && !everything) {
        if (all_some <= kFew) {
            for (int i = warp; i < all_some; i += warps) {
                const double x = exact_score<D>(p, tok, hk, sm.few_at[i]);
                if (lane == 0) sm.few[i] = x;
            }
            __syncthreads();
            // The rest-th in the order of score and place: pages at or before it are in.
            for (int i = tid; i < all_some; i += threads) {
                const double x = sm.few[i];
                const int e = sm.few_at[i];
                int better = 0;
                for (int j = 0; j < all_some; ++j) better += sm.few[j] > x || (sm.few[j] == x && sm.few_at[j] < e);
                exact[e] = better < rest ? 1.0 : 0.0;
            }
            __syncthreads();
        } else {
            // Many that differ by less than the error (alike, most of them): the rest-th largest of their exact scores, eight bits at a time, then
            // those above it and, of its own value, the first.
            for (int e = begin + warp; e < end; e += warps) {
                if (!doubtful(given[e])) continue;
                const double x = exact_score<D>(p, tok, hk, e);
                if (lane == 0) exact[e] = x;
            }
            __syncthreads();
            ties = rest;
            for (int shift = 56; shift >= 0; shift -= 8) {
                for (int i = tid; i < 256; i += threads) sm.bins[i] = 0;
                __syncthreads();
                each([&](int e, float x) {
                    if (!doubtful(x)) return;
                    const unsigned long long y = ordered(exact[e]);
                    if (shift == 56 || y >> (shift + 8) == value >> (shift + 8)) atomicAdd(&sm.bins[y >> shift & 255], 1);
                });
                __syncthreads();
                if (tid == 0) {
                    int bin = 255, left = ties;
                    while (sm.bins[bin] < left) left -= sm.bins[bin--];
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
            each([&](int e, float x) { equal += doubtful(x) && ordered(exact[e]) == value; });
            some_before = sum_before(equal, sm.sums, all);
        }
    }
    // Whether a doubtful page is in; asked in the order of a thread's pages.
    int equal = some_before;
    auto among = [&](int e) {
        if (everything) return true;
        if (all_some <= kFew) return exact[e] != 0.0;
        const unsigned long long y = ordered(exact[e]);
        return y > value || (y == value && equal++ < ties);
    };
    // The pages that are in, in their order: the first, those of [begin, end), the last.
    int own = in, all;
    if (some > 0) {
        each([&](int e, float x) {
            if (doubtful(x)) own += among(e);
        });
    }
    int at = p.first + sum_before(own, sm.sums, all);
    equal = some_before;
    if (own > 0) {
        each([&](int e, float x) {
            if (surely(x) || (doubtful(x) && among(e))) to[at++] = row[e];
        });
    }
    for (int i = tid; i < p.first; i += threads) to[i] = row[i];
    for (int i = tid; i < p.last; i += threads) to[top - p.last + i] = row[end + i];
}

// ---- host --------------------------------------------------------------------------------------

constexpr int kMaxEntries = 1 << 18;               // pages of a sequence
constexpr int64_t kWorkspace = 256ll << 20;        // bytes of scores at a time

struct SelectPlan {
    int64_t tokens, slice;   // of all, of a launch
    int blocks;
    int64_t most_at, exact_at, bytes;
};

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
    const int64_t one = static_cast<int64_t>(a->kv_heads) * s.blocks * (16 * 12 + 4);   // (scores, exact ones, magnitudes)
    int64_t most = kWorkspace / one;
    const int64_t pairs = (1ll << 30) / (static_cast<int64_t>(a->kv_heads) * s.blocks);   // CTAs of a launch
    if (most > pairs) most = pairs;
    s.slice = most < 1 ? 1 : (most < s.tokens ? most : s.tokens);
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t n = s.slice * a->kv_heads * s.blocks;
    s.exact_at = up(n * 64);
    s.most_at = s.exact_at + up(n * 128);
    s.bytes = s.most_at + up(n * 4);
    return s;
}

template <int D>
int run_select(SelectParams& p, const SelectPlan& plan, int width, cudaStream_t stream) {
    const int items = width <= 4096 ? 4 : (width <= 16384 ? 16 : 0);
    const int threads = items ? std::max(128, (width + 32 * items - 1) / (32 * items) * 32) : 1024;
    for (int64_t t0 = 0; t0 < plan.tokens; t0 += plan.slice) {
        const int64_t n = plan.tokens - t0 < plan.slice ? plan.tokens - t0 : plan.slice, pairs = n * p.kv_heads;
        p.token0 = t0;
        // Blocks of a warp: as few as there are warps for at a time (8 on an SM).
        const int64_t all = pairs * plan.blocks, warps = 148 * 8, each = (all + warps - 1) / warps;
        p.each = static_cast<int>(each > kEach ? kEach : each);
        p.lots = (plan.blocks + 4 * p.each - 1) / (4 * p.each);
        if (int rc = launch_dependent(score_kernel<D>, p, dim3(static_cast<unsigned>(pairs * p.lots)), dim3(128), stream, "paged_select launch")) return rc;
        auto kernel = items == 4 ? select_kernel<D, 4> : (items == 16 ? select_kernel<D, 16> : select_kernel<D, 0>);
        if (int rc = launch_dependent(kernel, p, dim3(static_cast<unsigned>(pairs)), dim3(static_cast<unsigned>(threads)), stream, "paged_select launch")) return rc;
    }
    return 0;
}

}  // namespace

int keep_bounds(const Pages& c, int bits, int d, int kv_heads, const Bounds& bounds, int batch, int64_t rows, const int32_t* cu, cudaStream_t stream) {
    if (rows == 0) return 0;
    BoundsParams p = {};
    p.c = c;
    p.bounds = bounds;
    p.batch = batch;
    p.kv_heads = kv_heads;
    p.rows = rows;
    p.cu = cu;
    return launch_bounds(p, bits, d, stream);
}

}  // namespace ktt

using namespace ktt;

extern "C" int ktt_b200_paged_bounds(const ktt_b200_bounds_args* a, void* stream) {
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_bounds: null arguments");
    BoundsParams p = {};
    if (const char* why = pages_of(p.c, a->cache, a->d)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_bounds: %s", why);
    if (a->batch < 1) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_bounds: sizes must be positive");
    if (a->batch > 65535) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_bounds: at most 65535 sequences");
    if (!a->cache.k || !a->cache.block_table || !a->cache.lengths || !a->bounds) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_bounds: null pointer");
    if (const char* why = bounds_of(p.bounds, a->bounds, a->bounds_strides)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_bounds: %s", why);
    p.batch = a->batch;
    p.kv_heads = a->cache.kv_heads;
    p.since = a->since;
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
    if (!a->workspace || a->workspace_bytes < s.bytes) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_select: workspace holds %lld bytes, %lld needed", static_cast<long long>(a->workspace_bytes), static_cast<long long>(s.bytes));
    }
    if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_select: the workspace must be 16-byte aligned");
    SelectParams p = {};
    if (const char* why = bounds_of(p.bounds, const_cast<void*>(a->bounds), a->bounds_strides)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_select: %s", why);
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
    unsigned char* base = static_cast<unsigned char*>(a->workspace);
    p.scores = reinterpret_cast<float*>(base);
    p.exact = reinterpret_cast<double*>(base + s.exact_at);
    p.most = reinterpret_cast<float*>(base + s.most_at);
    p.chosen = a->chosen;
    p.keys = a->keys;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->d == 64 ? run_select<64>(p, s, a->table_width, st) : run_select<128>(p, s, a->table_width, st);
}
