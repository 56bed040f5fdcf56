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
#include <cfloat>

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

// A warp takes `each` blocks of 16 pages of a (token, K / V head): its lanes load both bounds of pages g and g + 8 in pieces of 16 bytes
// as they lie (lane (g, t): channels 32 j + 8 t ..), which are the operands of m16n8k16 with the channels in that order; q+ and q- of 8 heads are
// its columns. Nothing goes through shared memory: no two warps read the same bounds.
template <int D>
__global__ void __launch_bounds__(128) score_kernel(const __grid_constant__ SelectParams p) {
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
    const int block1 = min(block0 + p.each, (count + 15) / 16);
    for (int h0 = 0; h0 < p.group; h0 += 8) {   // (more than 8 heads: the bounds come from the cache again)
        if (block0 >= block1) return;
        uint32_t up[J][4], down[J][4];
        {
            const bool there = h0 + g < p.group;
            const __nv_bfloat16* from = tok.q + static_cast<int64_t>(hk * p.group + (there ? h0 + g : 0)) * p.qs[1] + 8 * t;
            const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const uint4 x = *reinterpret_cast<const uint4*>(from + 32 * j);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __nv_bfloat162 y = *reinterpret_cast<const __nv_bfloat162*>(&w[i]), u = __hmax2_nan(y, zero), v = __hmin2_nan(y, zero);
                    up[j][i] = there ? *reinterpret_cast<const uint32_t*>(&u) : 0u;
                    down[j][i] = there ? *reinterpret_cast<const uint32_t*>(&v) : 0u;
                }
            }
        }
        for (int block = block0; block < block1; ++block) {
            const __nv_bfloat16* at[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int e = block * 16 + g + 8 * i;
                const int64_t page = e < count ? p.table[tok.b * p.table_stride + e] : -1;
                at[i] = page >= 0 && page < p.pages ? p.bounds.edge(page, hk, 0) + 8 * t : nullptr;
            }
            uint4 lo[J][2], hi[J][2];
#pragma unroll
            for (int j = 0; j < J; ++j) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    lo[j][i] = hi[j][i] = make_uint4(0u, 0u, 0u, 0u);
                    if (at[i]) {
                        lo[j][i] = *reinterpret_cast<const uint4*>(at[i] + 32 * j);
                        hi[j][i] = *reinterpret_cast<const uint4*>(at[i] + p.bounds.stride[2] + 32 * j);
                    }
                }
            }
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t most = 0u;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                auto product = [&](const uint4& x, const uint4& y, const uint32_t (&b)[4]) {
                    const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
                    mma_bf16(acc, a0, b[0], b[1]);
                    mma_bf16(acc, a1, b[2], b[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = max_magnitude(max_magnitude(most, a0[i]), a1[i]);
                };
                product(hi[j][0], hi[j][1], up[j]);
                product(lo[j][0], lo[j][1], down[j]);
            }
            // The largest of the columns that are heads.
            const bool c0 = h0 + 2 * t < p.group, c1 = h0 + 2 * t + 1 < p.group;
            float s[2] = {fmaxf(c0 ? acc[0] : -INFINITY, c1 ? acc[1] : -INFINITY), fmaxf(c0 ? acc[2] : -INFINITY, c1 ? acc[3] : -INFINITY)};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[i] = fmaxf(s[i], __shfl_xor_sync(0xffffffffu, s[i], 1));
                s[i] = fmaxf(s[i], __shfl_xor_sync(0xffffffffu, s[i], 2));
            }
            float* to = p.scores + (pair * p.blocks + block) * 16;
            if (t == 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (h0 > 0) s[i] = fmaxf(s[i], to[g + 8 * i]);
                    to[g + 8 * i] = s[i];
                }
            }
            if (h0 == 0) {
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) most = max_magnitude(most, __shfl_xor_sync(0xffffffffu, most, off));
                const __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&most);
                if (lane == 0) p.most[pair * p.blocks + block] = __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
            }
        }
    }
}

// ---- the selection -----------------------------------------------------------------------------

constexpr int kBins = 1024;
constexpr int kFew = 256;        // pages between in and out that are ranked one against the others

struct SelectShared {
    int bins[kBins];
    float fwarps[32];
    int iwarps[32];
    int few_at[kFew];
    double few[kFew];
    float lo, hi;                // fp32 scores that the last one selected lies between
    int lo_bits, hi_bits, need, above, in_bin, count;
    unsigned long long value;
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

template <typename T, typename Op>
__device__ __forceinline__ T over_block(T x, T* warps, Op op) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, off));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = x;
    __syncthreads();
    x = warps[0];
    for (int w = 1; w < blockDim.x / 32; ++w) x = op(x, warps[w]);
    return x;
}

// The exact score of a page: 64-bit sums of products that are exact themselves. By one warp.
template <int D>
__device__ __forceinline__ double exact_score(const SelectParams& p, const Token& tok, int hk, int e) {
    const int lane = threadIdx.x & 31;
    constexpr int kEach = D / 32;
    const int64_t page = p.table[tok.b * p.table_stride + e];
    if (page < 0 || page >= p.pages) return 0.0;
    double lo[kEach], hi[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        lo[i] = __bfloat162float(p.bounds.edge(page, hk, 0)[lane + 32 * i]);
        hi[i] = __bfloat162float(p.bounds.edge(page, hk, 1)[lane + 32 * i]);
    }
    double best = -INFINITY;
    for (int h = 0; h < p.group; ++h) {
        const __nv_bfloat16* q = tok.q + static_cast<int64_t>(hk * p.group + h) * p.qs[1];
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
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

// One CTA for a (token, K / V head). The fp32 scores lie in shared memory where they fit, else where they were written; `in` has a bit for each
// page that is selected.
template <int D>
__global__ void __launch_bounds__(1024) select_kernel(const __grid_constant__ SelectParams p, int in_shared) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ SelectShared sm;
    uint32_t* in = reinterpret_cast<uint32_t*>(dynamic);
    const int words = (p.blocks + 1) / 2;
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads / 32;
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
    float* held = reinterpret_cast<float*>(in + words);
    const float* s = in_shared ? held : given;
    const int begin = p.first, end = count - p.last, k = top - p.first - p.last;   // of [begin, end), more than k
    for (int w = tid; w < words; w += threads) in[w] = 0u;
    for (int i = tid; i < kBins; i += threads) sm.bins[i] = 0;
    if (tid == 0) {
        sm.need = k;
        sm.count = 0;
    }
    // The error of the fp32 scores.
    float norm = 0.f, most = 0.f, lo = INFINITY, hi = -INFINITY;
    constexpr int kHeadThreads = D / 8;
    for (int h0 = 0; h0 < p.group; h0 += threads / kHeadThreads) {
        const int h = h0 + tid / kHeadThreads;
        float sum = 0.f;
        if (h < p.group) {
            Eight<__nv_bfloat16> x;
            x.load(tok.q + static_cast<int64_t>(hk * p.group + h) * p.qs[1] + (tid % kHeadThreads) * 8);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += fabsf(__bfloat162float(x.get(e)));
        }
#pragma unroll
        for (int off = 1; off < kHeadThreads; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        norm = sum > norm || sum != sum ? sum : norm;
    }
    auto larger = [](float a, float b) { return a != a || a > b ? a : b; };   // (a NaN stays)
    for (int i = tid; i < (count + 15) / 16; i += threads) most = larger(p.most[pair * p.blocks + i], most);
    for (int e = begin + tid; e < end; e += threads) {
        const float x = given[e];
        if (in_shared) held[e] = x;
        lo = fminf(lo, x);
        hi = fmaxf(hi, x);
    }
    norm = over_block(norm, sm.fwarps, larger);
    most = over_block(most, sm.fwarps, larger);
    lo = over_block(lo, sm.fwarps, [](float a, float b) { return fminf(a, b); });
    hi = over_block(hi, sm.fwarps, [](float a, float b) { return fmaxf(a, b); });
    const float mass = norm * most;
    // (What the products could lose below fp32's least normal number is in the last terms.)
    const float off = fmaf(mass, 0x1p-17f, fmaf(norm + most, 0x1p-110f, 0x1p-110f));
    const bool sure = mass < 0x1p120f;   // else, and where it is no number: all in 64 bits
    // The value of the k-th largest is between lo and hi: bins of equal width, of which the one that has it is cut again while it holds many.
    for (int round = 0; round < 4 && sure && k > 0 && hi - lo > 4.f * off; ++round) {
        const float by = (kBins - 0.5f) / (hi - lo);
        if (!(by < 0x1p100f)) break;
        for (int e = begin + tid; e < end; e += threads) {
            const float x = s[e];
            if (x >= lo && x <= hi) atomicAdd(&sm.bins[static_cast<int>((x - lo) * by)], 1);
        }
        __syncthreads();
        if (warp == 0) {
            // From the top: lane l has bins [kBins - 32 (l + 1), kBins - 32 l), summed up.
            int sum = 0;
            for (int i = 0; i < kBins / 32; ++i) sum += sm.bins[kBins - 1 - (lane * (kBins / 32) + i)];
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const int need = sm.need;
            __syncwarp();
            if (upto - sum < need && upto >= need) {
                int above = upto - sum, bin = kBins - 1 - lane * (kBins / 32);
                while (above + sm.bins[bin] < need) above += sm.bins[bin--];
                sm.above = bin;
                sm.in_bin = sm.bins[bin];
                sm.need = need - above;
                sm.lo_bits = 0x7fffffff;
                sm.hi_bits = static_cast<int>(0x80000000);
            }
        }
        __syncthreads();
        const int bin = sm.above;
        for (int e = begin + tid; e < end; e += threads) {
            const float x = s[e];
            if (x >= lo && x <= hi && static_cast<int>((x - lo) * by) == bin) {
                atomicMin(&sm.lo_bits, ordered(x));
                atomicMax(&sm.hi_bits, ordered(x));
            }
        }
        for (int i = tid; i < kBins; i += threads) sm.bins[i] = 0;
        __syncthreads();
        lo = from_ordered(sm.lo_bits);
        hi = from_ordered(sm.hi_bits);
        const int many = sm.in_bin;
        __syncthreads();
        if (many <= 32) break;
    }
    // Pages above are in, pages below are out.
    const float above = sure ? hi + 2.f * off : INFINITY, below = sure ? lo - 2.f * off : -INFINITY;
    int mine = 0, doubtful = 0;
    if (k > 0) {
        for (int e0 = begin & ~31; e0 < end; e0 += threads) {
            const int e = e0 + tid;
            bool take = e < p.first || (e >= end && e < count);
            if (e >= begin && e < end) {
                const float x = s[e];
                take = sure && x > above;
                mine += take;
                if (!take && !(x < below)) {
                    const int at = atomicAdd(&sm.count, 1);
                    if (at < kFew) sm.few_at[at] = e;
                    ++doubtful;
                }
            }
            const uint32_t bits = __ballot_sync(0xffffffffu, take);
            if (lane == 0 && e < count) in[e >> 5] = bits;
        }
    }
    mine = over_block(mine, sm.iwarps, [](int a, int b) { return a + b; });
    for (int e = tid; e < p.first + p.last; e += threads) {   // (those that were not in a word above)
        const int at = e < p.first ? e : end + e - p.first;
        atomicOr(&in[at >> 5], 1u << (at & 31));
    }
    const int rest = k - mine, some = sm.count;
    if (k > 0 && some <= kFew) {
        if (some == rest) {
            for (int i = tid; i < some; i += threads) atomicOr(&in[sm.few_at[i] >> 5], 1u << (sm.few_at[i] & 31));
        } else {
            for (int i = warp; i < some; i += warps) {
                const double x = exact_score<D>(p, tok, hk, sm.few_at[i]);
                if (lane == 0) sm.few[i] = x;
            }
            __syncthreads();
            for (int i = tid; i < some; i += threads) {
                const double x = sm.few[i];
                const int e = sm.few_at[i];
                int better = 0;
                for (int j = 0; j < some; ++j) better += sm.few[j] > x || (sm.few[j] == x && sm.few_at[j] < e);
                if (better < rest) atomicOr(&in[e >> 5], 1u << (e & 31));
            }
        }
    } else if (k > 0) {
        // Many that differ by less than the error (alike, most of them): the rest-th largest of their exact scores, bits by bits from the top, then
        // those above it and, of its own value, the first.
        double* exact = p.exact + pair * p.blocks * 16;
        auto doubt = [&](int e) {
            const float x = s[e];
            return !(sure && x > above) && !(x < below);
        };
        for (int e = begin + warp; e < end; e += warps) {
            if (!doubt(e)) continue;
            const double x = exact_score<D>(p, tok, hk, e);
            if (lane == 0) exact[e] = x;
        }
        __syncthreads();
        int need = rest;
        unsigned long long value = 0;
        for (int shift = 56; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += threads) sm.bins[i] = 0;
            __syncthreads();
            for (int e = begin + tid; e < end; e += threads) {
                if (!doubt(e)) continue;
                const unsigned long long x = ordered(exact[e]);
                if (shift == 56 || x >> (shift + 8) == value >> (shift + 8)) atomicAdd(&sm.bins[x >> shift & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int bin = 255, left = need;
                while (sm.bins[bin] < left) left -= sm.bins[bin--];
                sm.need = left;
                sm.value = value | static_cast<unsigned long long>(bin) << shift;
            }
            __syncthreads();
            need = sm.need;
            value = sm.value;
            __syncthreads();
        }
        // need: how many of the value itself, in the order of their places.
        if (tid == 0) sm.count = 0;
        __syncthreads();
        for (int e0 = begin & ~31; e0 < end; e0 += threads) {
            const int e = e0 + tid;
            const bool here = e >= begin && e < end && doubt(e);
            const unsigned long long x = here ? ordered(exact[e]) : 0;
            const uint32_t ties = __ballot_sync(0xffffffffu, here && x == value);
            if (lane == 0) sm.iwarps[warp] = __popc(ties);
            __syncthreads();
            int before = sm.count + __popc(ties & ((1u << lane) - 1));
            for (int w = 0; w < warp; ++w) before += sm.iwarps[w];
            const bool take = here && (x > value || (x == value && before < need));
            const uint32_t bits = __ballot_sync(0xffffffffu, take);
            if (lane == 0 && bits) atomicOr(&in[e >> 5], bits);
            __syncthreads();
            if (tid == 0) {
                for (int w = 0; w < warps; ++w) sm.count += sm.iwarps[w];
            }
            __syncthreads();
        }
    }
    __syncthreads();
    // The bits in order: a thread has a word of 32 pages.
    int before = 0;
    for (int w0 = 0; w0 < words; w0 += threads) {
        const uint32_t bits = w0 + tid < words ? in[w0 + tid] : 0u;
        const int own = __popc(bits);
        int sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        if (lane == 31) sm.iwarps[warp] = sum;
        __syncthreads();
        int at = before + sum - own;
        for (int w = 0; w < warps; ++w) {
            const int x = sm.iwarps[w];
            at += w < warp ? x : 0;
            before += x;
        }
        for (uint32_t left = bits; left; left &= left - 1) {
            const int e = (w0 + tid) * 32 + __ffs(left) - 1;
            to[at++] = row[e];
        }
        __syncthreads();
    }
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
    const int threads = width <= 512 ? 256 : (width <= 2048 ? 512 : 1024);
    const int bits = (plan.blocks + 1) / 2 * 4, scores = plan.blocks * 64;
    constexpr int kMost = 200 * 1024;
    const bool in_shared = bits + scores <= kMost;
    const int smem = bits + (in_shared ? scores : 0);
    if (smem > 32 * 1024) {
        if (int rc = ensure_smem(select_kernel<D>, kMost, "cudaFuncSetAttribute(select)")) return rc;
    }
    for (int64_t t0 = 0; t0 < plan.tokens; t0 += plan.slice) {
        const int64_t n = plan.tokens - t0 < plan.slice ? plan.tokens - t0 : plan.slice, pairs = n * p.kv_heads;
        p.token0 = t0;
        // Blocks of a warp: as many warps as the GPU holds, and no more than four blocks one after another until it is full.
        const int64_t all = pairs * plan.blocks, warps = 148 * 16;
        const int64_t each = (all + warps - 1) / warps;
        p.each = static_cast<int>(each > 4 ? 4 : each);
        p.lots = (plan.blocks + 4 * p.each - 1) / (4 * p.each);
        if (int rc = launch_dependent(score_kernel<D>, p, dim3(static_cast<unsigned>(pairs * p.lots)), dim3(128), stream, "paged_select launch")) return rc;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(pairs));
        cfg.blockDim = dim3(static_cast<unsigned>(threads));
        cfg.dynamicSmemBytes = static_cast<size_t>(smem);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (int rc = check_cuda(cudaLaunchKernelEx(&cfg, select_kernel<D>, p, static_cast<int>(in_shared)), "paged_select launch")) return rc;
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
