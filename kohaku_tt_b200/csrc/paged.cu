// The paged cache: appending rows (with the rotation of the keys and of the step's queries) and reading it back.
#include <type_traits>

#include "four_bits.cuh"

namespace ktt {

const char* pages_of(Pages& c, const ktt_b200_pages& a, int d) {
    if (a.bits != 16 && a.bits != 4) return "pages hold 16 or 4 bits per value";
    if (d != 64 && d != 128) return "head dim 64 or 128";
    if (a.page_size < 16 || a.page_size % 16) return "the page size must be a multiple of 16";
    if (a.kv_heads < 1 || a.table_width < 1 || a.pages < 1) return "sizes must be positive";
    if (a.kv_heads > 4096) return "at most 4096 K / V heads";
    const int64_t all = static_cast<int64_t>(a.table_width) * a.page_size;
    if (all > (1 << 30)) return "at most 2^30 keys per sequence";
    const int size = a.bits == 16 ? 2 : 1;
    for (int i = 0; i < 3; ++i) {
        c.ks[i] = a.k_strides[i] * size;
        c.vs[i] = a.v_strides[i] * size;
        if (i < 2 || a.bits == 16) {
            if ((c.ks[i] | c.vs[i]) & 15) return "page strides must be multiples of 16 bytes";
        }
    }
    if ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15) return "pages must be 16-byte aligned";
    c.k = static_cast<unsigned char*>(a.k);
    c.v = static_cast<unsigned char*>(a.v);
    c.table = a.block_table;
    c.table_stride = a.table_stride;
    c.lengths = a.lengths;
    c.pages = a.pages;
    c.page_size = a.page_size;
    c.cap = static_cast<int>(a.max_keys > 0 && a.max_keys < all ? a.max_keys : all);
    return nullptr;
}

namespace {

struct AppendParams {
    Pages c;
    Turn turn;
    int batch, rows, heads, kv_heads;
    int groups;            // blocks of `loops` times kHeads queries' heads; those of the keys and of the values follow in the grid's y
    int loops;
    unsigned pair_blocks, pair_rows;   // blocks of the first part (append_queries), and of one group of heads there; the others follow in the grid's x, if any
    int64_t tokens;        // rows of all sequences
    const __nv_bfloat16* q;
    __nv_bfloat16* q_out;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    int64_t qs[3], qos[3], ks[3], vs[3];
    const int32_t* cu;
    int32_t* lengths_out;
    int vec;
};
// With positions of their own, and with bounds that a key of a sequence goes into on the way (one row for each sequence).
struct AppendAtParams : AppendParams {
    Placed positions;
    PairAxes axes;
    Bounds bounds;
};
// With how many of its new rows each sequence takes. (Kernels of their own: where a null pointer told them apart, one token of 64 sequences with
// positions and bounds took 4.2 us for 3.9. With bounds alone 3.1 us, granted 3.5.)
struct AppendGrantedParams : AppendAtParams {
    const int32_t* granted;
};

// Eight columns of one token in the cache's 4 bits. The 8 threads of a group of 64 columns are neighbours in a warp and
// all arrive here; `there`: the row has a place. Returns the codes and (step, least). The codes are those of (x - least) / step rounded as fp32 does, to the
// bit: the quotient is the product with 1 / step, corrected by its remainder (Markstein's theorem: with 1 / step correctly
// rounded and the remainder exact, the corrected quotient is the correctly rounded one), 6 operations for a column where a
// division takes some 12; a power of two keeps steps near the ends of fp32's range from taking the remainder out of it.
template <int D>
__device__ __forceinline__ uint2 put_four_bits(const Eight<__nv_bfloat16>& x, unsigned char* block, bool value, int token, int chunk, bool there) {
    const __nv_bfloat162* pair = reinterpret_cast<const __nv_bfloat162*>(x.raw);
    const __nv_bfloat162 lo = __hmin2_nan(__hmin2_nan(pair[0], pair[1]), __hmin2_nan(pair[2], pair[3]));
    const __nv_bfloat162 hi = __hmax2_nan(__hmax2_nan(pair[0], pair[1]), __hmax2_nan(pair[2], pair[3]));
    // (least, -most): a NaN anywhere makes both NaN.
    __nv_bfloat162 ends = __halves2bfloat162(__hmin_nan(__low2bfloat16(lo), __high2bfloat16(lo)), __hneg(__hmax_nan(__low2bfloat16(hi), __high2bfloat16(hi))));
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) ends = __hmin2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, off));
    const float least = __low2float(ends);
    const __nv_bfloat16 step = __float2bfloat16_rn(__fmul_rn(__fsub_rn(-__high2float(ends), least), 1.f / 15.f));
    const float s = __bfloat162float(step);
    uint32_t word = 0;
    auto encode = [&](auto coarse) {
        const float even = s < 0x1p-60f ? 0x1p100f : (s > 0x1p60f ? 0x1p-100f : 1.f), r = s * even, inv = __frcp_rn(r);
        const Pair least2(least), even2(even), inv2(inv), r2(-r), whole2(8388608.f);
        Pair codes(0.f);
#pragma unroll
        for (int n = 3; n >= 0; --n) {
            const Pair d = sub(Pair(to_f32(x.get(2 * n)), to_f32(x.get(2 * n + 1))), least2) * even2, q = d * inv2;
            Pair t = fma(fma(q, r2, d), inv2, q);
            if constexpr (decltype(coarse)::value) t = Pair(fminf(t.low(), 15.f), fminf(t.high(), 15.f));
            // To the nearest whole number, ties to even; four of them make one of 16 bits.
            codes = fma(codes, Pair(16.f), sub(t + whole2, whole2));
        }
        codes = codes + whole2;
        word = __byte_perm(__float_as_uint(codes.low()), __float_as_uint(codes.high()), 0x5410);
    };
    // t is at most 15 (1 + 2^-8), by half of a bf16 step's rounding; a subnormal step, which is rounded by up to half of 2^-133, can leave
    // values as far as 22 steps from the least, whose code is 15. (Else all codes are 0.)
    if (s >= 0x1p-126f && s < INFINITY) encode(std::false_type());
    else if (s > 0.f && s < INFINITY) encode(std::true_type());
    const uint2 held = make_uint2(word, static_cast<uint32_t>(__bfloat16_as_ushort(step)) | static_cast<uint32_t>(__bfloat16_as_ushort(__low2bfloat16(ends))) << 16);
    if (!there) return held;
    uint32_t* to = reinterpret_cast<uint32_t*>(block);
    to[value ? value_word<D>(token, chunk) : key_word<D>(token, chunk)] = held.x;
    if (chunk % 8 == 0) to[step_word<D>(token, chunk / 8)] = held.y;
    return held;
}

// Where row n of the new ones goes: its sequence and how many keys that has; kEach threads of a warp share a row.
struct Row {
    int b, cached;
    int64_t in;      // its place among the sequence's new ones
    bool there;
};
template <int kEach>
__device__ __forceinline__ Row row_at(const AppendParams& p, int64_t n, int b, int64_t r, bool in_range) {
    Row x = {b, 0, r, in_range};
    if (p.cu && p.batch < 32) {
        // A lane looks at one sequence each, its length with it: one trip where a search takes log2(batch) + 2 that wait for one
        // another (8 sequences, 10,240 tokens, 32 heads over 8, D 128, 4 bits: 61.5 us with a search).
        const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31, start = p.cu[min(lane, p.batch)], keys = cached_keys(p.c, min(lane, p.batch - 1));
#pragma unroll
        for (int i = 0; i < 32 / kEach; ++i) {   // (the last sequence that starts at or before the token)
            const int64_t token = __shfl_sync(0xffffffffu, n, i * kEach);
            const uint32_t before = __ballot_sync(0xffffffffu, lane <= p.batch && start <= token);
            if (token == n) x.b = __popc(before) - 1;
        }
        x.there = in_range && x.b >= 0 && x.b < p.batch;
        if (!x.there) x.b = 0;
        x.in = n - __shfl_sync(0xffffffffu, start, x.b);
        x.there = x.there && x.in >= 0;   // (offsets that decrease)
        x.cached = __shfl_sync(0xffffffffu, keys, x.b);
    } else if (in_range) {
        if (p.cu) {
            x.b = sequence_of(p.cu, p.batch, n);
            x.there = x.b >= 0;
            x.b = x.there ? x.b : 0;
            x.in = n - p.cu[x.b];
        }
        x.cached = cached_keys(p.c, x.b);
    }
    return x;
}

// What a row turns by: its place, or positions of its own. (Packed rows have one batch entry's positions; without any, the place is the only
// axis, and all pairs are of axis 0.)
template <bool kFast, typename Params>
__device__ __forceinline__ void turn_of(Turned<kFast>& turned, const Params& p, const Row& x, int64_t r, int col) {
    const int64_t pos = x.cached + x.in;
    if constexpr (std::is_base_of_v<AppendAtParams, Params>) {
        Positions<true> at = {};
        if (p.positions.at) at = p.positions.all(p.axes.axes, p.cu ? 0 : x.b, r);
        else at.at[0] = pos;
        turned.load(p.turn, p.axes, at, col);
    } else {
        turned.load(p.turn, pos, col);
    }
}

// Many queries in the half layout: a thread has eight pairs, both columns of each, of four heads of a token at a time, as in the rotation
// (rotary_pairs_kernel), or 16 columns that do not turn.
template <int D, typename Params>
__device__ __forceinline__ void append_queries(const Params& p) {
    constexpr int kEach = D / 16, kHeads = 4;
    const uint32_t group = blockIdx.x / p.pair_rows, rows = blockIdx.x - group * p.pair_rows;
    const int tid = threadIdx.y * blockDim.x + threadIdx.x, half = p.turn.half, pair = tid % kEach * 8;
    const int64_t n = static_cast<int64_t>(rows) * (256 / kEach) + tid / kEach;
    const bool in_range = n < p.tokens, turns = pair < half;
    const int b = in_range && !p.cu ? static_cast<int>(static_cast<uint32_t>(n) / static_cast<uint32_t>(p.rows)) : 0;
    const int64_t r = !in_range ? 0 : p.cu ? n : n - static_cast<int64_t>(b) * p.rows;
    const int col = turns ? pair : 2 * pair, other = turns ? pair + half : 2 * pair + 8;
    const __nv_bfloat16* from = p.q + (p.cu ? 0 : b * p.qs[0]) + r * p.qs[2];
    Eight<__nv_bfloat16> lo[kHeads], hi[kHeads];
    auto rows_of = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const __nv_bfloat16* row = from + static_cast<int64_t>(min(h0 + i, p.heads - 1)) * p.qs[1];
            lo[i].load(row + col);
            hi[i].load(row + other);
        }
    };
    int h0 = static_cast<int>(group) * (kHeads * p.loops);
    const Row x = row_at<kEach>(p, n, b, r, in_range);
    if (!x.there) return;
    Turned<true> turned;
    if (turns) turn_of(turned, p, x, r, col);
    __nv_bfloat16* out = p.q_out + (p.cu ? 0 : x.b * p.qos[0]) + r * p.qos[2];
    for (int loop = 0; loop < p.loops && h0 < p.heads; ++loop, h0 += kHeads) {
        rows_of(h0);
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            if (h0 + i >= p.heads) break;
            if (turns) turned.both(lo[i], hi[i]);
            __nv_bfloat16* to = out + (h0 + i) * p.qos[1];
            lo[i].store(to + col);
            hi[i].store(to + other);
        }
    }
}

// A thread has eight columns of kHeads heads of one token, and of the next kHeads, `loops` times: of queries, keys or values. Its first rows are
// requested before it knows where they go (a packed row's sequence takes a search). No thread leaves before the groups' shuffles.
template <int D, int kBits, bool kFast, int kHeads, typename Params>
__global__ void __launch_bounds__(256, kHeads == 4 ? 3 : 4) append_kernel(const __grid_constant__ Params p) {
    constexpr bool kAt = std::is_base_of_v<AppendAtParams, Params>, kGranted = std::is_same_v<Params, AppendGrantedParams>;
    const int chunk = threadIdx.x, col = chunk * 8;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (p.lengths_out && blockIdx.x == 0 && blockIdx.y == 0) {
        for (int b = threadIdx.y * blockDim.x + threadIdx.x; b < p.batch; b += blockDim.x * blockDim.y) {
            int64_t more = p.cu ? max(p.cu[b + 1] - p.cu[b], 0) : p.rows;
            if constexpr (kGranted) more = min(more, granted_to(p.granted, b));
            const int64_t all = cached_keys(p.c, b) + more;
            p.lengths_out[b] = static_cast<int32_t>(all < p.c.cap ? all : p.c.cap);
        }
    }
    if constexpr (kFast && kHeads > 1) {
        if (blockIdx.x < p.pair_blocks) return append_queries<D>(p);
    }
    // What the block has: queries, keys or values.
    const int loops = kHeads == 1 ? 1 : p.loops, per = kHeads * loops;
    const int kv = (p.kv_heads + per - 1) / per;
    uint32_t bx = blockIdx.x, y = blockIdx.y;
    if (kFast && kHeads > 1 && p.pair_blocks) {   // (keys and values, one group of heads after another)
        const uint32_t blocks = (gridDim.x - p.pair_blocks) / (2 * kv);
        y = (bx - p.pair_blocks) / blocks;
        bx -= p.pair_blocks + y * blocks;
        y += p.groups;
    }
    const int64_t n = static_cast<int64_t>(bx) * blockDim.y + threadIdx.y;
    const int what = static_cast<int>(y) < p.groups ? 0 : static_cast<int>(y) < p.groups + kv ? 1 : 2;
    int h0 = (static_cast<int>(y) - (what == 0 ? 0 : what == 1 ? p.groups : p.groups + kv)) * per;
    const int heads = what == 0 ? p.heads : p.kv_heads;
    const __nv_bfloat16* from = what == 0 ? p.q : what == 1 ? p.k : p.v;
    const int64_t sb = what == 0 ? p.qs[0] : what == 1 ? p.ks[0] : p.vs[0], sh = what == 0 ? p.qs[1] : what == 1 ? p.ks[1] : p.vs[1];
    const int64_t sr = what == 0 ? p.qs[2] : what == 1 ? p.ks[2] : p.vs[2];
    const bool in_range = n < p.tokens;
    const int b0 = in_range && !p.cu ? static_cast<int>(static_cast<uint32_t>(n) / static_cast<uint32_t>(p.rows)) : 0;   // (2^31 tokens at most)
    const int64_t r = !in_range ? 0 : p.cu ? n : n - static_cast<int64_t>(b0) * p.rows;
    from += (p.cu ? 0 : b0 * sb) + r * sr;
    Eight<__nv_bfloat16> x[kHeads], other[kHeads];
    const int partner = what == 2 || !p.turn.cos || p.turn.interleaved || col >= 2 * p.turn.half ? -1 : col < p.turn.half ? col + p.turn.half : col - p.turn.half;
    auto rows_of = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            if (!in_range || h0 + i >= heads) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i].set(e, __float2bfloat16_rn(0.f));
                continue;
            }
            const __nv_bfloat16* row = from + (h0 + i) * sh;
            if (kFast || p.vec) x[i].load(row + col); else x[i].load_some(row + col, 8);
            if (kFast && partner >= 0) other[i].load(row + partner);
        }
    };
    rows_of(h0);
    const Row x_row = row_at<D / 8>(p, n, b0, r, in_range);
    const int b = x_row.b;
    const bool row_there = x_row.there;
    const int64_t pos = row_there ? x_row.cached + x_row.in : 0;
    Turned<kFast> turned;
    turned.count = 0;
    if (what != 2 && row_there) turn_of(turned, p, x_row, r, col);
    if (what == 0) {
        if (!row_there) return;
        __nv_bfloat16* to = p.q_out + (p.cu ? 0 : b * p.qos[0]) + r * p.qos[2] + col;
        for (int loop = 0; loop < loops && h0 < heads; ++loop, h0 += kHeads) {
            if (loop) rows_of(h0);
#pragma unroll
            for (int i = 0; i < kHeads; ++i) {
                if (h0 + i >= heads) break;
                turned.apply(p.turn, x[i], other[i], from + (h0 + i) * sh, col);
                if (kFast || p.vec) x[i].store(to + (h0 + i) * p.qos[1]); else x[i].store_some(to + (h0 + i) * p.qos[1], 8);
            }
        }
        return;
    }
    int64_t page = -1;
    if (row_there && pos < p.c.cap) page = page_of(p.c, b, static_cast<int>(pos));
    if constexpr (kGranted) page = x_row.in < granted_to(p.granted, b) ? page : -1;   // (looked up beside it, not before it)
    const bool there = page >= 0;
    const int at = there ? static_cast<int>(pos) % p.c.page_size : 0;
    unsigned char* base = !there ? nullptr : what == 2 ? p.c.v + page * p.c.vs[0] : p.c.k + page * p.c.ks[0];
    const int64_t head_stride = what == 2 ? p.c.vs[1] : p.c.ks[1];
    for (int loop = 0; loop < loops && h0 < heads; ++loop, h0 += kHeads) {
        if (loop) rows_of(h0);
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            if (h0 + i >= heads) break;
            if (there && what == 1) turned.apply(p.turn, x[i], other[i], from + (h0 + i) * sh, col);
            unsigned char* to = there ? base + (h0 + i) * head_stride : nullptr;
            if constexpr (kBits == 16) {
                if (there) x[i].store(reinterpret_cast<__nv_bfloat16*>(to + at * (what == 2 ? p.c.vs[2] : p.c.ks[2])) + col);
            } else {
                if (there) to += static_cast<int64_t>(at >> 4) * (9 * D);
                const uint2 held = put_four_bits<D>(x[i], to, what == 2, at & 15, chunk, there);
                if constexpr (kAt) {
                    if (p.bounds.at && what == 1) x[i] = of_four_bits(held.x, held.y);
                }
            }
            if constexpr (kAt) {
                // The sequence's only new key: no other thread has these channels of its page's bounds.
                if (p.bounds.at && what == 1 && there) {
                    Edges e = {x[i], x[i]};
                    __nv_bfloat16 *lo = p.bounds.edge(page, h0 + i, 0) + col, *hi = p.bounds.edge(page, h0 + i, 1) + col;
                    if (at > 0) {
                        Edges old;
                        old.lo.load(lo);
                        old.hi.load(hi);
                        e.with(old.lo, old.hi);
                    }
                    e.lo.store(lo);
                    e.hi.store(hi);
                }
            }
        }
    }
}

struct ReadParams {
    Pages c;
    int batch, rows;
    ChunkHead head;
    __nv_bfloat16* k;
    __nv_bfloat16* v;
    int64_t ks[3], vs[3];
};

// The same in fp16, of a step and a least value times a power of two that leaves none of the sums at 2^15 or above. Both have 8 bits, so
// they are fp16's too but where they are under 2^-17, which is nothing beside 2^15; the sums are rounded once, by 2^-11 of them at most.
__device__ __forceinline__ Eight<__half> of_four_bits_f16(uint32_t word, uint32_t pair, float power) {
    const __half2 step = __float2half2_rn(step_of(pair) * power), least = __float2half2_rn(least_of(pair) * power), zero = __float2half2_rn(1024.f);
    Eight<__half> x;
    __half2* to = reinterpret_cast<__half2*>(x.raw);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const uint32_t two = ((word >> (4 * n)) & 0x000f000fu) | 0x64006400u;   // two codes as fp16 1024 + c
        to[n] = __hfma2(step, __hsub2(*reinterpret_cast<const __half2*>(&two), zero), least);
    }
    return x;
}

// A thread brings eight columns of kReadRows keys and their values, all requested before the first is used.
constexpr int kReadRows = 4;
// The power of two that brings numbers of up to this exponent (fp32's 8 bits) under 2^15: a multiple of 4, so that it changes
// seldom, 116 at most. What shares a power (a query row, 64 keys, 64 values) has 11 bits down to 2^-25 of the largest and fewer below, and
// under 2^-65 in any case, so that the sum of 2^30 weights over their power stays in range. (Keys whose values are all under 2^-110 of others' of
// the head weigh nothing beside them, in the sum of weights too.)
__device__ __forceinline__ int f16_power(int exponent) { return max((exponent - 127 + 1 - 15 + 3) & ~3, -80); }

// Queries in fp16 as the forward takes them beside such keys: rows [row][head][D], each times a power of two, by the blocks of a grid's planes
// from z on. D / 8 threads have kQueries of them.
constexpr int kQueries = 4;
template <int D>
__device__ __forceinline__ void f16_queries(const ChunkHead& p, int z) {
    constexpr int kThreads = D / 8, kRows = 256 / kThreads;
    const int col = threadIdx.x % kThreads * 8;
    const int64_t all = p.q_rows * p.heads, plane = static_cast<int64_t>(gridDim.x) * gridDim.y, step = plane * (gridDim.z - z) * (kQueries * kRows);
    for (int64_t n0 = ((blockIdx.z - z) * plane + static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * (kQueries * kRows); n0 < all; n0 += step) {
        Eight<__nv_bfloat16> x[kQueries];
#pragma unroll
        for (int i = 0; i < kQueries; ++i) {   // (all requested before the first is used)
            const int64_t n = n0 + i * kRows + threadIdx.x / kThreads;
            x[i].zero();
            if (n >= all) continue;
            // (64-bit quotients take some hundred instructions)
            const int64_t row = all >> 32 ? n / p.heads : static_cast<uint32_t>(n) / static_cast<uint32_t>(p.heads);
            const int64_t b = !p.sq ? 0 : all >> 32 ? row / p.sq : static_cast<uint32_t>(row) / static_cast<uint32_t>(p.sq);
            const __nv_bfloat16* from = p.q + b * p.qs[0] + (n - row * p.heads) * p.qs[1] + (row - b * p.sq) * p.qs[2] + col;
            if (p.q_vec) x[i].load(from); else x[i].load_some(from, 8);
        }
#pragma unroll
        for (int i = 0; i < kQueries; ++i) {
            const int64_t n = n0 + i * kRows + threadIdx.x / kThreads;
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(__bfloat162float(x[i].get(e))));
#pragma unroll
            for (int off = 1; off < kThreads; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            if (n >= all) continue;   // (the last in any case)
            const int power = f16_power(__float_as_int(top) >> 23);
            const float by = power_of_two(-power);
            Eight<__half> y;
#pragma unroll
            for (int e = 0; e < 8; ++e) y.set(e, __float2half_rn(__bfloat162float(x[i].get(e)) * by));
            y.store(p.q_out + n * D + col);
            if (col == 0) p.q_power[n] = power_of_two(power);
        }
    }
}

// kHalf: 4-bit keys and values as fp16 with powers of two for each 64 keys, for the forward (ChunkHead); else bf16.
template <int D, int kBits, bool kHalf>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadParams p) {
    constexpr int kChunks = D / 8, kTokens = 256 / kChunks;   // tokens of the block at a time
    const int chunk = threadIdx.x % kChunks, col = chunk * 8, head = blockIdx.y, b = blockIdx.z;
    const int first = blockIdx.x * (kReadRows * kTokens) + threadIdx.x / kChunks;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int batch = p.batch;
    if (kHalf && b >= batch) return f16_queries<D>(p.head, batch);
    const int len = cached_keys(p.c, b);
    if (p.head.words && blockIdx.x == 0 && head == 0) {
        if (threadIdx.x == 0) {
            const bool last = b == batch - 1;
            p.head.offsets()[b] = b * p.rows;
            if (last) p.head.offsets()[batch] = batch * p.rows;
            if (p.head.cu_q) {
                p.head.query_offsets(batch)[b] = static_cast<int32_t>(row_offset(p.head.cu_q, b, p.head.total_q));
                if (last) p.head.query_offsets(batch)[batch] = static_cast<int32_t>(row_offset(p.head.cu_q, batch, p.head.total_q));
            }
        }
        if (b == 0 && threadIdx.x < kHeadWords && (threadIdx.x == 0 || threadIdx.x > 2 || !p.head.most_parts)) p.head.words[threadIdx.x] = 0;
        int place = 0;
        for (int i0 = 0; i0 < batch; i0 += 256) {
            const int i = i0 + threadIdx.x, other = i < batch ? cached_keys(p.c, i) : -1;
            place += __syncthreads_count(other > len || (other == len && i < b));
        }
        if (threadIdx.x == 0) p.head.order(batch)[place] = b;
        if (threadIdx.x == 0 && place == 0 && p.head.most_parts) {   // (the longest)
            const int blocks = (max(len, 1) + 127) / 128, parts = parts_of_chunk(p.head.tiles, blocks, p.head.sms, p.head.d, p.head.most_parts);
            p.head.words[1] = parts;
            p.head.words[2] = (blocks + parts - 1) / parts * 128;
        }
    }
    const int rows = p.head.words ? min(len, p.rows) : p.rows;   // (what lies behind a length is nothing to the forward)
    if (blockIdx.x * (kReadRows * kTokens) >= rows) return;
    const unsigned char *kp[kReadRows], *vp[kReadRows];
    int token[kReadRows];
#pragma unroll
    for (int i = 0; i < kReadRows; ++i) {
        const int j = first + i * kTokens, entry = j / p.c.page_size, at = j - entry * p.c.page_size;
        int64_t page = -1;
        if (j < len && j < p.rows) page = p.c.table[b * p.c.table_stride + entry];
        kp[i] = vp[i] = nullptr;
        token[i] = at & 15;
        if (page >= 0 && page < p.c.pages) {
            kp[i] = p.c.k + page * p.c.ks[0] + head * p.c.ks[1] + (kBits == 16 ? at * p.c.ks[2] : static_cast<int64_t>(at >> 4) * (9 * D));
            vp[i] = p.c.v + page * p.c.vs[0] + head * p.c.vs[1] + (kBits == 16 ? at * p.c.vs[2] : static_cast<int64_t>(at >> 4) * (9 * D));
        }
    }
    Eight<__nv_bfloat16> k[kReadRows], v[kReadRows];
    uint32_t words[kReadRows][4];
#pragma unroll
    for (int i = 0; i < kReadRows; ++i) {
        if constexpr (kBits == 16) {
            k[i].zero();
            v[i].zero();
            if (kp[i]) {
                k[i].load(reinterpret_cast<const __nv_bfloat16*>(kp[i]) + col);
                v[i].load(reinterpret_cast<const __nv_bfloat16*>(vp[i]) + col);
            }
        } else {
            words[i][0] = words[i][1] = words[i][2] = words[i][3] = 0;   // (worth zeros)
            if (kp[i]) {
                const uint32_t *kw = reinterpret_cast<const uint32_t*>(kp[i]), *vw = reinterpret_cast<const uint32_t*>(vp[i]);
                words[i][0] = kw[key_word<D>(token[i], chunk)];
                words[i][1] = kw[step_word<D>(token[i], chunk / 8)];
                words[i][2] = vw[value_word<D>(token[i], chunk)];
                words[i][3] = vw[step_word<D>(token[i], chunk / 8)];
            }
        }
    }
    if constexpr (kHalf) {
        // The powers of each 64 keys, and of their values, from the largest end of a group among them (its exponent, over the block).
        constexpr int kKeys = 64, kOf = kReadRows * kTokens / kKeys, kEach = kReadRows / kOf;   // chunks of the block, a thread's keys of each
        static_assert(kKeys % kTokens == 0 && kOf >= 1, "a thread's keys are of whole chunks");
        __shared__ int tops[2 * kOf];
        if (threadIdx.x < 2 * kOf) tops[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2 * kOf; ++c) {   // keys of each chunk, then values
            float top = 0.f;
#pragma unroll
            for (int i = (c % kOf) * kEach; i < (c % kOf + 1) * kEach; ++i) {
                const uint32_t pair = words[i][c < kOf ? 1 : 3];
                const float end = fmaxf(fabsf(least_of(pair)), fabsf(fmaf(15.f, step_of(pair), least_of(pair))));
                if (end < INFINITY) top = fmaxf(top, end);   // (an infinity has no power, and takes none from the others)
            }
            const int most = __reduce_max_sync(0xffffffffu, __float_as_int(top) >> 23);
            if ((threadIdx.x & 31) == 0) atomicMax(&tops[c], most);
        }
        __syncthreads();
        const int first_chunk = blockIdx.x * kOf;
        int32_t* powers = p.head.powers + (static_cast<int64_t>(head) * batch + b) * p.head.chunks + first_chunk;
        if (threadIdx.x == 0) {
#pragma unroll
            for (int c = 0; c < kOf; ++c) powers[c] = static_cast<int>(__byte_perm(f16_power(tops[c]), f16_power(tops[kOf + c]), 0x5410));
            // The forward looks at chunks by two; the block of one without a key does not get here.
            if (kOf == 1 && !(first_chunk & 1) && (first_chunk + 1) * kKeys >= rows) powers[1] = powers[0];
        }
#pragma unroll
        for (int i = 0; i < kReadRows; ++i) {
            const int j = first + i * kTokens;
            if (j >= rows) break;
            const float kp2 = power_of_two(-f16_power(tops[i / kEach])), vp2 = power_of_two(-f16_power(tops[kOf + i / kEach]));
            of_four_bits_f16(words[i][0], words[i][1], kp2).store(reinterpret_cast<__half*>(p.k) + b * p.ks[0] + head * p.ks[1] + j * p.ks[2] + col);
            of_four_bits_f16(words[i][2], words[i][3], vp2).store(reinterpret_cast<__half*>(p.v) + b * p.vs[0] + head * p.vs[1] + j * p.vs[2] + col);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kReadRows; ++i) {
        const int j = first + i * kTokens;
        if (j >= rows) break;
        if constexpr (kBits == 4) {
            k[i] = of_four_bits(words[i][0], words[i][1]);
            v[i] = of_four_bits(words[i][2], words[i][3]);
        }
        k[i].store(p.k + b * p.ks[0] + head * p.ks[1] + j * p.ks[2] + col);
        v[i].store(p.v + b * p.vs[0] + head * p.vs[1] + j * p.vs[2] + col);
    }
}

template <int D, int kBits, typename Params>
int launch_append(const Params& given, cudaStream_t stream) {
    Params p = given;
    const dim3 block(D / 8, 256 / (D / 8));
    const int64_t blocks = (p.tokens + block.y - 1) / block.y;   // one at least: it writes the new lengths
    auto go = [&](auto kernel, int per, bool pairs) {   // pairs: queries by append_queries
        per *= p.loops;
        p.groups = (p.heads + per - 1) / per;
        const unsigned kv = 2 * ((p.kv_heads + per - 1) / per), rows = static_cast<unsigned>(blocks > 0 ? blocks : 1);
        p.pair_blocks = 0;
        if (pairs && p.heads) {
            p.pair_rows = static_cast<unsigned>((p.tokens + 4096 / D - 1) / (4096 / D));
            const int64_t all = static_cast<int64_t>(p.pair_rows) * p.groups + static_cast<int64_t>(rows) * kv;
            if (all < (1ll << 31)) {
                p.pair_blocks = p.pair_rows * p.groups;
                return launch_dependent(kernel, p, dim3(static_cast<unsigned>(all)), block, stream, "paged_append launch");
            }
        }
        return launch_dependent(kernel, p, dim3(rows, p.groups + kv), block, stream, "paged_append launch");
    };
    const bool fast = p.vec && turn_is_fast(p.turn);
    // Four heads to a thread once that makes threads enough, and four more after them: a token's place, page and table rows are looked up once for
    // all of them. 32 heads over 8, D 128, us for 1 and 4 heads: 256 tokens, 4 bits 4.6 and 5.4; 512, bf16 6.0 and 3.9; 1,024, 4 bits 11.5 and 7.7. For
    // 4, 8, 16 and 32 heads: 1,024 tokens, 4 bits 7.7, 10.1, 10.6, 14.3; 2,048, bf16 10.9, 9.8, 12.4, 18.2; 4,096, 4 bits 23.1, 22.4, 19.7, 20.6; 10,240
    // packed ones, 4 bits 54.4, 49.4, 48.1, 46.6 (bf16 42.0, 5.6 TB/s), by positions of three axes 67.4, 57.9, 56.7, 54.7. With queries in the
    // half layout as keys are, eight columns to a thread, 51.0 and 61.4.
    p.loops = 1;
    const int64_t threads = p.tokens * (D / 8) * (p.heads + 2 * p.kv_heads);
    if (threads >= 3 << 17) {
        p.loops = threads < 7 << 17 ? 1 : (threads < 1 << 21 ? 2 : (threads < 1 << 22 ? 4 : 8));
        if (fast) return go(append_kernel<D, kBits, true, 4, Params>, 4, p.turn.cos && !p.turn.interleaved);
        return go(append_kernel<D, kBits, false, 4, Params>, 4, false);
    }
    if (fast) return go(append_kernel<D, kBits, true, 1, Params>, 1, false);
    return go(append_kernel<D, kBits, false, 1, Params>, 1, false);
}

template <int D, int kBits>
int launch_read(const ReadParams& p, int kv_heads, cudaStream_t stream) {
    constexpr int kRows = kReadRows * (256 / (D / 8));
    dim3 grid(static_cast<unsigned>((p.rows + kRows - 1) / kRows), static_cast<unsigned>(kv_heads), static_cast<unsigned>(p.batch));
    if (p.head.q_rows > 0) {   // planes for the queries
        const int64_t one = static_cast<int64_t>(grid.x) * grid.y * (kQueries * 256 / (D / 8)), planes = (p.head.q_rows * p.head.heads + one - 1) / one;
        grid.z += static_cast<unsigned>(planes < 32768 ? planes : 32768);
    }
    if (kBits == 4 && p.head.powers) return launch_dependent(read_kernel<D, 4, true>, p, grid, dim3(256), stream, "paged_read launch");
    return launch_dependent(read_kernel<D, kBits, false>, p, grid, dim3(256), stream, "paged_read launch");
}

int launch_read(const ReadParams& p, int bits, int d, int kv_heads, cudaStream_t stream) {
    if (bits == 16) return d == 64 ? launch_read<64, 16>(p, kv_heads, stream) : launch_read<128, 16>(p, kv_heads, stream);
    return d == 64 ? launch_read<64, 4>(p, kv_heads, stream) : launch_read<128, 4>(p, kv_heads, stream);
}

}  // namespace

int read_pages(const Pages& c, int bits, int d, int batch, int kv_heads, int rows, void* k, void* v, const int64_t (&strides)[3], const ChunkHead& head, cudaStream_t stream) {
    ReadParams p = {};
    p.c = c;
    p.batch = batch;
    p.rows = rows;
    p.head = head;
    p.k = static_cast<__nv_bfloat16*>(k);
    p.v = static_cast<__nv_bfloat16*>(v);
    for (int i = 0; i < 3; ++i) p.ks[i] = p.vs[i] = strides[i];
    return launch_read(p, bits, d, kv_heads, stream);
}

}  // namespace ktt

using namespace ktt;

namespace {

// The checks of an append and its parameters; go: whether there is anything to launch.
template <typename Params>
int fill(Params& p, const ktt_b200_append_args* a, bool& go) {
    go = false;
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: null arguments");
    if (const char* why = pages_of(p.c, a->cache, a->d)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_append: %s", why);
    if (a->batch < 1 || a->rows < 0 || a->heads < 0) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: sizes must be positive");
    if (a->heads > 32768) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_append: at most 32768 heads");
    if (a->cos && (!a->sin || a->pairs < 1 || 2 * a->pairs > a->d || a->table_rows < 1)) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: 1 to D / 2 pairs of columns turn, by two tables");
    }
    if (!a->cache.k || !a->cache.v || !a->cache.block_table || !a->cache.lengths || (a->heads && a->rows && (!a->q || !a->q_out)) || (a->rows && (!a->k || !a->v))) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: null pointer");
    }
    if (a->lengths_out && a->lengths_out < a->cache.lengths + a->batch && a->cache.lengths < a->lengths_out + a->batch) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: lengths_out must not overlap the lengths");
    }
    if (a->heads && a->rows && a->q == a->q_out) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: q_out must not overlap q");
    p.turn = {a->cos, a->sin, a->table_stride, a->table_rows, a->pairs, a->interleaved, 0};
    p.batch = a->batch;
    p.rows = a->rows;
    p.heads = a->heads;
    p.kv_heads = a->cache.kv_heads;
    p.tokens = a->cu_seqlens ? a->rows : static_cast<int64_t>(a->batch) * a->rows;
    if (p.tokens > (1ll << 31)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_append: at most 2^31 rows");
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
    p.k = static_cast<const __nv_bfloat16*>(a->k);
    p.v = static_cast<const __nv_bfloat16*>(a->v);
    uintptr_t low = reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v);
    if (a->heads) low |= reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_out);
    bool vec = (low & 15) == 0;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a->q_strides[i]; p.qos[i] = a->q_out_strides[i];
        p.ks[i] = a->k_strides[i]; p.vs[i] = a->v_strides[i];
        vec = vec && p.ks[i] % 8 == 0 && p.vs[i] % 8 == 0 && (!a->heads || (p.qs[i] % 8 == 0 && p.qos[i] % 8 == 0));
    }
    p.vec = vec;
    p.cu = a->cu_seqlens;
    p.lengths_out = a->lengths_out;
    go = p.tokens > 0 || p.lengths_out;
    return 0;
}

template <typename Params>
int launch(const Params& p, int bits, int d, cudaStream_t st) {
    if (bits == 16) return d == 64 ? launch_append<64, 16>(p, st) : launch_append<128, 16>(p, st);
    return d == 64 ? launch_append<64, 4>(p, st) : launch_append<128, 4>(p, st);
}

}  // namespace

extern "C" int ktt_b200_paged_append(const ktt_b200_append_args* a, void* stream) {
    AppendParams p = {};
    bool go;
    if (int rc = fill(p, a, go)) return rc;
    return go ? launch(p, a->cache.bits, a->d, static_cast<cudaStream_t>(stream)) : 0;
}

extern "C" int ktt_b200_paged_append_at(const ktt_b200_append_at_args* x, void* stream) { return ktt_b200_paged_append_granted(x, nullptr, stream); }

extern "C" int ktt_b200_paged_append_granted(const ktt_b200_append_at_args* x, const int32_t* granted, void* stream) {
    if (!x) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: null arguments");
    const ktt_b200_append_args* a = &x->base;
    AppendGrantedParams p = {};
    bool go;
    if (int rc = fill(p, a, go)) return rc;
    if (granted && p.lengths_out && granted < p.lengths_out + a->batch && p.lengths_out < granted + a->batch) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: lengths_out must not overlap granted");
    }
    if (!go) return 0;
    p.granted = granted;
    p.axes.axes = 1;
    if (x->positions.positions && a->cos) {
        if (const char* why = axes_of(p.axes, x->positions, a->pairs)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_append: %s", why);
        p.positions = {x->positions.positions, x->positions.positions_are_64, {x->positions.strides[0], x->positions.strides[1], x->positions.strides[2]}};
    }
    Bounds bounds = {};
    if (x->bounds) {
        if (const char* why = bounds_of(bounds, x->bounds, x->bounds_strides, p.c, p.kv_heads, a->d)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_append: %s", why);
        if (a->batch > 65535) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_append: at most 65535 sequences with bounds");
    }
    // One new key of each sequence goes into its page's bounds as it passes; of several, those of a page meet in a launch behind this one, which
    // reads them back.
    const bool passing = !a->cu_seqlens && a->rows == 1;
    if (passing) p.bounds = bounds;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto behind = [&](bool go) {
        return bounds.at && !passing ? keep_bounds(p.c, a->cache.bits, a->d, p.kv_heads, bounds, a->batch, a->rows, a->cu_seqlens, granted, go, st) : 0;
    };
    if (int rc = behind(false)) return rc;   // (refused before anything is launched)
    if (int rc = granted ? launch(p, a->cache.bits, a->d, st) : launch(static_cast<const AppendAtParams&>(p), a->cache.bits, a->d, st)) return rc;
    return behind(true);
}

extern "C" int ktt_b200_paged_read(const ktt_b200_read_args* a, void* stream) {
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_read: null arguments");
    ReadParams p = {};
    if (const char* why = pages_of(p.c, a->cache, a->d)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_read: %s", why);
    if (a->batch < 1 || a->rows < 0) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_read: sizes must be positive");
    if (a->batch > 65535) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_read: at most 65535 sequences");
    if (a->rows == 0) return 0;
    if (!a->cache.k || !a->cache.v || !a->cache.block_table || !a->cache.lengths || !a->k_out || !a->v_out) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_read: null pointer");
    }
    uintptr_t low = reinterpret_cast<uintptr_t>(a->k_out) | reinterpret_cast<uintptr_t>(a->v_out);
    p.batch = a->batch;
    p.rows = a->rows;
    p.k = static_cast<__nv_bfloat16*>(a->k_out);
    p.v = static_cast<__nv_bfloat16*>(a->v_out);
    for (int i = 0; i < 3; ++i) {
        p.ks[i] = a->k_strides[i]; p.vs[i] = a->v_strides[i];
        low |= static_cast<uintptr_t>((p.ks[i] | p.vs[i]) * 2);
    }
    if (low & 15) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_read: outputs must be 16-byte aligned in every row");
    return launch_read(p, a->cache.bits, a->d, a->cache.kv_heads, static_cast<cudaStream_t>(stream));
}
