// Rotary positions: the tables of cosines and sines, and the rotation of queries and keys (its gradient too).
#include <cmath>
#include <type_traits>

#include "rotary.cuh"

namespace ktt {

const char* axes_of(PairAxes& x, const ktt_b200_axes& given, int pairs) {
    if (given.axes < 1 || given.axes > kMaxAxes) return "positions have 1 to 4 axes";
    if (!given.positions || (!given.of_pair && given.axes > 1)) return "null pointer";
    x.axes = given.axes;
    for (int i = 0; i < pairs && given.of_pair; ++i) {
        if (given.of_pair[i] >= given.axes) return "a pair's axis must be one of the positions'";
        x.of[i >> 4] |= static_cast<uint32_t>(given.of_pair[i]) << (2 * (i & 15));
    }
    return nullptr;
}

namespace {

// ---- tables ----------------------------------------------------------------------------------
//
// cos, sin[p][i] = scale * (cos, sin)(p f_i). What a position of 10^5 at f = 1 turns by is no 32-bit matter: a pair's turn
// per position, f / 2 pi, is a whole number of 2^-64 turns, and its multiples modulo 2^64 lose nothing, whole turns fall off
// by themselves, and the quarter turn nearest to what is left stands in two bits. The rest, at most an eighth of a turn, is
// read from the bits as a mantissa of 23 and a remainder of 23 more; sine and cosine of it are their Taylor sums to the 9th and
// 10th power (the next terms are 2^-29 and 2^-33 of the value).
// That is some 80 instructions a pair, so a block takes it for the first of every kSteps of its positions and for the first
// kSteps alone, each as an fp32 value and what it leaves, and the others by
//     cos(a + b) = cos a cos b - sin a sin b,   sin(a + b) = sin a cos b + cos a sin b
// with the leavings' products: 12 operations, two roundings that count (the larger product's sum and the result's), where each
// position by itself took 60 and had three. Bound: the writing of the tables, in 16-byte pieces.
constexpr int kMaxPairs = 256;
// Pairs in all from which a block has 256 positions, not 64. us for 64 and 256: 4,096 x 64 3.3 and 5.5, 16,384 x 64 4.3 and 5.5,
// 32,768 x 64 6.5 and 5.7, 131,072 x 64 17.2 and 14.0 (two fills of the same 67 MB 11.1; every position by itself 20.2).
constexpr int64_t kLargeTable = 3 << 19;
struct TableParams {
    float* cos;
    float* sin;
    int64_t positions;
    int pairs;
    float scale, scale_rest;   // as fp32, and what that leaves
    int vec;                   // both tables start at 16 bytes
    uint64_t turns[kMaxPairs];   // f_i / 2 pi in 2^-64 turns
};

constexpr int kTablePairs = 64;   // of a block

// An fp32 value and what it leaves of a number.
struct Two {
    float hi, lo;
};
__device__ __forceinline__ Two two_of(float hi, float lo) {
    const float s = hi + lo;
    return {s, lo - (s - hi)};
}
__device__ __forceinline__ Two times(const Two& x, const Two& y) {
    const float h = x.hi * y.hi;
    return {h, fmaf(x.hi, y.hi, -h) + fmaf(x.lo, y.hi, x.hi * y.lo)};
}

// Cosine and sine of an angle of `turn` 2^-64 turns.
__device__ __forceinline__ void cos_sin(uint64_t turn, Two& c, Two& s) {
    const uint64_t z = turn + (1ull << 61);
    const uint32_t quarter = static_cast<uint32_t>(z >> 62);
    // The rest and 2^61, as 62 bits: the upper 23 and the next 23 as fractions.
    const float hi = __uint_as_float(0x3f800000u | (static_cast<uint32_t>(z >> 39) & 0x7fffffu)) - 1.5f;
    const float lo = __uint_as_float(0x3f800000u | (static_cast<uint32_t>(z >> 16) & 0x7fffffu)) - 1.f;
    // Radians: a quarter turn times hi, rounded, and what the product and lo leave.
    constexpr float kQuarter = 1.57079632679489662f, kQuarterRest = -4.37113882867379e-8f;
    const float x = hi * kQuarter;
    const float rest = fmaf(lo, kQuarter * 0x1p-23f, fmaf(hi, kQuarterRest, fmaf(hi, kQuarter, -x)));
    const float q = x * x, more = fmaf(x, x, -q);   // (x^2 and its rounding)
    const float st = x * q * fmaf(q, fmaf(q, fmaf(q, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6);
    const float ct = q * q * fmaf(q, fmaf(q, fmaf(q, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24);
    const float half = fmaf(q, -0.5f, 1.f), left = (1.f - half) - 0.5f * q;
    const Two sr = two_of(x, fmaf(rest, half, st)), cr = two_of(half, left + fmaf(more, -0.5f, fmaf(-rest, x, ct)));
    c = quarter & 1 ? sr : cr;
    s = quarter & 1 ? cr : sr;
    if (quarter == 1 || quarter == 2) c = {-c.hi, -c.lo};
    if (quarter & 2) s = {-s.hi, -s.lo};
}

// The angles of a block, by pair: those of positions first + kSteps u, times the scale, then those of 0, 1, .. kSteps - 1.
template <int kSteps>
struct TableShared {
    alignas(16) float ch[2 * kSteps][kTablePairs], cl[2 * kSteps][kTablePairs], sh[2 * kSteps][kTablePairs], sl[2 * kSteps][kTablePairs];
};

template <int kVec>
__device__ __forceinline__ void table_load(float (&to)[kVec], const float* from) {
    if constexpr (kVec == 4) {
        const float4 x = *reinterpret_cast<const float4*>(from);
        to[0] = x.x; to[1] = x.y; to[2] = x.z; to[3] = x.w;
    } else if constexpr (kVec == 2) {
        const float2 x = *reinterpret_cast<const float2*>(from);
        to[0] = x.x; to[1] = x.y;
    } else {
        to[0] = *from;
    }
}
template <int kVec>
__device__ __forceinline__ void table_store(float* to, const float (&x)[kVec]) {
    if constexpr (kVec == 4) *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
    else if constexpr (kVec == 2) *reinterpret_cast<float2*>(to) = make_float2(x[0], x[1]);
    else *to = x[0];
}

// A block has kSteps * kSteps positions of up to 64 pairs; a thread kVec pairs of every position first + kSteps u + w of some
// of its (u, w).
template <int kSteps, int kVec>
__global__ void __launch_bounds__(256) rotary_table_kernel(const __grid_constant__ TableParams p) {
    __shared__ TableShared<kSteps> sm;
    __shared__ uint64_t turns[kTablePairs];   // (a warp's threads want different ones: no matter for constant memory)
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kSteps * kSteps);
    const int rows = static_cast<int>(p.positions - first < kSteps * kSteps ? p.positions - first : kSteps * kSteps);
    const int pair0 = blockIdx.y * kTablePairs, pairs = min(p.pairs - pair0, kTablePairs);
    if (threadIdx.x < pairs) turns[threadIdx.x] = p.turns[pair0 + threadIdx.x];
    __syncthreads();
    for (int at = threadIdx.x; at < 2 * kSteps * kTablePairs; at += 256) {
        const int row = at / kTablePairs, i = at % kTablePairs;
        if (i >= pairs) continue;
        const uint64_t pos = row < kSteps ? first + row * kSteps : row - kSteps;
        Two c, s;
        cos_sin(pos * turns[i], c, s);
        if (row < kSteps) {
            const Two scale = {p.scale, p.scale_rest};
            c = times(c, scale);
            s = times(s, scale);
        }
        sm.ch[row][i] = c.hi;
        sm.cl[row][i] = c.lo;
        sm.sh[row][i] = s.hi;
        sm.sl[row][i] = s.lo;
    }
    __syncthreads();
    const int chunks = pairs / kVec;   // (kVec divides the pairs)
    // Threads that share a u take every `parts`-th w.
    const int parts = min(max(256 / (kSteps * chunks), 1), kSteps);
    for (int at = threadIdx.x; at < kSteps * parts * chunks; at += 256) {
        const int group = at / chunks, i = (at - group * chunks) * kVec, u = group / parts;
        float ch[kVec], cl[kVec], sh[kVec], sl[kVec];
        table_load(ch, &sm.ch[u][i]);
        table_load(cl, &sm.cl[u][i]);
        table_load(sh, &sm.sh[u][i]);
        table_load(sl, &sm.sl[u][i]);
#pragma unroll 2
        for (int w = group - u * parts; w < kSteps; w += parts) {
            const int row = u * kSteps + w;
            if (row >= rows) break;
            float dh[kVec], dl[kVec], th[kVec], tl[kVec], c[kVec], s[kVec];
            table_load(dh, &sm.ch[kSteps + w][i]);
            table_load(dl, &sm.cl[kSteps + w][i]);
            table_load(th, &sm.sh[kSteps + w][i]);
            table_load(tl, &sm.sl[kSteps + w][i]);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const float cr = fmaf(ch[e], dl[e], fmaf(cl[e], dh[e], fmaf(-sh[e], tl[e], -sl[e] * th[e])));
                const float sr = fmaf(sh[e], dl[e], fmaf(sl[e], dh[e], fmaf(ch[e], tl[e], cl[e] * th[e])));
                c[e] = fmaf(ch[e], dh[e], fmaf(-sh[e], th[e], cr));
                s[e] = fmaf(sh[e], dh[e], fmaf(ch[e], th[e], sr));
            }
            const int64_t to = (first + row) * p.pairs + pair0 + i;
            table_store(p.cos + to, c);
            table_store(p.sin + to, s);
        }
    }
}

// ---- rotation --------------------------------------------------------------------------------

struct RotaryParams {
    Turn turn;
    const void* x[2];        // queries, keys
    void* y[2];
    int64_t xs[2][3], ys[2][3];   // (batch, head, row) strides
    int heads[2], groups[2];      // heads, and how many blocks of kHeads that is
    int64_t tokens;          // of all batch entries
    int rows;                // of one
    int d;
    Placed positions;        // none: the row
    int vec;                 // rows may be read and written in 16-byte pieces
    int loops;               // groups of kHeads that a thread goes through
};
struct RotaryAxesParams : RotaryParams {
    PairAxes axes;
};

// A thread turns eight columns of kHeads heads of one token, and of the next kHeads, `loops` times: the table is read once for all of them. A thread
// reads its partner columns too (its neighbour in the block brings the same line, so they come from L1).
template <typename T, bool kFast, int kHeads, typename Params>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ Params p) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const int col = threadIdx.x * 8;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (n >= p.tokens) return;
    const int which = static_cast<int>(blockIdx.y) >= p.groups[0];
    const int loops = kHeads == 1 ? 1 : p.loops;
    int h0 = (static_cast<int>(blockIdx.y) - (which ? p.groups[0] : 0)) * (kHeads * loops);
    const uint32_t entry = static_cast<uint32_t>(n) / static_cast<uint32_t>(p.rows);   // (2^31 tokens at most)
    const int64_t b = entry, r = static_cast<uint32_t>(n) - entry * static_cast<uint32_t>(p.rows);
    const T* x = static_cast<const T*>(p.x[which]) + b * p.xs[which][0] + r * p.xs[which][2];
    T* y = static_cast<T*>(p.y[which]) + b * p.ys[which][0] + r * p.ys[which][2];
    const int left = p.d - col, heads = p.heads[which], half = p.turn.half;
    const int partner = p.turn.interleaved || col >= 2 * half ? -1 : col < half ? col + half : col - half;
    Eight<T> v[kHeads], o[kHeads];
    auto rows_of = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const T* row = x + static_cast<int64_t>(min(h0 + i, heads - 1)) * p.xs[which][1];
            if (kFast || p.vec) v[i].load(row + col);
            else v[i].load_some(row + col, left);
            if (kFast && partner >= 0) o[i].load(row + partner);
        }
    };
    if (kHeads == 1) rows_of(h0);   // (requested before the positions, which the table's rows wait for)
    Turned<kFast> turned;
    if constexpr (std::is_same_v<Params, RotaryAxesParams>) turned.load(p.turn, p.axes, p.positions.all(p.axes.axes, b, r), col);
    else turned.load(p.turn, p.positions.at ? p.positions.get(0, b, r) : r, col);
    for (int loop = 0; loop < loops && h0 < heads; ++loop, h0 += kHeads) {
        if (kHeads > 1) rows_of(h0);
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = h0 + i;
            if (h >= heads) break;
            turned.apply(p.turn, v[i], o[i], x + h * p.xs[which][1], col);
            T* to = y + h * p.ys[which][1] + col;
            if (kFast || p.vec) v[i].store(to);
            else v[i].store_some(to, left);
        }
    }
}

// Half layout: a thread has eight pairs, both columns of each, so that no column is read twice and the table's entries are those of 16 columns; behind
// the pairs it copies 16 columns.
template <typename T, typename Params>
__global__ void __launch_bounds__(256) rotary_pairs_kernel(const __grid_constant__ Params p) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const int half = p.turn.half, pair = threadIdx.x * 8;
    const bool turns = pair < half;
    const int col = turns ? pair : 2 * pair, other = turns ? pair + half : 2 * pair + 8;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (n >= p.tokens) return;
    const int which = static_cast<int>(blockIdx.y) >= p.groups[0];
    const uint32_t entry = static_cast<uint32_t>(n) / static_cast<uint32_t>(p.rows);   // (2^31 tokens at most)
    const int64_t b = entry, r = static_cast<uint32_t>(n) - entry * static_cast<uint32_t>(p.rows);
    Turned<true> turned;   // (of the first columns; the others' sines have the other sign)
    if (turns) {
        if constexpr (std::is_same_v<Params, RotaryAxesParams>) turned.load(p.turn, p.axes, p.positions.all(p.axes.axes, b, r), col);
        else turned.load(p.turn, p.positions.at ? p.positions.get(0, b, r) : r, col);
    }
    const T* x = static_cast<const T*>(p.x[which]) + b * p.xs[which][0] + r * p.xs[which][2];
    T* y = static_cast<T*>(p.y[which]) + b * p.ys[which][0] + r * p.ys[which][2];
    constexpr int kHeads = 4;
    const int heads = p.heads[which];
    int h0 = (static_cast<int>(blockIdx.y) - (which ? p.groups[0] : 0)) * (kHeads * p.loops);
    for (int loop = 0; loop < p.loops && h0 < heads; ++loop, h0 += kHeads) {
        Eight<T> lo[kHeads], hi[kHeads];
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const T* row = x + static_cast<int64_t>(min(h0 + j, heads - 1)) * p.xs[which][1];
            lo[j].load(row + col);
            hi[j].load(row + other);
        }
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            if (h0 + j >= heads) break;
            if (turns) turned.both(lo[j], hi[j]);
            T* to = y + (h0 + j) * p.ys[which][1];
            lo[j].store(to + col);
            hi[j].store(to + other);
        }
    }
}

constexpr int64_t kManyThreads = 4 * 148 * 2048;

template <typename T, typename Params>
int launch_rotary(const Params& given, cudaStream_t stream) {
    Params p = given;
    const bool fast = p.vec && turn_is_fast(p.turn);
    constexpr bool kAxes = std::is_same_v<Params, RotaryAxesParams>;
    auto go = [&](auto kernel, int columns, int per) {   // of a thread
        const int x = (p.d + columns - 1) / columns, y = 256 / x > 0 ? 256 / x : 1;
        for (int i = 0; i < 2; ++i) p.groups[i] = (p.heads[i] + per - 1) / per;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>((p.tokens + y - 1) / y), static_cast<unsigned>(p.groups[0] + p.groups[1]));
        cfg.blockDim = dim3(static_cast<unsigned>(x), static_cast<unsigned>(y));
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return check_cuda(cudaLaunchKernelEx(&cfg, kernel, p), "rotary launch");
    };
    // Half layout: 16 columns and four heads to a thread as soon as that makes some 2^15 threads (one axis: 2^16), more heads one after another as
    // there are more. us for the pairs' kernel and the other, bf16, three axes taking turns: 512 rows, 32 heads over 8, D 128: 5.1 and 8.6; 2,048:
    // 8.2 and 11.0; 2,048 of 14 over 2, D 64: 5.3 and 6.4, with one axis 4.2 and 3.8; 77 of them 3.5 and 2.9. One, two and four
    // times four heads, three axes (one): 2,048 rows, 32 over 8, D 128: 8.2, 7.5, 11.5 (6.5, 6.4, 10.6); 8,192: 31.6, 30.3, 30.5 (28.0, 28.2, 29.0);
    // 65,536 of 16 + 16: 207, 170, 165 (182, 161, 163; a copy of the same bytes 165; the other kernel 264 and 215).
    p.loops = 1;
    if (fast && !p.turn.interleaved && p.d % 16 == 0) {
        const int64_t threads = p.tokens * (p.d / 16) * ((p.heads[0] + 3) / 4 + (p.heads[1] + 3) / 4);
        if (threads >= (kAxes ? 1 << 15 : 1 << 16)) {
            p.loops = threads < 1 << 19 ? 1 : (kAxes && threads >= 1 << 21 ? 4 : 2);
            return go(rotary_pairs_kernel<T, Params>, 16, 4 * p.loops);
        }
    }
    // Else four heads to a thread once that fills the GPU: a row's position and table entries are read once for all of them; and for the next four,
    // and as many again. 65,536 rows, 16 + 16 heads, D 128, neighbours, three axes (one), us for 4, 8 and 16 heads: 249, 191, 168 (211, 175, 162); 2,048 of
    // 32 over 8: 9.6, 8.1, 9.7 (7.1, 6.7, 8.8).
    // Where the pairs of the half layout are no multiple of 8 a thread goes for its columns' partners one by one, and reads the tables so:
    // 65,536 rows, 16 + 16 heads, D 128, 20 columns: 569, 406, 325 (443, 345, 296).
    const int64_t threads = p.tokens * ((p.d + 7) / 8) * (p.heads[0] + p.heads[1]);
    if (threads >= kManyThreads) {
        p.loops = threads < 1 << 21 ? 2 : 4;
        if (fast) return go(rotary_kernel<T, true, 4, Params>, 8, 4 * p.loops);
        return go(rotary_kernel<T, false, 4, Params>, 8, 4 * p.loops);
    }
    if (fast) return go(rotary_kernel<T, true, 1, Params>, 8, 1);
    return go(rotary_kernel<T, false, 1, Params>, 8, 1);
}

}  // namespace
}  // namespace ktt

using namespace ktt;

extern "C" int ktt_b200_rotary_frequencies(double* f, double* scale, int32_t dim, double base, int32_t scaling, double factor, double original, double fast, double slow) {
    if (!f || !scale) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary_frequencies: null pointer");
    if (dim < 2 || dim % 2 || dim > 2 * kMaxPairs) return fail(KTT_B200_ERR_BAD_ARGUMENT, "dim must be even, from 2 to %d", 2 * kMaxPairs);
    if (scaling < 0 || scaling > 3) return fail(KTT_B200_ERR_BAD_ARGUMENT, "unknown scaling");
    if (!(base > 0) || !(factor > 0) || std::isinf(base) || std::isinf(factor)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "base and factor must be positive");
    if (scaling == 2) {
        if (dim < 4) return fail(KTT_B200_ERR_BAD_ARGUMENT, "scaling of the base needs two pairs");
        base *= std::pow(factor, static_cast<double>(dim) / (dim - 2));
    }
    if (scaling == 3 && (!(original >= 1) || !(fast > slow) || !(factor >= 1))) {
        return fail(KTT_B200_ERR_BAD_ARGUMENT, "scaling by parts needs the original context's length, fast > slow and a factor of 1 or more");
    }
    for (int i = 0; i < dim / 2; ++i) {
        f[i] = std::pow(base, -2.0 * i / dim);
        if (scaling == 1) f[i] /= factor;
        if (scaling == 3) {
            double keep = (original * f[i] * 0.15915494309189533577 - slow) / (fast - slow);
            keep = keep < 0 ? 0 : (keep > 1 ? 1 : keep);
            f[i] = (1 - keep) * f[i] / factor + keep * f[i];
        }
    }
    *scale = scaling == 3 ? 0.1 * std::log(factor) + 1.0 : 1.0;
    return 0;
}

extern "C" int ktt_b200_rotary_table(float* cos, float* sin, int64_t positions, int32_t pairs, const double* frequencies, double scale, void* stream) {
    if (!cos || !sin || !frequencies) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary_table: null pointer");
    if (positions < 1 || pairs < 1 || pairs > kMaxPairs) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary_table: 1 or more positions and 1 to %d pairs", kMaxPairs);
    if (positions > (1ll << 31)) return fail(KTT_B200_ERR_UNSUPPORTED, "rotary_table: at most 2^31 positions");
    if (!std::isfinite(static_cast<float>(scale))) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary_table: the scale must be finite");
    TableParams p = {};
    p.cos = cos;
    p.sin = sin;
    p.positions = positions;
    p.pairs = pairs;
    p.scale = static_cast<float>(scale);
    p.scale_rest = static_cast<float>(scale - p.scale);
    for (int i = 0; i < pairs; ++i) {
        if (!std::isfinite(frequencies[i])) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary_table: frequencies must be finite");
        const long double turns = frequencies[i] * 0.159154943091895335768883763372514362L;   // f / 2 pi
        const long double part = turns - std::floor(turns);
        p.turns[i] = part < 1 ? static_cast<uint64_t>(part * 0x1p64L) : 0;   // (1: a frequency just below 0)
    }
    p.vec = ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15) == 0;
    auto go = [&](auto kernel, int rows) {
        const dim3 grid(static_cast<unsigned>((positions + rows - 1) / rows), static_cast<unsigned>((pairs + kTablePairs - 1) / kTablePairs));
        kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    };
    const int vec = !p.vec ? 1 : pairs % 4 == 0 ? 4 : pairs % 2 == 0 ? 2 : 1;
    if (positions * pairs >= kLargeTable) go(vec == 4 ? rotary_table_kernel<16, 4> : vec == 2 ? rotary_table_kernel<16, 2> : rotary_table_kernel<16, 1>, 256);
    else go(vec == 4 ? rotary_table_kernel<8, 4> : vec == 2 ? rotary_table_kernel<8, 2> : rotary_table_kernel<8, 1>, 64);
    return check_cuda(cudaGetLastError(), "rotary_table launch");
}

namespace {

// The checks of a rotation and its parameters; go: whether there is anything to launch.
template <typename Params>
int fill(Params& p, const ktt_b200_rotary_args* a, bool& go) {
    go = false;
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary: null arguments");
    if (a->batch < 0 || a->rows < 0 || a->heads < 1 || a->kv_heads < 0 || a->d < 1) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary: sizes must be positive");
    if (a->d > 1024) return fail(KTT_B200_ERR_UNSUPPORTED, "rotary: head dims above 1024 are not taken");
    if (a->pairs < 1 || 2 * a->pairs > a->d) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary: 1 to D / 2 pairs of columns turn");
    if (a->dtype < KTT_B200_MASK_BF16 || a->dtype > KTT_B200_MASK_F16) return fail(KTT_B200_ERR_UNSUPPORTED, "rotary: bf16, fp16 or fp32 operands");
    if (a->heads > 65535 - a->kv_heads) return fail(KTT_B200_ERR_UNSUPPORTED, "rotary: at most 65535 heads");
    const int64_t tokens = static_cast<int64_t>(a->batch) * a->rows;
    if (tokens == 0) return 0;
    if (tokens > (1ll << 31)) return fail(KTT_B200_ERR_UNSUPPORTED, "rotary: at most 2^31 tokens");
    if (!a->q || !a->q_out || !a->cos || !a->sin || (a->kv_heads && (!a->k || !a->k_out))) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary: null pointer");
    if (a->table_rows < 1) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary: the tables have no rows");
    if (a->q == a->q_out || (a->kv_heads && a->k == a->k_out)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary: outputs must not overlap inputs");
    p.turn = {a->cos, a->sin, a->table_stride, a->table_rows, a->pairs, a->interleaved, a->inverse};
    p.x[0] = a->q; p.x[1] = a->k;
    p.y[0] = a->q_out; p.y[1] = a->k_out;
    p.heads[0] = a->heads; p.heads[1] = a->kv_heads;
    const int size = a->dtype == KTT_B200_MASK_F32 ? 4 : 2, wide = 16 / size;
    uintptr_t low = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_out);
    if (a->kv_heads) low |= reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->k_out);
    bool vec = (low & 15) == 0 && a->d % 8 == 0;
    for (int i = 0; i < 3; ++i) {
        p.xs[0][i] = a->q_strides[i]; p.ys[0][i] = a->q_out_strides[i];
        p.xs[1][i] = a->k_strides[i]; p.ys[1][i] = a->k_out_strides[i];
        vec = vec && a->q_strides[i] % wide == 0 && a->q_out_strides[i] % wide == 0;
        if (a->kv_heads) vec = vec && a->k_strides[i] % wide == 0 && a->k_out_strides[i] % wide == 0;
    }
    p.tokens = tokens;
    p.rows = a->rows;
    p.d = a->d;
    p.positions = {a->positions, a->positions_are_64, {0, a->position_strides[0], a->position_strides[1]}};
    p.vec = vec;
    go = true;
    return 0;
}

template <typename Params>
int launch(const Params& p, int dtype, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == KTT_B200_MASK_F32) return launch_rotary<float>(p, st);
    if (dtype == KTT_B200_MASK_F16) return launch_rotary<__half>(p, st);
    return launch_rotary<__nv_bfloat16>(p, st);
}

}  // namespace

extern "C" int ktt_b200_rotary(const ktt_b200_rotary_args* a, void* stream) {
    RotaryParams p = {};
    bool go;
    if (int rc = fill(p, a, go)) return rc;
    return go ? launch(p, a->dtype, stream) : 0;
}

extern "C" int ktt_b200_rotary_axes(const ktt_b200_rotary_args* a, const ktt_b200_axes* axes, void* stream) {
    RotaryAxesParams p = {};
    bool go;
    if (int rc = fill(p, a, go)) return rc;
    if (!go) return 0;
    if (!axes) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary: null axes");
    if (const char* why = axes_of(p.axes, *axes, a->pairs)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "rotary: %s", why);
    p.positions = {axes->positions, axes->positions_are_64, {axes->strides[0], axes->strides[1], axes->strides[2]}};
    return launch(p, a->dtype, stream);
}
