// Rotary positions: the tables of cosines and sines, and the rotation of queries and keys (its gradient too).
#include <cmath>

#include "rotary.cuh"

namespace ktt {
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
    const void* positions;   // null: the row
    int wide_positions;      // int64, else int32
    int64_t ps[2];           // (batch, row) strides
    int vec;                 // rows may be read and written in 16-byte pieces
};

// A thread turns eight columns of kHeads heads of one token: the table is read once for all of them. A thread reads
// its partner columns too (its neighbour in the block brings the same line, so they come from L1).
template <typename T, bool kFast, int kHeads>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryParams p) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const int col = threadIdx.x * 8;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (n >= p.tokens) return;
    const int which = static_cast<int>(blockIdx.y) >= p.groups[0];
    const int h0 = (static_cast<int>(blockIdx.y) - (which ? p.groups[0] : 0)) * kHeads;
    const uint32_t entry = static_cast<uint32_t>(n) / static_cast<uint32_t>(p.rows);   // (2^31 tokens at most)
    const int64_t b = entry, r = static_cast<uint32_t>(n) - entry * static_cast<uint32_t>(p.rows);
    int64_t pos = r;
    if (p.positions) {
        const int64_t at = b * p.ps[0] + r * p.ps[1];
        pos = p.wide_positions ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
    }
    Turned<kFast> turned;
    turned.load(p.turn, pos, col);
    const T* x = static_cast<const T*>(p.x[which]) + b * p.xs[which][0] + r * p.xs[which][2];
    T* y = static_cast<T*>(p.y[which]) + b * p.ys[which][0] + r * p.ys[which][2];
    const int left = p.d - col;
    Eight<T> v[kHeads], o[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const T* row = x + static_cast<int64_t>(min(h0 + i, p.heads[which] - 1)) * p.xs[which][1];
        if (kFast || p.vec) v[i].load(row + col);
        else v[i].load_some(row + col, left);
        if (kFast && turned.partner >= 0) o[i].load(row + turned.partner);
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int h = h0 + i;
        if (h >= p.heads[which]) break;
        turned.apply(p.turn, v[i], o[i], x + h * p.xs[which][1], col);
        T* to = y + h * p.ys[which][1] + col;
        if (kFast || p.vec) v[i].store(to);
        else v[i].store_some(to, left);
    }
}

constexpr int64_t kManyThreads = 4 * 148 * 2048;

template <typename T>
int launch_rotary(const RotaryParams& given, cudaStream_t stream) {
    RotaryParams p = given;
    const int chunks = (p.d + 7) / 8;
    const int tokens_per_block = 256 / chunks > 0 ? 256 / chunks : 1;
    const int64_t blocks = (p.tokens + tokens_per_block - 1) / tokens_per_block;
    const bool fast = p.vec && turn_is_fast(p.turn);
    auto go = [&](auto kernel, int per) {
        for (int i = 0; i < 2; ++i) p.groups[i] = (p.heads[i] + per - 1) / per;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(p.groups[0] + p.groups[1]));
        cfg.blockDim = dim3(static_cast<unsigned>(chunks), static_cast<unsigned>(tokens_per_block));
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return check_cuda(cudaLaunchKernelEx(&cfg, kernel, p), "rotary launch");
    };
    // Four heads to a thread once that fills the GPU: a row's position and table entries are read once for all of them.
    // 4 x 4,096 tokens, 32 heads over 8, D 128, bf16, forward and gradient, us for 1 and 4 heads: 671 and 400. (Of the latter's
    // bytes 92 to 95 % of a copy's rate: forward alone, 16 x 4,096 tokens, 16 + 16 heads, 175.7 us, 6.1 TB/s.)
    // Where the pairs of the half layout are no multiple of 8 a thread goes for its columns' partners one by one, and reads the tables so:
    // 4 x 16 heads x 4,096, D 128, bf16, all columns turning 25.1, 20 or 40 of them 38.6; neighbours 24.3, and 26.3 with 20 columns.
    if (p.tokens * chunks * (p.heads[0] + p.heads[1]) >= kManyThreads) {
        if (fast) return go(rotary_kernel<T, true, 4>, 4);
        return go(rotary_kernel<T, false, 4>, 4);
    }
    if (fast) return go(rotary_kernel<T, true, 1>, 1);
    return go(rotary_kernel<T, false, 1>, 1);
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

extern "C" int ktt_b200_rotary(const ktt_b200_rotary_args* a, void* stream) {
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
    RotaryParams p = {};
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
    p.positions = a->positions;
    p.wide_positions = a->positions_are_64;
    p.ps[0] = a->position_strides[0]; p.ps[1] = a->position_strides[1];
    p.vec = vec;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->dtype == KTT_B200_MASK_F32) return launch_rotary<float>(p, st);
    if (a->dtype == KTT_B200_MASK_F16) return launch_rotary<__half>(p, st);
    return launch_rotary<__nv_bfloat16>(p, st);
}
