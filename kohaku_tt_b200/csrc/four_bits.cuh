// Codes of 4 bits as the bf16 values they stand for.
#pragma once
#include "paged.cuh"
#include "rotary.cuh"

namespace ktt {

// What eight codes are worth: bf16 products and sums of pairs, rounded once. (An fp32 sum rounded to bf16 would be the same but where the
// least value is under 2^-19 of the step: the sum then drops it, and a product that lies halfway between two bf16 values goes to the even one
// instead of to the side that the least value is on.)
__device__ __forceinline__ Eight<__nv_bfloat16> of_four_bits(uint32_t word, uint32_t pair) {
    const __nv_bfloat162 ends = *reinterpret_cast<const __nv_bfloat162*>(&pair), step = __low2bfloat162(ends), least = __high2bfloat162(ends);
    const __nv_bfloat162 zero = __float2bfloat162_rn(128.f);
    Eight<__nv_bfloat16> x;
    __nv_bfloat162* to = reinterpret_cast<__nv_bfloat162*>(x.raw);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const uint32_t two = ((word >> (4 * n)) & 0x000f000fu) | 0x43004300u;   // two codes as bf16 128 + c
        to[n] = __hfma2(step, __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&two), zero), least);
    }
    return x;
}

// Bounds of pages: the least and the largest value of each channel over a page's keys, bf16 [pages][kv heads][2][D].
struct Bounds {
    __nv_bfloat16* at;       // null: none are kept
    int64_t stride[3];       // (page, head, edge) in elements
    __device__ __forceinline__ __nv_bfloat16* edge(int64_t page, int head, int which) const { return at + page * stride[0] + head * stride[1] + which * stride[2]; }
};

// Eight channels of both edges with eight more channels of keys between them. A NaN stays.
struct Edges {
    Eight<__nv_bfloat16> lo, hi;
    __device__ __forceinline__ void with(const Eight<__nv_bfloat16>& least, const Eight<__nv_bfloat16>& most) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __nv_bfloat162 *l = reinterpret_cast<__nv_bfloat162*>(lo.raw) + i, *h = reinterpret_cast<__nv_bfloat162*>(hi.raw) + i;
            *l = __hmin2_nan(*l, reinterpret_cast<const __nv_bfloat162*>(least.raw)[i]);
            *h = __hmax2_nan(*h, reinterpret_cast<const __nv_bfloat162*>(most.raw)[i]);
        }
    }
};

// How many of its new rows a sequence takes.
__device__ __forceinline__ int64_t granted_to(const int32_t* granted, int b) { return max(granted[b], 0); }

// The bounds of the pages that keys of an append lie in (select.cu): those of sequence b from lengths[b] on, `rows` of each, or packed, as many as are
// granted; without `launch` the checks alone.
int keep_bounds(const Pages& c, int bits, int d, int kv_heads, const Bounds& bounds, int batch, int64_t rows, const int32_t* cu, const int32_t* granted, bool launch,
                cudaStream_t stream);
// Those of the pages that sequences are cut in, of their first kept[b] keys; without `launch` the checks alone.
int cut_bounds(const ktt_b200_bounds_args* a, const int32_t* kept, bool launch, cudaStream_t stream);
// Bounds from an argument block's fields after their checks; null, or why not.
const char* bounds_of(Bounds& b, void* at, const int64_t (&strides)[3]);
// Those that are written, of a cache of head dim d.
const char* bounds_of(Bounds& b, void* at, const int64_t (&strides)[3], const Pages& c, int kv_heads, int d);

}  // namespace ktt
