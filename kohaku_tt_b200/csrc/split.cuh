// Attention of a few queries over long caches, cut into equal shares: the (batch, kv head) pairs are laid end to end,
// a pair of n tiles of keys as n + kPairCost units, and CTA c owns units [c * upc, (c + 1) * upc). What the kernels of
// that kind (decode.cu, paged_attention.cu) have in common. `Params` has `batch` and `kv_heads`.
#pragma once
#include "common.cuh"

namespace ktt {

// prefix[b] = sum_{b' < b} (tiles of b' + kPairCost) for b in [0, batch], by one CTA of kThreads threads: the units of
// one kv head's pass over batch entries [0, b). lens[b] = length(b); a sequence has one tile at least.
template <int kThreads, int kMaxBatch, int kTile, int kPairCost, typename Length>
__device__ __forceinline__ void scan_lengths(int batch, Length length, int* prefix, int* lens, int* warp_sums) {
    constexpr int kPer = kMaxBatch / kThreads;  // consecutive entries per thread
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int tiles[kPer], mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = threadIdx.x * kPer + i;
        const int len = b < batch ? length(b) : 0;
        if (b < batch) lens[b] = len;
        tiles[i] = b < batch ? max((len + kTile - 1) / kTile, 1) + kPairCost : 0;
        mine += tiles[i];
    }
    int x = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int before = x - mine;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = threadIdx.x * kPer + i;
        if (b <= batch) prefix[b] = before;
        before += tiles[i];
    }
    if (threadIdx.x == kThreads - 1 && batch == kMaxBatch) prefix[kMaxBatch] = before;
    __syncthreads();
}

// Position inside the end-to-end sequence of (batch, kv head) pairs.
struct Cursor {
    int b, hk, tile, ntiles, len;
};

// Largest b with kv_heads * prefix[b] <= unit.
template <typename Params>
__device__ __forceinline__ int entry_of(const Params& p, const int* prefix, int unit) {
    int lo = 0, hi = p.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.kv_heads * prefix[mid] <= unit) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Tiles whose unit lies before `unit` (a pair's units: its tiles, then kPairCost units that
// belong to its last tile).
template <int kPairCost, typename Params>
__device__ __forceinline__ int tiles_before(const Params& p, const int* prefix, int unit) {
    const int b = entry_of(p, prefix, unit);
    const int span = prefix[b + 1] - prefix[b], ntiles = span - kPairCost;
    const int rem = unit - p.kv_heads * prefix[b];
    const int hk = rem / span, pos = rem % span;
    return p.kv_heads * (prefix[b] - kPairCost * b) + hk * ntiles + min(pos, ntiles);
}

// The first tile at or after `unit`.
template <int kPairCost, typename Params>
__device__ __forceinline__ void cursor_seek(const Params& p, const int* prefix, const int* lens, Cursor& c, int unit) {
    const int b = entry_of(p, prefix, unit);
    const int span = prefix[b + 1] - prefix[b];
    c.b = b;
    c.ntiles = span - kPairCost;
    c.len = lens[b];
    const int rem = unit - p.kv_heads * prefix[b];
    c.hk = rem / span;
    c.tile = rem % span;
    if (c.tile >= c.ntiles) {   // inside a pair's closing units: the next pair's first tile
        c.tile = 0;
        if (++c.hk == p.kv_heads) {
            c.hk = 0;
            if (++c.b < p.batch) {
                c.len = lens[c.b];
                c.ntiles = prefix[c.b + 1] - prefix[c.b] - kPairCost;
            }
        }
    }
}

template <int kPairCost, typename Params>
__device__ __forceinline__ void cursor_next(const Params& p, const int* prefix, const int* lens, Cursor& c) {
    if (++c.tile < c.ntiles) return;
    c.tile = 0;
    if (++c.hk < p.kv_heads) return;
    c.hk = 0;
    if (++c.b < p.batch) {
        c.len = lens[c.b];
        c.ntiles = prefix[c.b + 1] - prefix[c.b] - kPairCost;
    }
}

// The CTAs of a cluster meet; what each wrote to its shared memory before is visible to the others after.
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of `addr` (shared memory of this CTA) in CTA `rank` of the cluster, and loads from there.
__device__ __forceinline__ uint32_t in_rank(uint32_t addr, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

}  // namespace ktt
