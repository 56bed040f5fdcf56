// Block tables on the device: pages for the tokens that requests bring, with each token's place, and pages given back.
//
// With held_b = ceil(len_b / P) and wanted_b = ceil((len_b + added_b) / P) pages of P keys, sequence b takes wanted_b - held_b pages from the
// end of a list of free ones; before_b, the pages that sequences before it take, is an exclusive sum. So entry held_b + i of its row is
// free[count - 1 - before_b - i], a token's page is found without reading an entry that the same launch writes, and nothing waits for
// anything: every CTA sums up the lengths for itself. Bound: 12 bytes written for a token and 8 moved for a page, which is nothing; one trip for
// the lengths, a sum over the CTA and a search among the sequences are all that a call takes.
#include "four_bits.cuh"

namespace ktt {
namespace {

constexpr int kMaxSequences = 4096;   // their sums live in shared memory
constexpr int kThreads = 256;

struct ReserveParams {
    int batch, page_size;
    int64_t cap;             // keys that a row of the table has room for
    int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    const int32_t* added;
    const int32_t* free_pages;
    int64_t pool;
    const int32_t* count;
    int32_t* count_out;
    int64_t tokens;
    int32_t* cu;
    int32_t* positions;
    int64_t* slots;
    int32_t* granted;
};

__device__ __forceinline__ int clamped(int x, int64_t most) { return x < 0 ? 0 : (x > most ? static_cast<int>(most) : x); }
__device__ __forceinline__ int pages_for(int64_t keys, int page_size) {   // (2^30 keys at most)
    return static_cast<int>((static_cast<uint32_t>(keys) + page_size - 1) / static_cast<uint32_t>(page_size));
}

// Exclusive sums of x and y over the CTA's threads.
template <int N, typename X, typename Y>
__device__ __forceinline__ void sums_before(X& x, Y& y, X* x_warps, Y* y_warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    X sx = x;
    Y sy = y;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const X u = __shfl_up_sync(0xffffffffu, sx, off);
        const Y v = __shfl_up_sync(0xffffffffu, sy, off);
        if (lane >= off) {
            sx += u;
            sy += v;
        }
    }
    if (lane == 31) {
        x_warps[warp] = sx;
        y_warps[warp] = sy;
    }
    __syncthreads();
    x = sx - x;
    y = sy - y;
#pragma unroll
    for (int w = 0; w < N / 32; ++w) {
        x += w < warp ? x_warps[w] : 0;
        y += w < warp ? y_warps[w] : 0;
    }
}

// The last b with sums[b] <= n, of sequences lo to hi; sums do not decrease.
__device__ __forceinline__ int holder_of(const int* sums, int lo, int hi, int n) {
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= n) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// That of n + lane: a warp's lanes look at 32 sums that are evenly spaced, then between two of them, for the first; unless that has all of
// them, each lane for itself.
__device__ __forceinline__ int holders_of(const int* sums, int batch, int n) {
    const int lane = threadIdx.x & 31;
    int lo = 0, many = batch;
    while (many > 1) {
        const int step = (many + 31) / 32, i = lane * step;
        const uint32_t before = __ballot_sync(0xffffffffu, i < many && sums[lo + min(i, many - 1)] <= n);
        const int at = before ? (31 - __clz(before)) * step : 0;
        lo += at;
        many = min(step, many - at);
    }
    return n <= sums[lo + 1] - 32 ? lo : holder_of(sums, lo, batch - 1, n + lane);
}

__global__ void __launch_bounds__(kThreads) reserve_kernel(const __grid_constant__ ReserveParams p) {
    __shared__ int pages_s[kMaxSequences + 1], rows_s[kMaxSequences + 1];
    __shared__ int page_warps[kThreads / 32];
    __shared__ int64_t row_warps[kThreads / 32];
    __shared__ int short_s;   // the first sequence that gets nothing
    const int batch = p.batch;
    if (threadIdx.x == 0) short_s = batch;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int count = clamped(*p.count, p.pool);
    // Consecutive sequences to a thread; their pages and rows, then the sums before them.
    const int per = (batch + kThreads - 1) / kThreads, first = threadIdx.x * per, last = min(first + per, batch);
    auto wanted = [&](int b, int& len, int& more) {   // pages
        len = clamped(p.lengths[b], p.cap);
        more = max(p.added[b], 0);
        const int64_t all = static_cast<int64_t>(len) + more;
        return pages_for(all < p.cap ? all : p.cap, p.page_size) - pages_for(len, p.page_size);
    };
    int pages = 0;   // (under 2^31: a table of fewer entries)
    int64_t rows = 0;
    int len = 0, more = 0, one = 0;
    for (int b = first; b < last; ++b) {
        one = wanted(b, len, more);
        pages += one;
        rows += more;
    }
    sums_before<kThreads>(pages, rows, page_warps, row_warps);
    int over = batch;
    for (int b = first; b < last; ++b) {
        if (per > 1) one = wanted(b, len, more);
        pages_s[b] = pages;
        rows_s[b] = static_cast<int>(rows < INT32_MAX ? rows : INT32_MAX);
        pages += one;
        rows += more;
        if ((pages > count || static_cast<int64_t>(len) + more > p.cap) && over == batch) over = b;
        if (b == batch - 1) {
            pages_s[batch] = pages;
            rows_s[batch] = static_cast<int>(rows < INT32_MAX ? rows : INT32_MAX);
        }
    }
    if (over < batch) atomicMin(&short_s, over);
    __syncthreads();
    const int end = short_s;
    if (blockIdx.x == 0) {
        for (int b = threadIdx.x; b < batch; b += kThreads) {
            if (p.granted) p.granted[b] = b < end ? max(p.added[b], 0) : 0;
            if (p.cu) p.cu[b] = rows_s[b];
        }
        if (threadIdx.x == 0) {
            if (p.cu) p.cu[batch] = rows_s[batch];
            *p.count_out = count - pages_s[end];
        }
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads, warp_at = static_cast<int64_t>(blockIdx.x) * kThreads + (threadIdx.x & ~31);
    const int lane = threadIdx.x & 31, taken = pages_s[batch];
    for (int64_t n = warp_at; n < taken; n += step) {
        const int i = static_cast<int>(n) + lane, b = holders_of(pages_s, batch, static_cast<int>(n));
        if (i >= taken) continue;
        const int entry = pages_for(clamped(p.lengths[b], p.cap), p.page_size) + i - pages_s[b];
        p.table[b * p.table_stride + entry] = b < end ? p.free_pages[count - 1 - i] : -1;
    }
    if (!p.positions && !p.slots) return;
    const int packed = rows_s[batch];
    for (int64_t n = warp_at; n < p.tokens; n += step) {
        const int64_t row = n + lane;
        int position = -1;
        int64_t slot = -1;
        if (n < packed) {
            const int b = holders_of(rows_s, batch, static_cast<int>(n));
            if (row < packed) {
                const int keys = clamped(p.lengths[b], p.cap);
                const int64_t to = keys + row - rows_s[b];
                position = static_cast<int>(to < INT32_MAX ? to : INT32_MAX);
                if (b < end) {
                    const int entry = static_cast<int>(static_cast<uint32_t>(position) / static_cast<uint32_t>(p.page_size)), held = pages_for(keys, p.page_size);
                    const int64_t page = *(entry < held ? p.table + b * p.table_stride + entry : p.free_pages + (count - 1 - pages_s[b] - (entry - held)));
                    if (page >= 0) slot = page * p.page_size + (position - entry * p.page_size);
                }
            }
        }
        if (row >= p.tokens) continue;
        if (p.positions) p.positions[row] = position;
        if (p.slots) p.slots[row] = slot;
    }
}

// ---- pages given back --------------------------------------------------------------------------
//
// The entries that fall free are laid end to end and cut into equal runs for the threads of one cluster; what names a page is counted,
// the counts are summed over the CTA and, through the cluster's shared memory, over the CTAs before it, and a second look moves them.
struct ReleaseParams {
    int batch, page_size;
    int64_t cap;
    int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    const int32_t* kept;
    int32_t* free_pages;
    int64_t pool;
    const int32_t* count;
    int32_t* count_out;
};

constexpr int kReleaseThreads = 512;
constexpr int kReleaseCtas = 8;

__device__ __forceinline__ int in_cta(const int* here, int cta) {
    uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(here)), there;
    int x;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(cta));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(there) : "memory");
    return x;
}
__device__ __forceinline__ void ctas_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __cluster_dims__(kReleaseCtas, 1, 1) __launch_bounds__(kReleaseThreads) release_kernel(const __grid_constant__ ReleaseParams p) {
    __shared__ int entries_s[kMaxSequences + 1];
    __shared__ int64_t warps[kReleaseThreads / 32];
    __shared__ int none_warps[kReleaseThreads / 32], found_s;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int batch = p.batch, count = clamped(*p.count, p.pool);
    auto first_free = [&](int b, int& end) {
        const int len = clamped(p.lengths[b], p.cap);
        end = pages_for(len, p.page_size);
        return pages_for(clamped(p.kept[b], len), p.page_size);
    };
    const int per = (batch + kReleaseThreads - 1) / kReleaseThreads, first = threadIdx.x * per;
    int64_t mine = 0;
    for (int b = first; b < min(first + per, batch); ++b) {
        int end;
        const int begin = first_free(b, end);
        mine += end - begin;
    }
    int64_t before = mine;
    int none = 0;
    sums_before<kReleaseThreads>(before, none, warps, none_warps);
    __syncthreads();
    for (int b = first; b < min(first + per, batch); ++b) {
        int end;
        const int begin = first_free(b, end);
        entries_s[b] = static_cast<int>(before);
        before += end - begin;
        if (b == batch - 1) entries_s[batch] = static_cast<int>(before);
    }
    __syncthreads();
    const int all = entries_s[batch], each = (all + kReleaseCtas * kReleaseThreads - 1) / (kReleaseCtas * kReleaseThreads);
    const int64_t from = (static_cast<int64_t>(blockIdx.x) * kReleaseThreads + threadIdx.x) * each;
    const int n0 = static_cast<int>(from < all ? from : all), n1 = all - n0 < each ? all : n0 + each;
    auto visit = [&](auto use) {   // this thread's entries
        if (n0 >= n1) return;
        int b = holder_of(entries_s, 0, batch - 1, n0), end, entry = first_free(b, end) + n0 - entries_s[b];
        for (int n = n0; n < n1; ++n, ++entry) {
            while (entry >= end) entry = first_free(++b, end);
            use(p.table + b * p.table_stride + entry);
        }
    };
    int found = 0;
    visit([&](const int32_t* e) { found += *e >= 0 && *e < p.pool; });
    int64_t at = found;
    sums_before<kReleaseThreads>(at, none, warps, none_warps);
    if (threadIdx.x == kReleaseThreads - 1) found_s = static_cast<int>(at) + found;
    ctas_meet();
    int in_all = 0;
    for (int c = 0; c < kReleaseCtas; ++c) {
        const int there = in_cta(&found_s, c);
        if (c < static_cast<int>(blockIdx.x)) at += there;
        in_all += there;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const int64_t more = static_cast<int64_t>(count) + in_all;
        *p.count_out = static_cast<int32_t>(more < p.pool ? more : p.pool);
    }
    at += count;
    visit([&](int32_t* e) {
        const int page = *e;
        *e = -1;
        if (page < 0 || page >= p.pool) return;
        if (at < p.pool) p.free_pages[at] = page;
        ++at;
    });
    ctas_meet();   // nobody's shared memory goes away while another reads it
}

// Bytes of an argument. (CTAs read what is given after others may have written what is returned.)
struct Bytes {
    const void* at;   // null: none
    int64_t count;
};
bool meet(const Bytes& x, const Bytes& y) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x.at), b = reinterpret_cast<uintptr_t>(y.at);
    return a && b && x.count > 0 && y.count > 0 && a < b + static_cast<uintptr_t>(y.count) && b < a + static_cast<uintptr_t>(x.count);
}
template <int N, int M>
bool any_meet(const Bytes (&xs)[N], const Bytes (&ys)[M]) {
    for (const Bytes& x : xs) {
        for (const Bytes& y : ys) {
            if (meet(x, y)) return true;
        }
    }
    return false;
}

const char* tables_refusal(const ktt_b200_tables& a) {
    if (a.batch < 1 || a.table_width < 1 || a.pool < 0) return "sizes must be positive";
    if (a.page_size < 16 || a.page_size % 16) return "the page size must be a multiple of 16";
    if (a.batch > kMaxSequences) return "at most 4096 sequences";
    if (static_cast<int64_t>(a.table_width) * a.page_size > (1 << 30)) return "at most 2^30 keys per sequence";
    if (a.batch > 1 && a.table_stride < a.table_width && -a.table_stride < a.table_width) return "rows of the table must not lie on one another";
    if (static_cast<int64_t>(a.batch) * a.table_width >= (1ll << 31) || a.pool >= (1ll << 31)) return "fewer than 2^31 table entries and pages";
    return nullptr;
}

}  // namespace
}  // namespace ktt

using namespace ktt;

extern "C" int ktt_b200_paged_reserve(const ktt_b200_tables* a, const int32_t* added, int64_t tokens, int32_t* cu, int32_t* positions, int64_t* slots, int32_t* granted, void* stream) {
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_reserve: null arguments");
    if (const char* why = tables_refusal(*a)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_reserve: %s", why);
    if (tokens < 0 || tokens >= (1ll << 31)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_reserve: 0 to 2^31 - 1 tokens");
    if (!a->block_table || !a->lengths || !added || !a->count || !a->count_out || (a->pool && !a->free_pages)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_reserve: null pointer");
    if (a->count == a->count_out) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_reserve: count_out must be another word than count");
    const int64_t vector = 4 * static_cast<int64_t>(a->batch);
    const Bytes given[] = {{a->lengths, vector}, {added, vector}, {a->free_pages, 4 * a->pool}, {a->count, 4}};
    const Bytes returned[] = {{a->count_out, 4}, {cu, vector + 4}, {positions, 4 * tokens}, {slots, 8 * tokens}, {granted, vector}};
    if (any_meet(given, returned)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_reserve: outputs must not overlap inputs");
    ReserveParams p = {};
    p.batch = a->batch;
    p.page_size = a->page_size;
    p.cap = static_cast<int64_t>(a->table_width) * a->page_size;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.lengths = a->lengths;
    p.added = added;
    p.free_pages = a->free_pages;
    p.pool = a->pool;
    p.count = a->count;
    p.count_out = a->count_out;
    p.tokens = tokens;
    p.cu = cu;
    p.positions = positions;
    p.slots = slots;
    p.granted = granted;
    // A row to a thread at a time, two CTAs to an SM at most. 164,000 rows of 128 sequences, us with 1, 2, 4 and 6: 6.3, 5.1, 6.0, 5.6; with four rows to a
    // thread, looked up together, 7.1 with one and 8.2 with two.
    const int64_t blocks = (tokens + kThreads - 1) / kThreads;
    const dim3 grid(static_cast<unsigned>(blocks < 1 ? 1 : (blocks > 2 * 148 ? 2 * 148 : blocks)));
    return launch_dependent(reserve_kernel, p, grid, dim3(kThreads), static_cast<cudaStream_t>(stream), "paged_reserve launch");
}

extern "C" int ktt_b200_paged_release(const ktt_b200_tables* a, const int32_t* kept, void* stream) { return ktt_b200_paged_release_bounds(a, kept, nullptr, stream); }

extern "C" int ktt_b200_paged_release_bounds(const ktt_b200_tables* a, const int32_t* kept, const ktt_b200_bounds_args* bounds, void* stream) {
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_release: null arguments");
    if (const char* why = tables_refusal(*a)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_release: %s", why);
    if (!a->block_table || !a->lengths || !kept || !a->count || !a->count_out || (a->pool && !a->free_pages)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_release: null pointer");
    if (a->count == a->count_out) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_release: count_out must be another word than count");
    const int64_t vector = 4 * static_cast<int64_t>(a->batch);
    const Bytes given[] = {{a->lengths, vector}, {kept, vector}, {a->count, 4}}, returned[] = {{a->count_out, 4}, {a->free_pages, 4 * a->pool}};
    if (any_meet(given, returned) || meet(returned[0], returned[1])) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_release: outputs must not overlap inputs");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (bounds) {   // (refused before anything is launched)
        if (int rc = cut_bounds(bounds, kept, false, st)) return rc;
        const ktt_b200_pages& c = bounds->cache;
        if (bounds->batch != a->batch || c.page_size != a->page_size || c.table_width != a->table_width || c.block_table != a->block_table || c.table_stride != a->table_stride ||
            c.lengths != a->lengths || (c.max_keys > 0 && c.max_keys < static_cast<int64_t>(a->table_width) * a->page_size)) {
            return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_release: the bounds must be of the same table and lengths");
        }
    }
    ReleaseParams p = {};
    p.batch = a->batch;
    p.page_size = a->page_size;
    p.cap = static_cast<int64_t>(a->table_width) * a->page_size;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.lengths = a->lengths;
    p.kept = kept;
    p.free_pages = a->free_pages;
    p.pool = a->pool;
    p.count = a->count;
    p.count_out = a->count_out;
    if (int rc = launch_dependent(release_kernel, p, dim3(kReleaseCtas), dim3(kReleaseThreads), st, "paged_release launch")) return rc;
    return bounds ? cut_bounds(bounds, kept, true, st) : 0;   // (a page that is cut stays in its row)
}
