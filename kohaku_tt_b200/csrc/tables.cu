// Block tables on the device: pages for the tokens that requests bring, with each token's place, and pages given back.
//
// With held_b = ceil(len_b / P) and wanted_b = ceil((len_b + added_b) / P) pages of P keys, sequence b takes wanted_b - held_b pages from the
// end of a list of free ones; before_b, the pages that sequences before it take, is an exclusive sum. So entry held_b + i of its row is
// free[count - 1 - before_b - i], a token's page is found without reading an entry that the same launch writes, and nothing waits for
// anything: every CTA sums up the lengths for itself. Bound: 12 bytes written for a token and 8 moved for a page, which is nothing; one trip for
// the lengths, a sum over the CTA and a search among the sequences are all that a call takes.
#include "paged.cuh"

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
__device__ __forceinline__ int pages_for(int64_t keys, int page_size) { return static_cast<int>((keys + page_size - 1) / page_size); }

// Exclusive sum of x over the CTA's threads.
template <int N>
__device__ __forceinline__ int64_t sum_before(int64_t x, int64_t* warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t sum = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += y;
    }
    if (lane == 31) warps[warp] = sum;
    __syncthreads();
    int64_t before = sum - x;
#pragma unroll
    for (int w = 0; w < N / 32; ++w) before += w < warp ? warps[w] : 0;
    __syncthreads();
    return before;
}

// The last b with sums[b] <= n, of `batch` sequences; sums do not decrease.
__device__ __forceinline__ int holder_of(const int* sums, int batch, int n) {
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= n) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads) reserve_kernel(const __grid_constant__ ReserveParams p) {
    __shared__ int pages_s[kMaxSequences + 1], rows_s[kMaxSequences + 1];
    __shared__ int64_t warps[kThreads / 32];
    __shared__ int short_s;   // the first sequence that gets nothing
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int batch = p.batch;
    const int count = clamped(*p.count, p.pool);
    if (threadIdx.x == 0) short_s = batch;
    // Consecutive sequences to a thread; their pages and rows, then the sums before them.
    const int per = (batch + kThreads - 1) / kThreads, first = threadIdx.x * per;
    int64_t pages = 0, rows = 0;
    int over = batch;
    for (int i = 0; i < per; ++i) {
        const int b = first + i;
        if (b >= batch) break;
        const int len = clamped(p.lengths[b], p.cap), more = max(p.added[b], 0);
        const int64_t all = static_cast<int64_t>(len) + more;
        if (all > p.cap && over == batch) over = b;
        pages += pages_for(all < p.cap ? all : p.cap, p.page_size) - pages_for(len, p.page_size);
        rows += more;
    }
    int64_t pages_at = sum_before<kThreads>(pages, warps), rows_at = sum_before<kThreads>(rows, warps);
    for (int i = 0; i < per; ++i) {
        const int b = first + i;
        if (b >= batch) break;
        pages_s[b] = static_cast<int>(pages_at);   // (under 2^31: a table of fewer entries)
        rows_s[b] = static_cast<int>(rows_at < INT32_MAX ? rows_at : INT32_MAX);
        const int len = clamped(p.lengths[b], p.cap), more = max(p.added[b], 0);
        const int64_t all = static_cast<int64_t>(len) + more;
        pages_at += pages_for(all < p.cap ? all : p.cap, p.page_size) - pages_for(len, p.page_size);
        rows_at += more;
        if (pages_at > count && over == batch) over = b;
        if (b == batch - 1) {
            pages_s[batch] = static_cast<int>(pages_at);
            rows_s[batch] = static_cast<int>(rows_at < INT32_MAX ? rows_at : INT32_MAX);
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
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kThreads;
    const int taken = pages_s[batch];
    for (int64_t n = at; n < taken; n += step) {
        const int i = static_cast<int>(n), b = holder_of(pages_s, batch, i);
        const int entry = pages_for(clamped(p.lengths[b], p.cap), p.page_size) + i - pages_s[b];
        p.table[b * p.table_stride + entry] = b < end ? p.free_pages[count - 1 - i] : -1;
    }
    if (!p.positions && !p.slots) return;
    for (int64_t n = at; n < p.tokens; n += step) {
        int position = -1;
        int64_t slot = -1;
        if (n < rows_s[batch]) {
            const int b = holder_of(rows_s, batch, static_cast<int>(n));
            const int len = clamped(p.lengths[b], p.cap);
            const int64_t place = len + n - rows_s[b];
            position = static_cast<int>(place < INT32_MAX ? place : INT32_MAX);
            if (b < end) {
                const int entry = position / p.page_size, held = pages_for(len, p.page_size);
                const int64_t page = entry < held ? p.table[b * p.table_stride + entry] : p.free_pages[count - 1 - pages_s[b] - (entry - held)];
                if (page >= 0) slot = page * p.page_size + (position - entry * p.page_size);
            }
        }
        if (p.positions) p.positions[n] = position;
        if (p.slots) p.slots[n] = slot;
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
    __shared__ int found_s;
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
    int64_t before = sum_before<kReleaseThreads>(mine, warps);
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
    const int n0 = static_cast<int>(from < all ? from : all), n1 = min(n0 + each, all);
    auto visit = [&](auto use) {   // this thread's entries
        if (n0 >= n1) return;
        int b = holder_of(entries_s, batch, n0), end, entry = first_free(b, end) + n0 - entries_s[b];
        for (int n = n0; n < n1; ++n, ++entry) {
            while (entry >= end) entry = first_free(++b, end);
            use(p.table + b * p.table_stride + entry);
        }
    };
    int found = 0;
    visit([&](const int32_t* e) { found += *e >= 0 && *e < p.pool; });
    int64_t at = sum_before<kReleaseThreads>(found, warps);
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

const char* tables_refusal(const ktt_b200_tables& a) {
    if (a.batch < 1 || a.table_width < 1 || a.pool < 0) return "sizes must be positive";
    if (a.page_size < 16 || a.page_size % 16) return "the page size must be a multiple of 16";
    if (a.batch > kMaxSequences) return "at most 4096 sequences";
    if (static_cast<int64_t>(a.table_width) * a.page_size > (1 << 30)) return "at most 2^30 keys per sequence";
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
    // Four rows to a thread, two CTAs to an SM at most.
    const int64_t blocks = (tokens + 4 * kThreads - 1) / (4 * kThreads);
    const unsigned grid = static_cast<unsigned>(blocks < 1 ? 1 : (blocks > 296 ? 296 : blocks));
    return launch_dependent(reserve_kernel, p, dim3(grid), dim3(kThreads), static_cast<cudaStream_t>(stream), "paged_reserve launch");
}

extern "C" int ktt_b200_paged_release(const ktt_b200_tables* a, const int32_t* kept, void* stream) {
    if (!a) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_release: null arguments");
    if (const char* why = tables_refusal(*a)) return fail(KTT_B200_ERR_UNSUPPORTED, "paged_release: %s", why);
    if (!a->block_table || !a->lengths || !kept || !a->count || !a->count_out || (a->pool && !a->free_pages)) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_release: null pointer");
    if (a->count == a->count_out) return fail(KTT_B200_ERR_BAD_ARGUMENT, "paged_release: count_out must be another word than count");
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
    return launch_dependent(release_kernel, p, dim3(kReleaseCtas), dim3(kReleaseThreads), static_cast<cudaStream_t>(stream), "paged_release launch");
}
