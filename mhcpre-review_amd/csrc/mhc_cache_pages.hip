// The pages of a cache: a step's table (mhcCacheUpdate), compaction's plan
// (mhcCacheCompact) and the copying of contents (mhcCacheCopyPages).
//
// Which pages are held is not kept between calls: each call marks the pages
// that the rows hold in a bitmap (one bit per page, and in a second one the
// pages that two rows or more hold), from which ranks (how many held pages lie
// before this one) and selections (the k-th free page) follow by counting
// bits.  The counts up to every group of words are kept in LDS.

#include "mhc_pre_device.h"
#include "mhc_serve_internal.h"

namespace mhc {
namespace {

using dev::kWave;

constexpr int kGroups = 8192;  // of words whose counts LDS holds (32 KB)

__host__ __device__ __forceinline__ int64_t words_of(int64_t pages) { return (pages + 31) / 32; }

__device__ __forceinline__ int64_t clamped(int64_t v, int64_t most) { return v < 0 ? 0 : v > most ? most : v; }

// Row r of mhcCacheUpdate: what it goes on from and what it asks for.
struct Row {
    const int32_t *base;  // its parent's entries, or null
    int64_t length, held, grown;
    int add;  // tokens, 0 where they cannot fit the table's width

    __device__ Row(const CacheUpdateArgs &a, int64_t r)
    {
        const int64_t p = a.parents[r];
        const bool alive = p >= 0 && p < a.rows;
        length = alive ? clamped(a.lengths[p], (int64_t)a.width * a.pageSize) : 0;
        base = alive ? a.table + p * a.width : nullptr;
        held = (length + a.pageSize - 1) / a.pageSize;
        add = (int)clamped(a.counts[r], a.tokens);
        grown = (length + add + a.pageSize - 1) / a.pageSize;
        if (grown > a.width) {
            add = 0;
            grown = held;
        }
    }
    // The entry at column j < held, -1 for a hole.
    __device__ int entry(const CacheUpdateArgs &a, int64_t j) const
    {
        const int page = base[j];
        return page >= 0 && page < a.pages ? page : -1;
    }
    // The first column that the new tokens may change.
    __device__ int64_t open(const CacheUpdateArgs &a) const
    {
        return add > 0 && length % a.pageSize != 0 ? held - 1 : held;
    }
};

__global__ __launch_bounds__(256) void clear_words(uint32_t *words, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        words[i] = 0u;
    }
}

__device__ __forceinline__ void mark(int page, uint32_t *used, uint32_t *many)
{
    const uint32_t bit = 1u << (page % 32);
    const uint32_t before = __hip_atomic_fetch_or(used + page / 32, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (many != nullptr && (before & bit) != 0u) {
        (void)__hip_atomic_fetch_or(many + page / 32, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

// Marks a row's pages and writes the columns of its new row that the new
// tokens leave alone.
__global__ __launch_bounds__(256) void update_rows(CacheUpdateArgs a, uint32_t *used, uint32_t *many)
{
    const int64_t r = blockIdx.x;
    const Row row(a, r);
    const int64_t open = row.open(a), end = row.add > 0 ? row.grown : open;
    int32_t *out = a.newTable + r * a.width;
    for (int64_t j = threadIdx.x; j < a.width; j += 256) {
        const int page = j < row.held ? row.entry(a, j) : -1;
        if (page >= 0) {
            mark(page, used, many);
        }
        if (j < open || j >= end) {
            out[j] = page;
        }
    }
}

// Inclusive scan of v over the workgroup of 1024; *total gets the sum.
__device__ int64_t scan_1024(int64_t v, int64_t *total)
{
    __shared__ int64_t sums[16];
    const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) {
        const int64_t u = __shfl_up(v, m);
        v += lane >= m ? u : 0;
    }
    __syncthreads();
    if (lane == kWave - 1) {
        sums[wave] = v;
    }
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < 16; ++w) {
        v += w < wave ? sums[w] : 0;
        all += sums[w];
    }
    *total = all;
    return v;
}

// The held pages before each group of words, in LDS.
struct Counts {
    const uint32_t *used;
    int64_t pages, words, span;  // span: words of a group
    const int32_t *before;       // [kGroups + 1]

    // Called by all 1024 threads.
    __device__ Counts(const uint32_t *used_, int64_t pages_, int32_t *lds) : used(used_), pages(pages_), before(lds)
    {
        words = words_of(pages);
        span = (words + kGroups - 1) / kGroups;
        int64_t base = 0;
        for (int g = 0; g < kGroups; g += 1024) {
            const int64_t first = (g + (int64_t)threadIdx.x) * span;
            int n = 0;
            for (int64_t w = first; w < first + span && w < words; ++w) {
                n += __popc(used[w]);
            }
            int64_t total;
            lds[g + threadIdx.x + 1] = (int32_t)(base + scan_1024(n, &total));
            base += total;
            if (g == 0 && threadIdx.x == 0) {
                lds[0] = 0;
            }
        }
        __syncthreads();
    }
    __device__ int64_t held() const { return before[kGroups]; }
    // Held pages before `page`.
    __device__ int64_t rank(int64_t page) const
    {
        const int64_t word = page / 32, g = word / span;
        int64_t n = before[g];
        for (int64_t w = g * span; w < word; ++w) {
            n += __popc(used[w]);
        }
        return word < words ? n + __popc(used[word] & ((1u << (page % 32)) - 1u)) : n;
    }
    // The k-th free page (there is one).
    __device__ int64_t free_page(int64_t k) const
    {
        int low = 0, high = kGroups;  // free pages before group low <= k < before group high
        while (high - low > 1) {
            const int mid = (low + high) / 2;
            if ((int64_t)mid * span * 32 - before[mid] <= k) {
                low = mid;
            } else {
                high = mid;
            }
        }
        k -= (int64_t)low * span * 32 - before[low];
        for (int64_t w = low * span;; ++w) {
            uint32_t f = ~used[w];
            const int n = __popc(f);
            if (k >= n) {
                k -= n;
                continue;
            }
            for (; k > 0; --k) {
                f &= f - 1u;
            }
            return w * 32 + __ffs(f) - 1;
        }
    }
};

// Whether the row's partly filled page, which it would append to, is shared.
__device__ __forceinline__ bool wants_copy(const CacheUpdateArgs &a, const Row &row, const uint32_t *many, int *last)
{
    *last = -1;
    if (row.add == 0 || row.length % a.pageSize == 0) {
        return false;
    }
    *last = row.entry(a, row.held - 1);
    return *last >= 0 && (many[*last / 32] >> (*last % 32) & 1u) != 0u;
}

// One workgroup: which rows get their pages, first[r] = rank of the row's
// first free page or -1, and the list of the free pages given out.
__global__ __launch_bounds__(1024) void update_grants(CacheUpdateArgs a, const uint32_t *used, const uint32_t *many,
                                                      int32_t *first, int32_t *list)
{
    __shared__ int32_t lds[kGroups + 1];
    const Counts counts(used, a.pages, lds);
    const int64_t free = a.pages - counts.held();
    int64_t asked = 0;
    for (int64_t r0 = 0; r0 < a.rows; r0 += 1024) {
        const int64_t r = r0 + threadIdx.x;
        int64_t need = 0;
        bool any = false;
        if (r < a.rows) {
            const Row row(a, r);
            int last;
            need = wants_copy(a, row, many, &last) + row.grown - row.held;
            any = row.add > 0;
        }
        int64_t total;
        const int64_t upto = asked + scan_1024(need, &total);
        asked += total;
        if (r < a.rows) {
            const bool served = any && (need == 0 || upto <= free);
            first[r] = served ? (int32_t)(need == 0 ? 0 : upto - need) : -1;
        }
    }
    const int64_t given = asked < free ? asked : free;
    for (int g = (int)threadIdx.x; g < kGroups; g += 1024) {
        int64_t k = (int64_t)g * counts.span * 32 - lds[g];
        for (int64_t w = g * counts.span; w < (g + 1) * counts.span && w < counts.words && k < given; ++w) {
            for (uint32_t f = ~used[w]; f != 0u && k < given; f &= f - 1u) {
                const int64_t page = w * 32 + __ffs(f) - 1;
                if (page < a.pages) {
                    list[k++] = (int32_t)page;
                }
            }
        }
    }
}

// One wave per row: the columns that its new tokens change, its slots and
// the rest of its state.
__global__ __launch_bounds__(256) void update_finish(CacheUpdateArgs a, const uint32_t *many, const int32_t *first,
                                                     const int32_t *list)
{
    const int lane = (int)threadIdx.x % kWave;
    const int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (r >= a.rows) {
        return;
    }
    const Row row(a, r);
    int last;
    const bool copy = wants_copy(a, row, many, &last);
    const bool served = first[r] >= 0;
    const int32_t *mine = list + (served ? first[r] : 0);
    const auto column = [&](int64_t j) -> int {  // of the new row, j in [open, grown)
        if (j >= row.held) {
            return served ? mine[copy + j - row.held] : -1;
        }
        return served && copy ? mine[0] : last;
    };
    const int64_t open = row.open(a), end = row.add > 0 ? row.grown : open;
    for (int64_t j = open + lane; j < end; j += kWave) {
        a.newTable[r * a.width + j] = column(j);
    }
    const int granted = served ? row.add : 0;
    for (int64_t i = lane; i < a.tokens; i += kWave) {
        const int64_t t = row.length + i;
        const int page = i < granted ? column(t / a.pageSize) : -1;
        a.slots[r * a.tokens + i] = page >= 0 ? (int64_t)page * a.pageSize + t % a.pageSize : -1;
    }
    if (lane == 0) {
        a.newLengths[r] = (int32_t)(row.length + granted);
        a.granted[r] = granted;
        a.src[r] = served && copy ? last : -1;
        a.dst[r] = served && copy ? mine[0] : -1;
    }
}

// Column j of row r as mhcCacheCompact sees it.
__device__ __forceinline__ int held_entry(const CacheCompactArgs &a, int64_t r, int64_t j)
{
    const int64_t length = clamped(a.lengths[r], (int64_t)a.width * a.pageSize);
    if (j >= (length + a.pageSize - 1) / a.pageSize) {
        return -1;
    }
    const int page = a.table[r * a.width + j];
    return page >= 0 && page < a.pages ? page : -1;
}

__global__ __launch_bounds__(256) void compact_mark(CacheCompactArgs a, uint32_t *used)
{
    const int64_t r = blockIdx.x;
    for (int64_t j = threadIdx.x; j < a.width; j += 256) {
        const int page = held_entry(a, r, j);
        if (page >= 0) {
            mark(page, used, nullptr);
        }
    }
}

// Every workgroup counts for itself, then writes its part of the moves and of
// the table.
__global__ __launch_bounds__(1024) void compact_apply(CacheCompactArgs a, const uint32_t *used)
{
    __shared__ int32_t lds[kGroups + 1];
    const Counts counts(used, a.pages, lds);
    const int64_t U = counts.held(), stay = counts.rank(U), moves = U - stay;
    const int64_t at = (int64_t)blockIdx.x * 1024 + threadIdx.x, all = (int64_t)gridDim.x * 1024;
    if (at == 0) {
        a.used[0] = (int32_t)U;
    }
    for (int64_t page = U + at; page < a.pages; page += all) {
        if ((used[page / 32] >> (page % 32) & 1u) != 0u) {
            const int64_t k = counts.rank(page) - stay;
            a.src[k] = (int32_t)page;
            a.dst[k] = (int32_t)counts.free_page(k);
        }
    }
    for (int64_t k = moves + at; k < a.pages / 2; k += all) {
        a.src[k] = a.dst[k] = -1;
    }
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        for (int64_t j = threadIdx.x; j < a.width; j += 1024) {
            int page = held_entry(a, r, j);
            if (page >= U) {
                page = (int)counts.free_page(counts.rank(page) - stay);
            }
            a.newTable[r * a.width + j] = page;
        }
    }
}

// One workgroup per pair and cache.
__global__ __launch_bounds__(256) void copy_rows(CopyPagesArgs a)
{
    const CacheRows &c = blockIdx.y == 0 ? a.k : a.v;
    const int rows = a.kvHeads * a.pageSize;
    for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        const int64_t src = a.src[i], dst = a.dst[i];
        if (src < 0 || src >= a.pages || dst < 0 || dst >= a.pages) {
            continue;
        }
        char *base = static_cast<char *>(c.data);
        for (int64_t e = threadIdx.x; e < (int64_t)rows * (a.rowBytes / 2); e += 256) {
            const int64_t row = e / (a.rowBytes / 2), at = e % (a.rowBytes / 2) * 2;
            const int64_t inside = (row / a.kvHeads * c.slot + row % a.kvHeads * c.head) * a.elemBytes + at;
            *reinterpret_cast<uint16_t *>(base + dst * c.page * a.elemBytes + inside) =
                *reinterpret_cast<const uint16_t *>(base + src * c.page * a.elemBytes + inside);
        }
    }
}

size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

hipError_t clear(uint32_t *words, int64_t n, hipStream_t stream)
{
    const int64_t blocks = (n + 1023) / 1024;
    hipLaunchKernelGGL(clear_words, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, stream, words, n);
    return hipGetLastError();
}

}  // namespace

// [used bits][many bits][first: rows][list: pages]
size_t cache_update_workspace(const CacheUpdateArgs &a)
{
    return 2 * align_up(words_of(a.pages) * 4) + align_up((size_t)a.rows * 4) + align_up((size_t)a.pages * 4);
}

hipError_t launch_cache_update(const CacheUpdateArgs &a, void *workspace, int, hipStream_t stream)
{
    char *ws = static_cast<char *>(workspace);
    const size_t bits = align_up(words_of(a.pages) * 4);
    uint32_t *used = reinterpret_cast<uint32_t *>(ws), *many = reinterpret_cast<uint32_t *>(ws + bits);
    int32_t *first = reinterpret_cast<int32_t *>(ws + 2 * bits);
    int32_t *list = reinterpret_cast<int32_t *>(ws + 2 * bits + align_up((size_t)a.rows * 4));
    hipError_t err = clear(used, (int64_t)(2 * bits / 4), stream);
    if (err != hipSuccess) {
        return err;
    }
    hipLaunchKernelGGL(update_rows, dim3((unsigned)a.rows), dim3(256), 0, stream, a, used, many);
    if ((err = hipGetLastError()) != hipSuccess) {
        return err;
    }
    hipLaunchKernelGGL(update_grants, dim3(1), dim3(1024), 0, stream, a, used, many, first, list);
    if ((err = hipGetLastError()) != hipSuccess) {
        return err;
    }
    hipLaunchKernelGGL(update_finish, dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, stream, a, many, first, list);
    return hipGetLastError();
}

size_t cache_compact_workspace(const CacheCompactArgs &a) { return align_up(words_of(a.pages) * 4); }

hipError_t launch_cache_compact(const CacheCompactArgs &a, void *workspace, int cus, hipStream_t stream)
{
    uint32_t *used = static_cast<uint32_t *>(workspace);
    hipError_t err = clear(used, words_of(a.pages), stream);
    if (err != hipSuccess) {
        return err;
    }
    if (a.rows > 0) {
        hipLaunchKernelGGL(compact_mark, dim3((unsigned)a.rows), dim3(256), 0, stream, a, used);
        if ((err = hipGetLastError()) != hipSuccess) {
            return err;
        }
    }
    hipLaunchKernelGGL(compact_apply, dim3((unsigned)cus), dim3(1024), 0, stream, a, used);
    return hipGetLastError();
}

hipError_t launch_copy_pages(const CopyPagesArgs &a, int cus, hipStream_t stream)
{
    const int64_t blocks = a.n < 8 * (int64_t)cus ? a.n : 8 * (int64_t)cus;
    hipLaunchKernelGGL(copy_rows, dim3((unsigned)blocks, 2), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mhc
