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
template <typename Int>
__device__ Int scan_1024(Int v, Int *total)
{
    __shared__ Int sums[16];
    const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) {
        const Int u = __shfl_up(v, m);
        v += lane >= m ? u : 0;
    }
    __syncthreads();
    if (lane == kWave - 1) {
        sums[wave] = v;
    }
    __syncthreads();
    Int all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        v += w < wave ? sums[w] : 0;
        all += sums[w];
    }
    *total = all;
    return v;
}

// The held pages before each group of words, in LDS: kGroups + 1 counts, the
// groups as many words each as it takes.
struct Counts {
    const uint32_t *used;
    int64_t pages, words;
    int span, groups;  // words of a group; groups that have words
    const int32_t *before;

    // Called by all 1024 threads; each counts neighbouring groups.
    __device__ Counts(const uint32_t *used_, int64_t pages_, int32_t *lds) : used(used_), pages(pages_), before(lds)
    {
        constexpr int kEach = kGroups / 1024;
        words = words_of(pages);
        span = (int)((words + kGroups - 1) / kGroups);
        groups = (int)((words + span - 1) / span);
        int n[kEach], mine = 0;
        const int64_t first = (int64_t)threadIdx.x * kEach * span;
#pragma unroll
        for (int g = 0; g < kEach; ++g) {
            n[g] = 0;
            if (span == 1) {
                n[g] = first + g < words ? __popc(used[first + g]) : 0;
            } else {
                for (int64_t w = first + g * span; w < first + (g + 1) * span && w < words; ++w) {
                    n[g] += __popc(used[w]);
                }
            }
            mine += n[g];
        }
        int total;
        int base = scan_1024(mine, &total) - mine;
#pragma unroll
        for (int g = 0; g < kEach; ++g) {
            lds[threadIdx.x * kEach + g] = base;
            base += n[g];
        }
        if (threadIdx.x == 1023) {
            lds[kGroups] = total;
        }
        __syncthreads();
    }
    __device__ int held() const { return before[kGroups]; }
    // Held pages before `page`.
    __device__ int rank(int64_t page) const
    {
        const int64_t word = page / 32, g = word / span;
        int n = before[g];
        for (int64_t w = g * span; w < word; ++w) {
            n += __popc(used[w]);
        }
        return word < words ? n + __popc(used[word] & ((1u << (page % 32)) - 1u)) : n;
    }
    __device__ int free_before(int g) const { return (int)((int64_t)g * span * 32 - before[g]); }
    // The k-th free page (there is one).
    __device__ int free_page(int k) const
    {
        int low = 0, high = groups;  // free pages before group low <= k < before group high
        while (high - low > 1) {
            const int mid = (low + high) / 2;
            if (free_before(mid) <= k) {
                low = mid;
            } else {
                high = mid;
            }
        }
        k -= free_before(low);
        for (int64_t w = (int64_t)low * span;; ++w) {
            uint32_t f = ~used[w];
            const int n = __popc(f);
            if (k >= n) {
                k -= n;
                continue;
            }
            for (; k > 0; --k) {
                f &= f - 1u;
            }
            return (int)(w * 32) + __ffs(f) - 1;
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
        const int64_t upto = asked + scan_1024<int64_t>(need, &total);
        asked += total;
        if (r < a.rows) {
            const bool served = any && (need == 0 || upto <= free);
            first[r] = served ? (int32_t)(need == 0 ? 0 : upto - need) : -1;
        }
    }
    const int64_t given = asked < free ? asked : free;
    for (int g = (int)threadIdx.x; g < counts.groups; g += 1024) {
        int64_t k = counts.free_before(g);
        for (int64_t w = (int64_t)g * counts.span; w < (int64_t)(g + 1) * counts.span && w < counts.words && k < given;
             ++w) {
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
    const int U = counts.held(), stay = counts.rank(U), moves = U - stay;
    const int64_t at = (int64_t)blockIdx.x * 1024 + threadIdx.x, all = (int64_t)gridDim.x * 1024;
    if (at == 0) {
        a.used[0] = (int32_t)U;
    }
    for (int64_t page = U + at; page < a.pages; page += all) {
        if ((used[page / 32] >> (page % 32) & 1u) != 0u) {
            const int k = counts.rank(page) - stay;
            a.src[k] = (int32_t)page;
            a.dst[k] = counts.free_page(k);
        }
    }
    for (int64_t k = moves + at; k < a.pages / 2; k += all) {
        a.src[k] = a.dst[k] = -1;
    }
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        for (int64_t j = threadIdx.x; j < a.width; j += 1024) {
            int page = held_entry(a, r, j);
            if (page >= U) {
                page = counts.free_page(counts.rank(page) - stay);
            }
            a.newTable[r * a.width + j] = page;
        }
    }
}

// A page as n0 x n1 runs of `run` bytes, s0 and s1 bytes apart.
struct Runs {
    char *base;
    int64_t page;  // bytes
    int n0, n1;
    int64_t s0, s1, run;
};

// Vec-sized pieces of the pages, kPer a thread: a workgroup has 256 * kPer pieces of
// one pair's page in one cache.
constexpr int kPer = 4;

template <typename Vec>
__global__ __launch_bounds__(256) void copy_pieces(Runs k, Runs v, const int32_t *srcs, const int32_t *dsts, int64_t n,
                                                   int64_t pages, int64_t pieces, int64_t blocksPerPage)
{
    for (int64_t block = blockIdx.x; block < 2 * n * blocksPerPage; block += gridDim.x) {
        const int64_t pair = block / blocksPerPage, i = pair / 2;
        const int64_t src = srcs[i], dst = dsts[i];
        if (src < 0 || src >= pages || dst < 0 || dst >= pages) {
            continue;
        }
        const Runs &c = pair % 2 == 0 ? k : v;
        const int64_t first = block % blocksPerPage * (256 * kPer) + threadIdx.x;
        const int64_t inRun = c.run / (int64_t)sizeof(Vec);
        Vec held[kPer];
        int64_t at[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int64_t e = first + 256 * j;
            at[j] = -1;
            if (e < pieces) {
                int64_t inside = e * (int64_t)sizeof(Vec);
                if (c.n0 * (int64_t)c.n1 > 1) {
                    const int64_t row = e / inRun;
                    inside = row / c.n1 * c.s0 + row % c.n1 * c.s1 + e % inRun * (int64_t)sizeof(Vec);
                }
                at[j] = inside;
                held[j] = *reinterpret_cast<const Vec *>(c.base + src * c.page + inside);
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (at[j] >= 0) {
                *reinterpret_cast<Vec *>(c.base + dst * c.page + at[j]) = held[j];
            }
        }
    }
}

// The runs of a cache's pages, as long as they come.
Runs runs_of(const CacheRows &c, const CopyPagesArgs &a)
{
    Runs r;
    r.base = static_cast<char *>(c.data);
    r.page = c.page * a.elemBytes;
    int64_t slot = c.slot * a.elemBytes, head = c.head * a.elemBytes;
    r.run = a.rowBytes;
    int slots = a.pageSize, heads = a.kvHeads;
    for (int again = 0; again < 2; ++again) {
        if (heads > 1 && head == r.run) {
            r.run *= heads;
            heads = 1;
        }
        if (slots > 1 && slot == r.run) {
            r.run *= slots;
            slots = 1;
        }
    }
    r.n0 = slots;
    r.s0 = slots > 1 ? slot : 0;
    r.n1 = heads;
    r.s1 = heads > 1 ? head : 0;
    return r;
}

bool whole_pieces(const Runs &r, int64_t size)
{
    return reinterpret_cast<uintptr_t>(r.base) % size == 0 && r.page % size == 0 && r.s0 % size == 0 &&
           r.s1 % size == 0 && r.run % size == 0;
}

template <typename Vec>
hipError_t launch_pieces(const CopyPagesArgs &a, const Runs &k, const Runs &v, int cus, hipStream_t stream)
{
    const int64_t pieces = (int64_t)a.pageSize * a.kvHeads * a.rowBytes / (int64_t)sizeof(Vec);
    const int64_t perPage = (pieces + 256 * kPer - 1) / (256 * kPer);
    const int64_t blocks = 2 * a.n * perPage, most = (int64_t)cus * 1024;
    hipLaunchKernelGGL((copy_pieces<Vec>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, k, v,
                       a.src, a.dst, a.n, a.pages, pieces, perPage);
    return hipGetLastError();
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
    const Runs k = runs_of(a.k, a), v = runs_of(a.v, a);
    if (whole_pieces(k, 16) && whole_pieces(v, 16)) {
        return launch_pieces<dev::u32x4_t>(a, k, v, cus, stream);
    }
    if (whole_pieces(k, 4) && whole_pieces(v, 4)) {
        return launch_pieces<uint32_t>(a, k, v, cus, stream);
    }
    return launch_pieces<uint16_t>(a, k, v, cus, stream);
}

}  // namespace mhc
