// The pages of a cache: a step's table (mhcCacheUpdate), compaction's plan
// (mhcCacheCompact) and the copying of contents (mhcCacheCopyPages).
//
// Which pages are held is not kept between calls: each call marks the pages
// that the rows hold in a bitmap (one bit per page, and in a second one the
// pages that two rows or more hold), from which ranks (how many held pages lie
// before this one) and selections (the k-th free page) follow by counting
// bits.  The counts up to every group of words are kept in LDS.
//
// Bound: latencies.  Up to some entries one workgroup does all of it (64 rows of 128
// entries, us: 8.7, compaction 7.7); above, each launch waits for the one before.
// 1000 rows of up to 2048 entries, 200001 pages, us: clearing the bitmaps 2.0, marking
// and the columns that stay 11.1 (about 6 of it the atomics, which go past the L2s, for
// every XCD marks), who gets pages 6.0, the columns that change 3.3; compaction 1.9,
// 7.6 and 12.0.  What they read and write is 9 MB, 1.6 us.  A compaction of a nearly full
// pool takes longer, for its few free pages lie far apart (see index): 200001 pages, us,
// 40% free 23, 1% 67, 0.1% 166; 31 of 262144 free 675.  Copies are bound by the memory:
// 2000 pages of 128 KB twice, read and written, 194 us (5.4 TB/s).

#include "mhc_pre_device.h"
#include "mhc_serve_internal.h"

namespace mhc {
namespace {

using dev::kWave;

// What one workgroup does alone.  The rows, the bitmaps and a compaction's moves are held in its
// LDS; and the rest of the CUs pays for its launches above some entries (us of a call alone / by
// all CUs: 4 rows of 64 entries, update 8.6 / 19.1, compaction 8.1 / 13.9; 128 of 128 12.6 / 17.2,
// 12.6 / 14.0; 256 of 128 19.9 / 17.1, 20.9 / 14.8; 512 of 128 31.8 / 18.0, 37.0 / 15.7).
constexpr int kSmallPages = 1 << 16, kSmallWords = kSmallPages / 32, kSmallRows = 1024;
constexpr int64_t kSmallEntries = 1 << 14;
constexpr int kSmallBatch = 8;

constexpr int kGroups = 8192;  // of words whose counts LDS holds (32 KB)

__host__ __device__ __forceinline__ int64_t words_of(int64_t pages) { return (pages + 31) / 32; }

__device__ __forceinline__ int clamped(int v, int most) { return v < 0 ? 0 : v > most ? most : v; }

// Pages of `tokens` tokens (below 2^32).
__device__ __forceinline__ int pages_for(uint32_t tokens, int pageSize)
{
    return tokens == 0 ? 0 : (int)((tokens - 1) / (uint32_t)pageSize) + 1;
}

// A column of a table, or one some steps beyond the last: a table may have 2^31 - 1.
typedef uint32_t Column;

// Row r of mhcCacheUpdate: what it goes on from and what it asks for.
struct Row {
    int parent;       // row of the old table, or -1
    int length, held, grown;
    int full;         // pages that are filled; the next one holds `rest` tokens
    int rest;
    int add;          // tokens, 0 where they cannot fit the table's width
    int open, end;    // the columns that the new tokens may change

    Row() = default;
    __device__ Row(const CacheUpdateArgs &a, int64_t r)
    {
        parent = a.parents[r];
        parent = parent >= 0 && parent < a.rows ? parent : -1;
        length = parent >= 0 ? clamped(a.lengths[parent], a.width * a.pageSize) : 0;
        full = (int)((uint32_t)length / (uint32_t)a.pageSize);
        rest = length - full * a.pageSize;
        held = full + (rest > 0 ? 1 : 0);
        add = clamped(a.counts[r], a.tokens);
        const int64_t wanted = (int64_t)full + pages_for((uint32_t)rest + (uint32_t)add, a.pageSize);
        grown = (int)wanted;
        if (wanted > a.width) {
            add = 0;
            grown = held;
        }
        open = add > 0 ? full : held;
        end = add > 0 ? grown : held;
    }
    // The entry at column j < held, -1 for a hole.
    __device__ int entry(const CacheUpdateArgs &a, int j) const
    {
        const int page = a.table[(int64_t)parent * a.width + j];
        return page >= 0 && page < a.pages ? page : -1;
    }
    // The same where `on`, else -1: a load in any case (of the table's first entry), so that
    // a batch of them has no branches and all are on their way before the first is used.
    __device__ int entry_if(const CacheUpdateArgs &a, Column j, bool on) const
    {
        const int page = a.table[on ? (int64_t)parent * a.width + j : 0];
        return on && page >= 0 && page < a.pages ? page : -1;
    }
};

__global__ __launch_bounds__(256) void clear_words(uint32_t *words, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        words[i] = 0u;
    }
}

// Marks pages (-1: none), all of them on their way at once.
template <int N>
__device__ __forceinline__ void mark_all(const int (&page)[N], uint32_t *used, uint32_t *many)
{
    uint32_t before[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        before[n] = page[n] >= 0 ? __hip_atomic_fetch_or(used + page[n] / 32, 1u << (page[n] % 32), __ATOMIC_RELAXED,
                                                         __HIP_MEMORY_SCOPE_AGENT)
                                 : 0u;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (many != nullptr && page[n] >= 0 && (before[n] >> (page[n] % 32) & 1u) != 0u) {
            (void)__hip_atomic_fetch_or(many + page[n] / 32, 1u << (page[n] % 32), __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// One workgroup per row: marks its pages and writes the columns of its new row
// that the new tokens leave alone.  The entries are loaded kBatch at a time
// before the first is marked, for a mark waits for the word that was there.
constexpr int kBatch = 4;

// What update_rows finds out about a row, for the launches after it.
struct Found {
    Row row;
    int last;  // the partly filled page that the row appends to, or -1
};

// ... and what update_grants decides: the rank of the row's first free page (-1: it
// gets nothing), and whether that takes the place of `last`.
struct Grant {
    int32_t first, copy;
};

__global__ __launch_bounds__(256) void update_rows(CacheUpdateArgs a, uint32_t *used, uint32_t *many, Found *found)
{
    const int64_t r = blockIdx.x;
    const Row row(a, r);
    if (threadIdx.x == 0) {
        found[r] = Found{row, row.add > 0 && row.rest > 0 ? row.entry(a, row.held - 1) : -1};
    }
    int32_t *out = a.newTable + r * a.width;
    const Column width = (Column)a.width, held = (Column)row.held, open = (Column)row.open, end = (Column)row.end;
    for (Column j0 = threadIdx.x; j0 < width; j0 += 256 * kBatch) {
        int page[kBatch];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            const Column j = j0 + 256 * n;
            page[n] = row.entry_if(a, j, j < held);
        }
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            const Column j = j0 + 256 * n;
            if (j < width && (j < open || j >= end)) {
                out[j] = page[n];
            }
        }
        if (j0 - threadIdx.x < held) {
            mark_all(page, used, many);
        }
    }
}

// The bitmap's words into registers, neighbouring threads' neighbouring ones, and
// from there into LDS; words beyond it are 0.
struct Words {
    uint32_t held[kGroups / 1024];

    __device__ Words(const uint32_t *from, int words)
    {
#pragma unroll
        for (int n = 0; n < kGroups / 1024; ++n) {
            const int w = (int)threadIdx.x + 1024 * n;
            held[n] = from[w < words ? w : 0];  // (a load in any case)
            held[n] = w < words ? held[n] : 0u;
        }
    }
    __device__ void put(uint32_t *lds) const
    {
#pragma unroll
        for (int n = 0; n < kGroups / 1024; ++n) {
            lds[threadIdx.x + 1024 * n] = held[n];
        }
    }
};

// Inclusive scan of v over the workgroup of 1024; *total gets the sum.
template <typename Int>
__device__ Int scan_1024(Int v, Int *total)
{
    __shared__ Int sums[16];
    const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
    if constexpr (sizeof(Int) == 4) {
        v = dev::wave_scan(v);
    } else {
#pragma unroll
        for (int m = 1; m < kWave; m *= 2) {
            const Int u = __shfl_up(v, m);
            v += lane >= m ? u : 0;
        }
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

// The held pages before each group of words, in LDS: kMost + 1 counts, with
// kOne a word to a group and the words in LDS too (a copy, or there already), else
// as many words to a group as it takes (262144 pages, 512 rows of 1024, us, words in
// LDS / in memory: update 22.0 / 24.7, compaction 22.9 / 33.5).
template <int kMost, bool kOne>
struct Counts {
    const uint32_t *used;
    int pages, words;
    int span, groups;  // words of a group; groups that have words
    const int32_t *before;

    // Called by all 1024 threads; each counts neighbouring groups.  With kOne `from` is
    // in LDS, kMost words of which those beyond the pages are 0.
    __device__ Counts(const uint32_t *from, int64_t pages_, int32_t *lds) : used(from), pages((int)pages_), before(lds)
    {
        constexpr int kEach = kMost / 1024;
        words = (int)words_of(pages);
        span = kOne ? 1 : (words + kMost - 1) / kMost;
        groups = kOne ? words : (words + span - 1) / span;
        int n[kEach], mine = 0;
#pragma unroll
        for (int g = 0; g < kEach; ++g) {
            n[g] = 0;
            if constexpr (kOne) {
                n[g] = __popc(from[threadIdx.x * kEach + g]);
            } else {
                const int64_t first = ((int64_t)threadIdx.x * kEach + g) * span;
                for (int64_t w = first; w < first + span && w < words; ++w) {
                    n[g] += __popc(from[w]);
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
            lds[kMost] = total;
        }
        __syncthreads();
    }
    __device__ int held() const { return before[kMost]; }
    // Held pages before `page` (at most `pages`).
    __device__ int rank(int page) const
    {
        const int word = page / 32, g = kOne ? word : word / span;
        int n = before[g];
        if constexpr (!kOne) {
            for (int w = g * span; w < word; ++w) {
                n += __popc(used[w]);
            }
        }
        return page < pages ? n + __popc(used[word] & ((1u << (page % 32)) - 1u)) : held();
    }
    __device__ int free_before(int g) const { return (int)((int64_t)g * span * 32 - before[g]); }
    // LDS for `words` places; starts[k / 32] becomes the word of free page 32 (k / 32), from
    // where a search for the k-th goes word by word: 1 / 2 f words where a share f of the pages
    // is free and they lie evenly, all of them at worst.  All 1024 threads.
    __device__ void index(uint16_t *starts) const
    {
        static_assert(kOne, "a word to a group");
        for (int w = (int)threadIdx.x; w < words; w += 1024) {
            const int low = free_before(w), at = (low + 31) / 32;
            if (at * 32 < low + 32 - (int)__popc(used[w])) {
                starts[at] = (uint16_t)w;
            }
        }
        __syncthreads();
    }
    __device__ int free_page(int k, const uint16_t *starts) const
    {
        int w = starts[k / 32];
        while (w + 1 < words && free_before(w + 1) <= k) {
            ++w;
        }
        return free_in(w, k);
    }
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
        return free_in(low, k);
    }
    // ... which is in group low.
    __device__ int free_in(int low, int k) const
    {
        k -= free_before(low);
        int w = low * span;
        uint32_t f = ~used[w];
        if constexpr (!kOne) {
            for (int n = __popc(f); k >= n; n = __popc(f)) {
                k -= n;
                f = ~used[++w];
            }
        }
        int bit = 0;  // the k-th set bit of f
#pragma unroll
        for (int half = 16; half > 0; half /= 2) {
            const int n = __popc(f & ((1u << half) - 1u));
            if (k >= n) {
                k -= n;
                f >>= half;
                bit += half;
            }
        }
        return w * 32 + bit;
    }
};

// One workgroup: which rows get their pages, and the list of the free pages
// given out.
template <bool kOne>
__global__ __launch_bounds__(1024) void update_grants(CacheUpdateArgs a, const uint32_t *used, const uint32_t *many,
                                                      const Found *found, Grant *grants, int32_t *list)
{
    __shared__ __align__(16) int32_t lds[kGroups + 1];
    __shared__ __align__(16) uint32_t copy[kOne ? kGroups : 4], shared[kOne ? kGroups : 4];
    const int me = (int)threadIdx.x;
    const auto load = [&](int64_t r) {
        Found f{};
        f.last = -1;
        if (r < a.rows) {
            f.row.add = found[r].row.add;
            f.row.held = found[r].row.held;
            f.row.grown = found[r].row.grown;
            f.last = found[r].last;
        }
        return f;
    };
    Found next = load(me);  // (on its way while the words are counted)
    if constexpr (kOne) {
        const Words one(used, (int)words_of(a.pages)), two(many, (int)words_of(a.pages));
        one.put(copy);
        two.put(shared);
        __syncthreads();
    }
    const uint32_t *twice = kOne ? shared : many;
    const Counts<kGroups, kOne> counts(kOne ? copy : used, a.pages, lds);
    const int64_t free = a.pages - counts.held();
    int64_t asked = 0;
    for (int64_t r0 = 0; r0 < a.rows; r0 += 1024) {
        const int64_t r = r0 + me;
        const Found f = next;
        next = load(r + 1024);
        const int swap = f.last >= 0 ? (int)(twice[f.last / 32] >> (f.last % 32) & 1u) : 0;
        const int64_t need = swap + f.row.grown - f.row.held;
        int64_t total;
        const int64_t upto = asked + scan_1024<int64_t>(need, &total);
        asked += total;
        if (r < a.rows) {
            const bool served = f.row.add > 0 && (need == 0 || upto <= free);
            grants[r] = Grant{served ? (int32_t)(need == 0 ? 0 : upto - need) : -1, served ? swap : 0};
        }
    }
    const int64_t given = asked < free ? asked : free;
    for (int g = me; g < counts.groups; g += 1024) {
        int k = counts.free_before(g);
        for (int w = g * counts.span; w < (g + 1) * counts.span && w < counts.words && k < given; ++w) {
            for (uint32_t f = ~counts.used[w]; f != 0u && k < given; f &= f - 1u) {
                list[k++] = w * 32 + __ffs(f) - 1;
            }
        }
    }
}

// One wave per row: the columns that its new tokens change, its slots and the
// rest of its state.
__global__ __launch_bounds__(256) void update_finish(CacheUpdateArgs a, const Found *found, const Grant *grants,
                                                     const int32_t *list)
{
    const int lane = (int)threadIdx.x % kWave;
    const int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (r >= a.rows) {
        return;
    }
    const Row row = found[r].row;
    const int last = found[r].last;
    const Grant grant = grants[r];
    const bool served = grant.first >= 0, copy = grant.copy != 0;
    const int32_t *mine = list + (served ? grant.first : 0);
    const auto column = [&](int j) -> int {  // of the new row, j in [open, end)
        if (j >= row.held) {
            return served ? mine[copy + j - row.held] : -1;
        }
        return copy ? mine[0] : last;
    };
    for (Column j = (Column)row.open + lane; j < (Column)row.end; j += kWave) {
        a.newTable[r * a.width + j] = column((int)j);
    }
    const int granted = served ? row.add : 0;
    for (int i = lane; i < a.tokens; i += kWave) {
        const uint32_t t = (uint32_t)row.rest + (uint32_t)i, past = t / (uint32_t)a.pageSize;
        const int page = i < granted ? column(row.full + (int)past) : -1;
        a.slots[r * a.tokens + i] = page >= 0 ? (int64_t)page * a.pageSize + (t - past * (uint32_t)a.pageSize) : -1;
    }
    if (lane == 0) {
        a.newLengths[r] = row.length + granted;
        a.granted[r] = granted;
        a.src[r] = copy ? last : -1;
        a.dst[r] = copy ? mine[0] : -1;
    }
}

// The cells of a table as 1024 threads take them: narrow tables several rows at a
// time, wide ones 1024 columns.  f(j, r, step): the thread's cells at column j in rows
// r, r + step, ..., kSmallBatch of them (those below `rows`).
template <typename F>
__device__ __forceinline__ void each_cells(int rows, int width, F f)
{
    const int step = width < 1024 ? 1024 / width : 1;
    const int row0 = width < 1024 ? (int)threadIdx.x / width : 0;
    for (int j = (int)threadIdx.x - row0 * width; j < width; j += 1024) {
        for (int r = row0 < step ? row0 : rows; r < rows; r += step * kSmallBatch) {
            f(j, r, step);
        }
    }
}

// All of it by one workgroup, the bitmaps and the rows in its LDS.  `lanes`
// threads share a row's columns and slots.
__global__ __launch_bounds__(1024) void update_small(CacheUpdateArgs a, int lanes)
{
    __shared__ __align__(16) uint32_t used[kSmallWords], many[kSmallWords];
    __shared__ __align__(16) int32_t lds[kSmallWords + 1];
    __shared__ Row rows[kSmallRows];
    __shared__ int32_t lasts[kSmallRows], first[kSmallRows];
    const int me = (int)threadIdx.x;
    for (int w = me; w < kSmallWords; w += 1024) {
        used[w] = many[w] = 0u;
    }
    if (me < a.rows) {
        rows[me] = Row(a, me);
        lasts[me] = -1;
    }
    __syncthreads();
    each_cells(a.rows, a.width, [&](int j, int r0, int step) {
        int page[kSmallBatch];
#pragma unroll
        for (int n = 0; n < kSmallBatch; ++n) {
            const int r = r0 + n * step;
            const Row &row = rows[r < a.rows ? r : 0];
            page[n] = row.entry_if(a, j, r < a.rows && j < row.held);
        }
#pragma unroll
        for (int n = 0; n < kSmallBatch; ++n) {
            const int r = r0 + n * step;
            if (r < a.rows) {
                if (j < rows[r].open || j >= rows[r].end) {
                    a.newTable[r * a.width + j] = page[n];
                } else if (j < rows[r].held) {
                    lasts[r] = page[n];  // the partly filled page
                }
            }
        }
        mark_all(page, used, many);
    });
    __syncthreads();
    const Counts<kSmallWords, true> counts(used, a.pages, lds);
    const auto wants = [&](int r) { return lasts[r] >= 0 && (many[lasts[r] / 32] >> (lasts[r] % 32) & 1u) != 0u; };
    {
        const int need = me < a.rows ? wants(me) + rows[me].grown - rows[me].held : 0;
        int total;
        const int upto = scan_1024(need, &total);
        if (me < a.rows) {
            const bool served = rows[me].add > 0 && (need == 0 || upto <= a.pages - counts.held());
            first[me] = served ? upto - need : -1;
        }
    }
    __syncthreads();
    const int lane = me % lanes;
    for (int r = me / lanes; r < a.rows; r += 1024 / lanes) {
        const Row row = rows[r];
        const int from = first[r], last = lasts[r];
        const bool served = from >= 0, copy = served && wants(r);
        const int own = copy ? counts.free_page(from) : last;  // the page of the column before held
        const auto column = [&](int j) {
            return j < row.held ? own : served ? counts.free_page(from + copy + j - row.held) : -1;
        };
        for (int j = row.open + lane; j < row.end; j += lanes) {
            a.newTable[r * a.width + j] = column(j);
        }
        const int granted = served ? row.add : 0;
        for (int i = lane; i < a.tokens; i += lanes) {
            const uint32_t t = (uint32_t)row.rest + (uint32_t)i, past = t / (uint32_t)a.pageSize;
            const int page = i < granted ? column(row.full + (int)past) : -1;
            a.slots[(int64_t)r * a.tokens + i] =
                page >= 0 ? (int64_t)page * a.pageSize + (t - past * (uint32_t)a.pageSize) : -1;
        }
        if (lane == 0) {
            a.newLengths[r] = row.length + granted;
            a.granted[r] = granted;
            a.src[r] = copy ? last : -1;
            a.dst[r] = copy ? own : -1;
        }
    }
}

// Pages that row r holds as mhcCacheCompact sees it, and its column j < that.
__device__ __forceinline__ int held_pages(const CacheCompactArgs &a, int64_t r)
{
    return pages_for((uint32_t)clamped(a.lengths[r], a.width * a.pageSize), a.pageSize);
}

// (A load in any case, as Row::entry_if's.)
__device__ __forceinline__ int held_entry(const CacheCompactArgs &a, int64_t r, Column j, bool on)
{
    const int page = a.table[on ? r * a.width + j : 0];
    return on && page >= 0 && page < a.pages ? page : -1;
}

__global__ __launch_bounds__(256) void compact_mark(CacheCompactArgs a, uint32_t *used)
{
    const int64_t r = blockIdx.x;
    const Column held = (Column)held_pages(a, r);
    for (Column j0 = threadIdx.x; j0 < held; j0 += 256 * kBatch) {
        int page[kBatch];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            page[n] = held_entry(a, r, j0 + 256 * n, j0 + 256 * n < held);
        }
        mark_all(page, used, nullptr);
    }
}

// Every workgroup counts for itself, then does its part: of the moves, and of
// the table, cut into pieces of 512 columns of a row, a wave's each.
template <bool kOne>
__global__ __launch_bounds__(1024) void compact_apply(CacheCompactArgs a, const uint32_t *used)
{
    __shared__ __align__(16) int32_t lds[kGroups + 1];
    __shared__ __align__(16) uint32_t copy[kOne ? kGroups : 4];
    __shared__ uint16_t starts[kOne ? kGroups : 1];
    constexpr int kPieces = 8, kColumns = kWave * kPieces;
    const Column width = (Column)a.width;
    const int pieces = (int)((width + kColumns - 1) / kColumns);
    const int64_t waves = 16 * (int64_t)gridDim.x;
    int64_t n = (int64_t)blockIdx.x * 16 + threadIdx.x / kWave, r = 0;
    Column j0 = 0;
    int page[kPieces];
    const auto load = [&]() {
        r = n / pieces;
        j0 = (Column)(n - r * pieces) * kColumns + threadIdx.x % kWave;
        const Column held = r < a.rows ? (Column)held_pages(a, r) : 0;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            page[i] = held > 0 ? held_entry(a, r, j0 + i * kWave, j0 + i * kWave < held) : -1;
        }
    };
    load();  // (on its way while the words are counted)
    if constexpr (kOne) {
        const Words words(used, (int)words_of(a.pages));
        words.put(copy);
        __syncthreads();
    }
    const Counts<kGroups, kOne> counts(kOne ? copy : used, a.pages, lds);
    if constexpr (kOne) {
        counts.index(starts);
    }
    const auto to = [&](int k) {  // the k-th free page
        if constexpr (kOne) {
            return counts.free_page(k, starts);
        } else {
            return counts.free_page(k);
        }
    };
    const int U = counts.held(), stay = counts.rank(U);
    for (;;) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (page[i] >= U) {
                page[i] = to(counts.rank(page[i]) - stay);
            }
            if (r < a.rows && j0 + i * kWave < width) {
                a.newTable[r * a.width + j0 + i * kWave] = page[i];
            }
        }
        n += waves;
        if (n >= (int64_t)a.rows * pieces) {
            break;
        }
        load();
    }
    const int64_t at = (int64_t)blockIdx.x * 1024 + threadIdx.x, all = (int64_t)gridDim.x * 1024;
    if (at == 0) {
        a.used[0] = U;
    }
    for (int64_t x = U + at; x < a.pages; x += all) {
        if ((counts.used[x / 32] >> (x % 32) & 1u) != 0u) {
            const int k = counts.rank((int)x) - stay;
            a.src[k] = (int32_t)x;
            a.dst[k] = to(k);
        }
    }
    for (int64_t k = U - stay + at; k < a.pages / 2; k += all) {
        a.src[k] = a.dst[k] = -1;
    }
}

// All of it by one workgroup, the bitmap, the rows' pages and the moves'
// destinations in its LDS.
__global__ __launch_bounds__(1024) void compact_small(CacheCompactArgs a)
{
    __shared__ uint32_t used[kSmallWords];
    __shared__ int32_t lds[kSmallWords + 1], held[kSmallRows];
    __shared__ uint16_t to[kSmallPages / 2];
    const int me = (int)threadIdx.x;
    for (int w = me; w < kSmallWords; w += 1024) {
        used[w] = 0u;
    }
    if (me < a.rows) {
        held[me] = held_pages(a, me);
    }
    __syncthreads();
    int page[kSmallBatch];
    int pageColumn = -1, pageRow = -1;  // the cells of `page`: the last ones marked, for most the only ones
    const auto load = [&](int j, int r0, int step) {
        if (j == pageColumn && r0 == pageRow) {
            return;
        }
        pageColumn = j;
        pageRow = r0;
#pragma unroll
        for (int n = 0; n < kSmallBatch; ++n) {
            const int r = r0 + n * step;
            page[n] = held_entry(a, r, j, r < a.rows && j < held[r < a.rows ? r : 0]);
        }
    };
    each_cells(a.rows, a.width, [&](int j, int r, int step) {
        load(j, r, step);
        mark_all(page, used, nullptr);
    });
    __syncthreads();
    const Counts<kSmallWords, true> counts(used, a.pages, lds);
    const int U = counts.held(), stay = counts.rank(U), moves = U - stay;
    if (me == 0) {
        a.used[0] = U;
    }
    for (int w = me; w < counts.words; w += 1024) {
        // The free pages below U and the held ones from U on, in order.
        const int below = U - w * 32;  // the word's pages that are
        const uint32_t low = below >= 32 ? 0xFFFFFFFFu : below <= 0 ? 0u : (1u << below) - 1u;
        int k = counts.free_before(w);
        for (uint32_t f = ~used[w] & low; f != 0u; f &= f - 1u, ++k) {
            to[k] = (uint16_t)(w * 32 + __ffs(f) - 1);
            a.dst[k] = w * 32 + __ffs(f) - 1;
        }
        k = counts.rank(w * 32 < U ? U : w * 32) - stay;
        for (uint32_t f = used[w] & ~low; f != 0u; f &= f - 1u, ++k) {
            a.src[k] = w * 32 + __ffs(f) - 1;
        }
    }
    for (int k = moves + me; k < a.pages / 2; k += 1024) {
        a.src[k] = a.dst[k] = -1;
    }
    __syncthreads();
    each_cells(a.rows, a.width, [&](int j, int r0, int step) {
        load(j, r0, step);
#pragma unroll
        for (int n = 0; n < kSmallBatch; ++n) {
            if (r0 + n * step < a.rows) {
                a.newTable[(r0 + n * step) * a.width + j] =
                    page[n] >= U ? to[counts.rank(page[n]) - stay] : page[n];
            }
        }
    });
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
constexpr int64_t kCacheBytes = int64_t{256} << 20;  // the last-level cache

// The stores pass the caches by (nobody reads the copies soon); the loads too where
// more is moved than the last-level cache holds.  2000 pages of 128 KB twice, us:
// neither 208, stores 202.5, both 196.4; 480 pages of 32 KB twice 12.1 / 12.0 / 15.4.
template <typename Vec, bool kStream>
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
                const Vec *from = reinterpret_cast<const Vec *>(c.base + src * c.page + inside);
                held[j] = kStream ? __builtin_nontemporal_load(from) : *from;
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (at[j] >= 0) {
                __builtin_nontemporal_store(held[j], reinterpret_cast<Vec *>(c.base + dst * c.page + at[j]));
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
    const bool stream_by = 2 * a.n * pieces * (int64_t)sizeof(Vec) > kCacheBytes;
    hipLaunchKernelGGL((stream_by ? copy_pieces<Vec, true> : copy_pieces<Vec, false>),
                       dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, k, v, a.src, a.dst, a.n,
                       a.pages, pieces, perPage);
    return hipGetLastError();
}

size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

template <typename Args>
bool small(const Args &a)
{
    return a.rows <= kSmallRows && a.pages <= kSmallPages && (int64_t)a.rows * a.width <= kSmallEntries;
}

hipError_t clear(uint32_t *words, int64_t n, hipStream_t stream)
{
    const int64_t blocks = (n + 1023) / 1024;
    hipLaunchKernelGGL(clear_words, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, stream, words, n);
    return hipGetLastError();
}

}  // namespace

// [used bits][many bits][Found: rows][Grant: rows][list: pages]
size_t cache_update_workspace(const CacheUpdateArgs &a)
{
    return small(a) ? 0
                    : 2 * align_up(words_of(a.pages) * 4) + align_up((size_t)a.rows * sizeof(Found)) +
                          align_up((size_t)a.rows * sizeof(Grant)) + align_up((size_t)a.pages * 4);
}

hipError_t launch_cache_update(const CacheUpdateArgs &a, void *workspace, int, hipStream_t stream)
{
    char *ws = static_cast<char *>(workspace);
    if (small(a)) {
        int lanes = 1;
        while (lanes < kWave && lanes * 4 < a.tokens) {
            lanes *= 2;
        }
        hipLaunchKernelGGL(update_small, dim3(1), dim3(1024), 0, stream, a, lanes);
        return hipGetLastError();
    }
    const size_t bits = align_up(words_of(a.pages) * 4);
    uint32_t *used = reinterpret_cast<uint32_t *>(ws), *many = reinterpret_cast<uint32_t *>(ws + bits);
    ws += 2 * bits;
    Found *found = reinterpret_cast<Found *>(ws);
    ws += align_up((size_t)a.rows * sizeof(Found));
    Grant *grant = reinterpret_cast<Grant *>(ws);
    int32_t *list = reinterpret_cast<int32_t *>(ws + align_up((size_t)a.rows * sizeof(Grant)));
    hipError_t err = clear(used, (int64_t)(2 * bits / 4), stream);
    if (err != hipSuccess) {
        return err;
    }
    hipLaunchKernelGGL(update_rows, dim3((unsigned)a.rows), dim3(256), 0, stream, a, used, many, found);
    if ((err = hipGetLastError()) != hipSuccess) {
        return err;
    }
    const auto grants = words_of(a.pages) <= kGroups ? update_grants<true> : update_grants<false>;
    hipLaunchKernelGGL(grants, dim3(1), dim3(1024), 0, stream, a, used, many, found, grant, list);
    if ((err = hipGetLastError()) != hipSuccess) {
        return err;
    }
    hipLaunchKernelGGL(update_finish, dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, stream, a, found, grant, list);
    return hipGetLastError();
}

size_t cache_compact_workspace(const CacheCompactArgs &a) { return small(a) ? 0 : align_up(words_of(a.pages) * 4); }

hipError_t launch_cache_compact(const CacheCompactArgs &a, void *workspace, int cus, hipStream_t stream)
{
    if (small(a)) {
        hipLaunchKernelGGL(compact_small, dim3(1), dim3(1024), 0, stream, a);
        return hipGetLastError();
    }
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
    const auto apply = words_of(a.pages) <= kGroups ? compact_apply<true> : compact_apply<false>;
    hipLaunchKernelGGL(apply, dim3((unsigned)cus), dim3(1024), 0, stream, a, used);
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
