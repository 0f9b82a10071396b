// Attention over the pages that a score ranks highest (mhcSparseAttention): the
// scores, the selection, and the host side.  The attention itself is the kernel of
// single tokens (mhc_paged_attention.h) with a table of each kv head's own.
//
// A page's score is up . hi + down . lo with the sums of the positive and of the
// negative parts of the query heads that share the kv head, so that a page costs
// 2 d products however many heads there are.  It is computed in 64 bits, whose
// roundings lie far below the differences between pages: which page is the last one
// taken does not hang on the order of a sum.  A score becomes an integer of the
// same order; the top-th of them is found by histograms of 256 bins over a
// range that narrows to one bin, and what lies above it is written in order.
//
// 16 sequences of 131072 tokens at most, 64 heads to 8 of 128, 256 pages of 16 for each: scores
// 60 us (196 MB at 3.3 TB/s, bound by the 64-bit arithmetic and the loads together: alone these
// take 40 and 47), selection 13.5 (one workgroup a kv head: its rounds follow each other),
// attention 56 (244 MB at 4.4 TB/s).  One sequence, 64 pages of 64: 7.8, 9.0 and 12.2 us, all
// of them chains of loads.

#include "mhc_paged_attention.h"

namespace mhc {
namespace sparse {
namespace {

using dev::kWave;
using dev::u32x4_t;

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kBatch = 4;  // pages that a group of lanes scores at once

// Scores as ordered integers; what cannot be taken is 0.
constexpr uint64_t kAlways = ~0ull, kNotANumber = ~0ull - 1;

struct Args {
    SparseAttentionArgs a;
    uint64_t *keys;     // [B * kvHeads, width]
    int32_t *table;     // [B * kvHeads, top]: the pages taken
    int32_t *lengths;   // [B * kvHeads]: their tokens
    int columns;        // of a workgroup's item
    int heads;          // kv heads of a workgroup's item: 4, 2 or 1, of its waves each does one's
};

// Columns that row b of the batch holds, and its tokens.
struct Row {
    int length, held;
    __device__ Row(const PagedAttentionArgs &a, int b)
    {
        const int most = a.width * a.pageSize;
        length = a.lengths[b];
        length = length < 0 ? 0 : length > most ? most : length;
        held = length == 0 ? 0 : (length - 1) / a.pageSize + 1;
    }
};

__device__ __forceinline__ double shuffled(double v, int mask)
{
    const uint64_t bits = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)bits, mask), hi = (uint32_t)__shfl_xor((int)(bits >> 32), mask);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// kLanes lanes do a page, 8 dimensions each.
template <bool kBf16, int kLanes>
__global__ __launch_bounds__(kThreads) void score_pages(Args args)
{
    const SparseAttentionArgs &s = args.a;
    const PagedAttentionArgs &a = s.attention;
    constexpr int kPages = kWave / kLanes;  // of a wave at a time
    const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
    const int sub = lane % kLanes, e = 8 * sub;
    const bool on = e < a.d;
    const int group = a.heads / a.kvHeads, chunks = (a.width + args.columns - 1) / args.columns;
    const int headGroups = (a.kvHeads + args.heads - 1) / args.heads, perHead = kWaves / args.heads;
    const int64_t items = (int64_t)a.B * headGroups * chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int chunk = (int)(item % chunks), b = (int)(item / chunks / headGroups);
        const int kv = (int)(item / chunks % headGroups) * args.heads + wave / perHead, column0 = chunk * args.columns;
        const int64_t row = (int64_t)b * a.kvHeads + kv;
        const Row r(a, b);
        if (column0 >= r.held || kv >= a.kvHeads) {
            continue;
        }
        const int end = r.held - column0 < args.columns ? r.held : column0 + args.columns;
        const int32_t *table = a.table + (int64_t)b * a.width;
        // The pages of a step are known a step ahead.
        const int step = perHead * kPages;
        int c0 = column0 + wave % perHead * kPages + lane / kLanes;
        int next[kBatch];
        const auto find = [&](int from) {
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const int c = from + x * step;
                next[x] = table[c < end ? c : column0];
            }
        };
        find(c0);
        double up[8], down[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            up[x] = down[x] = 0;
        }
        const uint16_t *q = static_cast<const uint16_t *>(a.q.data) + b * a.q.row + (int64_t)kv * group * a.q.head +
                            (on ? e : 0);
        for (int h0 = 0; h0 < group; h0 += 4) {
            u32x4_t heads[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                heads[y] = *reinterpret_cast<const u32x4_t *>(q + (h0 + y < group ? h0 + y : h0) * a.q.head);
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                if (h0 + y < group) {
                    float f[8];
                    dev::unpack8<kBf16>(heads[y], f);
#pragma unroll
                    for (int x = 0; x < 8; ++x) {  // (NaN goes to both)
                        up[x] += f[x] < 0.f ? 0.0 : (double)f[x];
                        down[x] += f[x] > 0.f ? 0.0 : (double)f[x];
                    }
                }
            }
        }
        const uint16_t *loBase = static_cast<const uint16_t *>(s.lo.data) + kv * s.lo.head + (on ? e : 0);
        const uint16_t *hiBase = static_cast<const uint16_t *>(s.hi.data) + kv * s.hi.head + (on ? e : 0);
        struct Bounds {
            u32x4_t lo[kBatch], hi[kBatch];
            uint32_t good;  // pages there are, a bit each
        };
        const auto load = [&](Bounds &p, int from) {
            p.good = 0;
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const bool good = next[x] >= 0 && next[x] < a.pages && from + x * step < end;
                p.good |= good ? 1u << x : 0u;
                const int64_t page = good ? next[x] : 0;  // (no page: the first one is read, and not used)
                p.lo[x] = *reinterpret_cast<const u32x4_t *>(loBase + page * s.lo.row);
                p.hi[x] = *reinterpret_cast<const u32x4_t *>(hiBase + page * s.hi.row);
            }
            find(from + kBatch * step);
        };
        const auto score = [&](const Bounds &p, int from) {
            double sum[kBatch];
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                float l[8], h[8];
                dev::unpack8<kBf16>(p.lo[x], l);
                dev::unpack8<kBf16>(p.hi[x], h);
                sum[x] = 0;
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    sum[x] = __builtin_fma(up[y], (double)h[y], sum[x]);
                    sum[x] = __builtin_fma(down[y], (double)l[y], sum[x]);
                }
                sum[x] = on ? sum[x] : 0;  // (whatever lies behind a head's dimensions)
            }
            // Over the lanes: in the first two steps a lane gives its neighbour the sums of half of
            // the pages and goes on with the others', so that one is left, page sub % 4's.
            const bool odd = (sub & 1) != 0, second = (sub & 2) != 0;
            double two[2], one;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                two[x] = (odd ? sum[2 * x + 1] : sum[2 * x]) + shuffled(odd ? sum[2 * x] : sum[2 * x + 1], 1);
            }
            one = (second ? two[1] : two[0]) + shuffled(second ? two[0] : two[1], 2);
#pragma unroll
            for (int mask = 4; mask < kLanes; mask *= 2) {
                one += shuffled(one, mask);
            }
            one += 0.0;  // (-0 is 0)
            const uint64_t bits = (uint64_t)__double_as_longlong(one);
            uint64_t key = bits >> 63 != 0 ? ~bits : bits | 1ull << 63;
            key = one != one ? kNotANumber : key;
            const int c = from + sub * step;
            key = c < s.first || c >= r.held - s.last ? kAlways : key;
            if (sub < kBatch && c < end) {
                args.keys[row * a.width + c] = (p.good >> sub & 1u) != 0u ? key : 0;
            }
        };
        // The next pages' bounds are on their way while these are scored.
        Bounds here, ahead;
        load(here, c0);
        for (; c0 - lane / kLanes < end; c0 += 2 * kBatch * step) {
            load(ahead, c0 + kBatch * step);
            score(here, c0);
            load(here, c0 + 2 * kBatch * step);
            score(ahead, c0 + kBatch * step);
        }
    }
}

// The highest `top` keys of a (sequence, kv head), in order.  A thread has kHeld columns
// that follow each other (in registers; where the table is wider, segment by segment, read
// anew in each round).  Up to 2048 columns a thread has 2, which come sooner than 8: 64 of 2048
// 9.0 us, with 8 11.6.
constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave, kBins = 256;
constexpr int kMostHeld = 8;

template <typename F>
__device__ __forceinline__ uint64_t reduced(uint64_t v, F &&f)
{
#pragma unroll
    for (int mask = 1; mask < kWave; mask *= 2) {
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, mask), hi = (uint32_t)__shfl_xor((int)(v >> 32), mask);
        v = f(v, (uint64_t)hi << 32 | lo);
    }
    return v;
}

template <int kHeld, bool kOneSegment>
__global__ __launch_bounds__(kSelectThreads) void select_pages(Args args)
{
    constexpr int kSegment = kSelectThreads * kHeld;
    __shared__ uint64_t least[kSelectWaves], greatest[kSelectWaves], counts[kSelectWaves];
    __shared__ int bins[kBins];
    __shared__ uint64_t rangeLow;
    __shared__ int rangeNeed, rangeIn;
    __shared__ int before[kSelectWaves], tiesBefore[kSelectWaves];
    __shared__ int lastTaken;
    const SparseAttentionArgs &s = args.a;
    const PagedAttentionArgs &a = s.attention;
    const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
    const int64_t row = blockIdx.x;
    const int b = (int)(row / a.kvHeads);
    const Row r(a, b);
    const uint64_t *all = args.keys + row * a.width;
    uint64_t keys[kHeld];
    const int segments = kOneSegment ? 1 : (r.held + kSegment - 1) / kSegment;
    const auto read = [&](int segment) {
#pragma unroll
        for (int x = 0; x < kHeld; ++x) {
            const int c = segment * kSegment + (int)threadIdx.x * kHeld + x;
            keys[x] = c < r.held ? all[c] : 0;
        }
    };
    const auto each_segment = [&](auto &&f) {
        for (int segment = 0; segment < segments; ++segment) {
            if (!kOneSegment) {
                read(segment);
            }
            f(segment);
        }
    };
    if (kOneSegment) {
        read(0);
    }

    // How many can be taken, how many are in any case, and the others' range.
    uint64_t low = kAlways, high = 0, count = 0;  // count: of the first in the lower half, of the second in the upper
    each_segment([&](int) {
#pragma unroll
        for (int x = 0; x < kHeld; ++x) {
            const uint64_t key = keys[x];
            count += (key != 0 ? 1ull : 0ull) + (key == kAlways ? 1ull << 32 : 0ull);
            const bool ranked = key != 0 && key != kAlways;
            low = ranked && key < low ? key : low;
            high = ranked && key > high ? key : high;
        }
    });
    low = reduced(low, [](uint64_t x, uint64_t y) { return x < y ? x : y; });
    high = reduced(high, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
    count = reduced(count, [](uint64_t x, uint64_t y) { return x + y; });
    if (threadIdx.x == 0) {
        lastTaken = 0;
    }
    if (lane == 0) {
        least[wave] = low;
        greatest[wave] = high;
        counts[wave] = count;
    }
    if ((int)threadIdx.x < kBins) {
        bins[threadIdx.x] = 0;
    }
    __syncthreads();
    count = 0;
#pragma unroll
    for (int x = 0; x < kSelectWaves; ++x) {
        low = least[x] < low ? least[x] : low;
        high = greatest[x] > high ? greatest[x] : high;
        count += counts[x];
    }
    // Taken: keys above `floor`, and the first `ties` of those that equal it.
    uint64_t floor = 0;
    int ties = 0;
    if ((int)(uint32_t)count > s.top) {
        int need = s.top - (int)(count >> 32);  // of the keys in [low, high]
        if (need == 0) {
            floor = kAlways - 1;
        }
        while (need > 0) {
            int shift = 0;
            if ((high - low) / kBins != 0) {
                shift = 64 - __clzll((long long)((high - low) / kBins));
            }
            each_segment([&](int) {
#pragma unroll
                for (int x = 0; x < kHeld; ++x) {
                    if (keys[x] >= low && keys[x] <= high) {
                        atomicAdd(&bins[(keys[x] - low) >> shift], 1);
                    }
                }
            });
            __syncthreads();
            if (wave == 0) {
                // From the top: the bin at which `need` is reached.
                int mine[kBins / kWave], sum = 0;
#pragma unroll
                for (int x = 0; x < kBins / kWave; ++x) {
                    mine[x] = bins[kBins - 1 - (lane * (kBins / kWave) + x)];
                    sum += mine[x];
                }
                int above = dev::wave_scan(sum) - sum;
#pragma unroll
                for (int x = 0; x < kBins / kWave; ++x) {
                    const int bin = kBins - 1 - (lane * (kBins / kWave) + x);
                    if (above < need && above + mine[x] >= need) {
                        rangeLow = low + ((uint64_t)bin << shift);
                        rangeNeed = need - above;
                        rangeIn = mine[x];
                    }
                    above += mine[x];
                    bins[bin] = 0;
                }
            }
            __syncthreads();
            low = rangeLow;
            need = rangeNeed;
            const uint64_t wide = (1ull << shift) - 1;
            high = high - low < wide ? high : low + wide;
            if (rangeIn == need) {
                floor = low - 1;
                need = 0;
            } else if (shift == 0) {
                floor = low;
                ties = need;
                need = 0;
            }
            __syncthreads();  // (rangeLow and the others are read)
        }
    }
    // In the columns' order.
    int taken = 0, equal = 0;
    int32_t *columns = s.columns + row * s.top, *table = args.table + row * s.top;
    each_segment([&](int segment) {
        int tied = 0, takes = 0;
#pragma unroll
        for (int x = 0; x < kHeld; ++x) {
            tied += ties > 0 && keys[x] == floor ? 1 : 0;
        }
        int rank = 0;  // of the thread's first tie
        if (ties > 0) {
            const int upto = dev::wave_scan(tied);
            if (lane == kWave - 1) {
                tiesBefore[wave] = upto;
            }
            __syncthreads();
            rank = equal + upto - tied;
#pragma unroll
            for (int x = 0; x < kSelectWaves; ++x) {
                rank += x < wave ? tiesBefore[x] : 0;
                equal += tiesBefore[x];
            }
        }
        uint32_t mine = 0;
#pragma unroll
        for (int x = 0; x < kHeld; ++x) {
            const bool tie = ties > 0 && keys[x] == floor;
            const bool take = keys[x] > floor || (tie && rank < ties);
            rank += tie ? 1 : 0;
            mine |= take ? 1u << x : 0u;
        }
        takes = __popc(mine);
        const int upto = dev::wave_scan(takes);
        if (lane == kWave - 1) {
            before[wave] = upto;
        }
        __syncthreads();
        int at = taken + upto - takes;
#pragma unroll
        for (int x = 0; x < kSelectWaves; ++x) {
            at += x < wave ? before[x] : 0;
            taken += before[x];
        }
#pragma unroll
        for (int x = 0; x < kHeld; ++x) {
            if ((mine >> x & 1u) != 0u) {
                const int c = segment * kSegment + (int)threadIdx.x * kHeld + x;
                columns[at] = c;
                table[at] = a.table[(int64_t)b * a.width + c];
                ++at;
                if (c == r.held - 1) {
                    lastTaken = 1;
                }
            }
        }
        __syncthreads();
    });
    for (int x = taken + (int)threadIdx.x; x < s.top; x += kSelectThreads) {
        columns[x] = table[x] = -1;
    }
    if (threadIdx.x == 0) {  // (the last column may be filled in part)
        args.lengths[row] = taken * a.pageSize - (lastTaken != 0 ? r.held * a.pageSize - r.length : 0);
    }
}

// kv heads of a workgroup's item: those of a page lie together in memory (with 1 / 2 / 4: 210 /
// 147 / 130 us for the 16 sequences above, 39.7 / 33.3 / 32.1 for the one).
int heads_of(const PagedAttentionArgs &a) { return a.kvHeads >= 4 ? 4 : a.kvHeads >= 2 ? 2 : 1; }

// Columns of an item: enough items for all CUs, and beyond that long ones, whose start
// (lengths, query heads) costs as much as some dozens of columns.  us with 16 / 32 / 64 / 128 / 256:
// the 16 sequences above (8192 columns, 2 groups of heads) 191 / 142 / 130 / 133 / 139, the one
// (2048 columns) 32.0 / 31.6 / 33.2 / 37.3 / 44.7.
int columns_of(const PagedAttentionArgs &a)
{
    const int64_t all = (int64_t)a.B * a.kvHeads / heads_of(a) * a.width;
    return all <= (int64_t)16 * 2048 ? 16 : 64;
}

// The attention's call: a row for each kv head of a sequence.
PagedAttentionArgs rows_of(const SparseAttentionArgs &s, int32_t *table, int32_t *lengths)
{
    PagedAttentionArgs a = s.attention;
    a.B *= a.kvHeads;
    a.heads /= a.kvHeads;
    a.kvHeads = 1;
    a.width = s.top;
    a.table = table;
    a.lengths = lengths;
    a.window = 0;
    return a;
}

// The workspace: the attention's, then keys, the taken pages and their tokens.
struct Workspace {
    size_t keys, table, lengths, bytes;

    Workspace(const SparseAttentionArgs &s, int cus)
    {
        const PagedAttentionArgs &a = s.attention;
        const size_t rows = (size_t)a.B * a.kvHeads;
        const auto up = [](size_t x) { return (x + 255) / 256 * 256; };
        keys = up(paged_attention_workspace(rows_of(s, nullptr, nullptr), cus));
        table = keys + up(rows * a.width * 8);
        lengths = table + up(rows * s.top * 4);
        bytes = lengths + up(rows * 4);
    }
};

template <bool kBf16>
void launch_scores(const Args &args, unsigned grid, hipStream_t stream)
{
    const int d = args.a.attention.d;
    if (d <= 32) {
        hipLaunchKernelGGL((score_pages<kBf16, 4>), dim3(grid), dim3(kThreads), 0, stream, args);
    } else if (d <= 64) {
        hipLaunchKernelGGL((score_pages<kBf16, 8>), dim3(grid), dim3(kThreads), 0, stream, args);
    } else if (d <= 128) {
        hipLaunchKernelGGL((score_pages<kBf16, 16>), dim3(grid), dim3(kThreads), 0, stream, args);
    } else {
        hipLaunchKernelGGL((score_pages<kBf16, 32>), dim3(grid), dim3(kThreads), 0, stream, args);
    }
}

}  // namespace
}  // namespace sparse

bool sparse_attention_fits(const SparseAttentionArgs &s)
{
    const PagedAttentionArgs &a = s.attention;
    // (Columns are counted in steps that end behind the last one, in 32 bits.)
    return a.width <= (1 << 30) && (int64_t)a.B * a.kvHeads <= (1 << 20) &&
           paged_attention_units_fit(sparse::rows_of(s, nullptr, nullptr));
}

size_t sparse_attention_workspace(const SparseAttentionArgs &s, int cus) { return sparse::Workspace(s, cus).bytes; }

hipError_t launch_sparse_attention(const SparseAttentionArgs &s, void *workspace, int device, int cus,
                                   hipStream_t stream)
{
    const sparse::Workspace at(s, cus);
    char *base = static_cast<char *>(workspace);
    const sparse::Args args{s, reinterpret_cast<uint64_t *>(base + at.keys), reinterpret_cast<int32_t *>(base + at.table),
                            reinterpret_cast<int32_t *>(base + at.lengths), sparse::columns_of(s.attention),
                            sparse::heads_of(s.attention)};
    const PagedAttentionArgs &a = s.attention;
    const int64_t items = (int64_t)a.B * ((a.kvHeads + args.heads - 1) / args.heads) *
                          ((a.width + args.columns - 1) / args.columns);
    const unsigned grid = (unsigned)(items < (1 << 20) ? items : (1 << 20));
    if (a.isBf16) {
        sparse::launch_scores<true>(args, grid, stream);
    } else {
        sparse::launch_scores<false>(args, grid, stream);
    }
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        return err;
    }
    const dim3 rowsGrid((unsigned)(a.B * a.kvHeads)), threads(sparse::kSelectThreads);
    if (a.width <= 2 * sparse::kSelectThreads) {
        hipLaunchKernelGGL((sparse::select_pages<2, true>), rowsGrid, threads, 0, stream, args);
    } else if (a.width <= sparse::kMostHeld * sparse::kSelectThreads) {
        hipLaunchKernelGGL((sparse::select_pages<sparse::kMostHeld, true>), rowsGrid, threads, 0, stream, args);
    } else {
        hipLaunchKernelGGL((sparse::select_pages<sparse::kMostHeld, false>), rowsGrid, threads, 0, stream, args);
    }
    if ((err = hipGetLastError()) != hipSuccess) {
        return err;
    }
    const PagedAttentionArgs rows = sparse::rows_of(s, args.table, args.lengths);
    bool wide;
    attention::Args p = attention::plan(rows, cus, wide);
    p.each = a.kvHeads;
    if (!attention::short_rows(rows, p, wide)) {
        p.parts = base + kWsHeaderBytes;
        if ((err = make_launch_tag(next_launch_id(), device, p.most, workspace, stream, p.tag)) != hipSuccess) {
            return err;
        }
    }
    return a.isBf16 ? attention::launch_each_bf16(p, wide, stream) : attention::launch_each_f16(p, wide, stream);
}

}  // namespace mhc
