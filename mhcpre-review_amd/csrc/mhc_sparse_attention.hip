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

#include "mhc_paged_attention.h"

namespace mhc {
namespace sparse {
namespace {

using dev::kWave;
using dev::u32x4_t;

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kColumns = 64;  // columns of a workgroup's item

// Scores as ordered integers; what cannot be taken is 0.
constexpr uint64_t kAlways = ~0ull, kNotANumber = ~0ull - 1;

struct Args {
    SparseAttentionArgs a;
    uint64_t *keys;     // [B * kvHeads, width]
    int32_t *table;     // [B * kvHeads, top]: the pages taken
    int32_t *lengths;   // [B * kvHeads]: their tokens
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
    constexpr int kBatch = 2;
    const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
    const int sub = lane % kLanes, e = 8 * sub;
    const bool on = e < a.d;
    const int group = a.heads / a.kvHeads, chunks = (a.width + kColumns - 1) / kColumns;
    const int64_t items = (int64_t)a.B * a.kvHeads * chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t row = item / chunks;
        const int b = (int)(row / a.kvHeads), kv = (int)(row % a.kvHeads), column0 = (int)(item % chunks) * kColumns;
        const Row r(a, b);
        if (column0 >= r.held) {
            continue;
        }
        double up[8], down[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            up[x] = down[x] = 0;
        }
        const uint16_t *q = static_cast<const uint16_t *>(a.q.data) + b * a.q.row + (int64_t)kv * group * a.q.head + e;
        for (int h = 0; h < group && on; ++h) {
            float f[8];
            dev::unpack8<kBf16>(*reinterpret_cast<const u32x4_t *>(q + h * a.q.head), f);
#pragma unroll
            for (int x = 0; x < 8; ++x) {  // (NaN goes to both)
                up[x] += f[x] < 0.f ? 0.0 : (double)f[x];
                down[x] += f[x] > 0.f ? 0.0 : (double)f[x];
            }
        }
        const int end = r.held - column0 < kColumns ? r.held : column0 + kColumns;
        for (int c0 = column0 + wave * kPages + lane / kLanes; c0 - lane / kLanes < end; c0 += kBatch * kWaves * kPages) {
            int page[kBatch];
            u32x4_t lo[kBatch], hi[kBatch];
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const int c = c0 + x * kWaves * kPages;
                page[x] = c < end ? a.table[(int64_t)b * a.width + c] : -1;
            }
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const bool good = page[x] >= 0 && page[x] < a.pages;
                page[x] = good ? page[x] : -1;
                lo[x] = hi[x] = u32x4_t{0, 0, 0, 0};
                if (good && on) {
                    lo[x] = *reinterpret_cast<const u32x4_t *>(static_cast<const uint16_t *>(s.lo.data) +
                                                               page[x] * s.lo.row + kv * s.lo.head + e);
                    hi[x] = *reinterpret_cast<const u32x4_t *>(static_cast<const uint16_t *>(s.hi.data) +
                                                               page[x] * s.hi.row + kv * s.hi.head + e);
                }
            }
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                float l[8], h[8];
                dev::unpack8<kBf16>(lo[x], l);
                dev::unpack8<kBf16>(hi[x], h);
                double sum = 0;
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    sum = __builtin_fma(up[y], (double)h[y], sum);
                    sum = __builtin_fma(down[y], (double)l[y], sum);
                }
#pragma unroll
                for (int mask = 1; mask < kLanes; mask *= 2) {
                    sum += shuffled(sum, mask);
                }
                sum += 0.0;  // (-0 is 0)
                const uint64_t bits = (uint64_t)__double_as_longlong(sum);
                uint64_t key = bits >> 63 != 0 ? ~bits : bits | 1ull << 63;
                key = sum != sum ? kNotANumber : key;
                const int c = c0 + x * kWaves * kPages;
                key = c < s.first || c >= r.held - s.last ? kAlways : key;
                if (sub == 0 && c < end) {
                    args.keys[row * a.width + c] = page[x] >= 0 ? key : 0;
                }
            }
        }
    }
}

// The highest `top` keys of a (sequence, kv head), in order.
constexpr int kSelectThreads = 512, kSelectWaves = kSelectThreads / kWave, kBins = 256;

template <typename T, typename F>
__device__ __forceinline__ T reduced(T v, F &&f)
{
#pragma unroll
    for (int mask = 1; mask < kWave; mask *= 2) {
        const uint64_t bits = (uint64_t)v;
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)bits, mask),
                       hi = (uint32_t)__shfl_xor((int)(bits >> 32), mask);
        v = f(v, (T)((uint64_t)hi << 32 | lo));
    }
    return v;
}

__global__ __launch_bounds__(kSelectThreads) void select_pages(Args args)
{
    __shared__ uint64_t least[kSelectWaves], greatest[kSelectWaves];
    __shared__ int there[kSelectWaves], always[kSelectWaves];
    __shared__ int bins[kBins];
    __shared__ uint64_t rangeLow;
    __shared__ int rangeNeed, rangeIn;
    __shared__ int before[2][kSelectWaves];
    __shared__ int lastTaken;
    const SparseAttentionArgs &s = args.a;
    const PagedAttentionArgs &a = s.attention;
    const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
    const int64_t row = blockIdx.x;
    const int b = (int)(row / a.kvHeads);
    const Row r(a, b);
    const uint64_t *keys = args.keys + row * a.width;

    // How many can be taken, how many are in any case, and the others' range.
    uint64_t low = kAlways, high = 0;
    int some = 0, sure = 0;
    for (int c = (int)threadIdx.x; c < r.held; c += kSelectThreads) {
        const uint64_t key = keys[c];
        some += key != 0 ? 1 : 0;
        sure += key == kAlways ? 1 : 0;
        if (key != 0 && key != kAlways) {
            low = key < low ? key : low;
            high = key > high ? key : high;
        }
    }
    low = reduced(low, [](uint64_t x, uint64_t y) { return x < y ? x : y; });
    high = reduced(high, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
    some = reduced(some, [](int x, int y) { return x + y; });
    sure = reduced(sure, [](int x, int y) { return x + y; });
    if (threadIdx.x == 0) {
        lastTaken = 0;
    }
    if (lane == 0) {
        least[wave] = low;
        greatest[wave] = high;
        there[wave] = some;
        always[wave] = sure;
    }
    __syncthreads();
    some = sure = 0;
#pragma unroll
    for (int x = 0; x < kSelectWaves; ++x) {
        low = least[x] < low ? least[x] : low;
        high = greatest[x] > high ? greatest[x] : high;
        some += there[x];
        sure += always[x];
    }
    // Taken: keys above `floor`, and the first `ties` of those that equal it.
    uint64_t floor = 0;
    int ties = 0;
    if (some > s.top) {
        int need = s.top - sure;  // of the keys in [low, high]
        if (need == 0) {
            floor = kAlways - 1;
        }
        while (need > 0) {
            int shift = 0;
            if ((high - low) / kBins != 0) {
                shift = 64 - __clzll((long long)((high - low) / kBins));
            }
            __syncthreads();
            for (int x = (int)threadIdx.x; x < kBins; x += kSelectThreads) {
                bins[x] = 0;
            }
            __syncthreads();
            for (int c = (int)threadIdx.x; c < r.held; c += kSelectThreads) {
                const uint64_t key = keys[c];
                if (key >= low && key <= high) {
                    atomicAdd(&bins[(key - low) >> shift], 1);
                }
            }
            __syncthreads();
            if (wave == 0) {
                // From the top: the bin at which `need` is reached.
                int mine[kBins / kWave], all = 0;
#pragma unroll
                for (int x = 0; x < kBins / kWave; ++x) {
                    mine[x] = bins[kBins - 1 - (lane * (kBins / kWave) + x)];
                    all += mine[x];
                }
                int above = dev::wave_scan(all) - all;
#pragma unroll
                for (int x = 0; x < kBins / kWave; ++x) {
                    if (above < need && above + mine[x] >= need) {
                        rangeLow = low + ((uint64_t)(kBins - 1 - (lane * (kBins / kWave) + x)) << shift);
                        rangeNeed = need - above;
                        rangeIn = mine[x];
                    }
                    above += mine[x];
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
        }
    }
    // In the columns' order.
    int taken = 0, equal = 0;
    int32_t *columns = s.columns + row * s.top, *table = args.table + row * s.top;
    for (int c0 = 0; c0 < r.held; c0 += kSelectThreads) {
        const int c = c0 + (int)threadIdx.x;
        const uint64_t key = c < r.held ? keys[c] : 0;
        const bool tie = ties > 0 && key == floor;
        const uint64_t tied = __ballot(tie);
        __syncthreads();
        if (lane == 0) {
            before[0][wave] = __popcll(tied);
        }
        __syncthreads();
        int rank = equal + __popcll(tied & ((1ull << lane) - 1));
#pragma unroll
        for (int x = 0; x < kSelectWaves; ++x) {
            rank += x < wave ? before[0][x] : 0;
            equal += before[0][x];
        }
        const bool take = key > floor || (tie && rank < ties);
        const uint64_t takes = __ballot(take);
        if (lane == 0) {
            before[1][wave] = __popcll(takes);
        }
        __syncthreads();
        int at = taken + __popcll(takes & ((1ull << lane) - 1));
#pragma unroll
        for (int x = 0; x < kSelectWaves; ++x) {
            at += x < wave ? before[1][x] : 0;
            taken += before[1][x];
        }
        if (take) {
            columns[at] = c;
            table[at] = a.table[(int64_t)b * a.width + c];
            if (c == r.held - 1) {
                lastTaken = 1;
            }
        }
    }
    for (int x = taken + (int)threadIdx.x; x < s.top; x += kSelectThreads) {
        columns[x] = table[x] = -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) {  // (the last column may be filled in part)
        args.lengths[row] = taken * a.pageSize - (lastTaken != 0 ? r.held * a.pageSize - r.length : 0);
    }
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
    return (int64_t)a.B * a.kvHeads <= (1 << 20) && paged_attention_units_fit(sparse::rows_of(s, nullptr, nullptr));
}

size_t sparse_attention_workspace(const SparseAttentionArgs &s, int cus) { return sparse::Workspace(s, cus).bytes; }

hipError_t launch_sparse_attention(const SparseAttentionArgs &s, void *workspace, int device, int cus,
                                   hipStream_t stream)
{
    const sparse::Workspace at(s, cus);
    char *base = static_cast<char *>(workspace);
    const sparse::Args args{s, reinterpret_cast<uint64_t *>(base + at.keys), reinterpret_cast<int32_t *>(base + at.table),
                            reinterpret_cast<int32_t *>(base + at.lengths)};
    const PagedAttentionArgs &a = s.attention;
    const int64_t items = (int64_t)a.B * a.kvHeads * ((a.width + sparse::kColumns - 1) / sparse::kColumns);
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
    hipLaunchKernelGGL(sparse::select_pages, dim3((unsigned)(a.B * a.kvHeads)), dim3(sparse::kSelectThreads), 0, stream,
                       args);
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
