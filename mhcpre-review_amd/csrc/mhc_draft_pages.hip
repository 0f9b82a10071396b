// What stands around attention over drafted tokens and selected pages: the path of
// a tree that the model's choices confirm (mhcDraftAccept), its keys and values to
// their places (mhcCacheKeep), and the bounds of the pages' keys (mhcCacheBounds).

#include "mhc_pre_device.h"
#include "mhc_serve_internal.h"

namespace mhc {
namespace {

using dev::kWave;
using dev::u32x4_t;

__device__ __forceinline__ int clamped(int v, int most) { return v < 0 ? 0 : v > most ? most : v; }

// ---- accept ------------------------------------------------------------------

// A wave does a row; a lane holds nodes lane + 64 k with their parents, tokens and
// choices.  A step of the path asks all nodes at once whether they are a child with
// the wanted token, and takes the first.  Bound by the launch and one load: 3.0 us for
// 32 trees of 32 nodes, 3.7 for 1000 of 256 (6.2 MB).
constexpr int kAcceptWaves = 4, kHeld = kDraftNodes / kWave;

template <typename Token>
__global__ __launch_bounds__(kAcceptWaves *kWave) void accept_rows(DraftAcceptArgs a)
{
    const int lane = (int)threadIdx.x % kWave;
    const int64_t b = (int64_t)blockIdx.x * kAcceptWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    if (b >= a.B) {
        return;
    }
    const int L = a.lengths[b] < 0 ? 0 : a.lengths[b];
    const int drafted = clamped(a.drafted[b], a.S), n = drafted < L ? drafted : L;
    int parent[kHeld], path[kHeld];
    Token token[kHeld], chosen[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int i = k * kWave + lane;
        parent[k] = path[k] = -1;
        token[k] = chosen[k] = 0;
        if (i < n) {
            parent[k] = a.parents != nullptr ? a.parents[b * a.S + i] : i - 1;
            parent[k] = parent[k] < i ? parent[k] : -1;
            token[k] = static_cast<const Token *>(a.tokens)[b * a.S + i];
            chosen[k] = static_cast<const Token *>(a.chosen)[b * a.S + i];
        }
    }
    Token wanted = -1;
    int accepted = 0;
    for (int node = n > 0 ? 0 : -1; node >= 0;) {
        int next = -1;
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            if (node / kWave == k) {
                if constexpr (sizeof(Token) == 8) {
                    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)chosen[k], node % kWave);
                    const uint32_t hi = __builtin_amdgcn_readlane((int)(chosen[k] >> 32), node % kWave);
                    wanted = (Token)((uint64_t)hi << 32 | lo);
                } else {
                    wanted = __builtin_amdgcn_readlane(chosen[k], node % kWave);
                }
            }
            path[k] = accepted == k * kWave + lane ? node : path[k];
        }
        ++accepted;
#pragma unroll
        for (int k = kHeld - 1; k >= 0; --k) {
            const uint64_t children = __ballot(parent[k] == node && token[k] == wanted);
            next = children != 0 ? k * kWave + __ffsll((unsigned long long)children) - 1 : next;
        }
        node = next;
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int i = k * kWave + lane;
        if (i < a.S) {
            a.path[b * a.S + i] = path[k];
        }
    }
    if (lane == 0) {
        a.accepted[b] = accepted;
        a.newLengths[b] = L - n + accepted;
        static_cast<Token *>(a.next)[b] = wanted;
    }
}

// ---- keep --------------------------------------------------------------------

// A workgroup does a row of the batch and some columns (bytes of a slot, of both
// caches, or of the one that is both: two threads at one place would not keep the
// order).  Its path goes through LDS in pieces as pairs of offsets.  A node moves
// towards the front only and paths ascend, so a thread that goes along the path with
// loads before stores never reads what it has written.  Bound by its chain (lengths,
// path, table, values): 6.0 us for 32 rows with 5 nodes of 32 (8 kv heads of 128), 13.3
// for 500 with 17 of 101, 31.7 MB at 2.4 TB/s; with 16 or 32 nodes on their way at
// once 13.6.
constexpr int kKeepThreads = 256, kKeepBatch = 8;

template <typename Piece>
__global__ __launch_bounds__(kKeepThreads) void keep_rows(CacheKeepArgs a)
{
    __shared__ int fromPage[kKeepThreads], toPage[kKeepThreads], fromSlot[kKeepThreads], toSlot[kKeepThreads];
    __shared__ int broken;
    const int64_t b = blockIdx.x;
    const int L = clamped(a.lengths[b], a.width * a.pageSize);
    const int drafted = clamped(a.drafted[b], a.S), n = drafted < L ? drafted : L, c = L - n;
    const uint32_t pieces = (uint32_t)a.rowBytes / (uint32_t)sizeof(Piece), half = (uint32_t)a.kvHeads * pieces;
    for (int k0 = 0; k0 < n; k0 += kKeepThreads) {
        __syncthreads();
        if (threadIdx.x == 0) {
            broken = kKeepThreads;
        }
        __syncthreads();
        const int k = k0 + (int)threadIdx.x;
        int node = -1;
        if (k < n) {
            node = a.path[b * a.S + k];
            const int before = k > 0 ? a.path[b * a.S + k - 1] : -1;
            if (node < 0 || node >= n || node <= before) {
                atomicMin(&broken, (int)threadIdx.x);
            }
        } else {
            atomicMin(&broken, (int)threadIdx.x);
        }
        int pages[2] = {-1, -1}, slots[2] = {0, 0};
        if (node > k && node < n) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t t = (uint32_t)(c + (x == 0 ? node : k)), column = t / (uint32_t)a.pageSize;
                slots[x] = (int)(t - column * (uint32_t)a.pageSize);
                pages[x] = a.table[b * a.width + column];
            }
        }
        const bool good = pages[0] >= 0 && pages[0] < a.pages && pages[1] >= 0 && pages[1] < a.pages;
        fromPage[threadIdx.x] = good ? pages[0] : -1;
        toPage[threadIdx.x] = pages[1];
        fromSlot[threadIdx.x] = slots[0];
        toSlot[threadIdx.x] = slots[1];
        __syncthreads();
        const int count = broken;
        for (uint64_t at = (uint64_t)blockIdx.y * kKeepThreads + threadIdx.x; at < (uint64_t)a.caches * half;
             at += (uint64_t)gridDim.y * kKeepThreads) {
            const CacheRows &cache = at < half ? a.k : a.v;
            const uint32_t in = (uint32_t)(at < half ? at : at - half);
            char *const base = static_cast<char *>(cache.data) + (int64_t)(in / pieces) * cache.head * a.elemBytes +
                               (int64_t)(in % pieces) * (int)sizeof(Piece);
            const int64_t pageBytes = cache.page * a.elemBytes, slotBytes = cache.slot * a.elemBytes;
            for (int x0 = 0; x0 < count; x0 += kKeepBatch) {
                Piece held[kKeepBatch];
#pragma unroll
                for (int x = 0; x < kKeepBatch; ++x) {
                    if (x0 + x < count && fromPage[x0 + x] >= 0) {
                        held[x] = *reinterpret_cast<const Piece *>(base + fromPage[x0 + x] * pageBytes +
                                                                   fromSlot[x0 + x] * slotBytes);
                    }
                }
#pragma unroll
                for (int x = 0; x < kKeepBatch; ++x) {
                    if (x0 + x < count && fromPage[x0 + x] >= 0) {
                        *reinterpret_cast<Piece *>(base + toPage[x0 + x] * pageBytes + toSlot[x0 + x] * slotBytes) =
                            held[x];
                    }
                }
            }
        }
        if (count < kKeepThreads) {
            return;
        }
    }
}

// ---- bounds ------------------------------------------------------------------

// A 16-bit floating value as an integer of the same order (NaN beyond infinity on its
// sign's side), two at a time; its own inverse.
typedef short s16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ s16x2_t ordered(uint32_t two)
{
    const s16x2_t v = __builtin_bit_cast(s16x2_t, two);
    return v ^ ((v >> 15) & (s16x2_t){0x7FFF, 0x7FFF});
}

struct Range {
    s16x2_t lo[4], hi[4];

    __device__ void clear()
    {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            lo[x] = (s16x2_t){0x7FFF, 0x7FFF};
            hi[x] = (s16x2_t){-0x8000, -0x8000};
        }
    }
    __device__ void add(const u32x4_t &low, const u32x4_t &high)
    {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            lo[x] = __builtin_elementwise_min(lo[x], ordered(low[x]));
            hi[x] = __builtin_elementwise_max(hi[x], ordered(high[x]));
        }
    }
    __device__ void add(const Range &r)
    {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            lo[x] = __builtin_elementwise_min(lo[x], r.lo[x]);
            hi[x] = __builtin_elementwise_max(hi[x], r.hi[x]);
        }
    }
    // Where one bound is NaN both are, lo a value below all and hi one above all: what
    // is added later does not hide it.  (Below -infinity and above infinity lie NaN.)
    template <bool kBf16>
    __device__ void mark()
    {
        constexpr short kInf = kBf16 ? 0x7F80 : 0x7C00;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const bool nan = lo[x][y] < (short)~kInf || lo[x][y] > kInf || hi[x][y] < (short)~kInf || hi[x][y] > kInf;
                lo[x][y] = nan ? (short)-0x8000 : lo[x][y];
                hi[x][y] = nan ? (short)0x7FFF : hi[x][y];
            }
        }
    }
    __device__ Range shuffled(int mask) const
    {
        Range r;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            r.lo[x] = __builtin_bit_cast(s16x2_t, __shfl_xor(__builtin_bit_cast(int, lo[x]), mask));
            r.hi[x] = __builtin_bit_cast(s16x2_t, __shfl_xor(__builtin_bit_cast(int, hi[x]), mask));
        }
        return r;
    }
};

// kLanes lanes do 16 bytes (of a head's dimensions) of a page of a row, each every
// kLanes-th token; neighbouring groups have neighbouring pieces.  A lane has kBoundsBatch
// tokens on their way at once.  Bound by memory for prompts, 8 of 8192 tokens in pages of 16
// (64.6 MB) 13.9 us, 4.6 TB/s; by its chain of loads for a step of 64 tokens, 4.0.
constexpr int kBoundsThreads = 256, kBoundsBatch = 8;

template <bool kBf16, int kLanes>
__global__ __launch_bounds__(kBoundsThreads) void bounds_pages(CacheBoundsArgs a)
{
    constexpr int kPieces = kBoundsThreads / kLanes;  // of a workgroup
    // Lanes of a piece lie kStride lanes apart in a wave.
    constexpr int kStride = kWave / kLanes;
    const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
    const int split = lane / kStride, inGroup = wave * kStride + lane % kStride;
    for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t perRow = (int64_t)a.columns * a.pieceGroups;
        const int64_t b = a.B == 1 ? 0 : item / perRow;
        // (A row's items may be more than 2^31.  A 64-bit division where they need it only.)
        const int64_t inRow = item - b * perRow;
        const int64_t ofRow = inRow <= INT32_MAX ? (int)inRow / a.pieceGroups : inRow / a.pieceGroups;
        const int pieceGroup = (int)(inRow - ofRow * a.pieceGroups);
        const int L = clamped(a.lengths[b], a.width * a.pageSize);
        const int wanted = clamped(a.counts[b], a.tokens), count = wanted < L ? wanted : L, begin = L - count;
        const int64_t column = begin / a.pageSize + ofRow;
        const int64_t start = column * a.pageSize;
        if (count == 0 || start >= L) {
            continue;
        }
        const int page = a.table[b * a.width + column];
        if (page < 0 || page >= a.pages) {
            continue;
        }
        const int chunks = a.d / 8, piece = pieceGroup * kPieces + inGroup;
        const bool on = piece < a.kvHeads * chunks;
        const int head = on ? piece / chunks : 0, e = on ? piece % chunks * 8 : 0;
        const uint32_t first = begin > start ? (uint32_t)(begin - start) : 0u;
        const uint32_t end = L - start < a.pageSize ? (uint32_t)(L - start) : (uint32_t)a.pageSize;
        const uint16_t *from = static_cast<const uint16_t *>(a.k.data) + page * a.k.page + head * a.k.head + e;
        uint16_t *lo = static_cast<uint16_t *>(a.lo.data) + page * a.lo.row + head * a.lo.head + e;
        uint16_t *hi = static_cast<uint16_t *>(a.hi.data) + page * a.hi.row + head * a.hi.head + e;
        Range range;
        range.clear();
        const bool old = split == 0 && first > 0;
        u32x4_t oldLow = {0, 0, 0, 0}, oldHigh = oldLow;
        if (old) {
            oldLow = *reinterpret_cast<const u32x4_t *>(lo);
            oldHigh = *reinterpret_cast<const u32x4_t *>(hi);
        }
        for (uint32_t t0 = first + split; t0 < end; t0 += kLanes * kBoundsBatch) {
            u32x4_t k[kBoundsBatch];
#pragma unroll
            for (int x = 0; x < kBoundsBatch; ++x) {
                const uint32_t t = t0 + x * kLanes < end ? t0 + x * kLanes : t0;
                k[x] = *reinterpret_cast<const u32x4_t *>(from + t * a.k.slot);
            }
#pragma unroll
            for (int x = 0; x < kBoundsBatch; ++x) {
                range.add(k[x], k[x]);
            }
        }
        if (old) {
            Range before;
            before.clear();
            before.add(oldLow, oldHigh);
            before.mark<kBf16>();
            range.add(before);
        }
#pragma unroll
        for (int mask = kStride; mask < kWave; mask *= 2) {
            range.add(range.shuffled(mask));
        }
        if (split != 0 || !on) {
            continue;
        }
        range.mark<kBf16>();
        constexpr uint32_t kNan = kBf16 ? 0x7FC0 : 0x7E00;
        u32x4_t low, high;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            low[x] = __builtin_bit_cast(uint32_t, ordered(__builtin_bit_cast(uint32_t, range.lo[x])));
            high[x] = __builtin_bit_cast(uint32_t, ordered(__builtin_bit_cast(uint32_t, range.hi[x])));
            low[x] = range.lo[x][0] == -0x8000 ? (low[x] & 0xFFFF0000u) | kNan : low[x];
            low[x] = range.lo[x][1] == -0x8000 ? (low[x] & 0xFFFFu) | kNan << 16 : low[x];
            high[x] = range.lo[x][0] == -0x8000 ? (high[x] & 0xFFFF0000u) | kNan : high[x];
            high[x] = range.lo[x][1] == -0x8000 ? (high[x] & 0xFFFFu) | kNan << 16 : high[x];
        }
        *reinterpret_cast<u32x4_t *>(lo) = low;
        *reinterpret_cast<u32x4_t *>(hi) = high;
    }
}

}  // namespace

hipError_t launch_draft_accept(const DraftAcceptArgs &a, hipStream_t stream)
{
    const dim3 grid((unsigned)((a.B + kAcceptWaves - 1) / kAcceptWaves));
    if (a.tokens64) {
        hipLaunchKernelGGL((accept_rows<int64_t>), grid, dim3(kAcceptWaves * kWave), 0, stream, a);
    } else {
        hipLaunchKernelGGL((accept_rows<int32_t>), grid, dim3(kAcceptWaves * kWave), 0, stream, a);
    }
    return hipGetLastError();
}

namespace {

bool divides(const CacheRows &c, int elemBytes, uintptr_t by)
{
    return reinterpret_cast<uintptr_t>(c.data) % by == 0 && c.page * elemBytes % (int64_t)by == 0 &&
           c.slot * elemBytes % (int64_t)by == 0 && c.head * elemBytes % (int64_t)by == 0;
}

template <typename Piece>
hipError_t launch_keep(const CacheKeepArgs &a, hipStream_t stream)
{
    const int64_t pieces = (int64_t)a.caches * a.kvHeads * (a.rowBytes / (int)sizeof(Piece));
    const int64_t groups = (pieces + kKeepThreads - 1) / kKeepThreads;
    hipLaunchKernelGGL((keep_rows<Piece>), dim3((unsigned)a.B, (unsigned)(groups < 256 ? groups : 256)),
                       dim3(kKeepThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_keep(const CacheKeepArgs &a, hipStream_t stream)
{
    // Pieces of 16 bytes where sizes, strides and addresses allow it, else single values.
    if (a.rowBytes % 16 == 0 && divides(a.k, a.elemBytes, 16) && divides(a.v, a.elemBytes, 16)) {
        return launch_keep<u32x4_t>(a, stream);
    }
    return a.elemBytes == 4 ? launch_keep<uint32_t>(a, stream) : launch_keep<uint16_t>(a, stream);
}

namespace {

// Workgroups of a launch: what is on the CUs at once, a few times over.
constexpr int64_t kBoundsMost = 8192;

template <bool kBf16, int kLanes>
hipError_t launch_bounds(CacheBoundsArgs a, hipStream_t stream)
{
    constexpr int kPieces = kBoundsThreads / kLanes;
    const int64_t columns = ((int64_t)a.tokens + a.pageSize - 2) / a.pageSize + 1;
    a.columns = (int)(columns < a.width ? columns : (int64_t)a.width);
    a.pieceGroups = (a.kvHeads * (a.d / 8) + kPieces - 1) / kPieces;
    a.items = (int64_t)a.B * a.columns * a.pieceGroups;
    hipLaunchKernelGGL((bounds_pages<kBf16, kLanes>), dim3((unsigned)(a.items < kBoundsMost ? a.items : kBoundsMost)),
                       dim3(kBoundsThreads), 0, stream, a);
    return hipGetLastError();
}

template <bool kBf16>
hipError_t launch_bounds_type(const CacheBoundsArgs &a, hipStream_t stream)
{
    // Tokens of a page that a call may bring: several lanes to a piece where they are many.  us, 1 /
    // 4 / 16 lanes, 8 prompts of 8192 tokens: pages of 16 14.6 / 20.8 / 59.9, of 64 16.4 / 13.6 /
    // 21.3, of 128 16.1 / 14.5 / 14.7, of 256 23.9 / 14.3 / 13.6, of 1024 74 / 23 / 15.8; one prompt,
    // pages of 128 11.3 / 8.2 / 6.1.
    const int64_t tokens = a.tokens < a.pageSize ? a.tokens : a.pageSize;
    return tokens <= 16 ? launch_bounds<kBf16, 1>(a, stream)
           : tokens <= 64 ? launch_bounds<kBf16, 4>(a, stream) : launch_bounds<kBf16, 16>(a, stream);
}

}  // namespace

hipError_t launch_cache_bounds(const CacheBoundsArgs &a, hipStream_t stream)
{
    return a.isBf16 ? launch_bounds_type<true>(a, stream) : launch_bounds_type<false>(a, stream);
}

}  // namespace mhc
