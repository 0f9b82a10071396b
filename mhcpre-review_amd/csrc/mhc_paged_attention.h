// Attention of one new token per sequence over a paged cache
// (mhcPagedAttention): the kernels, instantiated per element type.
//
// The keys of a row are cut into units of 128 (aligned to multiples of 128, so
// a unit never changes with the row's length).  All units of all (row, kv head,
// group of query heads) in that order form one line, which is shared out evenly
// to a fixed grid: the lengths are on the device, and so is this arithmetic.  A
// workgroup walks its stretch; a (row, kv head, group) that lies in one
// stretch is finished there, the others leave their maximum, sum and output per
// stretch in the workspace and count them, and the workgroup that counts the last
// one joins them, in the order of the keys (many of them in spans first, each
// joined by its own last workgroup).  Nobody waits.  What tells this
// launch's counts from what the workspace held before is the launch's tag
// (LaunchTag); a count that is complete is taken away.
//
// In a unit each of the 4 waves has 32 keys of its own.  The scores are S^T =
// K Q^T, 16 keys by 16 query heads (a wave's K rows go straight from memory to
// the operand's registers), so a lane has the scores of one head, and the
// probabilities are, as they lie in its registers, the operand of O^T = V^T
// P^T: the order of the keys within a product is free.  V goes through LDS,
// rows as they come, and is read transposed (ds_read_b64_tr_b16); the region is
// the wave's own, so the loop has no barrier.  A probability is the sum of as many
// 16-bit terms as hold it, three in bf16 (24 bits) and two in fp16 (21): one alone
// would add an error as large as the output's own rounding, two of bf16 an error of
// 2^-16 that shows where values cancel; the matrix cores have time (32 bf16 heads
// at a time, with two / three, us: of 64 31 / 33, of 128 51.7 / 54.5; all else the
// same). fp16 ends at 2^-24, so there they are lifted by 2^15 (at most 32768):
// small weights are held to 2^-39 of the largest, of which 131072 keys' are 2^-22
// of it.  All terms but the last are cut, not rounded, and all but the first are
// above 0 wherever the weight is: with one at 0 or below, an infinite value would
// come out as NaN.  (Looking for such values in every tile instead took 10% of the
// time with 32 heads at a time, 3% of one short row's.)
//
// Bound: the cache is read once, 4 bytes a value pair for at most 4 * 16
// flops, so the memory's rate decides (6.05 TB/s for a cold read of two
// tensors of 0.5 GB in the same pieces).  Measured: 64 rows of 1 to 8192 keys,
// 32 heads to 8 of 128, 734 MB, 139 us (5.3 TB/s); 4 rows up to 131072 keys, 1007 MB,
// 184 us (5.5 TB/s).  The rest is the start and the join.  The same launches with one
// key a row take 7.2 us (a launch, lengths, pages, keys, output).  The join's chain of
// store, count and load, left out in a copy, is 2.1 us of one row of 1000 keys
// (9.2 in all), 2.8 of the 64 rows, 7 of the 4, whose 64 heads' parts are the largest.
#pragma once

#include "mhc_pre_device.h"
#include "mhc_serve_internal.h"

namespace mhc {
namespace attention {

using dev::f32x4_t;
using dev::kWave;
using dev::u32x4_t;

constexpr int kWaves = 4;
constexpr int kTile = 32;               // keys of a wave at a time
constexpr int kUnit = kWaves * kTile;   // keys of a unit
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

// What the probabilities, and with them the outputs' sums (not the weights' sums), are
// multiplied by until they are put out.
template <bool kBf16>
constexpr float kLift = kBf16 ? 1.f : 32768.f;

// The 16-bit terms of a probability.
template <bool kBf16>
constexpr int kTerms = kBf16 ? 3 : 2;

// Workgroups that a CU's registers hold.  A product with 32 query heads reads the cache once
// where two with 16 read it twice: 64 rows of 8192 keys, 32 heads to one, us, 32 at a
// time / 16, bf16: d = 64 33 / 46, 128 54.5 / 85.4, 192 87 / 123; fp16: 31.2 / 45.4,
// 51.5 / 84.7, 85.8 / 121.  At d = 256 its registers spill (285 / 166).
constexpr int workgroups_per_cu(int d, bool wide) { return d <= (wide ? 64 : 128) ? 2 : 1; }
constexpr int kWideMost = 192;  // the largest d with 32 query heads at a time

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8v_t __attribute__((ext_vector_type(8)));

// How the units are shared out.
struct Shares {
    int units, grid;  // all units; workgroups that have some (each has at least one)

    __device__ Shares(int units_, int most) : units(units_), grid(units_ < most ? units_ : most) {}
    __device__ int start(int w) const
    {
        const int q = units / grid, r = units % grid;
        return w * q + (w < r ? w : r);
    }
    __device__ int owner(int u) const
    {
        const int q = units / grid, r = units % grid;
        return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q;
    }
};

struct Args {
    PagedAttentionArgs a;
    int group;    // query heads of a kv head
    int blocks;   // blocks of 16 * RT query heads in a group
    int most;     // workgroups of the launch
    char *parts;  // see Parts; null: the kernel of short rows
    LaunchTag tag;
    int each = 1;  // kEach: kv heads of a sequence
};

// A stretch leaves at most two parts in the workspace, of the (row, kv head,
// group) that it begins in and of the one that it ends in: [2 * most] outputs [16
// RT][D], maxima (base 2) and sums [16 RT][2]; and an 8-byte word, of those of
// the parts that are joined together the first one's, that counts the parts that are
// there: its upper 52 bits are the launch's and the place's, so that the first to come
// sees that the word is not yet this launch's and sets it to none.  The last to come
// sets it to 0: a captured launch's tag returns after 2048 replays, and which words a
// replay uses goes by its lengths, so one that still held an old count under the same
// tag would be taken for this replay's.  Many parts are
// joined in spans: a span's result takes the place of its first output, its maxima,
// sums and word are a second [2 * most] ones.  All of it is stored through to memory
// and read from there: the reader may be on another XCD.
template <int D, int RT>
struct Parts {
    static constexpr int kRows = 16 * RT;
    __amdgpu_buffer_rsrc_t outs, ends;
    uint64_t *words;

    __device__ Parts(char *base, int most)
        : outs(dev::make_rsrc(base, 2 * most * kRows * D * 4)),
          ends(dev::make_rsrc(base + (size_t)2 * most * kRows * D * 4, 4 * most * kRows * 8)),
          words(reinterpret_cast<uint64_t *>(base + (size_t)2 * most * kRows * (D + 4) * 4))
    {
    }
    static constexpr uint64_t kCount = 0xFFF;
    // Counts one of `all` parts at the word, which was found as `found`; whether it is the
    // last.
    __device__ bool count(uint32_t tag, int slot, uint64_t found, int all) const
    {
        const uint64_t none = sign(tag, slot);
        if ((found & ~kCount) != none) {  // (fails where another workgroup was first)
            (void)__hip_atomic_compare_exchange_strong(words + slot, &found, none, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_AGENT);
        }
        const uint64_t before = __hip_atomic_fetch_add(words + slot, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = (int)(before & kCount) == all - 1;
        if (last) {
            __hip_atomic_store(words + slot, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        return last;
    }
    __device__ uint64_t word(int slot) const
    {
        return __hip_atomic_load(words + slot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // A word of this launch before the first part is counted.
    __device__ static uint64_t sign(uint32_t tag, int slot)
    {
        return ((uint64_t)mix32(tag ^ (2u * (uint32_t)slot + 1u)) << 32 | tag) & ~kCount;
    }
    __device__ void put(int slot, int row, int e, f32x4_t out) const
    {
        dev::store16<dev::kCpolDev>(__builtin_bit_cast(u32x4_t, out), outs, ((slot * kRows + row) * D + e) * 4);
    }
    __device__ void put_ends(int slot, int row, float top, float sum) const
    {
        const u32x2_t v = {__float_as_uint(top), __float_as_uint(sum)};
        __builtin_amdgcn_raw_buffer_store_b64(v, ends, (slot * kRows + row) * 8, 0, dev::kCpolDev);
    }
    __device__ f32x4_t out(int slot, int row, int e) const
    {
        return __builtin_bit_cast(f32x4_t, dev::load16<dev::kCpolDev>(outs, ((slot * kRows + row) * D + e) * 4));
    }
    __device__ u32x2_t end(int slot, int row) const
    {
        return __builtin_bit_cast(
            u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(ends, (slot * kRows + row) * 8, 0, dev::kCpolDev));
    }
};


// The keys of a row of length L: [low, high), and its units' number (one at least).
struct Keys {
    int low, high, first, units;

    Keys() = default;
    // unit: keys of a unit.
    __device__ Keys(const PagedAttentionArgs &a, int L, int unit)
    {
        const int most = a.width * a.pageSize;
        L = L < 0 ? 0 : L > most ? most : L;
        low = a.window > 0 && L > a.window ? L - (int)a.window : 0;
        high = L;
        first = low / unit;
        units = high > low ? (high - 1) / unit + 1 - first : 1;  // (high may be 2^31 - 1)
    }
};

__device__ __forceinline__ int64_t shfl64(int64_t v, int lane)
{
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)v, lane), hi = (uint32_t)__shfl((int)(v >> 32), lane);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

// LDS bytes between two rows of V: 8 banks off a multiple of 16 or 32, so that
// the four rows that 16 lanes read together lie in different banks.
template <int D>
constexpr int pitch()
{
    return 2 * D + (D == 112 ? 0 : 32);
}

// Bytes of a wave's LDS: V's tile, then the wave's output for the join.
template <int D>
constexpr int region()
{
    constexpr int v = kTile * pitch<D>(), o = 16 * (D + 4) * 4;
    return v > o ? v : o;
}

template <bool kBf16>
__device__ __forceinline__ f32x4_t mfma32(u32x4_t a, u32x4_t b, f32x4_t c)
{
    if constexpr (kBf16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v_t, a),
                                                       __builtin_bit_cast(bf16x8v_t, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b),
                                                      c, 0, 0, 0);
    }
}

// 4 values at the same column of 4 rows of LDS (the lane's column of 16).
__device__ __forceinline__ u32x2_t read_transposed(const char *p)
{
    return __builtin_bit_cast(
        u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t *)p));
}

template <int D>
struct Shape {
    static constexpr int kSteps = (D + 31) / 32;     // of 32 values in a product over d
    static constexpr int kChunks = D / 8;            // 16-byte chunks of a row
    static constexpr int kLoads = kTile * kChunks / kWave;  // of V, by a wave
    static constexpr int kDims = D / 16;
};

// 16 rows of K or Q: lane l has row l % 16, values 32 s + 8 (l / 16) .. + 7.
// Where D % 32 == 16 the last step's upper half is zero in both.  (A 16x16x16
// product in its place, added to the sum of the 16x16x32 ones, came out wrong.)
template <int D>
struct Fragment {
    u32x4_t step[Shape<D>::kSteps];

    __device__ void load(const uint16_t *row, int lane)
    {
        const int c = lane / 16;
#pragma unroll
        for (int s = 0; s < Shape<D>::kSteps; ++s) {
            const bool half = 32 * s + 32 > D;
            step[s] = *reinterpret_cast<const u32x4_t *>(row + 32 * s + 8 * (half ? c % 2 : c));
            if (half && c >= 2) {
                step[s] = u32x4_t{0, 0, 0, 0};
            }
        }
    }
    __device__ void clear()
    {
#pragma unroll
        for (int s = 0; s < Shape<D>::kSteps; ++s) {
            step[s] = u32x4_t{0, 0, 0, 0};
        }
    }
};

// Two values (0 at least) cut to the 16-bit type.
template <bool kBf16>
__device__ __forceinline__ uint32_t cut2(float p0, float p1)
{
    if constexpr (kBf16) {
        return __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302u);
    } else {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    }
}

// Two 16-bit values (0 at least), and where p is not 0 the type's smallest at least.
__device__ __forceinline__ uint32_t at_least(uint32_t two, float p0, float p1)
{
    const u16x2_t some = __builtin_bit_cast(u16x2_t, __builtin_amdgcn_cvt_pk_u16(__float_as_uint(p0), __float_as_uint(p1)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, two),
                                                                  __builtin_elementwise_min(some, u16x2_t{1, 1})));
}

// Where the query heads of row b and kv head `kv` begin in q or out.  kEach: a row is one
// kv head of a sequence of `each` (its own page table and length; a.kvHeads is 1).
template <bool kEach>
__device__ __forceinline__ int64_t first_head(const HeadRows &t, int b, int kv, int group, int each)
{
    return kEach ? b / each * t.row + (int64_t)(b % each * group) * t.head : b * t.row + (int64_t)(kv * group) * t.head;
}

// 4 values of the output from their sum, its weights' sum and their maximum; the
// first ones' thread also writes the head's lse.
template <bool kBf16, bool kEach = false>
__device__ __forceinline__ void finish(const PagedAttentionArgs &a, int b, int head, int e, f32x4_t all, float top,
                                       float total, int each = 1)
{
    const float inv = total == 0.f ? 0.f : 1.f / kLift<kBf16> / total;
    uint16_t *out = static_cast<uint16_t *>(a.out.data) +
                    (kEach ? first_head<true>(a.out, b, 0, a.heads, each) : b * a.out.row) + head * a.out.head + e;
    *reinterpret_cast<u32x2_t *>(out) =
        u32x2_t{dev::pack2_x<kBf16>(all[0] * inv, all[1] * inv), dev::pack2_x<kBf16>(all[2] * inv, all[3] * inv)};
    if (e == 0 && a.lse != nullptr) {
        a.lse[(int64_t)b * a.heads + head] = (top + __builtin_amdgcn_logf(total)) * kLn2;
    }
}

// What a stretch leaves of the (row, kv head, block) that it begins in, or of
// the one that it ends in, whose parts are those of workgroups first to last.
struct Part {
    bool on;
    int b, hg, first, last, firstSlot;
    __device__ int slot(int x) const { return x == first ? firstSlot : 2 * x; }
    // Parts that are joined together (2 to this power): all of them where one round of loads
    // takes them, or spans of about the root of their number, whose results are joined then.
    int spanBits;
    __device__ int span_first(int w) const { return first + (((w - first) >> spanBits) << spanBits); }
    __device__ int span_last(int w) const
    {
        const int after = (last - span_first(w)) >> spanBits;
        return after == 0 ? last : span_first(w) + (1 << spanBits) - 1;
    }
    __device__ int spans() const { return ((last - first) >> spanBits) + 1; }
};

// us, all at once / in spans: 64 parts of 16 heads of 128 47.4 / 36.8, of 256 74.4 / 46.8; 32 parts of 4
// heads of 128 (one round) 11.8 / 13.2.
constexpr int kAllBits = 30;  // (parts are at most 2048)
__device__ __forceinline__ int span_bits(int parts, int round)
{
    return parts <= round ? kAllBits : parts <= 64 ? 3 : parts <= 256 ? 4 : 5;
}


// kShort: rows of few keys (by the table's width or the window) in large batches.  Each
// wave is on its own: a share of the (row, kv head, block)s, each of which it does
// alone, 32 keys at a time, with no join and no workspace.  (Otherwise a row of up
// to 32 keys leaves three waves of its workgroup without any.)
// kEach: rows are the kv heads of sequences, each with a table and a length of its own.
template <bool kBf16, int D, int RT, bool kShort, bool kEach = false>
__global__ __launch_bounds__(64 * kWaves, workgroups_per_cu(D, RT > 1)) void attention_units(Args args)
{
    using S = Shape<D>;
    using Left = Parts<D, RT>;
    constexpr int P = pitch<D>();
    __shared__ __align__(16) char lds[kWaves][region<D>()];
    __shared__ float tops[kWaves][16 * RT], sums[kWaves][16 * RT];
    __shared__ uint32_t tag;
    __shared__ bool complete[2], spansComplete;
    __shared__ Part left[2];
    const PagedAttentionArgs &a = args.a;
    const int w = (int)blockIdx.x;
    const int lane = (int)threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int c = lane / 16, col = lane % 16;
    const int perRow = a.kvHeads * args.blocks;
    constexpr int kPer = kShort ? kTile : kUnit;  // keys of a unit
    const Left parts(args.parts, args.most);

    // A place in the line: unit `tile` of (row b, its hg-th kv head and block).
    struct Place {
        int b, hg, tile;
        Keys keys;
    };
    // Heads of a block; parts that a round of loads takes in a join of more than one task a thread.
    const auto heads_of = [&](int hg) {
        const int h = args.group - hg % args.blocks * 16 * RT;
        return h < 16 * RT ? h : 16 * RT;
    };
    constexpr int kManyTasks = D > 128 ? 4 : 2, kRound = 32 / kManyTasks;
    const auto row_keys = [&](int x) { return Keys(a, __builtin_amdgcn_readfirstlane(a.lengths[x]), kPer); };

    // The workgroup's stretch of units (the wave's, of (row, kv head, block)s) and where it
    // begins.
    Shares shares(1, 1);
    int begin, end;
    Place first{};
    if constexpr (kShort) {
        shares = Shares(a.B * perRow, args.most * kWaves);
        const int worker = w * kWaves + wave;
        if (worker >= shares.grid) {
            return;
        }
        begin = shares.start(worker);
        end = shares.start(worker + 1);
        first.b = begin / perRow;
        first.hg = begin % perRow;
        first.keys = row_keys(first.b);
    } else {
        const uint32_t replay = threadIdx.x == 0 ? dev::replay_load(args.tag.words, w) : 0u;
        const int firstLength = a.lengths[lane < a.B ? lane : 0];
        const int firstUnits = lane < a.B ? Keys(a, firstLength, kPer).units : 0, firstUpto = dev::wave_scan(firstUnits);
        int all = __builtin_amdgcn_readlane(firstUpto, kWave - 1);
        for (int b0 = kWave; b0 < a.B; b0 += kWave) {
            const int x = b0 + lane, L = a.lengths[x < a.B ? x : 0];
            all += __builtin_amdgcn_readlane(dev::wave_scan(x < a.B ? Keys(a, L, kPer).units : 0), kWave - 1);
        }
        shares = Shares(all * perRow, args.most);
        if (threadIdx.x == 0) {
            tag = dev::launch_epoch<Args>(w, replay);
            left[0].on = left[1].on = false;
        }
        if (w >= shares.grid) {
            return;
        }
        begin = shares.start(w);
        end = shares.start(w + 1);
        int b = 0, base = 0, length = 0;  // base: the row's first unit
        int L = firstLength, units = firstUnits, upto = firstUpto;
        for (int b0 = 0;;) {
            const uint64_t past = __ballot(base + upto * perRow > begin);
            if (past != 0) {
                const int at = __ffsll((unsigned long long)past) - 1;
                b = b0 + at;
                base += __builtin_amdgcn_readlane(upto - units, at) * perRow;
                length = __builtin_amdgcn_readlane(L, at);
                break;
            }
            base += __builtin_amdgcn_readlane(upto, kWave - 1) * perRow;
            b0 += kWave;
            L = a.lengths[b0 + lane < a.B ? b0 + lane : 0];
            units = b0 + lane < a.B ? Keys(a, L, kPer).units : 0;
            upto = dev::wave_scan(units);
        }
        first.b = b;
        first.keys = Keys(a, length, kPer);
        first.hg = (begin - base) / first.keys.units;
        first.tile = (begin - base) % first.keys.units;
    }
    const auto advance = [&](Place &x) {
        if (++x.tile < x.keys.units) {
            return;
        }
        x.tile = 0;
        if (++x.hg == perRow) {
            x.hg = 0;
            if (++x.b < a.B) {
                x.keys = row_keys(x.b);
            }
        }
    };
    const auto inside = [&](const Place &x, int unit) { return kShort ? x.b * perRow + x.hg < end : unit < end; };
    Place place = first;

    // The loads run ahead of the products, over the ends of rows: a unit's pages are
    // looked up three units ahead, its rows' addresses found two ahead, and its
    // keys and values leave memory one ahead.
    Place ahead = place;
    int unit = begin;  // the unit at `ahead`
    struct Found {     // lane's key (lane % 32) of a unit
        int page, slot, kvHead;
    };
    const auto find_page = [&]() {
        Found f{-1, 0, 0};
        if (inside(ahead, unit)) {
            const int t = (ahead.keys.first + ahead.tile) * kPer + (kShort ? 0 : wave * kTile) + lane % kTile;
            f.kvHead = kEach ? ahead.b % args.each : ahead.hg / args.blocks;
            if (t >= ahead.keys.low && t < ahead.keys.high) {
                const uint32_t at = (uint32_t)t / (uint32_t)a.pageSize;
                f.page = a.table[(int64_t)ahead.b * a.width + at];
                f.slot = t - (int)(at * (uint32_t)a.pageSize);
            }
            ++unit;
            advance(ahead);
        }
        return f;
    };
    Fragment<D> k[2];
    u32x4_t v[S::kLoads];
    const uint16_t *kFrom[2], *vFrom[S::kLoads];
    uint32_t mask = 0;  // keys at kFrom and vFrom that the row sees
    const auto find_rows = [&](const Found &f) {
        const bool seen = f.page >= 0 && f.page < a.pages;
        mask = __builtin_amdgcn_readfirstlane((int)(uint32_t)__ballot(seen));
        // Where there is no key the first row of the cache is read instead, and not used.
        const int64_t kAt = seen ? f.page * a.kCache.page + f.slot * a.kCache.slot : 0;
        const int64_t vAt = seen ? f.page * a.vCache.page + f.slot * a.vCache.slot : 0;
        const uint16_t *kBase = static_cast<const uint16_t *>(a.kCache.data) + f.kvHead * a.kCache.head;
        const uint16_t *vBase = static_cast<const uint16_t *>(a.vCache.data) + f.kvHead * a.vCache.head;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            kFrom[kt] = kBase + shfl64(kAt, kt * 16 + col);
        }
#pragma unroll
        for (int n = 0; n < S::kLoads; ++n) {
            const int at = n * kWave + lane;
            vFrom[n] = vBase + shfl64(vAt, at / S::kChunks) + at % S::kChunks * 8;
        }
    };
    const auto load = [&]() {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            k[kt].load(kFrom[kt], lane);
        }
#pragma unroll
        for (int n = 0; n < S::kLoads; ++n) {
            v[n] = *reinterpret_cast<const u32x4_t *>(vFrom[n]);
        }
    };
    Fragment<D> q[RT];
    const auto load_q = [&](const Place &x) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int h = x.hg % args.blocks * 16 * RT + rt * 16 + col;
            q[rt].clear();
            if (h < args.group) {
                q[rt].load(static_cast<const uint16_t *>(a.q.data) +
                               first_head<kEach>(a.q, x.b, x.hg / args.blocks, args.group, args.each) + h * a.q.head,
                           lane);
            }
        }
    };
    f32x4_t o[RT][S::kDims];
    float top[RT], sum[RT];
    const auto clear = [&]() {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            top[rt] = -INFINITY;
            sum[rt] = 0.f;
#pragma unroll
            for (int j = 0; j < S::kDims; ++j) {
                o[rt][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            }
        }
    };

    Found found = find_page();
    Found second = find_page(), third = find_page();
    find_rows(found);
    load();
    load_q(place);
    uint32_t now = mask;
    find_rows(second);
    found = third;
    clear();
    bool partial = false;
    int from = begin;  // the first unit of the (row, kv head, block) in this stretch
    char *mine = lds[wave];
    for (int u = begin; inside(place, u); ++u) {
        // V to LDS; what the row does not see is zero there, whatever the cache holds.
        if (now != 0xFFFFFFFFu) {
#pragma unroll
            for (int n = 0; n < S::kLoads; ++n) {
                if ((now >> ((n * kWave + lane) / S::kChunks) & 1u) == 0u) {
                    v[n] = u32x4_t{0, 0, 0, 0};
                }
            }
        }
#pragma unroll
        for (int n = 0; n < S::kLoads; ++n) {
            const int at = n * kWave + lane;
            *reinterpret_cast<u32x4_t *>(mine + at / S::kChunks * P + at % S::kChunks * 16) = v[n];
        }
        f32x4_t s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                s[rt][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < S::kSteps; ++x) {
                    s[rt][kt] = mfma32<kBf16>(k[kt].step[x], q[rt].step[x], s[rt][kt]);
                }
            }
        }
        const uint32_t seen = now;
        const Place here = place;
        advance(place);
        const bool more = inside(place, u + 1);
        const bool ends = here.tile + 1 == here.keys.units || !more;
        if (more) {
            load();
            if (ends) {
                load_q(place);
            }
            now = mask;
            find_rows(found);
            found = find_page();
        }
        if (seen != 0u) {
            u32x4_t p[RT][kTerms<kBf16>];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float x[8], most = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = s[rt][e / 4][e % 4] * (a.scale * kLog2e);
                }
                if (seen != 0xFFFFFFFFu) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = (seen >> (e / 4 * 16 + 4 * c + e % 4) & 1u) != 0u ? x[e] : -INFINITY;
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    most = fmaxf(most, x[e]);
                }
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                const float next = fmaxf(top[rt], most);
                const float zero = next == -INFINITY ? 0.f : next;
                if (__any(next > top[rt])) {  // (else the sums are on the right scale)
                    const float keep = __builtin_amdgcn_exp2f(top[rt] - zero);
                    top[rt] = next;
                    sum[rt] *= keep;
#pragma unroll
                    for (int j = 0; j < S::kDims; ++j) {
                        o[rt][j] *= keep;
                    }
                }
                float part = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(x[e] - zero);
                    part += x[e];
                }
                sum[rt] += part;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p0 = x[2 * e] * kLift<kBf16>, p1 = x[2 * e + 1] * kLift<kBf16>;
                    float rest0 = p0, rest1 = p1;
#pragma unroll
                    for (int n = 0; n < kTerms<kBf16>; ++n) {
                        const uint32_t h =
                            n + 1 < kTerms<kBf16> ? cut2<kBf16>(rest0, rest1) : dev::pack2_x<kBf16>(rest0, rest1);
                        p[rt][n][e] = n == 0 ? h : at_least(h, p0, p1);
                        rest0 -= dev::x_to_f32<kBf16>(h & 0xFFFFu);
                        rest1 -= dev::x_to_f32<kBf16>(h >> 16);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < S::kDims; ++j) {
                const char *at = mine + (4 * c + col / 4) * P + (16 * j + col % 4 * 4) * 2;
                const u32x2_t v0 = read_transposed(at), v1 = read_transposed(at + 16 * P);
                const u32x4_t vt = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                    for (int n = 0; n < kTerms<kBf16>; ++n) {
                        o[rt][j] = mfma32<kBf16>(vt, p[rt][n], o[rt][j]);
                    }
                }
            }
        }
        if (!ends) {
            continue;
        }

        if constexpr (kShort) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                sum[rt] += __shfl_xor(sum[rt], 16);
                sum[rt] += __shfl_xor(sum[rt], 32);
                const int h = here.hg % args.blocks * 16 * RT + rt * 16 + col;
                if (h < args.group) {
#pragma unroll
                    for (int j = 0; j < S::kDims; ++j) {
                        finish<kBf16, kEach>(a, here.b, here.hg / args.blocks * args.group + h, 16 * j + 4 * c,
                                             o[rt][j], top[rt] == -INFINITY ? 0.f : top[rt], sum[rt], args.each);
                    }
                }
            }
            clear();
            continue;
        }

        // The waves' results together, 16 query heads at a time.
        const int kvHead = here.hg / args.blocks, head0 = here.hg % args.blocks * 16 * RT;
        const int u0 = u - here.tile;  // where it begins, in this stretch or before
        const bool whole = from == u0 && here.tile + 1 == here.keys.units;
        const int slot = 2 * w + (from == begin ? 0 : 1);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int rows = heads_of(here.hg) - rt * 16 < 16 ? heads_of(here.hg) - rt * 16 : 16;
            if (rows <= 0) {
                break;
            }
            sum[rt] += __shfl_xor(sum[rt], 16);
            sum[rt] += __shfl_xor(sum[rt], 32);
            if (c == 0) {
                tops[wave][rt * 16 + col] = top[rt];
                sums[wave][rt * 16 + col] = sum[rt];
            }
            float *row = reinterpret_cast<float *>(mine) + col * (D + 4);
            if (col < rows) {
#pragma unroll
                for (int j = 0; j < S::kDims; ++j) {
                    *reinterpret_cast<f32x4_t *>(row + 16 * j + 4 * c) = o[rt][j];
                }
            }
            __syncthreads();
            for (int at = (int)threadIdx.x; at < rows * (D / 4); at += 64 * kWaves) {
                const int row = at / (D / 4), e = at % (D / 4) * 4;
                float most = -INFINITY;
#pragma unroll
                for (int x = 0; x < kWaves; ++x) {
                    most = fmaxf(most, tops[x][rt * 16 + row]);
                }
                const float zero = most == -INFINITY ? 0.f : most;
                float total = 0.f;
                f32x4_t all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < kWaves; ++x) {
                    const float f = __builtin_amdgcn_exp2f(tops[x][rt * 16 + row] - zero);
                    total += f * sums[x][rt * 16 + row];
                    all += f * *reinterpret_cast<const f32x4_t *>(reinterpret_cast<const float *>(lds[x]) +
                                                                  row * (D + 4) + e);
                }
                const int h = head0 + rt * 16 + row;
                if (!whole) {
                    parts.put(slot, rt * 16 + row, e, all);
                    if (e == 0) {
                        parts.put_ends(slot, rt * 16 + row, most, total);
                    }
                } else {
                    finish<kBf16, kEach>(a, here.b, kvHead * args.group + h, e, all, zero, total, args.each);
                }
            }
            __syncthreads();
        }
        if (!whole) {
            partial = true;
            if (threadIdx.x == 0) {
                const int first = shares.owner(u0), last = shares.owner(u0 + here.keys.units - 1);
                left[from == begin ? 0 : 1] =
                    Part{true, here.b, here.hg, first, last, 2 * first + (shares.start(first) == u0 ? 0 : 1),
                         span_bits(last - first + 1, heads_of(here.hg) * (D / 4) <= 64 * kWaves ? 32 : kRound)};
            }
        }
        from = u + 1;
        clear();
    }
    if (kShort || !partial) {
        return;
    }

    // The parts are there once their stores have ended; then they are counted.
    uint64_t found_word = 0;
    int wordSlot = 0;
    if (wave == 0 && lane < 2 && left[lane].on) {
        wordSlot = left[lane].slot(left[lane].span_first(w));
        found_word = parts.word(wordSlot);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (wave == 0 && lane < 2) {
        bool all = false;
        if (left[lane].on) {
            all = parts.count(tag, wordSlot, found_word, left[lane].span_last(w) - left[lane].span_first(w) + 1);
        }
        complete[lane] = all;
    }
    __syncthreads();
    // A thread's tasks (4 values of a head each) times 32 / tasks parts are on their way at once,
    // in groups: those beyond the last part are left out.
    // `spans`: the parts are the results of the spans; `whole`: what comes out is the output.
    const auto join = [&](const Part &part, int head0, int rows, int first, int last, int step, bool spans, bool whole,
                          auto tasks) {
        const int second = spans ? 2 * args.most : 0;
        constexpr int kTasks = decltype(tasks)::value, kBlock = 32 / kTasks, kGroup = kBlock / 4;
        for (int at0 = (int)threadIdx.x; at0 < rows * (D / 4); at0 += 64 * kWaves * kTasks) {
            int row[kTasks], e[kTasks];
            float most[kTasks], zero[kTasks], total[kTasks];
            f32x4_t all[kTasks];
#pragma unroll
            for (int t = 0; t < kTasks; ++t) {
                const int at = at0 + t * 64 * kWaves < rows * (D / 4) ? at0 + t * 64 * kWaves : at0;
                row[t] = at / (D / 4);
                e[t] = at % (D / 4) * 4;
                most[t] = -INFINITY;
                zero[t] = total[t] = 0.f;
                all[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            }
            for (int x0 = first; x0 <= last; x0 += kBlock * step) {
                u32x2_t ends[kTasks][kBlock];
                f32x4_t outs[kTasks][kBlock];
#pragma unroll
                for (int m0 = 0; m0 < kBlock; m0 += kGroup) {
                    if (x0 + m0 * step <= last) {
#pragma unroll
                        for (int m = m0; m < m0 + kGroup; ++m) {
                            const int slot = part.slot(x0 + m * step <= last ? x0 + m * step : x0 + m0 * step);
#pragma unroll
                            for (int t = 0; t < kTasks; ++t) {
                                ends[t][m] = parts.end(slot + second, row[t]);
                                outs[t][m] = parts.out(slot, row[t], e[t]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int m = m0; m < m0 + kGroup; ++m) {
#pragma unroll
                            for (int t = 0; t < kTasks; ++t) {
                                ends[t][m] = u32x2_t{0xFF800000u, 0u};  // (-inf: weight 0)
                                outs[t][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                            }
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < kTasks; ++t) {
                    float next = most[t];
#pragma unroll
                    for (int m = 0; m < kBlock; ++m) {
                        next = fmaxf(next, __uint_as_float(ends[t][m][0]));
                    }
                    zero[t] = next == -INFINITY ? 0.f : next;
                    const float keep = __builtin_amdgcn_exp2f(most[t] - zero[t]);
                    most[t] = next;
                    total[t] *= keep;
                    all[t] *= keep;
#pragma unroll
                    for (int m = 0; m < kBlock; ++m) {
                        if (x0 + m * step <= last) {
                            const float f = __builtin_amdgcn_exp2f(__uint_as_float(ends[t][m][0]) - zero[t]);
                            total[t] += f * __uint_as_float(ends[t][m][1]);
                            all[t] += f * outs[t][m];
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < kTasks; ++t) {
                if (at0 + t * 64 * kWaves >= rows * (D / 4)) {
                } else if (whole) {
                    finish<kBf16, kEach>(a, part.b, part.hg / args.blocks * args.group + head0 + row[t], e[t], all[t],
                                         zero[t], total[t], args.each);
                } else {
                    parts.put(part.slot(first), row[t], e[t], all[t]);
                    if (e[t] == 0) {
                        parts.put_ends(part.slot(first) + 2 * args.most, row[t], most[t], total[t]);
                    }
                }
            }
        }
    };
    for (int n = 0; n < 2; ++n) {
        if (!complete[n]) {
            continue;
        }
        const Part part = left[n];
        const int head0 = part.hg % args.blocks * 16 * RT;
        const int rows = heads_of(part.hg);
        const auto join_all = [&](int first, int last, int step, bool spans, bool whole) {
            if (rows * (D / 4) <= 64 * kWaves) {
                join(part, head0, rows, first, last, step, spans, whole, std::integral_constant<int, 1>{});
            } else {
                join(part, head0, rows, first, last, step, spans, whole, std::integral_constant<int, kManyTasks>{});
            }
        };
        const bool one = part.spans() == 1;
        join_all(part.span_first(w), part.span_last(w), 1, false, one);
        if (one) {
            continue;
        }
        const int slot = part.firstSlot + 2 * args.most;
        uint64_t found = 0;
        if (threadIdx.x == 0) {
            found = parts.word(slot);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            spansComplete = parts.count(tag, slot, found, part.spans());
        }
        __syncthreads();
        if (spansComplete) {
            join_all(part.first, part.last, 1 << part.spanBits, true, true);
        }
        __syncthreads();
    }
}

template <bool kBf16, int D, int RT, bool kEach>
hipError_t launch_size(const Args &args, hipStream_t stream)
{
    int grid = args.most;
    auto kernel = attention_units<kBf16, D, RT, false, kEach>;
    if constexpr (RT == 1) {
        if (args.parts == nullptr) {
            kernel = attention_units<kBf16, D, RT, true, kEach>;
            const int items = args.a.B * args.a.kvHeads * args.blocks;
            grid = (items + kWaves - 1) / kWaves < grid ? (items + kWaves - 1) / kWaves : grid;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * kWaves), 0, stream, args);
    return hipGetLastError();
}

template <bool kBf16, int RT, bool kEach = false>
hipError_t launch_heads(const Args &args, hipStream_t stream)
{
    switch (args.a.d) {
    case 32: return launch_size<kBf16, 32, RT, kEach>(args, stream);
    case 64: return launch_size<kBf16, 64, RT, kEach>(args, stream);
    case 80: return launch_size<kBf16, 80, RT, kEach>(args, stream);
    case 96: return launch_size<kBf16, 96, RT, kEach>(args, stream);
    case 112: return launch_size<kBf16, 112, RT, kEach>(args, stream);
    case 128: return launch_size<kBf16, 128, RT, kEach>(args, stream);
    case 160: return launch_size<kBf16, 160, RT, kEach>(args, stream);
    case 192: return launch_size<kBf16, 192, RT, kEach>(args, stream);
    case 256:
        if constexpr (RT == 1) {
            return launch_size<kBf16, 256, RT, kEach>(args, stream);
        }
        return hipErrorInvalidValue;
    default: return hipErrorInvalidValue;
    }
}

// One file per instance: mhc_paged_attention_{bf16,f16}.hip, RT 1 and 2.
hipError_t launch_bf16(const Args &args, bool wide, hipStream_t stream);
hipError_t launch_f16(const Args &args, bool wide, hipStream_t stream);
// kEach's: mhc_sparse_attention_{bf16,f16}.hip.
hipError_t launch_each_bf16(const Args &args, bool wide, hipStream_t stream);
hipError_t launch_each_f16(const Args &args, bool wide, hipStream_t stream);

// How a call is laid out (mhc_paged_attention_bf16.hip): 32 query heads at a time or 16, and
// whether rows are short enough for a wave each.
Args plan(const PagedAttentionArgs &a, int cus, bool &wide);
bool short_rows(const PagedAttentionArgs &a, const Args &p, bool wide);

}  // namespace attention
}  // namespace mhc
