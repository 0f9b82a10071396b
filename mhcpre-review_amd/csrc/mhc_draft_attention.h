// Attention of several new tokens per sequence over a paged cache
// (mhcDraftAttention): the kernels, instantiated per element type.
//
// The rows of a (sequence, kv head) are its new tokens' query heads that share the
// kv head, token by token; a block of them (32 a wave) goes over the keys in
// tiles.  As in the kernel of single tokens, all units (tiles) of all (sequence,
// kv head, block)s form one line that is shared out evenly to a fixed grid, what a
// stretch leaves of a row that it does not finish goes to the workspace, and a
// second launch joins these parts in the order of the keys.
//
// In a tile the scores are S^T = K Q^T, 32 keys by 32 rows, so that a lane has
// half of one row's scores (lane l: row l % 32) and the probabilities, as they lie
// in its registers, are the operand of O^T = V^T P^T: the order of the keys within
// a product is free.  K and V go through LDS, where kRowWaves waves share them; V
// is read transposed (ds_read_b64_tr_b16).  A probability is the sum of two 16-bit
// terms, the first one cut, the second rounded: bf16 holds 16 bits, fp16 (lifted, for
// its range ends at 2^-24) 22.  One term alone would add an error of the size of the
// output's own rounding; it took 237 us where two took 297 (2 of 65536, below).
//
// What a row sees is all of the context in front of the new tokens (but for a
// window), and of the new tokens its ancestors, found from the parents by
// doubling (the ancestors of my farthest known ancestor are mine), 256 bits a token.
// Tiles that all rows see whole have no masks.  The loop takes V as finite: an
// infinite or NaN value times a weight of zero would reach rows that do not see
// it.  Where a block's output is not finite (or near the end of fp32), the block is done
// again with such values taken out of the products and added to the rows that see them
// alone.
//
// What bounds it, and what it reaches (8 kv heads of 128; a copy reaches 4.9 TB/s, a
// product of 8192^3 1140 TFLOP/s): memory for few rows, 32 sequences of 8192 tokens with
// trees of 8 nodes of 4 heads each 202 to 212 us, 5.1 to 5.3 TB/s; the matrix cores for many,
// 2 of up to 65536 with trees of 64 of 8 heads each 265 us, and 285 to 300 where calls follow each
// other without a pause (the clock falls): 490 to 550 TFLOP/s of the formulas' operations, half
// as many again with the second term's.  There a tile's exponentials, splits and LDS reads
// stand between its products: they are written among each other, and half of the time is
// the products' own.  A chunk of 2048 tokens behind 6144, 4 heads each, 370 us, 650 TFLOP/s.  A
// single small sequence costs two launches, one chain of loads and the join: 17 us.
//
// What is not used, and could be: a wave without rows that are there does all products
// (a block is 256 rows for a tree of 64 of 8 heads, of which 52 nodes may be there), a window's
// whole tiles are taken to begin where the last new token's window does, and every workgroup
// counts all blocks of a sequence before its first tile (a call for 2048 tokens of 16 heads to
// one of which one is there 70 us, for 8192 242).
#pragma once

#include "mhc_paged_attention.h"

namespace mhc {
namespace draft {

using attention::bf16x8v_t;
using attention::f16x8_t;
using attention::kLn2;
using attention::kLog2e;
using attention::shfl64;
using attention::u32x2_t;
using dev::f32x4_t;
using dev::kWave;
using dev::u32x4_t;

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kRows = 32;  // of a wave

// What is loaded in the place of keys that nobody sees (a row of the largest size).
__device__ const uint32_t kZeros[128] = {};

// 16 bytes a lane from memory to LDS, lane by lane from `to` on.  In assembly, for the
// compiler would let every read of LDS wait for all such loads: the caller waits
// (dev::wait_vm) before a tile is read.  (m0 is no register that the compiler hands out.)
__device__ __forceinline__ void load_to_lds(const void *from, __attribute__((address_space(3))) char *to)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"((uint32_t)(uintptr_t)to), "v"(from)
                 : "memory");
}
// The same from `base`, which all lanes share, and an offset of the lane's.
__device__ __forceinline__ void load_to_lds(uint64_t base, uint32_t offset, __attribute__((address_space(3))) char *to)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"((uint32_t)(uintptr_t)to), "v"(offset), "s"(base)
                 : "memory");
}

// How a workgroup's waves are laid out: kRowWaves share a tile, each with rows of its
// own, and kKeyWaves such groups have tiles of their own.  Tiles come from memory
// straight into LDS, the next one while this one is worked on.
template <int D_, int kRowWaves_, int kKeyWaves_, int kTile_>
struct Layout {
    static constexpr int D = D_, kRowWaves = kRowWaves_, kKeyWaves = kKeyWaves_, kTile = kTile_;
    static constexpr int kWaves = kRowWaves * kKeyWaves, kThreads = kWave * kWaves;
    static constexpr int kUnit = kTile * kKeyWaves;  // keys of a unit
    static constexpr int kBlock = kRows * kRowWaves;
    static constexpr int kChunks = D / 8;                       // 16-byte chunks of a row
    static constexpr int kSide = kTile * kChunks * 16;          // bytes of a tile of K or V
    static constexpr int kBuffer = 2 * kSide;                   // K, then V
    static constexpr int kLoads = kSide / 1024 / kRowWaves;     // of a wave, for either
    static constexpr int kLds = 2 * kBuffer * kKeyWaves;
    static constexpr int kMore = kDraftNodes * 36 + kKeyWaves * kBlock * 8 + 256;  // the other LDS
    // Workgroups of a CU: what its registers (two waves a SIMD up to D = 128) and LDS hold.
    static constexpr int kPerCu = kThreads == 256 && D <= 128 && 2 * (kLds + kMore) <= 160 * 1024 ? 2 : 1;
    static_assert(kLoads * kRowWaves * 1024 == kSide && kLds + kMore <= 160 * 1024);
    // What a group's waves leave to be joined fits a buffer.
    static_assert(kKeyWaves == 1 || (kRowWaves == 1 && kRows * D * 4 <= kBuffer) ||
                  kRowWaves * kRows * D * 4 / kKeyWaves <= kBuffer);

    // Rows that whole loads of 64 chunks cover together: in a page of a multiple of these the
    // loads of such a group have one page.
    static constexpr int kGroupRows = kChunks % 16 == 0 ? 64 / kChunks : kChunks % 8 == 0 ? 8 : 16;

    // Where chunk c of row r lies among its row's chunks: turned so that what 16 lanes read at
    // a time lies in different banks, of K the same chunk of 16 rows, of V 64 bytes of 4 rows.
    __device__ static constexpr int turn(int r)
    {
        return kChunks % 16 == 0  ? (r & 3) << 2 | (r >> 2 & 3)
               : kChunks % 8 == 0 ? (r >> 1 & 1) << 2 | (r >> 2 & 3)
                                  : r >> 2 & 3;
    }
    __device__ static constexpr uint32_t at(int r, int c) { return (r * kChunks + (c ^ turn(r))) * 16; }
    // A constant step of `by` chunks (a multiple of the lanes' own range) from place p of a row
    // whose turn is in p: what the turn reaches changes by an exclusive or, the rest by a sum.
    static constexpr int kTurned = kChunks % 16 == 0 ? 16 : kChunks % 8 == 0 ? 8 : 4;
    __device__ static uint32_t step(uint32_t p, int by) { return (p ^ by % kTurned * 16) + by / kTurned * kTurned * 16; }
};

// What a (sequence, kv head, block) costs beside its tiles (its start and end), in tiles: it
// stands for that in the line, in front of its tiles.  (32 sequences of 1 to 8192 tokens with
// trees of 8: 206 us if it stands for nothing, 99 so.)
constexpr int kItemUnits = 3;

// What a stretch begins and does not finish: a (sequence, kv head, block), the stretch that
// finishes it, and the slot of its first part.  last < 0: nothing.
struct Open {
    int last, b, kv, block, slot, none[3];
};

struct Args {
    DraftAttentionArgs a;
    int group;   // query heads of a kv head
    int blocks;  // blocks of rows of a (sequence, kv head)
    int rows;    // of a block
    int unit;    // keys of a unit
    int most;    // workgroups of the launch
    bool grouped;  // pages of whole groups of rows (Layout::kGroupRows), the caches' strides alike
    float *outs, *ends;  // the parts: [2 * most][rows / 32][D / 8][64][4], [2 * most][rows][2]
    Open *open;          // [most]
};

// The kernel's arguments, and the lane's number, for what is done once a block: read and
// derived there.  (Derived from what is known at the kernel's start, all of it would be
// computed in front of the loop and held over it, and registers be spilled in it, whose
// reloads wait for the tile on its way.)
__device__ __forceinline__ const Args &late() { return *(const Args *)dev::late_args<Args>(); }
__device__ __forceinline__ int late_lane()
{
    int lane = (int)threadIdx.x % kWave;
    asm volatile("" : "+v"(lane));
    return lane;
}
__device__ __forceinline__ int late_thread()
{
    int thread = (int)threadIdx.x;
    asm volatile("" : "+v"(thread));
    return thread;
}

// The keys of a block of a sequence with c + n tokens, n of them new: [low, high), in
// `tiles` (units of the launch, one at least) from `first` on.
struct Keys {
    int low, high, first, tiles;
};

struct Sequence {
    int c, n;  // tokens in front of the new ones, new ones

    __device__ Sequence(int c_, int n_) : c(c_), n(n_) {}
    __device__ Sequence(const DraftAttentionArgs &a, int L, int m)
    {
        const int most = a.width * a.pageSize;
        L = L < 0 ? 0 : L > most ? most : L;
        m = m < 0 ? 0 : m > a.S ? a.S : m;
        n = m < L ? m : L;
        c = L - n;
    }
    // A lane's own row, and the same row for all lanes (by scalar loads, which do not wait for
    // vector ones).
    __device__ static Sequence of(const DraftAttentionArgs &a, int b) { return {a, a.lengths[b], a.drafted[b]}; }
    __device__ static Sequence same(const DraftAttentionArgs &a, int b)
    {
        typedef const __attribute__((address_space(4))) int32_t *Scalar;
        return {a, ((Scalar)(uintptr_t)a.lengths)[b], ((Scalar)(uintptr_t)a.drafted)[b]};
    }
    __device__ Keys keys(const Args &args, int block) const
    {
        // (rows of a kv head stay below 2^30)
        const uint32_t group = (uint32_t)args.group, row0 = (uint32_t)(block * args.rows);
        const int i0 = args.blocks == 1 ? 0 : (int)(row0 / group);
        const int last = args.blocks == 1 ? n : (int)((row0 + (uint32_t)args.rows + group - 1) / group);
        const int i1 = last < n ? last : n;
        Keys k{0, 0, 0, 1};
        if (i0 < n) {
            // A chain's token i is at position c + i, a tree's at c or later.
            const int64_t from = (int64_t)c + (args.a.parents == nullptr ? i0 : 0) + 1 - args.a.window;
            k.low = args.a.window > 0 && from > 0 ? (int)from : 0;
            k.high = c + i1;
            k.first = k.low / args.unit;
            k.tiles = (k.high - 1) / args.unit + 1 - k.first;
        }
        return k;
    }
    // Of a kv head, in the line.
    __device__ int units(const Args &args) const
    {
        int all = args.blocks * kItemUnits;
        for (int x = 0; x < args.blocks; ++x) {
            all += keys(args, x).tiles;
        }
        return all;
    }
};

template <bool kBf16>
__device__ __forceinline__ f32x16_t mfma(u32x4_t a, u32x4_t b, f32x16_t c)
{
    if constexpr (kBf16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v_t, a),
                                                       __builtin_bit_cast(bf16x8v_t, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b),
                                                      c, 0, 0, 0);
    }
}

// Weights are relative to a reference near the maximum, which follows it only where it
// has grown by more than kSlack bits: a weight may be as large as 2^kSlack, and in fp16 with
// what all of them are multiplied by (2^kLiftBits, for the type ends at 2^-24) 2^15.
constexpr float kSlack = 5.f;
template <bool kBf16>
constexpr float kLiftBits = kBf16 ? 0.f : 15.f - kSlack;

// bf16 values end where fp32 does, so that sums of finite ones may pass its end before they
// are divided.  Below 2^116 at a block's end they do not later: up to 4 waves' and 512
// workgroups' are added.  Where one is not, the block is done again, and the reference is then
// kRaised + log2 n bits above the scores of the values that are large: n of them below 2^128, with
// weights of at most 2^(kSlack - kRaised) / n, and n others of weights up to 2^kSlack, sum up to
// less than 2^116.  (Weights of less than 2^-108 n of a large value's may then count as 0:
// whatever their values, n of them are not n^3 2^-90 of that value's product.)  fp16's have room.
template <bool kBf16>
constexpr float kFar = kBf16 ? 8192.f : 1.f;  // (2^116 times this takes any finite sum beyond the end)
constexpr float kRaised = 18.f;
// log2 n, rounded up, and the exponent bits of a large value, 2^110 / n.
__device__ __forceinline__ int bits_of(int n) { return 32 - __clz(n); }
__device__ __forceinline__ uint32_t large_from(int n) { return (uint32_t)(127 + 110 - bits_of(n)) << 7; }

template <bool kBf16>
__device__ __forceinline__ bool infinite(uint32_t bits)
{
    constexpr uint32_t kExponent = kBf16 ? 0x7F80u : 0x7C00u;
    return (bits & kExponent) == kExponent;
}

__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }

// A factor of at most 1 for a sum whose infinite values stay infinite.
__device__ __forceinline__ float scaled(float x, float f)
{
    return __builtin_isfinite(x) ? x * f : x * fmaxf(f, 1e-30f);
}

// A tile of the line: sequence (its context and new tokens), kv head, block, and the tile of
// its keys.
struct Place {
    int b, kv, block, tile;
    int start;  // the line's unit of tile 0
    int c, n;
    Keys keys;

    __device__ void enter(const Args &args)
    {
        const Sequence s = Sequence::same(args.a, b);
        c = s.c;
        n = s.n;
        keys = s.keys(args, block);
    }
    __device__ bool inside(int end) const { return start + tile < end; }
    // (Behind the last sequence: at the line's end, which is inside of no stretch.)
    __device__ void advance()
    {
        if (++tile < keys.tiles) {
            return;
        }
        const Args &args = late();
        tile = 0;
        start += keys.tiles + kItemUnits;
        if (++block == args.blocks) {
            block = 0;
            if (++kv == args.a.kvHeads) {
                kv = 0;
                ++b;
            }
        }
        if (b < args.a.B) {
            enter(args);
        } else {
            start = INT32_MAX;
            keys.tiles = INT32_MAX;
        }
    }
};

// The line of all tiles, 64 sequences at a time: a lane has one's context, new tokens and
// units, and the units up to it.
struct Line {
    int all;  // all units
    int c, n, units, upto;  // of sequences 0 to 63

    __device__ explicit Line(const Args &args) : all(0)
    {
        for (int b0 = 0; b0 < args.a.B; b0 += kWave) {
            Line part;
            part.read(args, b0);
            all += __builtin_amdgcn_readlane(part.upto, kWave - 1);
            if (b0 == 0) {
                c = part.c;
                n = part.n;
                units = part.units;
                upto = part.upto;
            }
        }
    }
    // The first tile at unit `at` of the line or behind it.
    __device__ Place find(const Args &args, int at) const
    {
        const DraftAttentionArgs &a = args.a;
        int base = 0;
        Line part = *this;
        for (int b0 = 0;;) {
            const uint64_t past = __ballot(base + part.upto > at);
            if (past == 0 && b0 + kWave < a.B) {
                base += __builtin_amdgcn_readlane(part.upto, kWave - 1);
                b0 += kWave;
                part.read(args, b0);
                continue;
            }
            const int hit = __ffsll((unsigned long long)past) - 1;
            Place p;
            p.b = b0 + hit;
            p.c = __builtin_amdgcn_readlane(part.c, hit);
            p.n = __builtin_amdgcn_readlane(part.n, hit);
            const int row = __builtin_amdgcn_readlane(part.units, hit);
            base += __builtin_amdgcn_readlane(part.upto, hit) - row;
            const uint32_t one = (uint32_t)row / (uint32_t)a.kvHeads;
            p.kv = (int)((uint32_t)(at - base) / one);
            base += p.kv * (int)one;
            for (p.block = 0;; ++p.block) {
                p.keys = Sequence(p.c, p.n).keys(args, p.block);
                if (at < base + kItemUnits + p.keys.tiles) {
                    break;
                }
                base += kItemUnits + p.keys.tiles;
            }
            p.start = base + kItemUnits;
            p.tile = at > p.start ? at - p.start : 0;
            return p;
        }
    }

private:
    Line() = default;
    __device__ void read(const Args &args, int b0)
    {
        const int x = b0 + (int)threadIdx.x % kWave;
        const Sequence s = Sequence::of(args.a, x < args.a.B ? x : 0);
        c = s.c;
        n = s.n;
        units = x < args.a.B ? s.units(args) * args.a.kvHeads : 0;
        upto = dev::wave_scan(units);
    }
};

// 4 values of row `row` of a block, from their sum and its weights' sum and maximum.
template <bool kBf16>
__device__ __forceinline__ void finish(const Args &args, const Place &p, int node, int head, int e, f32x4_t all,
                                       float top, float total)
{
    const DraftAttentionArgs &a = args.a;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int h = p.kv * args.group + head;
    if (e < a.d) {
        uint16_t *out = static_cast<uint16_t *>(a.out.data) + p.b * a.out.row + node * a.out.token + h * a.out.head + e;
        *reinterpret_cast<u32x2_t *>(out) =
            u32x2_t{dev::pack2_x<kBf16>(all[0] * inv, all[1] * inv), dev::pack2_x<kBf16>(all[2] * inv, all[3] * inv)};
    }
    if (e == 0 && a.lse != nullptr) {
        a.lse[((int64_t)p.b * a.S + node) * a.heads + h] =
            ((top == -INFINITY ? 0.f : top) + (__builtin_amdgcn_logf(total) - kLiftBits<kBf16>)) * kLn2;
    }
}

// The ancestors of every node of a row, 256 bits each (itself among them), from the parents
// of a thread's nodes.  A node's farthest known ancestor's are its own too: each round doubles
// how far.
template <int kThreads, int kNodes>
__device__ __forceinline__ void find_ancestors(const int (&parents)[kNodes], int n, uint64_t (&known)[kDraftNodes][4],
                                               int (&farthest)[kDraftNodes])
{
    const int thread = late_thread();
    uint64_t own[kNodes][4];
    int far[kNodes];
#pragma unroll
    for (int k = 0; k < kNodes; ++k) {
        const int i = k * kThreads + thread;
        far[k] = -1;
        if (i < n) {
            const int p = parents[k];
            far[k] = p >= 0 && p < i ? p : -1;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            own[k][x] = i / 64 == x ? 1ull << (i % 64) : 0ull;
        }
    }
    for (int reach = 1;; reach *= 2) {
#pragma unroll
        for (int k = 0; k < kNodes; ++k) {
            const int i = k * kThreads + thread;
            if (i < n) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    known[i][x] = own[k][x];
                }
                farthest[i] = far[k];
            }
        }
        __syncthreads();
        if (reach >= n) {
            return;
        }
#pragma unroll
        for (int k = 0; k < kNodes; ++k) {
            if (far[k] >= 0) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    own[k][x] |= known[far[k]][x];
                }
                far[k] = farthest[far[k]];
            }
        }
        __syncthreads();
    }
}

// Which of the 64 keys from t0 on a node sees: the context from `from` on, and of the new
// tokens its ancestors but the first `over`, or in a chain those from `from` up to itself.
__device__ __forceinline__ uint64_t seen_keys(bool tree, int c, int node, uint32_t from, int over, int64_t t0,
                                              const uint64_t (&known)[kDraftNodes][4])
{
    // (positions below 2^31 and their differences fit 33 bits)
    const int64_t to = (tree ? c : (int64_t)c + node + 1) - t0, first = (int64_t)from - t0;
    uint64_t seen = low_bits(to > 64 ? 64 : to < 0 ? 0 : (int)to) & ~low_bits(first > 64 ? 64 : first < 0 ? 0 : (int)first);
    if (tree && t0 + 64 > c) {
        // Bit x of the tile is node x + t0 - c.
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int64_t by = t0 - c - 64 * x;
            uint64_t own = known[node][x];
            while (over > 0 && own != 0) {
                own &= own - 1;
                --over;
            }
            if (by > -64 && by < 64) {
                seen |= by >= 0 ? own >> by : own << -by;
            }
        }
    }
    return seen;
}

// What the first of a weight's two terms leaves: x without its upper 8 (bf16) or 11 (fp16)
// bits.  (An fp16 below 2^-14 holds fewer: then up to 2^-24 is lost, 2^-34 of the largest
// weight.)
template <bool kBf16>
__device__ __forceinline__ float rest(float x)
{
    return x - __uint_as_float(__float_as_uint(x) & (kBf16 ? 0xFFFF0000u : 0xFFFFE000u));
}

// 4 values at the same column of 4 rows of LDS (the lane's column of 16).
__device__ __forceinline__ u32x2_t transposed(uint32_t at)
{
    return __builtin_bit_cast(
        u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attention::s16x4_t *)(uintptr_t)at));
}

// Keeps the instructions on both sides in the order that they are written in.  (Left to
// itself the compiler waits for every operand where registers are short.)
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

template <bool kBf16, typename L>
__global__ __launch_bounds__(L::kThreads, (L::kThreads * L::kPerCu + 255) / 256) void draft_units(Args args)
{
    constexpr int D = L::D, kTile = L::kTile, kKt = kTile / 32, kSteps = D / 16, kDims = D / 32;
    __shared__ __align__(256) char lds[L::kLds];
    __shared__ uint64_t known[kDraftNodes][4];  // the new tokens' ancestors
    __shared__ int farthest[kDraftNodes];
    __shared__ uint64_t setApart[L::kKeyWaves][2];  // keys of a tile with infinite and NaN values, and with large ones
    __shared__ float2 ends[L::kKeyWaves][L::kBlock];
    __shared__ bool odd[L::kWaves];
    const DraftAttentionArgs &a = args.a;
    const int w = (int)blockIdx.x;
    const int lane = (int)threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int rowWave = wave % L::kRowWaves, keyWave = wave / L::kRowWaves;
    const int half = lane / 32, col = lane % 32;
    auto *const mine = (__attribute__((address_space(3))) char *)lds + keyWave * 2 * L::kBuffer;
    // Where a lane reads in a tile: of K row `col` and every second chunk from `half` on; of V
    // (turned) rows 4 half + .. and + 8, 4 columns of 32.
    const uint32_t kPlace = L::at(col, half);
    const uint32_t vPlace = L::at(4 * half + lane % 16 / 4, lane / 16 % 2 * 2 + lane % 4 / 2) + lane % 2 * 8;
    const bool tree = a.parents != nullptr;
    // (The scale's sign goes to q, for the maximum wants a factor above 0; with a scale of 0 q is 0.)
    const float factor = a.scale == 0.f ? 1.f : fabsf(a.scale * kLog2e);

    const Line line(args);
    const attention::Shares shares(line.all, args.most);
    if (threadIdx.x == 0) {
        args.open[w].last = -1;
    }
    if (w >= shares.grid) {
        return;
    }
    const int begin = shares.start(w), end = shares.start(w + 1);
    Place here = line.find(args, begin);
    if (!here.inside(end)) {
        return;
    }

    // The lane's key (lane % kTile) of the tile at `ahead`: its page and slot.
    Place ahead = here;
    const int32_t *table = a.table + (int64_t)here.b * a.width;
    uint32_t page = 0, t = 0, column = 0, slot = 0;
    int foundKv = here.kv;
    bool key = false, enters = true;  // enters: `ahead` is the first tile of its block here
    const uint32_t pageSize = (uint32_t)a.pageSize, stepColumns = L::kUnit / pageSize, stepSlots = L::kUnit % pageSize;
    const auto find_page = [&]() {
        key = false;
        if (ahead.inside(end)) {
            if (enters) {
                t = (uint32_t)(ahead.keys.first + ahead.tile) * L::kUnit + keyWave * kTile + lane % kTile;
                column = t / pageSize;
                slot = t - column * pageSize;
                table = a.table + (int64_t)ahead.b * a.width;
                foundKv = ahead.kv;
            } else {
                t += L::kUnit;
                slot += stepSlots;
                const bool over_ = slot >= pageSize;
                column += stepColumns + (over_ ? 1u : 0u);
                slot -= over_ ? pageSize : 0u;
            }
            key = t >= (uint32_t)ahead.keys.low && t < (uint32_t)ahead.keys.high;
            ahead.advance();
            enters = ahead.tile == 0;
        }
        // (Always a load, of the row's first entry where there is no key: under a branch it would
        // be waited for at once.)
        page = (uint32_t)table[key ? column : 0u];
    };
    uint64_t loaded = 0;  // keys of the tile on its way
    const auto load = [&](int buffer) {
        const bool seen = key && page < (uint64_t)a.pages;
        loaded = __ballot(seen);
        if constexpr (kTile == 32) {
            loaded &= 0xFFFFFFFFull;
        }
        const uint64_t kAt = 2 * (page * (uint64_t)a.kCache.page + slot * (uint64_t)a.kCache.slot);
        const uint64_t kFirst = (uint64_t)a.kCache.data + 2 * foundKv * a.kCache.head;
        const uint64_t vFirst = (uint64_t)a.vCache.data + 2 * foundKv * a.vCache.head;
        auto *const to = mine + buffer * L::kBuffer;
        if (args.grouped && loaded == (kTile == 64 ? ~0ull : 0xFFFFFFFFull)) {
            // The row where a group of rows begins is found by one lane for all, and the others lie
            // behind it: no address is a lane's own.
            const uint32_t slotBytes = 2 * (uint32_t)a.kCache.slot;
#pragma unroll
            for (int n = 0; n < L::kLoads; ++n) {
                const int first = (n * L::kRowWaves + rowWave) * kWave, at = first + lane;
                const int r = at / L::kChunks, ch = at % L::kChunks ^ L::turn(r), group = first / L::kChunks & -L::kGroupRows;
                const uint64_t row = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(kAt >> 32), group) << 32 |
                                     (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)kAt, group);
                const uint32_t offset = (uint32_t)(r - group) * slotBytes + ch * 16;
                load_to_lds(kFirst + row, offset, to + first * 16);
                load_to_lds(vFirst + row, offset, to + L::kSide + first * 16);
            }
            return;
        }
        const uint64_t vAt = 2 * (page * (uint64_t)a.vCache.page + slot * (uint64_t)a.vCache.slot);
        const uint64_t zeros = (uint64_t)kZeros;
        const int64_t kRow = (int64_t)(seen ? kFirst + kAt : zeros), vRow = (int64_t)(seen ? vFirst + vAt : zeros);
        uint64_t k[L::kLoads], v[L::kLoads];
#pragma unroll
        for (int n = 0; n < L::kLoads; ++n) {
            const int at = (n * L::kRowWaves + rowWave) * kWave + lane;
            const int r = at / L::kChunks, ch = at % L::kChunks ^ L::turn(r);
            k[n] = (uint64_t)shfl64(kRow, r) + ch * 16;
            v[n] = (uint64_t)shfl64(vRow, r) + ch * 16;
            if (ch * 8 >= a.d) {
                k[n] = v[n] = zeros;
            }
        }
#pragma unroll
        for (int n = 0; n < L::kLoads; ++n) {
            const int first = (n * L::kRowWaves + rowWave) * kWave;
            load_to_lds((const void *)k[n], to + first * 16);
            load_to_lds((const void *)v[n], to + L::kSide + first * 16);
        }
    };
    // The operand of the rows of a place's block.  (It is turned where it is used first: what a
    // load brings must not be touched before the wait at the loop's head.)
    u32x4_t q[kSteps];
    constexpr int kNodes = kDraftNodes / L::kThreads > 0 ? kDraftNodes / L::kThreads : 1;  // of a thread
    int parents[kNodes];
    const auto load_q = [&](const Place &p) {
        const Args &l = late();
        const int ln = late_lane();
        const int row = p.block * L::kBlock + rowWave * kRows + ln % 32;
        const int node = row / l.group, head = row - node * l.group;
        const uint16_t *from = static_cast<const uint16_t *>(l.a.q.data) + p.b * l.a.q.row + node * l.a.q.token +
                               (int64_t)(p.kv * l.group + head) * l.a.q.head + ln / 32 * 8;
        const bool on = node < p.n && l.a.scale != 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q[s] = *reinterpret_cast<const u32x4_t *>(on && 16 * s < l.a.d ? from + 16 * s
                                                                           : reinterpret_cast<const uint16_t *>(kZeros));
        }
        // (and the parents, which are asked for where the block is entered)
        const int32_t *const row_ = l.a.parents != nullptr ? l.a.parents + (int64_t)p.b * l.a.S
                                                           : reinterpret_cast<const int32_t *>(kZeros);
#pragma unroll
        for (int k = 0; k < kNodes; ++k) {
            const int i = k * L::kThreads + (int)threadIdx.x;
            parents[k] = row_[l.a.parents != nullptr && i < l.a.S ? i : 0];
        }
    };
    const auto turn_q = [&]() {
        const uint32_t flip = late().a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q[s] ^= u32x4_t{flip, flip, flip, flip};
        }
    };

    f32x16_t o[kDims];
    float top, sum;
    const auto clear = [&]() {
#pragma unroll
        for (int j = 0; j < kDims; ++j) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                o[j][i] = 0.f;
            }
        }
        top = -INFINITY;
        sum = 0.f;
    };
    // The lane's row of the block at `here`: its node, where its context begins, how many of its
    // first ancestors lie in front of its window; and tiles in [wholeFrom, wholeTo) that all rows
    // of the wave see whole.
    int node = 0, over = 0, maskedRow = -1;
    bool there = false;
    uint32_t from = 0;
    int wholeFrom = 0, wholeTo = 0;  // (a chain's last block may say one more than there are)
    const auto enter = [&]() {
        const Args &l = late();
        const int row0 = here.block * L::kBlock + rowWave * kRows;
        node = (row0 + late_lane() % 32) / l.group;
        there = node < here.n;
        int depth = node;
        const int lastTile = end - 1 - here.start < here.keys.tiles - 1 ? end - 1 - here.start : here.keys.tiles - 1;
        if (tree && here.n > 0 &&
            (l.a.window > 0 || (int64_t)(here.keys.first + lastTile + 1) * L::kUnit > here.c)) {
            if (maskedRow != here.b) {
                __syncthreads();  // (the ones before are read)
                find_ancestors<L::kThreads>(parents, here.n, known, farthest);
                maskedRow = here.b;
            }
            if (l.a.window > 0) {
                depth = -1;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    depth += there ? __popcll(known[node][x]) : 0;
                }
            }
        }
        over = l.a.window > 0 && l.a.window < depth + 1 ? depth + 1 - (int)l.a.window : 0;
        // (The context that the row sees: [from, c); a chain's row: [from, c + node].)
        const int64_t from64 = (int64_t)here.c + depth + 1 - l.a.window;
        from = l.a.window > 0 && from64 > 0 ? (uint32_t)from64 : 0u;
        wholeTo = tree ? here.c : here.c + row0 / l.group + 1;
        const int64_t all = (int64_t)here.c + here.n - l.a.window;
        wholeFrom = l.a.window > 0 && all > 0 ? (int)all : 0;
    };

    // A tile: its keys from t0 on, of which `valid` are in the cache.  kChecked: with infinite and
    // NaN values of V set apart, at the keys set[0], and large ones at the keys set[1].
    const auto attend = [&](auto kChecked, uint32_t buffer, int64_t t0, uint64_t valid, const uint64_t *set) {
        constexpr bool checked = decltype(kChecked)::value;
        const uint32_t kFrom = buffer + kPlace, vFrom = buffer + L::kSide + vPlace;
        constexpr uint64_t kAll = kTile == 64 ? ~0ull : 0xFFFFFFFFull;
        const bool whole = valid == kAll && t0 >= wholeFrom && t0 + kTile <= wholeTo;
        uint64_t seen = kAll;
        if (!whole) {
            seen = there ? seen_keys(tree, here.c, node, from, over, t0, known) & valid : 0ull;
            if (!__any((int)(seen != 0ull))) {
                return;
            }
        }

        f32x16_t s[kKt] = {};
        {
            constexpr int kReads = kSteps * kKt, kAhead = kReads < 6 ? kReads : 6;
            u32x4_t k[kAhead];
            const auto read = [&](int x) {
                return *(__attribute__((address_space(3))) const u32x4_t *)(uintptr_t)(
                    L::step(kFrom, 2 * (x / kKt)) + x % kKt * 32 * L::kChunks * 16);
            };
#pragma unroll
            for (int x = 0; x < kAhead; ++x) {
                k[x] = read(x);
            }
            in_order();
#pragma unroll
            for (int x = 0; x < kReads; ++x) {
                s[x % kKt] = mfma<kBf16>(k[x % kAhead], q[x / kKt], s[x % kKt]);
                if (x + kAhead < kReads) {
                    k[x % kAhead] = read(x + kAhead);
                }
                in_order();
            }
        }
        if (!whole) {
#pragma unroll
            for (int kt = 0; kt < kKt; ++kt) {
                const uint32_t bits = (uint32_t)(seen >> (32 * kt)) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[kt][i] = (int)(bits << (31 - (8 * (i / 4) + i % 4))) < 0 ? s[kt][i] : -INFINITY;
                }
            }
        }
        float most = s[0][0];
#pragma unroll
        for (int kt = 0; kt < kKt; ++kt) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                most = fmaxf(most, s[kt][i]);
            }
        }
        most = fmaxf(most, __shfl_xor(most, 32));
        most *= factor;
        if constexpr (checked && kBf16) {
            if (set[1] != 0) {
                float high = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < kKt; ++kt) {
                    const uint32_t bits = (uint32_t)(set[1] >> (32 * kt)) >> (late_lane() / 32 * 4);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        high = (int)(bits << (31 - (8 * (i / 4) + i % 4))) < 0 ? fmaxf(high, s[kt][i]) : high;
                    }
                }
                high = fmaxf(high, __shfl_xor(high, 32)) * factor;
                most = fmaxf(most, high + (kRaised + (float)bits_of(here.keys.high - here.keys.low)));
            }
        }
        if (__any((int)(most > top + kSlack))) {
            const float next = most > top + kSlack ? most : top;
            const float keep = __builtin_amdgcn_exp2f(top - (next == -INFINITY ? 0.f : next));
            top = next;
            sum *= keep;
#pragma unroll
            for (int j = 0; j < kDims; ++j) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    o[j][i] = checked ? scaled(o[j][i], keep) : o[j][i] * keep;
                }
            }
        }
        const float shift = kLiftBits<kBf16> - (top == -INFINITY ? 0.f : top);
        // The weights of 16 keys, two at a time, between the products of the 16 before, whose
        // values of V are read ahead.
        constexpr int kGroups = kTile / 16, kProducts = kGroups * kDims, kAhead = kProducts < 4 ? kProducts : 4;
        u32x4_t p[kGroups][2], v[kAhead];
        float x0 = 0.f, x1 = 0.f;
        const auto raise = [&](int t, int x) {  // (keys 2 x and 2 x + 1 of the lane's 8)
            x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t / 2][t % 2 * 8 + 2 * x], factor, shift));
            x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t / 2][t % 2 * 8 + 2 * x + 1], factor, shift));
        };
        const auto split = [&](int t, int x) {
            sum += x0;
            sum += x1;
            p[t][0][x] = attention::cut2<kBf16>(x0, x1);
            p[t][1][x] = dev::pack2_x<kBf16>(rest<kBf16>(x0), rest<kBf16>(x1));
        };
        const auto read = [&](int x) {  // (rows r and r + 8 of the tile, the lane's 4 columns of 32)
            const uint32_t rows = x / kDims * 16 * L::kChunks * 16;
            const u32x2_t v0 = transposed(L::step(vFrom, 4 * (x % kDims)) + rows);
            const u32x2_t v1 = transposed(L::step(vFrom ^ 32, 4 * (x % kDims)) + rows + 8 * L::kChunks * 16);
            return u32x4_t{v0[0], v0[1], v1[0], v1[1]};
        };
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            v[x] = read(x);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            raise(0, x);
            split(0, x);
        }
        in_order();
#pragma unroll
        for (int x = 0; x < kProducts; ++x) {
            const int t = x / kDims, j = x % kDims;
            // (This product's share of the next 16 keys' four pairs.)
            const int y0 = t + 1 < kGroups ? j * 4 / kDims : 0, y1 = t + 1 < kGroups ? (j + 1) * 4 / kDims : 0;
            o[j] = mfma<kBf16>(v[x % kAhead], p[t][0], o[j]);
            if (y0 < y1) {
                raise(t + 1, y0);
            }
            in_order();
            o[j] = mfma<kBf16>(v[x % kAhead], p[t][1], o[j]);
            if (x + kAhead < kProducts) {
                v[x % kAhead] = read(x + kAhead);
            }
#pragma unroll
            for (int y = y0; y < y1; ++y) {
                if (y > y0) {
                    raise(t + 1, y);
                }
                split(t + 1, y);
            }
            in_order();
        }
        if constexpr (checked) {
            // The infinite and NaN values of the rows that see them.
            uint64_t bad = set[0];
            while (bad != 0) {
                const int at = __ffsll((unsigned long long)bad) - 1;
                bad &= bad - 1;
                float weight = 0.f;
#pragma unroll
                for (int kt = 0; kt < kKt; ++kt) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (32 * kt + 8 * (i / 4) + i % 4 == (at & ~4)) {
                            const uint32_t hi = p[2 * kt + i / 8][0][i % 8 / 2] >> (i % 2 * 16) & 0xFFFFu;
                            const uint32_t lo = p[2 * kt + i / 8][1][i % 8 / 2] >> (i % 2 * 16) & 0xFFFFu;
                            weight = dev::x_to_f32<kBf16>(hi) + dev::x_to_f32<kBf16>(lo);
                        }
                    }
                }
                weight = __shfl(weight, col + 32 * (at >> 2 & 1));
                const bool on = (seen >> at & 1u) != 0u;
                // (a weight that is 0 in 32 bits is above 0 all the same)
                weight = weight == 0.f ? 1e-30f : weight;
                const DraftAttentionArgs &l = late().a;
                const uint32_t t = (uint32_t)t0 + at, column = t / (uint32_t)l.pageSize;
                const uint16_t *value = static_cast<const uint16_t *>(l.vCache.data) + here.kv * l.vCache.head +
                                        l.table[(int64_t)here.b * l.width + column] * l.vCache.page +
                                        (t - column * (uint32_t)l.pageSize) * l.vCache.slot;
#pragma unroll
                for (int j = 0; j < kDims; ++j) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = 32 * j + 8 * (i / 4) + 4 * (late_lane() / 32) + i % 4;
                        if (32 * j + i / 8 * 16 < l.d) {  // (e < d, for d % 16 is 0)
                            const uint32_t bits = value[e];
                            if (on && infinite<kBf16>(bits)) {
                                o[j][i] += weight * dev::x_to_f32<kBf16>(bits);
                            }
                        }
                    }
                }
            }
        }
    };

    // The block at `here` again, tile `firstTile` to the one at `here`.
    const auto again = [&](int firstTile) {
        const int lastTile = here.tile;
        clear();
        load_q(here);
        ahead = here;
        ahead.tile = firstTile;
        enters = true;
        for (int tile = firstTile; tile <= lastTile; ++tile) {
            find_page();
            __syncthreads();  // (the tile before is done)
            load(0);
            const uint64_t valid = loaded;
            if (rowWave == 0 && lane == 0) {
                setApart[keyWave][0] = 0;
                if (kBf16) {
                    setApart[keyWave][1] = 0;
                }
            }
            const uint32_t least = large_from(here.keys.high - here.keys.low);
            dev::wait_vm<0>();
            if (tile == firstTile) {
                turn_q();
            }
            __syncthreads();
            const uint32_t buffer = (uint32_t)(uintptr_t)mine;
#pragma unroll 1
            for (int n = 0; n < L::kLoads; ++n) {
                const int at = (n * L::kRowWaves + rowWave) * kWave + lane;
                auto *const place16 = (__attribute__((address_space(3))) u32x4_t *)(uintptr_t)(buffer + L::kSide + at * 16);
                u32x4_t v = *place16;
                bool bad = false, large = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t low = v[e] & 0x7FFFu, high = v[e] >> 16 & 0x7FFFu;
                    large = large || (low >= least && low < 0x7F80u) || (high >= least && high < 0x7F80u);
                    if (infinite<kBf16>(v[e])) {
                        v[e] &= 0xFFFF0000u;
                        bad = true;
                    }
                    if (infinite<kBf16>(v[e] >> 16)) {
                        v[e] &= 0xFFFFu;
                        bad = true;
                    }
                }
                if (__builtin_expect(bad, 0)) {
                    *place16 = v;
                    atomicOr(reinterpret_cast<unsigned long long *>(&setApart[keyWave][0]), 1ull << (at / L::kChunks));
                }
                if (kBf16 && large) {
                    atomicOr(reinterpret_cast<unsigned long long *>(&setApart[keyWave][1]), 1ull << (at / L::kChunks));
                }
            }
            __syncthreads();
            attend(std::true_type{}, buffer, (int64_t)(here.keys.first + tile) * L::kUnit + keyWave * kTile, valid,
                   setApart[keyWave]);
        }
        __syncthreads();
    };

    find_page();
    load(0);
    find_page();
    load_q(here);
    clear();
    int firstTile = here.tile;  // of the block, in this stretch
    bool fresh = true, firstBlock = true;
    for (int buffer = 0;; buffer ^= 1) {
        const uint64_t valid = loaded;
        dev::wait_vm<0>();  // (the tile is there, the next one's pages are known, and so is q)
        if constexpr (L::kRowWaves > 1) {
            __syncthreads();
        }
        if (fresh) {
            enter();
            turn_q();
            fresh = false;
        }
        // The next tile, of this block or the next one (behind the last one rows of zeros: under a
        // branch the page would be waited for).
        load(buffer ^ 1);
        find_page();
        attend(std::false_type{}, (uint32_t)(uintptr_t)mine + buffer * L::kBuffer,
               (int64_t)(here.keys.first + here.tile) * L::kUnit + keyWave * kTile, valid, nullptr);
        if (here.tile + 1 < here.keys.tiles && here.start + here.tile + 1 < end) {
            ++here.tile;
            continue;
        }

        // The block's end, or the stretch's.
        float far = 0.f;  // (not finite where one of the sums is not, or is 2^116 or more)
#pragma unroll
        for (int j = 0; j < kDims; ++j) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                far = __builtin_fmaf(o[j][i], kFar<kBf16>, far);
            }
        }
        const bool finite = __all((int)__builtin_isfinite(far));
        if (lane == 0) {
            odd[wave] = !finite;
        }
        Place next = here;
        next.advance();
        const bool more = next.inside(end);
        if (more) {
            load_q(next);
        }
        __syncthreads();
        bool redo = false;
#pragma unroll
        for (int x = 0; x < L::kWaves; ++x) {
            redo = redo || odd[x];
        }
        if (__builtin_expect(redo, 0)) {
            dev::wait_vm<0>();  // (the tile on its way)
            again(firstTile);
            // The next one anew.
            ahead = next;
            enters = true;
            find_page();
            load(buffer ^ 1);
            find_page();
            if (more) {
                load_q(next);
            }
        }

        sum += __shfl_xor(sum, 32);
        if (!there) {  // (its scores of 0 count in tiles without masks)
            top = -INFINITY;
            sum = 0.f;
#pragma unroll
            for (int j = 0; j < kDims; ++j) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    o[j][i] = 0.f;
                }
            }
        }
        const bool all = firstTile == 0 && here.tile + 1 == here.keys.tiles;
        const int slot = 2 * w + (firstBlock ? 0 : 1);
        if (threadIdx.x == 0 && firstTile == 0 && !all) {
            late().open[w] = Open{shares.owner(here.start + here.keys.tiles - 1), here.b, here.kv, here.block, slot, {}};
        }
        // The lane's four x of values: of a row's dimension 32 (x / 4) + 8 (x % 4) + 4 upper on.
        // A part lies in the workspace as in the registers, so that a wave writes 1 KB at a time.
        const Args &l = late();
        const int ln = late_lane(), r = rowWave * kRows + ln % 32, upper = ln / 32;
        const int head = here.block * L::kBlock + r - node * l.group;
        float *const parts = l.outs + (int64_t)slot * L::kBlock * D + rowWave * kRows * D + ln * 4;
        const auto put = [&](int x, f32x4_t value, float t, float total) {
            const int e = x / 4 * 32 + x % 4 * 8 + 4 * upper;
            if (node >= l.a.S) {
            } else if (all) {
                finish<kBf16>(l, here, node, head, e, value, t, total);
            } else {
                *reinterpret_cast<f32x4_t *>(parts + x * kWave * 4) = value;
                if (e == 0) {
                    *reinterpret_cast<float2 *>(l.ends + ((int64_t)slot * L::kBlock + r) * 2) = float2{t, total};
                }
            }
        };
        if constexpr (L::kKeyWaves == 1) {
#pragma unroll
            for (int j = 0; j < kDims; ++j) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    put(4 * j + i / 4, f32x4_t{o[j][i], o[j][i + 1], o[j][i + 2], o[j][i + 3]}, top, sum);
                }
            }
        } else {
            // The groups' results together: each has a share of the values and leaves the others',
            // as they lie in its registers, in the buffer that it has read.
            constexpr int kShare = kDims * 4 / L::kKeyWaves;  // fours of values
            const auto left = [&](int k, int x) {
                return (__attribute__((address_space(3))) f32x4_t *)(uintptr_t)(
                    (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + (2 * k + buffer) * L::kBuffer +
                    ((L::kRowWaves == 1 ? x : rowWave * kShare + x % kShare) * kWave + ln) * 16);
            };
            __syncthreads();  // (the tiles are read)
            if (upper == 0) {
                ends[keyWave][r] = float2{top, sum};
            }
#pragma unroll
            for (int share = 0; share < L::kKeyWaves; ++share) {
                if (share != keyWave) {
#pragma unroll
                    for (int x = share * kShare; x < (share + 1) * kShare; ++x) {
                        const f32x16_t &from_ = o[x / 4];
                        const int i = x % 4 * 4;
                        *left(keyWave, x) = f32x4_t{from_[i], from_[i + 1], from_[i + 2], from_[i + 3]};
                    }
                }
            }
            __syncthreads();
            float f[L::kKeyWaves], total = 0.f, most = -INFINITY;
            float2 end_[L::kKeyWaves];
#pragma unroll
            for (int k = 0; k < L::kKeyWaves; ++k) {
                end_[k] = ends[k][r];
                most = fmaxf(most, end_[k].x);
            }
#pragma unroll
            for (int k = 0; k < L::kKeyWaves; ++k) {
                f[k] = __builtin_amdgcn_exp2f(end_[k].x - (most == -INFINITY ? 0.f : most));
                total += f[k] * end_[k].y;
            }
            const auto join = [&](auto kInfinite) {
#pragma unroll
                for (int share = 0; share < L::kKeyWaves; ++share) {
                    if (share == keyWave) {
#pragma unroll
                        for (int x = share * kShare; x < (share + 1) * kShare; ++x) {
                            f32x4_t value = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int k = 0; k < L::kKeyWaves; ++k) {
                                const f32x16_t &own = o[x / 4];
                                const int i = x % 4 * 4;
                                const f32x4_t v = k == share ? f32x4_t{own[i], own[i + 1], own[i + 2], own[i + 3]}
                                                             : *left(k, x);
#pragma unroll
                                for (int y = 0; y < 4; ++y) {
                                    value[y] += decltype(kInfinite)::value ? scaled(v[y], f[k]) : v[y] * f[k];
                                }
                            }
                            put(x, value, most, total);
                        }
                    }
                }
            };
            if (redo) {
                join(std::true_type{});
            } else {
                join(std::false_type{});
            }
        }
        if (!more) {
            break;
        }
        if constexpr (L::kKeyWaves > 1) {
            __syncthreads();  // (what the groups left is read)
        }
        here = next;
        firstTile = 0;
        fresh = true;
        firstBlock = false;
        clear();
    }
    dev::wait_vm<0>();  // (the rows of zeros, before the LDS is another workgroup's)
}

// Joins the parts of the (sequence, kv head, block)s that no stretch finished: a workgroup
// for some rows of the one that stretch `first` began.  Where one has more than kJoinBatch
// parts, the workgroups of the next three stretches, which begin none, help: each has a quarter of
// the values, and its waves a quarter of the parts each (256 parts, one sequence of 131072 tokens
// with 16 heads to one of 128, a chain of 4: the call 90.8 us without them, 48.8 so; 47 parts of one
// row 28.3 and 19.2).  Bound by its chain of loads (what there is to join, then up to 16 parts at
// once) for one small sequence, 4.0 us, and by memory for many, 12 to 14 with 40 to 50 MB of parts.
constexpr int kJoinThreads = 256, kJoinWaves = kJoinThreads / kWave;
constexpr int kJoinBatch = 16;

// What some parts amount to, of four values of a row.
struct Joined {
    float top, total;
    f32x4_t all;

    // To a reference of `next` (which is 0 where nothing is seen).
    __device__ void turn(float next)
    {
        const float keep = __builtin_amdgcn_exp2f(top - (next == -INFINITY ? 0.f : next));
        top = next;
        total *= keep;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            all[y] = scaled(all[y], keep);
        }
    }
    __device__ void add(float factor, float weights, f32x4_t values)
    {
        total += factor * weights;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            all[y] += scaled(values[y], factor);
        }
    }
};

template <bool kBf16, int D>
__global__ __launch_bounds__(kJoinThreads) void draft_join(Args args)
{
    __shared__ Joined shared[kJoinWaves][kWave];
    const DraftAttentionArgs &a = args.a;
    // (Turned by blockIdx.y: the stretches that begin parts may lie 8 apart, and so all on one XCD.
    // 32 blocks of 8 parts each: 21.8 us not turned, 12.4 so.)
    const int own = (int)((blockIdx.x + blockIdx.y) % gridDim.x);
    // The one to join: begun by this stretch, or one of many parts begun by a stretch just before.
    // (Its stretches begin nothing else, so there is one at most.)
    int first = -1, last = -1;
#pragma unroll
    for (int k = 0; k < kJoinWaves; ++k) {
        const int begun = own >= k ? own - k : 0, to = args.open[begun].last;
        if (k == 0 ? to >= 0 : to - begun >= kJoinBatch) {
            first = begun;
            last = to;
        }
    }
    if (first < 0) {
        return;
    }
    const Open open = args.open[first];
    const bool shares = last - first >= kJoinBatch;
    const int wave = (int)threadIdx.x / kWave;
    // (32 rows, four x of each, of each lane of a wave.)
    const int at = (int)blockIdx.y * kJoinThreads + (shares ? own - first : wave) * kWave + (int)threadIdx.x % kWave;
    const int lane = at % kWave, x = at / kWave % (D / 8);
    const int r = at / (kRows * D / 4) * kRows + lane % 32, e = x / 4 * 32 + x % 4 * 8 + lane / 32 * 4;
    Place p{};
    p.b = open.b;
    p.kv = open.kv;
    p.block = open.block;
    const uint32_t row = (uint32_t)p.block * args.rows + r, group = (uint32_t)args.group;  // (below 2^30)
    const int node = (int)(row / group), head = (int)(row % group);
    const bool there = node < a.S;
    const int quarter = (last - first) / kJoinWaves + 1;
    const int from = shares ? first + wave * quarter : first;
    const int to = !there ? from - 1 : shares && from + quarter - 1 < last ? from + quarter - 1 : last;
    Joined sum{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}};
    for (int x0 = from; x0 <= to; x0 += kJoinBatch) {
        float2 ends[kJoinBatch];
        f32x4_t outs[kJoinBatch];
#pragma unroll
        for (int m = 0; m < kJoinBatch; ++m) {
            ends[m] = float2{-INFINITY, 0.f};
            outs[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (x0 + m <= to) {
                const int64_t slot = x0 + m == first ? open.slot : 2 * (x0 + m);
                ends[m] = *reinterpret_cast<const float2 *>(args.ends + (slot * args.rows + r) * 2);
                outs[m] = *reinterpret_cast<const f32x4_t *>(args.outs + slot * args.rows * D + at * 4);
            }
        }
        float next = sum.top;
#pragma unroll
        for (int m = 0; m < kJoinBatch; ++m) {
            next = fmaxf(next, ends[m].x);
        }
        sum.turn(next);
#pragma unroll
        for (int m = 0; m < kJoinBatch; ++m) {
            if (x0 + m <= to) {
                sum.add(__builtin_amdgcn_exp2f(ends[m].x - (next == -INFINITY ? 0.f : next)), ends[m].y, outs[m]);
            }
        }
    }
    if (shares) {
        shared[wave][lane] = sum;
        __syncthreads();
        if (wave != 0) {
            return;
        }
        float next = sum.top;
#pragma unroll
        for (int k = 1; k < kJoinWaves; ++k) {
            next = fmaxf(next, shared[k][lane].top);
        }
        sum.turn(next);
#pragma unroll
        for (int k = 1; k < kJoinWaves; ++k) {
            const Joined other = shared[k][lane];
            sum.add(__builtin_amdgcn_exp2f(other.top - (next == -INFINITY ? 0.f : next)), other.total, other.all);
        }
    }
    if (there) {
        finish<kBf16>(args, p, node, head, e, sum.all, sum.top, sum.total);
    }
}

template <bool kBf16, typename L>
hipError_t launch_layout(const Args &args, hipStream_t stream)
{
    if (args.rows != L::kBlock || args.unit != L::kUnit || args.a.d > L::D) {
        return hipErrorInvalidValue;  // (planned for another layout, and so is the workspace)
    }
    hipLaunchKernelGGL((draft_units<kBf16, L>), dim3((unsigned)args.most), dim3(L::kThreads), 0, stream, args);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        return err;
    }
    static_assert(kRows * (L::D / 4) % kJoinThreads == 0);
    const int64_t rows = (int64_t)args.a.S * args.group < args.rows ? (int64_t)args.a.S * args.group : args.rows;
    hipLaunchKernelGGL((draft_join<kBf16, L::D>),
                       dim3((unsigned)args.most, (unsigned)((rows + kRows - 1) / kRows) * (kRows * (L::D / 4) / kJoinThreads)),
                       dim3(kJoinThreads), 0, stream, args);
    return hipGetLastError();
}

// The layouts by rows of a (sequence, kv head).
enum class Kind { kOne, kTwo, kFour, kEight };

template <int D, Kind kKind>
struct LayoutOf;
template <int D>
struct LayoutOf<D, Kind::kOne> : Layout<D, 1, (D > 128 ? 2 : 4), 32> {};
template <int D>
struct LayoutOf<D, Kind::kTwo> : Layout<D, 2, 2, 32> {};
template <int D>
struct LayoutOf<D, Kind::kFour> : Layout<D, 4, 1, 64> {};
// (For heads of 64 and 128 only: other sizes' tiles do not split into 8 waves' whole loads, and
// larger ones' registers do not hold it.)
template <int D>
struct LayoutOf<D, Kind::kEight> : Layout<D, 8, 1, 64> {};

// The sizes that there are layouts for.
inline int padded(int d)
{
    return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 160 ? 160 : d <= 192 ? 192 : 256;
}

// Calls f(layout) for a kind and head size.
template <Kind kKind, typename F>
auto with_size(int d, F &&f)
{
    if constexpr (kKind == Kind::kEight) {
        return padded(d) == 64 ? f(LayoutOf<64, kKind>{}) : f(LayoutOf<128, kKind>{});
    } else {
        switch (padded(d)) {
        case 32: return f(LayoutOf<32, kKind>{});
        case 64: return f(LayoutOf<64, kKind>{});
        case 96: return f(LayoutOf<96, kKind>{});
        case 128: return f(LayoutOf<128, kKind>{});
        case 160: return f(LayoutOf<160, kKind>{});
        case 192: return f(LayoutOf<192, kKind>{});
        default: return f(LayoutOf<256, kKind>{});
        }
    }
}

// One file per instance: mhc_draft_attention_{bf16,f16}_{one,two,four,eight}.hip.
template <bool kBf16, Kind kKind>
hipError_t launch_kind(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<true, Kind::kOne>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<true, Kind::kTwo>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<true, Kind::kFour>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<true, Kind::kEight>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<false, Kind::kEight>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<false, Kind::kOne>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<false, Kind::kTwo>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<false, Kind::kFour>(const Args &args, hipStream_t stream);

}  // namespace draft
}  // namespace mhc
