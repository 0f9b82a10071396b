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
// terms, the first one cut, the second rounded: bf16 holds 16 bits, fp16 (lifted by
// 2^15, for its range ends at 2^-24) 22.  One term alone would add an error of the
// size of the output's own rounding.
//
// What a row sees is all of the context in front of the new tokens (but for a
// window), and of the new tokens its ancestors, found from the parents by
// doubling (the ancestors of my farthest known ancestor are mine), 256 bits a token.
// Tiles that all rows see whole have no masks.  The loop takes V as finite: an
// infinite or NaN value times a weight of zero would reach rows that do not see
// it.  Where a block's output is not finite, the block is done again with such
// values taken out of the products and added to the rows that see them alone.
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
    static constexpr int kTiles = 2 * kBuffer * kKeyWaves;
    static constexpr int kJoin = kKeyWaves > 1 ? kRows * (D + 4) * 4 * kWaves : 0;
    static constexpr int kSetup = kDraftNodes * (32 + 4);
    static constexpr int kLds = kTiles > kJoin ? (kTiles > kSetup ? kTiles : kSetup) : (kJoin > kSetup ? kJoin : kSetup);
    // Workgroups of a CU: what its registers (two waves a SIMD up to D = 128) and LDS hold.
    static constexpr int kPerCu = kThreads == 256 && D <= 128 && 2 * (kLds + kBlock * 48) <= 160 * 1024 ? 2 : 1;
    static_assert(kLoads * kRowWaves * 1024 == kSide && kLds + kBlock * 48 <= 160 * 1024);

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

// What a stretch begins and does not finish: a (sequence, kv head, block), the line's unit
// at which it begins and its units, and the units of the line.  units 0: nothing.
struct Open {
    int b, kv, block, start, units, all;
};

struct Args {
    DraftAttentionArgs a;
    int group;   // query heads of a kv head
    int blocks;  // blocks of rows of a (sequence, kv head)
    int rows;    // of a block
    int unit;    // keys of a unit
    int most;    // workgroups of the launch
    float *outs, *ends;  // the parts: [2 * most][rows][D], [2 * most][rows][2]
    Open *open;          // [most]
};

// The keys of a block of a sequence with c + n tokens, n of them new: [low, high).
struct Keys {
    int low, high, first, units;
};

struct Sequence {
    int c, n;  // tokens in front of the new ones, new ones

    __device__ Sequence(const DraftAttentionArgs &a, int b)
    {
        const int most = a.width * a.pageSize;
        int L = a.lengths[b], m = a.drafted[b];
        L = L < 0 ? 0 : L > most ? most : L;
        m = m < 0 ? 0 : m > a.S ? a.S : m;
        n = m < L ? m : L;
        c = L - n;
    }
    __device__ Keys keys(const Args &args, int block) const
    {
        const int i0 = (int)((int64_t)block * args.rows / args.group);
        const int64_t last = ((int64_t)(block + 1) * args.rows + args.group - 1) / args.group;
        const int i1 = last < n ? (int)last : n;
        Keys k{0, 0, 0, 1};
        if (i0 < n) {
            // A chain's token i is at position c + i, a tree's at c or later.
            const int64_t from = (int64_t)c + (args.a.parents == nullptr ? i0 : 0) + 1 - args.a.window;
            k.low = args.a.window > 0 && from > 0 ? (int)from : 0;
            k.high = c + i1;
            k.first = k.low / args.unit;
            k.units = (k.high - 1) / args.unit + 1 - k.first;
        }
        return k;
    }
    __device__ int units(const Args &args) const
    {
        int all = 0;
        for (int x = 0; x < args.blocks; ++x) {
            all += keys(args, x).units;
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

// log2 of what the probabilities are multiplied by.
template <bool kBf16>
constexpr float kLiftBits = kBf16 ? 0.f : 15.f;

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

// Place of a stretch's first unit: sequence, kv head, block, and the unit in its keys.
struct Place {
    int b, kv, block, tile;
    int start;  // the line's unit at which the (sequence, kv head, block) begins
    Keys keys;
};

// The place of unit `at` of the line, from the units of sequences (lane's: of `first`).
__device__ __forceinline__ Place find_place(const Args &args, int at)
{
    const DraftAttentionArgs &a = args.a;
    const int lane = (int)threadIdx.x % kWave;
    int base = 0;
    for (int b0 = 0;; b0 += kWave) {
        const int x = b0 + lane;
        const int units = x < a.B ? Sequence(a, x).units(args) * a.kvHeads : 0;
        const int upto = dev::wave_scan(units);
        const uint64_t past = __ballot(base + upto > at);
        if (past == 0 && b0 + kWave < a.B) {
            base += __builtin_amdgcn_readlane(upto, kWave - 1);
            continue;
        }
        const int hit = __ffsll((unsigned long long)past) - 1;
        Place p;
        p.b = b0 + hit;
        const int all = __builtin_amdgcn_readlane(units, hit) / a.kvHeads;
        base += __builtin_amdgcn_readlane(upto, hit) - all * a.kvHeads;
        p.kv = (at - base) / all;
        base += p.kv * all;
        const Sequence s(a, p.b);
        for (p.block = 0;; ++p.block) {
            p.keys = s.keys(args, p.block);
            if (at < base + p.keys.units) {
                break;
            }
            base += p.keys.units;
        }
        p.start = base;
        p.tile = at - base;
        return p;
    }
}

__device__ __forceinline__ int all_units(const Args &args)
{
    const int lane = (int)threadIdx.x % kWave;
    int all = 0;
    for (int b0 = 0; b0 < args.a.B; b0 += kWave) {
        const int x = b0 + lane;
        all += __builtin_amdgcn_readlane(
            dev::wave_scan(x < args.a.B ? Sequence(args.a, x).units(args) * args.a.kvHeads : 0), kWave - 1);
    }
    return all;
}

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

// The ancestors of every node of row b, 256 bits each (itself among them), at the start of
// `lds`.  A node's farthest known ancestor's are its own too: each round doubles how far.
template <int kThreads>
__device__ __forceinline__ void find_ancestors(const DraftAttentionArgs &a, int b, int n, char *lds)
{
    constexpr int kNodes = kDraftNodes / kThreads > 0 ? kDraftNodes / kThreads : 1;  // of a thread
    uint64_t *known = reinterpret_cast<uint64_t *>(lds);
    int *farthest = reinterpret_cast<int *>(lds + kDraftNodes * 32);
    uint64_t own[kNodes][4];
    int far[kNodes];
#pragma unroll
    for (int k = 0; k < kNodes; ++k) {
        const int i = k * kThreads + (int)threadIdx.x;
        far[k] = -1;
        if (i < n) {
            const int p = a.parents[(int64_t)b * a.S + i];
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
            const int i = k * kThreads + (int)threadIdx.x;
            if (i < n) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    known[4 * i + x] = own[k][x];
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
                    own[k][x] |= known[4 * far[k] + x];
                }
                far[k] = farthest[far[k]];
            }
        }
        __syncthreads();
    }
}

// Which of the 64 keys from t0 on a node sees: the context from `from` on, and of the new
// tokens its ancestors, or in a chain those up to itself.
__device__ __forceinline__ uint64_t seen_keys(bool tree, int c, int node, uint32_t from, int64_t t0,
                                              const uint64_t (&ancestors)[4])
{
    // (positions below 2^31 and their differences fit 33 bits)
    const int64_t to = (tree ? c : (int64_t)c + node + 1) - t0, first = (int64_t)from - t0;
    uint64_t seen = low_bits(to > 64 ? 64 : to < 0 ? 0 : (int)to) & ~low_bits(first > 64 ? 64 : first < 0 ? 0 : (int)first);
    if (tree) {
        // Bit x of the tile is node x + t0 - c.
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int64_t by = t0 - c - 64 * x;
            if (by > -64 && by < 64) {
                seen |= by >= 0 ? ancestors[x] >> by : ancestors[x] << -by;
            }
        }
    }
    return seen;
}

// What one of two packed 16-bit values leaves of x.
template <bool kBf16>
__device__ __forceinline__ float rest(float x, uint32_t two, int which)
{
    if constexpr (kBf16) {  // (cut: the upper half of x itself)
        return x - __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    } else {
        const _Float16 h = __builtin_bit_cast(_Float16, (uint16_t)(which == 0 ? two : two >> 16));
        return __builtin_fmaf(-(float)h, 1.f, x);
    }
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
    __shared__ uint64_t rowMasks[L::kBlock][4];  // the rows' ancestors
    __shared__ uint64_t badKeys[L::kKeyWaves][2];
    __shared__ float tops[L::kKeyWaves][L::kBlock], sums[L::kKeyWaves][L::kBlock];
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

    const attention::Shares shares(all_units(args), args.most);
    if (threadIdx.x == 0) {
        args.open[w].units = 0;
    }
    if (w >= shares.grid) {
        return;
    }
    const int begin = shares.start(w), end = shares.start(w + 1);
    Place place = find_place(args, begin);

    for (int unit = begin; unit < end;) {
        const Sequence seq(a, place.b);
        const int tiles = end - unit < place.keys.units - place.tile ? end - unit : place.keys.units - place.tile;
        const int row = place.block * L::kBlock + rowWave * kRows + col;
        const int node = row / args.group, head = row % args.group;
        const bool there = node < seq.n;

        // The node's ancestors (itself one of them) among the new tokens, and its depth.
        int depth = node;
        const bool tree = a.parents != nullptr;
        const int draftFrom = (place.keys.first + place.tile) * L::kUnit;
        __syncthreads();  // (the LDS is free)
        if (tree && seq.n > 0 && (a.window > 0 || (int64_t)draftFrom + (int64_t)tiles * L::kUnit > seq.c)) {
            find_ancestors<L::kThreads>(a, place.b, seq.n, lds);
            const uint64_t *known = reinterpret_cast<const uint64_t *>(lds);
            depth = 0;
            if (there) {
                uint64_t own[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    own[x] = known[4 * node + x];
                    depth += __popcll(own[x]);
                }
                depth -= 1;
                // Of the path only the window's length, from the node up: the lower numbers go.
                int over = a.window > 0 && a.window < depth + 1 ? depth + 1 - (int)a.window : 0;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    while (over > 0 && own[x] != 0) {
                        own[x] &= own[x] - 1;
                        --over;
                    }
                    rowMasks[rowWave * kRows + col][x] = own[x];  // (by all key waves, the same)
                }
            }
            __syncthreads();
        }
        // The context that the row sees: [from, c).  (A chain's row: [from, c + node].)
        const int64_t from64 = (int64_t)seq.c + depth + 1 - a.window;
        const uint32_t from = a.window > 0 && from64 > 0 ? (uint32_t)from64 : 0u;
        // Tiles in [wholeFrom, wholeTo) all rows of the wave see whole.
        const int64_t wholeTo =
            tree ? seq.c : (int64_t)seq.c + (place.block * L::kBlock + rowWave * kRows) / args.group + 1;
        const int64_t wholeFrom = a.window > 0 ? (int64_t)seq.c + seq.n - a.window : 0;

        u32x4_t q[kSteps];
        // (Its sign goes to q, for the maximum wants a factor above 0; with a scale of 0 q is 0.)
        const float c = a.scale == 0.f ? 1.f : fabsf(a.scale * kLog2e);
        {
            const uint16_t *at = static_cast<const uint16_t *>(a.q.data) + place.b * a.q.row + node * a.q.token +
                                 (int64_t)(place.kv * args.group + head) * a.q.head;
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                q[s] = u32x4_t{0, 0, 0, 0};
                if (there && a.scale != 0.f && 16 * s < a.d) {
                    q[s] = *reinterpret_cast<const u32x4_t *>(at + 16 * s + 8 * half);
                    q[s] ^= u32x4_t{flip, flip, flip, flip};
                }
            }
        }

        const char *kBase = static_cast<const char *>(a.kCache.data) + 2 * place.kv * a.kCache.head;
        const char *vBase = static_cast<const char *>(a.vCache.data) + 2 * place.kv * a.vCache.head;
        const int32_t *table = a.table + (int64_t)place.b * a.width;
        f32x16_t o[kDims];
        float top, sum;
        // kChecked: with infinite and NaN values of V set apart.
        const auto pass = [&](auto kChecked) {
            constexpr bool checked = decltype(kChecked)::value;
#pragma unroll
            for (int j = 0; j < kDims; ++j) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    o[j][i] = 0.f;
                }
            }
            top = -INFINITY;
            sum = 0.f;

            // The lane's key (lane % kTile) of a tile: its page and slot, then its rows.
            uint32_t t = (uint32_t)(place.keys.first + place.tile) * L::kUnit + keyWave * kTile + lane % kTile;
            // (Always a load, of the row's first entry where there is no key: under a branch it
            // would be waited for at once.)
            int page = -1, slot = 0;
            bool key = false;
            const auto find_page = [&](bool more) {
                key = more && t >= (uint32_t)place.keys.low && t < (uint32_t)place.keys.high;
                const uint32_t at = (key ? t : 0u) / (uint32_t)a.pageSize;
                page = table[at];
                slot = (int)(t - at * (uint32_t)a.pageSize);
                t += L::kUnit;
            };
            uint64_t loaded = 0;  // keys of the tile on its way
            const auto load = [&](int buffer) {
                const bool seen = key && page >= 0 && page < a.pages;
                loaded = __ballot(seen);
                if constexpr (kTile == 32) {
                    loaded &= 0xFFFFFFFFull;
                }
                const char *kRow = seen ? kBase + 2 * (page * a.kCache.page + slot * a.kCache.slot)
                                        : reinterpret_cast<const char *>(kZeros);
                const char *vRow = seen ? vBase + 2 * (page * a.vCache.page + slot * a.vCache.slot)
                                        : reinterpret_cast<const char *>(kZeros);
                auto *const to = mine + buffer * L::kBuffer;
#pragma unroll
                for (int n = 0; n < L::kLoads; ++n) {
                    const int first = (n * L::kRowWaves + rowWave) * kWave, at = first + lane;
                    const int r = at / L::kChunks, ch = at % L::kChunks ^ L::turn(r);
                    const char *k = reinterpret_cast<const char *>(shfl64(reinterpret_cast<int64_t>(kRow), r)) + ch * 16;
                    const char *v = reinterpret_cast<const char *>(shfl64(reinterpret_cast<int64_t>(vRow), r)) + ch * 16;
                    if (ch * 8 >= a.d) {
                        k = v = reinterpret_cast<const char *>(kZeros);
                    }
                    load_to_lds(k, to + first * 16);
                    load_to_lds(v, to + L::kSide + first * 16);
                }
            };
            find_page(true);
            load(0);
            find_page(tiles > 1);
            for (int tile = 0; tile < tiles; ++tile) {
                const uint32_t buffer = (uint32_t)(uintptr_t)mine + tile % 2 * L::kBuffer;
                const uint32_t kFrom = buffer + kPlace, vFrom = buffer + L::kSide + vPlace;
                const uint64_t valid = loaded;
                const int64_t t0 = (int64_t)(place.keys.first + place.tile + tile) * L::kUnit + keyWave * kTile;
                dev::wait_vm<0>();  // (the tile is there, and the next one's pages are known)
                if constexpr (L::kRowWaves > 1 || checked) {
                    __syncthreads();
                }
                if constexpr (checked) {
                    if (rowWave == 0 && lane == 0) {
                        badKeys[keyWave][tile % 2] = 0;
                    }
                    __syncthreads();
#pragma unroll 1
                    for (int n = 0; n < L::kLoads; ++n) {
                        const int at = (n * L::kRowWaves + rowWave) * kWave + lane;
                        auto *const place16 = (__attribute__((address_space(3))) u32x4_t *)(uintptr_t)(buffer + L::kSide + at * 16);
                        u32x4_t v = *place16;
                        bool bad = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (infinite<kBf16>(v[e])) {
                                v[e] &= 0xFFFF0000u;
                                bad = true;
                            }
                            if (infinite<kBf16>(v[e] >> 16)) {
                                v[e] &= 0xFFFFu;
                                bad = true;
                            }
                        }
                        if (bad) {
                            *place16 = v;
                            atomicOr(reinterpret_cast<unsigned long long *>(&badKeys[keyWave][tile % 2]),
                                     1ull << (at / L::kChunks));
                        }
                    }
                    __syncthreads();
                }
                // (After the last tile: rows of zeros.  Under a branch the page would be waited for.)
                load((tile + 1) % 2);
                find_page(tile + 2 < tiles);

                // What the row sees of the tile (its keys from t0 on).
                constexpr uint64_t kAll = kTile == 64 ? ~0ull : 0xFFFFFFFFull;
                const bool whole = valid == kAll && t0 >= wholeFrom && t0 + kTile <= wholeTo;
                uint64_t seen = kAll;
                if (!whole) {
                    seen = seen_keys(tree, seq.c, node, from, t0, rowMasks[rowWave * kRows + col]);
                    seen = there ? seen & valid : 0ull;
                    if (!__any((int)(seen != 0ull))) {
                        continue;
                    }
                }

                f32x16_t s[kKt] = {};
                {
                    constexpr int kAll = kSteps * kKt, kAhead = kAll < 6 ? kAll : 6;
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
                    for (int x = 0; x < kAll; ++x) {
                        s[x % kKt] = mfma<kBf16>(k[x % kAhead], q[x / kKt], s[x % kKt]);
                        if (x + kAhead < kAll) {
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
                            s[kt][i] = (bits >> (8 * (i / 4) + i % 4) & 1u) != 0u ? s[kt][i] : -INFINITY;
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
                const float next_top = fmaxf(top, most * c);
                const float zero = next_top == -INFINITY ? 0.f : next_top;
                if (__any((int)(next_top > top))) {  // (else the sums are on the right scale)
                    const float keep = __builtin_amdgcn_exp2f(top - zero);
                    top = next_top;
                    sum *= keep;
#pragma unroll
                    for (int j = 0; j < kDims; ++j) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            o[j][i] = checked ? scaled(o[j][i], keep) : o[j][i] * keep;
                        }
                    }
                }
                const float shift = kLiftBits<kBf16> - zero;
                // The weights of 16 keys, two at a time, between the products of the 16 before, whose
                // values of V are read ahead.
                constexpr int kGroups = kTile / 16, kProducts = kGroups * kDims, kAhead = kProducts < 4 ? kProducts : 4;
                u32x4_t p[kGroups][2], v[kAhead];
                const auto weigh = [&](int t, int x) {  // (keys 2 x and 2 x + 1 of the lane's 8)
                    const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t / 2][t % 2 * 8 + 2 * x], c, shift));
                    const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t / 2][t % 2 * 8 + 2 * x + 1], c, shift));
                    sum += x0;
                    sum += x1;
                    const uint32_t first = attention::cut2<kBf16>(x0, x1);
                    p[t][0][x] = first;
                    p[t][1][x] = dev::pack2_x<kBf16>(rest<kBf16>(x0, first, 0), rest<kBf16>(x1, first, 1));
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
                    weigh(0, x);
                }
                in_order();
#pragma unroll
                for (int x = 0; x < kProducts; ++x) {
                    const int t = x / kDims, j = x % kDims;
                    o[j] = mfma<kBf16>(v[x % kAhead], p[t][0], o[j]);
                    o[j] = mfma<kBf16>(v[x % kAhead], p[t][1], o[j]);
                    if (x + kAhead < kProducts) {
                        v[x % kAhead] = read(x + kAhead);
                    }
                    if (t + 1 < kGroups) {
#pragma unroll
                        for (int y = j * 4 / kDims; y < (j + 1) * 4 / kDims; ++y) {
                            weigh(t + 1, y);
                        }
                    }
                    in_order();
                }
                if constexpr (checked) {
                    // The infinite and NaN values of the rows that see them.
                    uint64_t bad = badKeys[keyWave][tile % 2];
                    while (bad != 0) {
                        const int key = __ffsll((unsigned long long)bad) - 1;
                        bad &= bad - 1;
                        float weight = 0.f;
#pragma unroll
                        for (int kt = 0; kt < kKt; ++kt) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                if (32 * kt + 8 * (i / 4) + i % 4 == (key & ~4)) {
                                    const uint32_t hi = p[2 * kt + i / 8][0][i % 8 / 2] >> (i % 2 * 16) & 0xFFFFu;
                                    const uint32_t lo = p[2 * kt + i / 8][1][i % 8 / 2] >> (i % 2 * 16) & 0xFFFFu;
                                    weight = dev::x_to_f32<kBf16>(hi) + dev::x_to_f32<kBf16>(lo);
                                }
                            }
                        }
                        weight = __shfl(weight, col + 32 * (key >> 2 & 1));
                        const bool on = (seen >> key & 1u) != 0u;
                        // (a weight that is 0 in 32 bits is above 0 all the same)
                        weight = weight == 0.f ? 1e-30f : weight;
                        const uint32_t at = (uint32_t)t0 + key, column = at / (uint32_t)a.pageSize;
                        const uint16_t *v = reinterpret_cast<const uint16_t *>(
                            vBase + 2 * (table[column] * a.vCache.page + (at - column * (uint32_t)a.pageSize) * a.vCache.slot));
#pragma unroll
                        for (int j = 0; j < kDims; ++j) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int e = 32 * j + 8 * (i / 4) + 4 * half + i % 4;
                                if (32 * j + i / 8 * 16 < a.d) {  // (e < d, for d % 16 is 0)
                                    const uint32_t bits = v[e];
                                    if (on && infinite<kBf16>(bits)) {
                                        o[j][i] += weight * dev::x_to_f32<kBf16>(bits);
                                    }
                                }
                            }
                        }
                    }
                }
            }
            dev::wait_vm<0>();  // (the rows of zeros, before the LDS serves for something else)
        };
        pass(std::false_type{});
        bool all = true;
#pragma unroll
        for (int j = 0; j < kDims; ++j) {
            float none = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                none += o[j][i] * 0.f;
            }
            all = all && none == 0.f;
        }
        if (lane == 0) {
            odd[wave] = false;
        }
        if (!all) {
            odd[wave] = true;
        }
        __syncthreads();
        bool again = false;
#pragma unroll
        for (int x = 0; x < L::kWaves; ++x) {
            again = again || odd[x];
        }
        if (again) {
            pass(std::true_type{});
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
        const bool whole = place.tile == 0 && tiles == place.keys.units;
        if (threadIdx.x == 0 && place.tile == 0 && !whole) {
            args.open[w] = Open{place.b, place.kv, place.block, place.start, place.keys.units, shares.units};
        }
        const int slot = 2 * w + (unit == begin ? 0 : 1);
        // 4 values of row r of the block.
        const auto put = [&](int r, int e, f32x4_t all, float t, float s) {
            const int x = place.block * L::kBlock + r;
            const int i = x / args.group, h = x % args.group;
            if (i >= a.S) {
            } else if (whole) {
                finish<kBf16>(args, place, i, h, e, all, t, s);
            } else {
                *reinterpret_cast<f32x4_t *>(args.outs + ((int64_t)slot * L::kBlock + r) * D + e) = all;
                if (e == 0) {
                    *reinterpret_cast<float2 *>(args.ends + ((int64_t)slot * L::kBlock + r) * 2) = float2{t, s};
                }
            }
        };
        if constexpr (L::kKeyWaves == 1) {
#pragma unroll
            for (int j = 0; j < kDims; ++j) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    put(rowWave * kRows + col, 32 * j + 2 * i + 4 * half,
                        f32x4_t{o[j][i], o[j][i + 1], o[j][i + 2], o[j][i + 3]}, top, sum);
                }
            }
        } else {
            // The groups' results together.
            constexpr int kPitch = D + 4;
            if (half == 0) {
                tops[keyWave][rowWave * kRows + col] = top;
                sums[keyWave][rowWave * kRows + col] = sum;
            }
            float *out = reinterpret_cast<float *>(lds) + (keyWave * L::kBlock + rowWave * kRows + col) * kPitch;
            __syncthreads();  // (the tiles are read)
#pragma unroll
            for (int j = 0; j < kDims; ++j) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    *reinterpret_cast<f32x4_t *>(out + 32 * j + 2 * i + 4 * half) =
                        f32x4_t{o[j][i], o[j][i + 1], o[j][i + 2], o[j][i + 3]};
                }
            }
            __syncthreads();
            for (int at = (int)threadIdx.x; at < L::kBlock * (D / 4); at += L::kThreads) {
                const int r = at / (D / 4), e = at % (D / 4) * 4;
                float most = -INFINITY;
#pragma unroll
                for (int x = 0; x < L::kKeyWaves; ++x) {
                    most = fmaxf(most, tops[x][r]);
                }
                const float zero = most == -INFINITY ? 0.f : most;
                float total = 0.f;
                f32x4_t all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < L::kKeyWaves; ++x) {
                    const float f = __builtin_amdgcn_exp2f(tops[x][r] - zero);
                    total += f * sums[x][r];
                    const f32x4_t v = *reinterpret_cast<const f32x4_t *>(
                        reinterpret_cast<const float *>(lds) + (x * L::kBlock + r) * kPitch + e);
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        all[y] += scaled(v[y], f);
                    }
                }
                put(r, e, all, most, total);
            }
            __syncthreads();
        }

        unit += tiles;
        if (unit < end) {
            place.start += place.keys.units;
            place.tile = 0;
            if (++place.block == args.blocks) {
                place.block = 0;
                if (++place.kv == a.kvHeads) {
                    place.kv = 0;
                    ++place.b;
                }
            }
            place.keys = Sequence(a, place.b).keys(args, place.block);
        }
    }
}

// Joins the parts of the (sequence, kv head, block)s that no stretch finished: a workgroup
// for some rows of the one that stretch blockIdx.x began.
constexpr int kJoinThreads = 256;
constexpr int kJoinBatch = 8;

template <bool kBf16, int D>
__global__ __launch_bounds__(kJoinThreads) void draft_join(Args args)
{
    const DraftAttentionArgs &a = args.a;
    const Open open = args.open[blockIdx.x];
    if (open.units == 0) {
        return;
    }
    const int r = (int)blockIdx.y * (kJoinThreads / (D / 4)) + (int)threadIdx.x / (D / 4);
    const int e = (int)threadIdx.x % (D / 4) * 4;
    const attention::Shares shares(open.all, args.most);
    Place p{};
    p.b = open.b;
    p.kv = open.kv;
    p.block = open.block;
    const int base = open.start, first = (int)blockIdx.x, last = shares.owner(open.start + open.units - 1);
    const int64_t row = (int64_t)p.block * args.rows + r;
    const int node = (int)(row / args.group), head = (int)(row % args.group);
    if (r >= args.rows || node >= a.S || (int)threadIdx.x >= kJoinThreads / (D / 4) * (D / 4)) {
        return;
    }
    const int firstSlot = 2 * first + (shares.start(first) == base ? 0 : 1);
    float top = -INFINITY, total = 0.f;
    f32x4_t all = {0.f, 0.f, 0.f, 0.f};
    for (int x0 = first; x0 <= last; x0 += kJoinBatch) {
        float2 ends[kJoinBatch];
        f32x4_t outs[kJoinBatch];
#pragma unroll
        for (int m = 0; m < kJoinBatch; ++m) {
            const int x = x0 + m <= last ? x0 + m : last;
            const int64_t slot = x == first ? firstSlot : 2 * x;
            ends[m] = *reinterpret_cast<const float2 *>(args.ends + (slot * args.rows + r) * 2);
            outs[m] = *reinterpret_cast<const f32x4_t *>(args.outs + (slot * args.rows + r) * D + e);
        }
        float next = top;
#pragma unroll
        for (int m = 0; m < kJoinBatch; ++m) {
            next = fmaxf(next, ends[m].x);
        }
        const float zero = next == -INFINITY ? 0.f : next;
        const float keep = __builtin_amdgcn_exp2f(top - zero);
        top = next;
        total *= keep;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            all[y] = scaled(all[y], keep);
        }
#pragma unroll
        for (int m = 0; m < kJoinBatch; ++m) {
            if (x0 + m <= last) {
                const float f = __builtin_amdgcn_exp2f(ends[m].x - zero);
                total += f * ends[m].y;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    all[y] += scaled(outs[m][y], f);
                }
            }
        }
    }
    finish<kBf16>(args, p, node, head, e, all, top, total);
}

template <bool kBf16, typename L>
hipError_t launch_layout(const Args &args, hipStream_t stream)
{
    hipLaunchKernelGGL((draft_units<kBf16, L>), dim3((unsigned)args.most), dim3(L::kThreads), 0, stream, args);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        return err;
    }
    constexpr int kPer = kJoinThreads / (L::D / 4);
    const int64_t rows = (int64_t)args.a.S * args.group < args.rows ? (int64_t)args.a.S * args.group : args.rows;
    hipLaunchKernelGGL((draft_join<kBf16, L::D>),
                       dim3((unsigned)args.most, (unsigned)((rows + kPer - 1) / kPer)), dim3(kJoinThreads), 0, stream, args);
    return hipGetLastError();
}

// The layouts by rows of a (sequence, kv head).
enum class Kind { kOne, kTwo, kFour };

template <int D, Kind kKind>
struct LayoutOf;
template <int D>
struct LayoutOf<D, Kind::kOne> : Layout<D, 1, (D > 128 ? 2 : 4), 32> {};
template <int D>
struct LayoutOf<D, Kind::kTwo> : Layout<D, 2, 2, 32> {};
template <int D>
struct LayoutOf<D, Kind::kFour> : Layout<D, 4, 1, 64> {};

// Calls f(layout) for a kind and (padded) head size.
template <Kind kKind, typename F>
auto with_size(int d, F &&f)
{
    const int padded = d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 160 ? 160 : d <= 192 ? 192 : 256;
    switch (padded) {
    case 32: return f(LayoutOf<32, kKind>{});
    case 64: return f(LayoutOf<64, kKind>{});
    case 96: return f(LayoutOf<96, kKind>{});
    case 128: return f(LayoutOf<128, kKind>{});
    case 160: return f(LayoutOf<160, kKind>{});
    case 192: return f(LayoutOf<192, kKind>{});
    default: return f(LayoutOf<256, kKind>{});
    }
}

// One file per instance: mhc_draft_attention_{bf16,f16}_{one,two,four}.hip.
template <bool kBf16, Kind kKind>
hipError_t launch_kind(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<true, Kind::kOne>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<true, Kind::kTwo>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<true, Kind::kFour>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<false, Kind::kOne>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<false, Kind::kTwo>(const Args &args, hipStream_t stream);
template <>
hipError_t launch_kind<false, Kind::kFour>(const Args &args, hipStream_t stream);

}  // namespace draft
}  // namespace mhc
