// Norms of queries and keys per head, rotary positions and the cache write
// (mhcQkNormRope): y = x w / sqrt(mean(x^2) + eps), each pair of y's first rot
// values turned by its angle.
//
// A row is read once, into the registers of the lanes that write it, for its sum of
// squares and the products; sums, angles' sines and products are fp32, each output is
// rounded once.  An angle is position * frequency / (2 pi) in 64 bits, of which the
// nearest whole number is taken away before it is rounded to fp32 (in 32 bits a
// position of 10^6 would have lost the phase: 2^-4 of a radian); the hardware's sine and
// cosine take turns, and are within 1.3e-7 there.
//
// Bound: the memory (2 bytes in, 2 out a value, and 6 flops).  Measured: 8192 tokens, 64 + 8
// heads of 128, 302 MB, 58 us (5.2 TB/s; a copy of 2 GiB reaches 4.8); one
// token each for 64 rows, 32 + 8 + 8 heads of 128 into the cache 5.6 us, which is a
// launch and two latencies.

#include "mhc_pre_device.h"
#include "mhc_serve_internal.h"

namespace mhc {
namespace {

using dev::kWave;

constexpr int kMaxPairs = 1024 / 2 / kWave;  // of a lane, at d = 1024

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) {
        v += __shfl_xor(v, m);
    }
    return v;
}

// Where the row of v or k of the token's slot goes, or null.
__device__ __forceinline__ uint16_t *cache_at(const CacheRows &c, const NormRopeArgs &a, int64_t t, int h)
{
    const int64_t slot = a.slots[t];
    if (slot < 0) {
        return nullptr;
    }
    // (A 64-bit division takes ten times as long.)
    const int64_t page = slot >> 32 == 0 ? (uint32_t)slot / (uint32_t)a.pageSize : slot / a.pageSize;
    if (page >= a.pages) {
        return nullptr;
    }
    return static_cast<uint16_t *>(c.data) + page * c.page + (slot - page * a.pageSize) * c.slot + h * c.head;
}

// Row `row` of the tokens' heads of q, k and v, one wave: any size, stride and
// alignment.
template <bool kBf16>
__device__ void one_row(const NormRopeArgs &a, int64_t row, int perToken, int lane)
{
    const int64_t t = row / perToken;
    int h = (int)(row % perToken);
    const bool isQ = h < a.heads;
    const bool isV = h >= a.heads + a.kvHeads;
    const HeadRows &in = isQ ? a.q : isV ? a.v : a.k;
    h -= isQ ? 0 : isV ? a.heads + a.kvHeads : a.heads;
    const uint16_t *x = static_cast<const uint16_t *>(in.data) + t * in.row + h * in.head;
    uint16_t *y;
    if (isQ) {
        y = static_cast<uint16_t *>(a.qOut.data) + t * a.qOut.row + h * a.qOut.head;
    } else if (a.kOut.data != nullptr) {
        y = static_cast<uint16_t *>(a.kOut.data) + t * a.kOut.row + h * a.kOut.head;
    } else {
        y = cache_at(isV ? a.vCache : a.kCache, a, t, h);
    }
    if (y == nullptr) {
        return;
    }
    if (isV) {  // bits as they are
        for (int e = lane; e < a.d; e += kWave) {
            y[e] = x[e];
        }
        return;
    }
    const int half = a.rot / 2, pairs = a.d / 2;
    float va[kMaxPairs], vb[kMaxPairs];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
        const int p = lane + i * kWave;
        va[i] = vb[i] = 0.f;
        if (p < pairs) {
            const bool split = p < half && !a.interleaved;
            va[i] = dev::x_to_f32<kBf16>(x[split ? p : 2 * p]);
            vb[i] = dev::x_to_f32<kBf16>(x[split ? p + half : 2 * p + 1]);
            sum += va[i] * va[i] + vb[i] * vb[i];
        }
    }
    const float *w = isQ ? a.qWeight : a.kWeight;
    float inv = 1.f;
    if (w != nullptr) {
        inv = 1.f / __builtin_sqrtf(wave_sum(sum) / (float)a.d + a.eps);
    }
    const double pos = a.positions64 ? (double)static_cast<const int64_t *>(a.positions)[t]
                                     : (double)static_cast<const int32_t *>(a.positions)[t];
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
        const int p = lane + i * kWave;
        if (p >= pairs) {
            continue;
        }
        const bool turn = p < half;
        const bool split = p < half && !a.interleaved;
        const int ia = split ? p : 2 * p, ib = split ? p + half : 2 * p + 1;
        float u = va[i], v = vb[i];
        if (w != nullptr) {
            u *= inv * w[ia];
            v *= inv * w[ib];
        }
        if (turn) {
            const double turns = pos * (a.invFreq[p] * 0.15915494309189533577);
            const float f = (float)(turns - __builtin_rint(turns));
            const float c = __builtin_amdgcn_cosf(f) * a.amplitude, s = __builtin_amdgcn_sinf(f) * a.amplitude;
            const float u0 = u;
            u = u0 * c - v * s;
            v = u0 * s + v * c;
        }
        y[ia] = (uint16_t)dev::f32_to_x<kBf16>(u);
        y[ib] = (uint16_t)dev::f32_to_x<kBf16>(v);
    }
}

// One wave per token and head of q, k or v.
template <bool kBf16>
__global__ __launch_bounds__(256) void norm_rope_rows(NormRopeArgs a, int64_t rows, int perToken)
{
    const int lane = (int)threadIdx.x % kWave;
    for (int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave; row < rows; row += (int64_t)gridDim.x * 4) {
        one_row<kBf16>(a, row, perToken, lane);
    }
}

// Sum over the aligned group of L lanes that the lane is in.
template <int L>
__device__ __forceinline__ float group_sum(float v)
{
    const auto add = [&](auto ctrl) {
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    if constexpr (L >= 2) {
        add(std::integral_constant<int, 0xB1>{});  // quad_perm [1, 0, 3, 2]
    }
    if constexpr (L >= 4) {
        add(std::integral_constant<int, 0x4E>{});  // quad_perm [2, 3, 0, 1]
    }
    if constexpr (L >= 8) {
        add(std::integral_constant<int, 0x141>{});  // row_half_mirror: the other quad, all alike
    }
    if constexpr (L >= 16) {
        add(std::integral_constant<int, 0x140>{});  // row_mirror
    }
    if constexpr (L >= 32) {
        v += __shfl_xor(v, 16);
    }
    if constexpr (L >= 64) {
        v += __shfl_xor(v, 32);
    }
    return v;
}

// 1 / sqrt(v): the instruction takes values below the normal ones for 0, which a tiny row's mean
// square is where eps is as small.
__device__ __forceinline__ float rsqrt_any(float v)
{
    const bool tiny = v < 0x1p-100f;
    return __builtin_amdgcn_rsqf(tiny ? v * 0x1p100f : v) * (tiny ? 0x1p50f : 1.f);
}

constexpr int kSteps = 4;

struct Split {
    int parts;       // of a token's rows, each a wave's
    int q, k, all;   // steps of 64 / L rows: of q, of k, with v's
};

// Rows whose 16-byte pieces are aligned (a value at a time as above, 8192 tokens of 72 heads
// of 128 take 345 us, so 60.6): L lanes to a row (d / 16 of them with
// work), each with 8 pairs in two pieces: at 8 c and rot / 2 + 8 c (the half layout;
// beyond rot likewise, half of the rest apart), or at 8 c and d / 2 + 8 c
// (interleaved), so that neighbouring lanes have neighbouring pieces.  A wave has
// some of a token's rows, 64 / L at a time, and computes the token's 8 angles per
// lane once for all of them.
//
// kBy: the stores pass the caches by (1: more is written than the L2s keep for the
// reader), and the loads too (2: more is read than the last-level cache holds).
// 8192 tokens, 72 heads of 128, us: neither 64.2, stores 61.1, both 58.9; 4096 tokens,
// 20 + 4 heads of 256 into the cache 31.8 / 25.4 / 28.8.
template <bool kBf16, int L, bool kInterleaved, int kBy>
__global__ __launch_bounds__(256) void norm_rope_pieces(NormRopeArgs a, Split split)
{
    constexpr int kRows = kWave / L;
    const int lane = (int)threadIdx.x % kWave, c = lane % L, sub = lane / L;
    const int half = a.rot / 2;
    const bool on = 16 * c < a.d;
    const bool turned = 8 * c < half;  // (the half layout: a lane's pairs all are or none is)
    const int at0 = kInterleaved || turned ? 8 * c : half + 8 * c;
    const int at1 = kInterleaved ? a.d / 2 + 8 * c : turned ? half + 8 * c : a.d / 2 + 8 * c;
    const float perValue = 1.f / (float)a.d;
    const auto pair = [&](int j) { return !kInterleaved ? 8 * c + j : j < 4 ? 4 * c + j : a.d / 4 + 4 * c + j - 4; };
    double freq[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int p = pair(j);
        freq[j] = p < half ? a.invFreq[p] * 0.15915494309189533577 : 0.0;
    }
    const int64_t items = a.T * split.parts, step = (int64_t)gridDim.x * 4;
    for (int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave); item < items;
         item += step) {
        const int64_t t = split.parts == 1 ? item : item / split.parts;
        const int part = split.parts == 1 ? 0 : (int)(item - t * split.parts);
        const int begin = part * split.all / split.parts, end = (part + 1) * split.all / split.parts;
        float cosine[8], sine[8];
        const double pos = a.positions64 ? (double)static_cast<const int64_t *>(a.positions)[t]
                                         : (double)static_cast<const int32_t *>(a.positions)[t];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double turns = pos * freq[j];
            const float f = (float)(turns - __builtin_rint(turns));
            cosine[j] = __builtin_amdgcn_cosf(f) * a.amplitude;
            sine[j] = __builtin_amdgcn_sinf(f) * a.amplitude;
        }
        // Norm and rotation of the lane's two pieces.
        const auto turn_row = [&](dev::u32x4_t &r0, dev::u32x4_t &r1, bool norm, const float (&w)[16]) {
            float u[8], v[8];
            dev::unpack8<kBf16>(r0, u);
            dev::unpack8<kBf16>(r1, v);
            if (norm) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    sum = __builtin_fmaf(u[j], u[j], sum);
                    sum = __builtin_fmaf(v[j], v[j], sum);
                }
                const float inv = rsqrt_any(group_sum<L>(sum) * perValue + a.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    u[j] *= inv * w[j];
                    v[j] *= inv * w[8 + j];
                }
            }
            if constexpr (kInterleaved) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float &first = j < 4 ? u[2 * j] : v[2 * j - 8], &second = j < 4 ? u[2 * j + 1] : v[2 * j - 7];
                    const float u0 = first, v0 = second;
                    const bool turn = pair(j) < half;
                    first = turn ? u0 * cosine[j] - v0 * sine[j] : u0;
                    second = turn ? u0 * sine[j] + v0 * cosine[j] : v0;
                }
            } else if (turned) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float u0 = u[j];
                    u[j] = u0 * cosine[j] - v[j] * sine[j];
                    v[j] = u0 * sine[j] + v[j] * cosine[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                r0[j] = dev::pack2_x<kBf16>(u[2 * j], u[2 * j + 1]);
                r1[j] = dev::pack2_x<kBf16>(v[2 * j], v[2 * j + 1]);
            }
        };
        // kSteps steps' rows are on their way at once.
        const auto rows = [&](auto kind, const HeadRows &in, const HeadRows &out, int heads, const float *w, int first,
                              int last) {
            constexpr bool isV = decltype(kind)::value == 2;
            float weights[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                weights[j] = !isV && w != nullptr && on ? w[at0 + j] : 0.f;
                weights[8 + j] = !isV && w != nullptr && on ? w[at1 + j] : 0.f;
            }
            for (int i = first; i < last; i += kSteps) {
                dev::u32x4_t r0[kSteps], r1[kSteps];
#pragma unroll
                for (int n = 0; n < kSteps; ++n) {
                    const int h = (i + n) * kRows + sub;
                    // (Lanes without values stay: their row's sum goes through them.)
                    r0[n] = r1[n] = dev::u32x4_t{0, 0, 0, 0};
                    if (on && i + n < last && h < heads) {
                        const uint16_t *x = static_cast<const uint16_t *>(in.data) + t * in.row + h * in.head;
                        const auto *x0 = reinterpret_cast<const dev::u32x4_t *>(x + at0);
                        const auto *x1 = reinterpret_cast<const dev::u32x4_t *>(x + at1);
                        r0[n] = kBy == 2 ? __builtin_nontemporal_load(x0) : *x0;
                        r1[n] = kBy == 2 ? __builtin_nontemporal_load(x1) : *x1;
                    }
                }
#pragma unroll
                for (int n = 0; n < kSteps; ++n) {
                    if (i + n >= last) {
                        break;
                    }
                    const int h = (i + n) * kRows + sub;
                    if constexpr (!isV) {
                        turn_row(r0[n], r1[n], w != nullptr, weights);
                    }
                    if (on && h < heads) {
                        uint16_t *y = static_cast<uint16_t *>(out.data) + h * out.head;
                        auto *y0 = reinterpret_cast<dev::u32x4_t *>(y + at0), *y1 = reinterpret_cast<dev::u32x4_t *>(y + at1);
                        if constexpr (kBy > 0) {
                            __builtin_nontemporal_store(r0[n], y0);
                            __builtin_nontemporal_store(r1[n], y1);
                        } else {
                            *y0 = r0[n];
                            *y1 = r1[n];
                        }
                    }
                }
            }
        };
        const auto clip = [](int v, int low, int high) { return v < low ? low : v > high ? high : v; };
        const int q0 = clip(begin, 0, split.q), q1 = clip(end, 0, split.q);
        if (q0 < q1) {
            HeadRows out = a.qOut;
            out.data = static_cast<uint16_t *>(out.data) + t * out.row;
            rows(std::integral_constant<int, 0>{}, a.q, out, a.heads, a.qWeight, q0, q1);
        }
        const int k0 = clip(begin - split.q, 0, split.k), k1 = clip(end - split.q, 0, split.k);
        const int v0 = clip(begin - split.q - split.k, 0, split.k), v1 = clip(end - split.q - split.k, 0, split.k);
        if (a.kOut.data != nullptr) {
            HeadRows out = a.kOut;
            out.data = static_cast<uint16_t *>(out.data) + t * out.row;
            rows(std::integral_constant<int, 1>{}, a.k, out, a.kvHeads, a.kWeight, k0, k1);
        } else if (k0 < k1 || v0 < v1) {
            // No slot: neither k nor v of this token goes anywhere.
            uint16_t *y = cache_at(a.kCache, a, t, 0);
            if (y != nullptr) {
                rows(std::integral_constant<int, 1>{}, a.k, HeadRows{y, 0, a.kCache.head}, a.kvHeads, a.kWeight, k0, k1);
                rows(std::integral_constant<int, 2>{}, a.v, HeadRows{cache_at(a.vCache, a, t, 0), 0, a.vCache.head},
                     a.kvHeads, nullptr, v0, v1);
            }
        }
    }
}

bool even_rows(const HeadRows &r)
{
    return (reinterpret_cast<uintptr_t>(r.data) % 16 | r.row % 8 | r.head % 8) == 0;
}

bool even_cache(const CacheRows &r)
{
    return (reinterpret_cast<uintptr_t>(r.data) % 16 | r.page % 8 | r.slot % 8 | r.head % 8) == 0;
}

template <bool kBf16, int L>
hipError_t launch_pieces(const NormRopeArgs &a, int cus, hipStream_t stream)
{
    constexpr int kRows = kWave / L;
    Split s;
    s.q = (a.heads + kRows - 1) / kRows;
    s.k = (a.kvHeads + kRows - 1) / kRows;
    s.all = s.q + s.k * (a.kOut.data != nullptr ? 1 : 2);
    // A token's rows are shared out until each SIMD has a wave; more waves would each compute
    // the token's angles again (1024 tokens of 40 heads of 128, us: 16 waves a CU 13.1, 4 9.0;
    // 2048 tokens into the cache 13.8 / 12.7).
    const int64_t fill = (int64_t)cus * 4;
    const int64_t want = a.T < fill ? (fill + a.T - 1) / a.T : 1;
    s.parts = want < s.all ? (int)want : s.all;
    const int64_t blocks = (a.T * s.parts + 3) / 4, most = (int64_t)cus * 8;
    const int64_t bytes = 2 * a.T * a.d * (a.heads + (int64_t)a.kvHeads * (a.kOut.data != nullptr ? 1 : 2));
    const int by = bytes > (int64_t{128} << 20) ? 2 : bytes > (int64_t{4} << 20) ? 1 : 0;
    const auto pick = [&](auto interleaved) {
        constexpr bool kInterleaved = decltype(interleaved)::value;
        return by == 2   ? norm_rope_pieces<kBf16, L, kInterleaved, 2>
               : by == 1 ? norm_rope_pieces<kBf16, L, kInterleaved, 1>
                         : norm_rope_pieces<kBf16, L, kInterleaved, 0>;
    };
    const auto kernel = a.interleaved ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, a, s);
    return hipGetLastError();
}

template <bool kBf16>
hipError_t launch_pieces_of(const NormRopeArgs &a, int cus, hipStream_t stream)
{
    const int lanes = a.d / 16;
    return lanes <= 1    ? launch_pieces<kBf16, 1>(a, cus, stream)
           : lanes <= 2  ? launch_pieces<kBf16, 2>(a, cus, stream)
           : lanes <= 4  ? launch_pieces<kBf16, 4>(a, cus, stream)
           : lanes <= 8  ? launch_pieces<kBf16, 8>(a, cus, stream)
           : lanes <= 16 ? launch_pieces<kBf16, 16>(a, cus, stream)
           : lanes <= 32 ? launch_pieces<kBf16, 32>(a, cus, stream)
                         : launch_pieces<kBf16, 64>(a, cus, stream);
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeArgs &a, int cus, hipStream_t stream)
{
    const bool append = a.kOut.data == nullptr;
    if (a.d % 16 == 0 && (a.interleaved || a.rot % 16 == 0) && even_rows(a.q) && even_rows(a.k) && even_rows(a.qOut) &&
        (append ? even_rows(a.v) && even_cache(a.kCache) && even_cache(a.vCache) : even_rows(a.kOut))) {
        return a.isBf16 ? launch_pieces_of<true>(a, cus, stream) : launch_pieces_of<false>(a, cus, stream);
    }
    const int perToken = a.heads + a.kvHeads * (a.kOut.data != nullptr ? 1 : 2);
    const int64_t rows = a.T * perToken;
    const int64_t most = int64_t{1} << 22, blocks = (rows + 3) / 4 < most ? (rows + 3) / 4 : most;
    const auto kernel = a.isBf16 ? norm_rope_rows<true> : norm_rope_rows<false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a, rows, perToken);
    return hipGetLastError();
}

}  // namespace mhc
