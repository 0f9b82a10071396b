// Norms of queries and keys per head, rotary positions and the cache write
// (mhcQkNormRope).

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
    if (slot < 0 || slot / a.pageSize >= a.pages) {
        return nullptr;
    }
    return static_cast<uint16_t *>(c.data) + slot / a.pageSize * c.page + slot % a.pageSize * c.slot + h * c.head;
}

// Row `row` of the tokens' heads of q, k and v, one wave.
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

}  // namespace

hipError_t launch_norm_rope(const NormRopeArgs &a, int cus, hipStream_t stream)
{
    (void)cus;
    const int perToken = a.heads + a.kvHeads * (a.kOut.data != nullptr ? 1 : 2);
    const int64_t rows = a.T * perToken;
    const int64_t most = int64_t{1} << 22, blocks = (rows + 3) / 4 < most ? (rows + 3) / 4 : most;
    const auto kernel = a.isBf16 ? norm_rope_rows<true> : norm_rope_rows<false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a, rows, perToken);
    return hipGetLastError();
}

}  // namespace mhc
