// Attention of one new token per sequence over a paged cache
// (mhcPagedAttention).

#include "mhc_pre_device.h"
#include "mhc_serve_internal.h"

namespace mhc {
namespace {

using dev::kWave;

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) {
        v += __shfl_xor(v, m);
    }
    return v;
}

// One wave per row and query head: the keys one after the other, with the
// running maximum and sum of the softmax.
template <bool kBf16>
__global__ __launch_bounds__(64) void attention_rows(PagedAttentionArgs a)
{
    const int lane = (int)threadIdx.x, b = (int)blockIdx.y, h = (int)blockIdx.x;
    const int kvHead = h / (a.heads / a.kvHeads);
    const int64_t most = (int64_t)a.width * a.pageSize;
    int64_t L = a.lengths[b];
    L = L < 0 ? 0 : L > most ? most : L;
    const uint16_t *q = static_cast<const uint16_t *>(a.q.data) + b * a.q.row + h * a.q.head;
    float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = lane + i * kWave;
        qv[i] = e < a.d ? dev::x_to_f32<kBf16>(q[e]) : 0.f;
    }
    float top = -INFINITY, sum = 0.f;
    for (int64_t t = a.window > 0 && L > a.window ? L - a.window : 0; t < L; ++t) {
        const int64_t page = a.table[(int64_t)b * a.width + t / a.pageSize], slot = t % a.pageSize;
        if (page < 0 || page >= a.pages) {
            continue;
        }
        const uint16_t *k = static_cast<const uint16_t *>(a.kCache.data) + page * a.kCache.page +
                            slot * a.kCache.slot + kvHead * a.kCache.head;
        const uint16_t *v = static_cast<const uint16_t *>(a.vCache.data) + page * a.vCache.page +
                            slot * a.vCache.slot + kvHead * a.vCache.head;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = lane + i * kWave;
            if (e < a.d) {
                dot += qv[i] * dev::x_to_f32<kBf16>(k[e]);
            }
        }
        const float s = wave_sum(dot) * a.scale;
        const float next = fmaxf(top, s);
        const float keep = __expf(top - next), p = __expf(s - next);
        sum = sum * keep + p;
        top = next;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = lane + i * kWave;
            acc[i] = acc[i] * keep + (e < a.d ? p * dev::x_to_f32<kBf16>(v[e]) : 0.f);
        }
    }
    uint16_t *out = static_cast<uint16_t *>(a.out.data) + b * a.out.row + h * a.out.head;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = lane + i * kWave;
        if (e < a.d) {
            out[e] = (uint16_t)dev::f32_to_x<kBf16>(sum > 0.f ? acc[i] / sum : 0.f);
        }
    }
    if (lane == 0 && a.lse != nullptr) {
        a.lse[(int64_t)b * a.heads + h] = sum > 0.f ? top + __logf(sum) : -INFINITY;
    }
}

}  // namespace

bool paged_attention_head_size(int d)
{
    return d == 32 || d == 64 || d == 80 || d == 96 || d == 112 || d == 128 || d == 160 || d == 192 || d == 256;
}

size_t paged_attention_workspace(const PagedAttentionArgs &, int) { return 0; }

hipError_t launch_paged_attention(const PagedAttentionArgs &a, void *, int, hipStream_t stream)
{
    const auto kernel = a.isBf16 ? attention_rows<true> : attention_rows<false>;
    const int most = a.heads < 1024 ? 32768 : 512;  // work-items of a launch below 2^32
    for (int b = 0; b < a.B; b += most) {
        PagedAttentionArgs part = a;
        part.B = a.B - b < most ? a.B - b : most;
        part.q.data = static_cast<uint16_t *>(a.q.data) + b * a.q.row;
        part.out.data = static_cast<uint16_t *>(a.out.data) + b * a.out.row;
        part.table = a.table + (int64_t)b * a.width;
        part.lengths = a.lengths + b;
        part.lse = a.lse != nullptr ? a.lse + (int64_t)b * a.heads : nullptr;
        hipLaunchKernelGGL(kernel, dim3(a.heads, part.B), dim3(64), 0, stream, part);
        if (const hipError_t err = hipGetLastError(); err != hipSuccess) {
            return err;
        }
    }
    return hipSuccess;
}

}  // namespace mhc
