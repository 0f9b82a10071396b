// Launch arguments of the serving operators (include/mhc_serve.h), shared by
// the host library and their kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

namespace mhc {

// A [rows, heads, d] tensor: strides in elements, that of d is 1.
struct HeadRows {
    void *data;
    int64_t row, head;
};

// A cache [pages, pageSize, kvHeads, d].
struct CacheRows {
    void *data;
    int64_t page, slot, head;
};

struct NormRopeArgs {
    bool isBf16;
    int64_t T;
    int heads, kvHeads, d, rot;
    HeadRows q, k, v, qOut, kOut;  // kOut.data null: k and v go to the caches
    const void *positions;
    bool positions64;
    const double *invFreq;
    const float *qWeight, *kWeight;  // null: no norm
    float eps, amplitude;
    bool interleaved;
    const int64_t *slots;
    CacheRows kCache, vCache;
    int64_t pages;
    int pageSize;
};

struct PagedAttentionArgs {
    bool isBf16;
    int B, heads, kvHeads, d;
    HeadRows q, out;
    CacheRows kCache, vCache;
    int64_t pages;
    int pageSize, width;
    const int32_t *table, *lengths;
    float scale;
    int64_t window;
    float *lse;  // or null
};

struct CacheUpdateArgs {
    int rows, width, tokens;
    int64_t pages;
    int pageSize;
    const int32_t *table, *lengths, *parents, *counts;
    int32_t *newTable, *newLengths, *granted, *src, *dst;
    int64_t *slots;
};

struct CacheCompactArgs {
    int rows, width;
    int64_t pages;
    int pageSize;
    const int32_t *table, *lengths;
    int32_t *newTable, *src, *dst, *used;
};

struct CopyPagesArgs {
    CacheRows k, v;
    int64_t pages;
    int pageSize, kvHeads, rowBytes;  // bytes of a head's slot: d elements
    int elemBytes;
    int64_t n;
    const int32_t *src, *dst;
};

// Each launcher enqueues on the current device and returns the first HIP
// error.  cus: compute units of the device.
hipError_t launch_norm_rope(const NormRopeArgs &a, int cus, hipStream_t stream);
size_t paged_attention_workspace(const PagedAttentionArgs &a, int cus);
bool paged_attention_head_size(int64_t d);
// Whether the kernels' counts of work fit 31 bits.
bool paged_attention_units_fit(const PagedAttentionArgs &a);
hipError_t launch_paged_attention(const PagedAttentionArgs &a, void *workspace, int device, int cus,
                                  hipStream_t stream);
size_t cache_update_workspace(const CacheUpdateArgs &a);
hipError_t launch_cache_update(const CacheUpdateArgs &a, void *workspace, int cus, hipStream_t stream);
size_t cache_compact_workspace(const CacheCompactArgs &a);
hipError_t launch_cache_compact(const CacheCompactArgs &a, void *workspace, int cus, hipStream_t stream);
hipError_t launch_copy_pages(const CopyPagesArgs &a, int cus, hipStream_t stream);

}  // namespace mhc
