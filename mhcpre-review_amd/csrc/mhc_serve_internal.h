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

// A [B, S, heads, d] tensor.
struct TokenRows {
    void *data;
    int64_t row, token, head;
};

struct DraftAttentionArgs {
    bool isBf16;
    int B, S, heads, kvHeads, d;
    TokenRows q, out;
    CacheRows kCache, vCache;
    int64_t pages;
    int pageSize, width;
    const int32_t *table, *lengths, *drafted;
    const int32_t *parents;  // null: a chain
    float scale;
    int64_t window;
    float *lse;  // or null
};

struct DraftAcceptArgs {
    int B, S;
    bool tokens64;
    const void *tokens, *chosen;
    const int32_t *parents;  // null: a chain
    const int32_t *drafted, *lengths;
    int32_t *path, *accepted, *newLengths;
    void *next;
};

struct CacheKeepArgs {
    CacheRows k, v;
    int caches;  // 1: v is k
    int64_t pages;
    int pageSize, width, kvHeads, rowBytes, elemBytes;
    int B, S;
    const int32_t *table, *lengths, *drafted, *path;
};

struct CacheBoundsArgs {
    bool isBf16;
    int B, kvHeads, d;
    CacheRows k;
    HeadRows lo, hi;  // [pages, kvHeads, d]
    int64_t pages;
    int pageSize, width, tokens;
    const int32_t *table, *lengths, *counts;
    // The launch's: columns of a row, groups of pieces of a page, all of them.
    int columns, pieceGroups;
    int64_t items;
};

struct SparseAttentionArgs {
    PagedAttentionArgs attention;  // without a window
    HeadRows lo, hi;
    int top, first, last;
    int32_t *columns;
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
// Whether the kernels' counts of work fit 31 bits.
bool draft_attention_units_fit(const DraftAttentionArgs &a);
size_t draft_attention_workspace(const DraftAttentionArgs &a, int cus);
hipError_t launch_draft_attention(const DraftAttentionArgs &a, void *workspace, int cus, hipStream_t stream);
constexpr int kDraftNodes = 256;  // the most nodes of a tree
hipError_t launch_draft_accept(const DraftAcceptArgs &a, hipStream_t stream);
hipError_t launch_cache_keep(const CacheKeepArgs &a, hipStream_t stream);
hipError_t launch_cache_bounds(const CacheBoundsArgs &a, hipStream_t stream);
bool sparse_attention_fits(const SparseAttentionArgs &a);
size_t sparse_attention_workspace(const SparseAttentionArgs &a, int cus);
hipError_t launch_sparse_attention(const SparseAttentionArgs &a, void *workspace, int device, int cus,
                                   hipStream_t stream);
size_t cache_update_workspace(const CacheUpdateArgs &a);
hipError_t launch_cache_update(const CacheUpdateArgs &a, void *workspace, int cus, hipStream_t stream);
size_t cache_compact_workspace(const CacheCompactArgs &a);
hipError_t launch_cache_compact(const CacheCompactArgs &a, void *workspace, int cus, hipStream_t stream);
hipError_t launch_copy_pages(const CopyPagesArgs &a, int cus, hipStream_t stream);

}  // namespace mhc
