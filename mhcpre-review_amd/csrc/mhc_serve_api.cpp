// Host side of the serving operators (include/mhc_serve.h): validation,
// executors, workspace sizes and launches.

#include "mhc_serve.h"
#include "mhc_pre_internal.h"
#include "mhc_serve_internal.h"

#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <new>

namespace {

enum class Op { kNormRope, kAttention, kUpdate, kCompact, kCopy, kDraft, kAccept, kKeep, kBounds, kSparse };

// The most rows, pages and elements a tensor may have: every index below fits
// its kernel's type, every byte offset 62 bits.
constexpr int64_t kMaxCount = (int64_t{1} << 31) - 1;
constexpr int64_t kMaxElements = int64_t{1} << 60;
constexpr int64_t kMaxTableRows = int64_t{1} << 22;
constexpr int kPlanCus = 256;  // MI355X, where the runtime cannot tell the device

}  // namespace

struct mhcServeExecutor {
    Op op;
    int device = -1;  // device of the tensors (-1: the runtime could not tell)
    int cus = kPlanCus;
    uint64_t workspace = 0;
    bool empty = false;  // nothing to do: no rows
    union {
        mhc::NormRopeArgs rope;
        mhc::PagedAttentionArgs attention;
        mhc::CacheUpdateArgs update;
        mhc::CacheCompactArgs compact;
        mhc::CopyPagesArgs copy;
        mhc::DraftAttentionArgs draft;
        mhc::DraftAcceptArgs accept;
        mhc::CacheKeepArgs keep;
        mhc::CacheBoundsArgs bounds;
        mhc::SparseAttentionArgs sparse;
    };
    mhcServeExecutor() : rope{} {}
};

namespace {

bool aligned(const void *p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// The device that holds `p`, and its compute units.
void find_device(const void *p, mhcServeExecutor &ex)
{
    hipPointerAttribute_t attr;
    if (hipPointerGetAttributes(&attr, p) != hipSuccess || attr.type != hipMemoryTypeDevice) {
        (void)hipGetLastError();
        return;
    }
    ex.device = attr.device;
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];
    if (ex.device < 0 || ex.device >= kDevices) {
        return;
    }
    int cus = known[ex.device].load(std::memory_order_relaxed);
    if (cus == 0) {
        if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, ex.device) != hipSuccess || cus <= 0) {
            (void)hipGetLastError();
            return;
        }
        known[ex.device].store(cus, std::memory_order_relaxed);
    }
    ex.cus = cus;
}

int first_of(std::initializer_list<int> statuses)
{
    for (int s : statuses) {
        if (s != MHC_STATUS_SUCCESS) {
            return s;
        }
    }
    return MHC_STATUS_SUCCESS;
}

// A dense tensor of one of `dtypes` and exactly these dims; with no elements
// its data may be null.
int check_dense(const mhcTensor *t, std::initializer_list<int32_t> dtypes, std::initializer_list<int64_t> dims)
{
    if (t == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    if (t->ndim != static_cast<int32_t>(dims.size())) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    int i = 0;
    int64_t n = 1;
    for (int64_t want : dims) {
        if (t->dims[i++] != want || want < 0 || __builtin_mul_overflow(n, want, &n) || n > kMaxElements) {
            return MHC_STATUS_INVALID_SHAPE;
        }
    }
    bool known = false;
    for (int32_t d : dtypes) {
        known = known || t->dtype == d;
    }
    if (!known) {
        return MHC_STATUS_INVALID_DTYPE;
    }
    if (t->data == nullptr && n > 0) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    const uintptr_t size = t->dtype == MHC_DTYPE_INT64 || t->dtype == MHC_DTYPE_DOUBLE ? 8 : 4;
    return aligned(t->data, size) ? MHC_STATUS_SUCCESS : MHC_STATUS_MISALIGNED;
}

int elem_bytes(int32_t dtype)
{
    switch (dtype) {
    case MHC_DTYPE_FLOAT16:
    case MHC_DTYPE_BF16:
        return 2;
    case MHC_DTYPE_FLOAT:
        return 4;
    default:
        return 0;
    }
}

// A strided tensor of type `dtype` and these dims whose elements lie within
// 2^60 of its first one; non-negative strides.  `align`: of its data and, in
// bytes, of its strides.
int check_strided(const mhcStridedTensor *t, int32_t dtype, std::initializer_list<int64_t> dims, int align)
{
    if (t == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    if (t->ndim != static_cast<int32_t>(dims.size())) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (t->dtype != dtype || elem_bytes(dtype) == 0) {
        return MHC_STATUS_INVALID_DTYPE;
    }
    int i = 0;
    int64_t n = 1, reach = 0;
    bool even = true;
    for (int64_t want : dims) {
        int64_t step = 0;
        const int64_t stride = t->strides[i];
        if (t->dims[i] != want || want < 0 || __builtin_mul_overflow(n, want, &n) || n > kMaxElements) {
            return MHC_STATUS_INVALID_SHAPE;
        }
        if (want > 1) {
            if (stride < 0 || __builtin_mul_overflow(stride, want - 1, &step) ||
                __builtin_add_overflow(reach, step, &reach) || reach > kMaxElements) {
                return MHC_STATUS_INVALID_SHAPE;
            }
            const bool last = i + 1 == t->ndim;
            if (last && stride != 1) {
                return MHC_STATUS_INVALID_SHAPE;
            }
            even = even && (last || stride * elem_bytes(dtype) % align == 0);
        }
        ++i;
    }
    if (n == 0) {
        return MHC_STATUS_SUCCESS;
    }
    if (t->data == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    return even && aligned(t->data, align) ? MHC_STATUS_SUCCESS : MHC_STATUS_MISALIGNED;
}

// Strides of dimensions of size 1 are never used: 0, so that no offset is
// formed from what a caller left there.
int64_t stride_of(const mhcStridedTensor *t, int i) { return t->dims[i] > 1 ? t->strides[i] : 0; }

mhc::HeadRows head_rows(const mhcStridedTensor *t)
{
    return {t->data, stride_of(t, 0), stride_of(t, 1)};
}

mhc::TokenRows token_rows(const mhcStridedTensor *t)
{
    return {t->data, stride_of(t, 0), stride_of(t, 1), stride_of(t, 2)};
}

mhc::CacheRows cache_rows(const mhcStridedTensor *t)
{
    return {t->data, stride_of(t, 0), stride_of(t, 1), stride_of(t, 2)};
}

// Looks the device's replay words up (once per device), so that a launch under
// stream capture does not have to.
void prime_replay_words(const mhcServeExecutor &ex)
{
    int current = -1;
    uint32_t *words = nullptr;
    if (ex.device >= 0 && hipGetDevice(&current) == hipSuccess && current == ex.device) {
        (void)mhc::replay_words_address(current, &words);
    }
    (void)hipGetLastError();
}

// Hands a filled executor out.
int finish(mhcServeExecutor *ex, const void *someTensor, uint64_t *workspaceSize, mhcServeExecutor **executor)
{
    if (!ex->empty) {
        find_device(someTensor, *ex);
    }
    switch (ex->op) {
    case Op::kAttention:
        ex->workspace = ex->empty ? 0 : mhc::paged_attention_workspace(ex->attention, ex->cus);
        prime_replay_words(*ex);
        break;
    case Op::kUpdate:
        ex->workspace = ex->empty ? 0 : mhc::cache_update_workspace(ex->update);
        break;
    case Op::kCompact:
        ex->workspace = mhc::cache_compact_workspace(ex->compact);
        break;
    case Op::kDraft:
        ex->workspace = ex->empty ? 0 : mhc::draft_attention_workspace(ex->draft, ex->cus);
        break;
    case Op::kSparse:
        ex->workspace = ex->empty ? 0 : mhc::sparse_attention_workspace(ex->sparse, ex->cus);
        prime_replay_words(*ex);
        break;
    case Op::kNormRope:
    case Op::kCopy:
    case Op::kAccept:
    case Op::kKeep:
    case Op::kBounds:
        break;
    }
    *workspaceSize = ex->workspace;
    *executor = ex;
    return MHC_STATUS_SUCCESS;
}

int launch(Op op, void *workspace, uint64_t workspaceSize, mhcServeExecutor *ex, hipStream_t stream)
{
    if (ex == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    if (ex->op != op) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (ex->workspace > 0 && (workspace == nullptr || workspaceSize < ex->workspace || !aligned(workspace, 256))) {
        return MHC_STATUS_WORKSPACE_TOO_SMALL;
    }
    if (ex->empty) {
        return MHC_STATUS_SUCCESS;
    }
    int current = -1;
    if (hipGetDevice(&current) != hipSuccess) {
        (void)hipGetLastError();
        return MHC_STATUS_HIP_ERROR;
    }
    if (ex->device >= 0 && current != ex->device) {
        return MHC_STATUS_DEVICE_MISMATCH;
    }
    (void)hipGetLastError();  // an earlier call's error is not this launch's
    hipError_t err = hipSuccess;
    switch (op) {
    case Op::kNormRope:
        err = mhc::launch_norm_rope(ex->rope, ex->cus, stream);
        break;
    case Op::kAttention:
        err = mhc::launch_paged_attention(ex->attention, workspace, current, ex->cus, stream);
        break;
    case Op::kUpdate:
        err = mhc::launch_cache_update(ex->update, workspace, ex->cus, stream);
        break;
    case Op::kCompact:
        err = mhc::launch_cache_compact(ex->compact, workspace, ex->cus, stream);
        break;
    case Op::kCopy:
        err = mhc::launch_copy_pages(ex->copy, ex->cus, stream);
        break;
    case Op::kDraft:
        err = mhc::launch_draft_attention(ex->draft, workspace, ex->cus, stream);
        break;
    case Op::kAccept:
        err = mhc::launch_draft_accept(ex->accept, stream);
        break;
    case Op::kKeep:
        err = mhc::launch_cache_keep(ex->keep, stream);
        break;
    case Op::kBounds:
        err = mhc::launch_cache_bounds(ex->bounds, stream);
        break;
    case Op::kSparse:
        err = mhc::launch_sparse_attention(ex->sparse, workspace, current, ex->cus, stream);
        break;
    }
    return err == hipSuccess ? MHC_STATUS_SUCCESS : MHC_STATUS_HIP_ERROR;
}

// [pages, pageSize, kvHeads, d] of a cache whose sizes fit the kernels.
int cache_limits(const mhcStridedTensor *c)
{
    if (c == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    if (c->ndim != 4) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    for (int i = 0; i < 4; ++i) {
        if (c->dims[i] < 1) {
            return MHC_STATUS_INVALID_SHAPE;
        }
        if (c->dims[i] > kMaxCount) {
            return MHC_STATUS_UNSUPPORTED_SHAPE;
        }
    }
    return MHC_STATUS_SUCCESS;
}

// The page table [rows, width] and lengths [rows] of a pool of `pages` pages.
int table_limits(const mhcTensor *table, const mhcTensor *lengths, int64_t pages, int64_t pageSize)
{
    if (table == nullptr || lengths == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    if (table->ndim != 2 || table->dims[0] < 0 || table->dims[1] < 1 || pages < 1 || pageSize < 1) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (table->dims[0] > kMaxTableRows || table->dims[1] > kMaxCount || pages > kMaxCount || pageSize > kMaxCount ||
        table->dims[1] > kMaxCount / pageSize) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    return first_of({check_dense(table, {MHC_DTYPE_INT32}, {table->dims[0], table->dims[1]}),
                     check_dense(lengths, {MHC_DTYPE_INT32}, {table->dims[0]})});
}

// The arguments that attention of single tokens takes, checked.
int attention_args(const mhcStridedTensor *q, const mhcStridedTensor *kCache, const mhcStridedTensor *vCache,
                   const mhcTensor *pageTable, const mhcTensor *lengths, float scale, int64_t window,
                   const mhcStridedTensor *out, const mhcTensor *lse, uint64_t *workspaceSize,
                   mhcServeExecutor **executor, mhc::PagedAttentionArgs &a)
{
    if (q == nullptr || out == nullptr || vCache == nullptr || workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    int st = cache_limits(kCache);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t pages = kCache->dims[0], pageSize = kCache->dims[1], kvHeads = kCache->dims[2], d = kCache->dims[3];
    if (q->ndim != 3 || window < 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (q->dtype != MHC_DTYPE_FLOAT16 && q->dtype != MHC_DTYPE_BF16) {
        return MHC_STATUS_INVALID_DTYPE;
    }
    const int64_t B = q->dims[0], heads = q->dims[1];
    if (B < 0 || heads < 1 || heads % kvHeads != 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if ((st = table_limits(pageTable, lengths, pages, pageSize)) != MHC_STATUS_SUCCESS) {
        return st;
    }
    if (pageTable->dims[0] != B) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (!mhc::paged_attention_head_size(d) || heads > 65536 || B > (1 << 20)) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    st = first_of({check_strided(q, q->dtype, {B, heads, d}, 16), check_strided(out, q->dtype, {B, heads, d}, 16),
                   check_strided(kCache, q->dtype, {pages, pageSize, kvHeads, d}, 16),
                   check_strided(vCache, q->dtype, {pages, pageSize, kvHeads, d}, 16),
                   lse != nullptr ? check_dense(lse, {MHC_DTYPE_FLOAT}, {B, heads}) : MHC_STATUS_SUCCESS});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    a.isBf16 = q->dtype == MHC_DTYPE_BF16;
    a.B = static_cast<int>(B);
    a.heads = static_cast<int>(heads);
    a.kvHeads = static_cast<int>(kvHeads);
    a.d = static_cast<int>(d);
    a.q = head_rows(q);
    a.out = head_rows(out);
    a.kCache = cache_rows(kCache);
    a.vCache = cache_rows(vCache);
    a.pages = pages;
    a.pageSize = static_cast<int>(pageSize);
    a.width = static_cast<int>(pageTable->dims[1]);
    a.table = static_cast<const int32_t *>(pageTable->data);
    a.lengths = static_cast<const int32_t *>(lengths->data);
    a.scale = scale;
    a.window = window;
    a.lse = lse != nullptr ? static_cast<float *>(lse->data) : nullptr;
    return MHC_STATUS_SUCCESS;
}

}  // namespace

extern "C" {

int mhcServeExecutorDestroy(mhcServeExecutor *executor)
{
    if (executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    delete executor;
    return MHC_STATUS_SUCCESS;
}

int mhcQkNormRopeGetWorkspaceSize(const mhcStridedTensor *q, const mhcStridedTensor *k, const mhcStridedTensor *v,
                                  const mhcTensor *positions, const mhcTensor *invFreq, const mhcTensor *qWeight,
                                  const mhcTensor *kWeight, float eps, int32_t interleaved, float amplitude,
                                  const mhcTensor *slots, const mhcStridedTensor *qOut, const mhcStridedTensor *kOut,
                                  const mhcStridedTensor *kCache, const mhcStridedTensor *vCache,
                                  uint64_t *workspaceSize, mhcServeExecutor **executor)
{
    if (q == nullptr || k == nullptr || qOut == nullptr || workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    // Either kOut, or v, slots and both caches.
    const bool append = kOut == nullptr;
    if (append != (v != nullptr) || append != (slots != nullptr) || append != (kCache != nullptr) ||
        append != (vCache != nullptr) || (qWeight == nullptr) != (kWeight == nullptr)) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    if (q->ndim != 3 || k->ndim != 3) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (q->dtype != MHC_DTYPE_FLOAT16 && q->dtype != MHC_DTYPE_BF16) {
        return MHC_STATUS_INVALID_DTYPE;
    }
    const int64_t T = q->dims[0], heads = q->dims[1], d = q->dims[2], kvHeads = k->dims[1];
    if (T < 0 || heads < 1 || kvHeads < 1 || d < 1) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (d % 2 != 0 || d > 1024 || heads > 65536 || kvHeads > 65536 || T > kMaxCount) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    int64_t rot = 0;
    if (invFreq != nullptr) {
        if (invFreq->ndim != 1 || invFreq->dims[0] < 0 || invFreq->dims[0] > d / 2) {
            return MHC_STATUS_INVALID_SHAPE;
        }
        rot = 2 * invFreq->dims[0];
        if (const int st = check_dense(invFreq, {MHC_DTYPE_DOUBLE}, {rot / 2})) {
            return st;
        }
    }
    int st = first_of({check_strided(q, q->dtype, {T, heads, d}, 2), check_strided(k, q->dtype, {T, kvHeads, d}, 2),
                       check_strided(qOut, q->dtype, {T, heads, d}, 2),
                       check_dense(positions, {MHC_DTYPE_INT32, MHC_DTYPE_INT64}, {T})});
    if (st == MHC_STATUS_SUCCESS && qWeight != nullptr) {
        st = first_of({check_dense(qWeight, {MHC_DTYPE_FLOAT}, {d}), check_dense(kWeight, {MHC_DTYPE_FLOAT}, {d})});
    }
    if (st == MHC_STATUS_SUCCESS && !append) {
        st = check_strided(kOut, q->dtype, {T, kvHeads, d}, 2);
    }
    if (st == MHC_STATUS_SUCCESS && append) {
        st = cache_limits(kCache);
    }
    if (st == MHC_STATUS_SUCCESS && append) {
        const int64_t pages = kCache->dims[0], pageSize = kCache->dims[1];
        st = first_of({check_strided(v, q->dtype, {T, kvHeads, d}, 2), check_dense(slots, {MHC_DTYPE_INT64}, {T}),
                       check_strided(kCache, q->dtype, {pages, pageSize, kvHeads, d}, 2),
                       check_strided(vCache, q->dtype, {pages, pageSize, kvHeads, d}, 2)});
    }
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kNormRope;
    ex->empty = T == 0;
    mhc::NormRopeArgs &a = ex->rope;
    a.isBf16 = q->dtype == MHC_DTYPE_BF16;
    a.T = T;
    a.heads = static_cast<int>(heads);
    a.kvHeads = static_cast<int>(kvHeads);
    a.d = static_cast<int>(d);
    a.rot = static_cast<int>(rot);
    a.q = head_rows(q);
    a.k = head_rows(k);
    a.qOut = head_rows(qOut);
    a.positions = positions->data;
    a.positions64 = positions->dtype == MHC_DTYPE_INT64;
    a.invFreq = rot > 0 ? static_cast<const double *>(invFreq->data) : nullptr;
    if (qWeight != nullptr) {
        a.qWeight = static_cast<const float *>(qWeight->data);
        a.kWeight = static_cast<const float *>(kWeight->data);
    }
    a.eps = eps;
    a.amplitude = amplitude;
    a.interleaved = interleaved != 0;
    if (append) {
        a.v = head_rows(v);
        a.slots = static_cast<const int64_t *>(slots->data);
        a.kCache = cache_rows(kCache);
        a.vCache = cache_rows(vCache);
        a.pages = kCache->dims[0];
        a.pageSize = static_cast<int>(kCache->dims[1]);
    } else {
        a.kOut = head_rows(kOut);
    }
    return finish(ex, q->data, workspaceSize, executor);
}

int mhcQkNormRope(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kNormRope, workspace, workspaceSize, executor, stream);
}

int mhcRotaryFrequencies(int32_t rot, double base, int32_t kind, double factor, double low, double high,
                         double trainedLength, double *invFreq)
{
    if (invFreq == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    const bool ramp = kind == MHC_ROTARY_RAMP || kind == MHC_ROTARY_INDEX_RAMP;
    if (rot < 2 || rot % 2 != 0 || kind < MHC_ROTARY_PLAIN || kind > MHC_ROTARY_INDEX_RAMP || !(base > 1) ||
        !std::isfinite(base) || !(factor > 0) || !std::isfinite(factor) || (kind == MHC_ROTARY_BASE && rot < 4) ||
        (ramp && (!(low > 0) || !(high > low) || !std::isfinite(high) || !(trainedLength > 0) ||
                  !std::isfinite(trainedLength)))) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    constexpr double kTurn = 6.283185307179586476925;
    if (kind == MHC_ROTARY_BASE) {
        base *= std::pow(factor, static_cast<double>(rot) / (rot - 2));
    }
    double first = 0, last = 0;  // MHC_ROTARY_INDEX_RAMP's ends
    if (kind == MHC_ROTARY_INDEX_RAMP) {
        const auto index = [&](double turns) {
            return rot * std::log(trainedLength / (kTurn * turns)) / (2 * std::log(base));
        };
        first = std::fmax(std::floor(index(high)), 0.0);
        last = std::fmin(std::ceil(index(low)), rot - 1.0);
        if (!(last > first)) {
            last = first + 1e-3;  // a step
        }
    }
    for (int i = 0; i < rot / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / rot);
        double keep = 1;  // weight of f; the rest is f / factor's
        if (kind == MHC_ROTARY_LINEAR) {
            keep = 0;
        } else if (kind == MHC_ROTARY_RAMP) {
            keep = (trainedLength * f / kTurn - low) / (high - low);
        } else if (kind == MHC_ROTARY_INDEX_RAMP) {
            keep = 1 - (i - first) / (last - first);
        }
        keep = std::fmin(std::fmax(keep, 0.0), 1.0);
        invFreq[i] = keep * f + (1 - keep) * (f / factor);
    }
    return MHC_STATUS_SUCCESS;
}

int mhcPagedAttentionGetWorkspaceSize(const mhcStridedTensor *q, const mhcStridedTensor *kCache,
                                      const mhcStridedTensor *vCache, const mhcTensor *pageTable,
                                      const mhcTensor *lengths, float scale, int64_t window,
                                      const mhcStridedTensor *out, const mhcTensor *lse, uint64_t *workspaceSize,
                                      mhcServeExecutor **executor)
{
    mhc::PagedAttentionArgs a{};
    const int st = attention_args(q, kCache, vCache, pageTable, lengths, scale, window, out, lse, workspaceSize, executor, a);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    if (!mhc::paged_attention_units_fit(a)) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kAttention;
    ex->empty = a.B == 0;
    ex->attention = a;
    return finish(ex, q->data, workspaceSize, executor);
}

int mhcPagedAttention(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kAttention, workspace, workspaceSize, executor, stream);
}

int mhcCacheUpdateGetWorkspaceSize(const mhcTensor *pageTable, const mhcTensor *lengths, const mhcTensor *parents,
                                   const mhcTensor *counts, int64_t pages, int64_t pageSize, const mhcTensor *newTable,
                                   const mhcTensor *newLengths, const mhcTensor *slots, const mhcTensor *granted,
                                   const mhcTensor *src, const mhcTensor *dst, uint64_t *workspaceSize,
                                   mhcServeExecutor **executor)
{
    if (slots == nullptr || workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    int st = table_limits(pageTable, lengths, pages, pageSize);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t R = pageTable->dims[0], W = pageTable->dims[1];
    if (slots->ndim != 2 || slots->dims[1] < 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    const int64_t tokens = slots->dims[1];
    if (tokens > kMaxCount / 2) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    st = first_of({check_dense(parents, {MHC_DTYPE_INT32}, {R}), check_dense(counts, {MHC_DTYPE_INT32}, {R}),
                   check_dense(newTable, {MHC_DTYPE_INT32}, {R, W}), check_dense(newLengths, {MHC_DTYPE_INT32}, {R}),
                   check_dense(slots, {MHC_DTYPE_INT64}, {R, tokens}), check_dense(granted, {MHC_DTYPE_INT32}, {R}),
                   check_dense(src, {MHC_DTYPE_INT32}, {R}), check_dense(dst, {MHC_DTYPE_INT32}, {R})});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kUpdate;
    ex->empty = R == 0;
    ex->update = {static_cast<int>(R),
                  static_cast<int>(W),
                  static_cast<int>(tokens),
                  pages,
                  static_cast<int>(pageSize),
                  static_cast<const int32_t *>(pageTable->data),
                  static_cast<const int32_t *>(lengths->data),
                  static_cast<const int32_t *>(parents->data),
                  static_cast<const int32_t *>(counts->data),
                  static_cast<int32_t *>(newTable->data),
                  static_cast<int32_t *>(newLengths->data),
                  static_cast<int32_t *>(granted->data),
                  static_cast<int32_t *>(src->data),
                  static_cast<int32_t *>(dst->data),
                  static_cast<int64_t *>(slots->data)};
    return finish(ex, pageTable->data, workspaceSize, executor);
}

int mhcCacheUpdate(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kUpdate, workspace, workspaceSize, executor, stream);
}

int mhcCacheCompactGetWorkspaceSize(const mhcTensor *pageTable, const mhcTensor *lengths, int64_t pages,
                                    int64_t pageSize, const mhcTensor *newTable, const mhcTensor *src,
                                    const mhcTensor *dst, const mhcTensor *used, uint64_t *workspaceSize,
                                    mhcServeExecutor **executor)
{
    if (workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    int st = table_limits(pageTable, lengths, pages, pageSize);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t R = pageTable->dims[0], W = pageTable->dims[1];
    st = first_of({check_dense(newTable, {MHC_DTYPE_INT32}, {R, W}), check_dense(src, {MHC_DTYPE_INT32}, {pages / 2}),
                   check_dense(dst, {MHC_DTYPE_INT32}, {pages / 2}), check_dense(used, {MHC_DTYPE_INT32}, {1})});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kCompact;
    ex->compact = {static_cast<int>(R),
                   static_cast<int>(W),
                   pages,
                   static_cast<int>(pageSize),
                   static_cast<const int32_t *>(pageTable->data),
                   static_cast<const int32_t *>(lengths->data),
                   static_cast<int32_t *>(newTable->data),
                   static_cast<int32_t *>(src->data),
                   static_cast<int32_t *>(dst->data),
                   static_cast<int32_t *>(used->data)};
    return finish(ex, used->data, workspaceSize, executor);
}

int mhcCacheCompact(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kCompact, workspace, workspaceSize, executor, stream);
}

int mhcCacheCopyPagesGetWorkspaceSize(const mhcStridedTensor *kCache, const mhcStridedTensor *vCache,
                                      const mhcTensor *src, const mhcTensor *dst, uint64_t *workspaceSize,
                                      mhcServeExecutor **executor)
{
    if (vCache == nullptr || src == nullptr || dst == nullptr || workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    int st = cache_limits(kCache);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    if (src->ndim != 1 || src->dims[0] < 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    const int64_t pages = kCache->dims[0], pageSize = kCache->dims[1], kvHeads = kCache->dims[2], d = kCache->dims[3];
    const int64_t n = src->dims[0];
    const int size = elem_bytes(kCache->dtype);
    if (n > kMaxCount || d > (1 << 16) || kvHeads > 65536) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    st = first_of({check_strided(kCache, kCache->dtype, {pages, pageSize, kvHeads, d}, size > 0 ? size : 2),
                   check_strided(vCache, kCache->dtype, {pages, pageSize, kvHeads, d}, size > 0 ? size : 2),
                   check_dense(src, {MHC_DTYPE_INT32}, {n}), check_dense(dst, {MHC_DTYPE_INT32}, {n})});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kCopy;
    ex->empty = n == 0;
    ex->copy = {cache_rows(kCache),
                cache_rows(vCache),
                pages,
                static_cast<int>(pageSize),
                static_cast<int>(kvHeads),
                static_cast<int>(d) * size,
                size,
                n,
                static_cast<const int32_t *>(src->data),
                static_cast<const int32_t *>(dst->data)};
    return finish(ex, kCache->data, workspaceSize, executor);
}

int mhcCacheCopyPages(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kCopy, workspace, workspaceSize, executor, stream);
}

int mhcDraftAttentionGetWorkspaceSize(const mhcStridedTensor *q, const mhcStridedTensor *kCache,
                                      const mhcStridedTensor *vCache, const mhcTensor *pageTable,
                                      const mhcTensor *lengths, const mhcTensor *drafted, const mhcTensor *parents,
                                      float scale, int64_t window, const mhcStridedTensor *out, const mhcTensor *lse,
                                      uint64_t *workspaceSize, mhcServeExecutor **executor)
{
    if (q == nullptr || out == nullptr || vCache == nullptr || workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    int st = cache_limits(kCache);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t pages = kCache->dims[0], pageSize = kCache->dims[1], kvHeads = kCache->dims[2], d = kCache->dims[3];
    if (q->ndim != 4 || window < 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (q->dtype != MHC_DTYPE_FLOAT16 && q->dtype != MHC_DTYPE_BF16) {
        return MHC_STATUS_INVALID_DTYPE;
    }
    const int64_t B = q->dims[0], S = q->dims[1], heads = q->dims[2];
    if (B < 0 || S < 0 || heads < 1 || heads % kvHeads != 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if ((st = table_limits(pageTable, lengths, pages, pageSize)) != MHC_STATUS_SUCCESS) {
        return st;
    }
    if (pageTable->dims[0] != B) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (!mhc::paged_attention_head_size(d) || heads > 65536 || B > (1 << 20) || S > (1 << 20) ||
        (parents != nullptr && S > mhc::kDraftNodes)) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    st = first_of(
        {check_strided(q, q->dtype, {B, S, heads, d}, 16), check_strided(out, q->dtype, {B, S, heads, d}, 16),
         check_strided(kCache, q->dtype, {pages, pageSize, kvHeads, d}, 16),
         check_strided(vCache, q->dtype, {pages, pageSize, kvHeads, d}, 16),
         check_dense(drafted, {MHC_DTYPE_INT32}, {B}),
         parents != nullptr ? check_dense(parents, {MHC_DTYPE_INT32}, {B, S}) : MHC_STATUS_SUCCESS,
         lse != nullptr ? check_dense(lse, {MHC_DTYPE_FLOAT}, {B, S, heads}) : MHC_STATUS_SUCCESS});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kDraft;
    ex->empty = B == 0 || S == 0;
    ex->draft = mhc::DraftAttentionArgs{};
    mhc::DraftAttentionArgs &a = ex->draft;
    a.isBf16 = q->dtype == MHC_DTYPE_BF16;
    a.B = static_cast<int>(B);
    a.S = static_cast<int>(S);
    a.heads = static_cast<int>(heads);
    a.kvHeads = static_cast<int>(kvHeads);
    a.d = static_cast<int>(d);
    a.q = token_rows(q);
    a.out = token_rows(out);
    a.kCache = cache_rows(kCache);
    a.vCache = cache_rows(vCache);
    a.pages = pages;
    a.pageSize = static_cast<int>(pageSize);
    a.width = static_cast<int>(pageTable->dims[1]);
    a.table = static_cast<const int32_t *>(pageTable->data);
    a.lengths = static_cast<const int32_t *>(lengths->data);
    a.drafted = static_cast<const int32_t *>(drafted->data);
    a.parents = parents != nullptr ? static_cast<const int32_t *>(parents->data) : nullptr;
    a.scale = scale;
    a.window = window;
    a.lse = lse != nullptr ? static_cast<float *>(lse->data) : nullptr;
    if (!ex->empty && !mhc::draft_attention_units_fit(a)) {
        delete ex;
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    return finish(ex, q->data, workspaceSize, executor);
}

int mhcDraftAttention(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kDraft, workspace, workspaceSize, executor, stream);
}

int mhcDraftAcceptGetWorkspaceSize(const mhcTensor *tokens, const mhcTensor *parents, const mhcTensor *drafted,
                                   const mhcTensor *chosen, const mhcTensor *lengths, const mhcTensor *path,
                                   const mhcTensor *accepted, const mhcTensor *next, const mhcTensor *newLengths,
                                   uint64_t *workspaceSize, mhcServeExecutor **executor)
{
    if (tokens == nullptr || workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    if (tokens->ndim != 2 || tokens->dims[0] < 0 || tokens->dims[1] < 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    const int64_t B = tokens->dims[0], S = tokens->dims[1];
    if (B > kMaxTableRows || S > mhc::kDraftNodes) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    const int32_t type = tokens->dtype;
    const int st = first_of(
        {check_dense(tokens, {MHC_DTYPE_INT32, MHC_DTYPE_INT64}, {B, S}), check_dense(chosen, {type}, {B, S}),
         parents != nullptr ? check_dense(parents, {MHC_DTYPE_INT32}, {B, S}) : MHC_STATUS_SUCCESS,
         check_dense(drafted, {MHC_DTYPE_INT32}, {B}), check_dense(lengths, {MHC_DTYPE_INT32}, {B}),
         check_dense(path, {MHC_DTYPE_INT32}, {B, S}), check_dense(accepted, {MHC_DTYPE_INT32}, {B}),
         check_dense(next, {type}, {B}), check_dense(newLengths, {MHC_DTYPE_INT32}, {B})});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kAccept;
    ex->empty = B == 0;
    ex->accept = {static_cast<int>(B),
                  static_cast<int>(S),
                  type == MHC_DTYPE_INT64,
                  tokens->data,
                  chosen->data,
                  parents != nullptr ? static_cast<const int32_t *>(parents->data) : nullptr,
                  static_cast<const int32_t *>(drafted->data),
                  static_cast<const int32_t *>(lengths->data),
                  static_cast<int32_t *>(path->data),
                  static_cast<int32_t *>(accepted->data),
                  static_cast<int32_t *>(newLengths->data),
                  next->data};
    return finish(ex, accepted->data, workspaceSize, executor);
}

int mhcDraftAccept(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kAccept, workspace, workspaceSize, executor, stream);
}

int mhcCacheKeepGetWorkspaceSize(const mhcStridedTensor *kCache, const mhcStridedTensor *vCache,
                                 const mhcTensor *pageTable, const mhcTensor *lengths, const mhcTensor *drafted,
                                 const mhcTensor *path, uint64_t *workspaceSize, mhcServeExecutor **executor)
{
    if (vCache == nullptr || path == nullptr || workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    int st = cache_limits(kCache);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t pages = kCache->dims[0], pageSize = kCache->dims[1], kvHeads = kCache->dims[2], d = kCache->dims[3];
    if (path->ndim != 2 || path->dims[1] < 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if ((st = table_limits(pageTable, lengths, pages, pageSize)) != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t B = pageTable->dims[0], S = path->dims[1];
    const int size = elem_bytes(kCache->dtype);
    if (S > (1 << 30) || d > (1 << 16) || kvHeads > 65536 || kvHeads * d > kMaxCount) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    st = first_of({check_strided(kCache, kCache->dtype, {pages, pageSize, kvHeads, d}, size > 0 ? size : 2),
                   check_strided(vCache, kCache->dtype, {pages, pageSize, kvHeads, d}, size > 0 ? size : 2),
                   check_dense(drafted, {MHC_DTYPE_INT32}, {B}), check_dense(path, {MHC_DTYPE_INT32}, {B, S})});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kKeep;
    ex->empty = B == 0 || S == 0;
    const mhc::CacheRows k = cache_rows(kCache), v = cache_rows(vCache);
    const bool one = k.data == v.data && k.page == v.page && k.slot == v.slot && k.head == v.head;
    ex->keep = {k,
                v,
                one ? 1 : 2,
                pages,
                static_cast<int>(pageSize),
                static_cast<int>(pageTable->dims[1]),
                static_cast<int>(kvHeads),
                static_cast<int>(d) * size,
                size,
                static_cast<int>(B),
                static_cast<int>(S),
                static_cast<const int32_t *>(pageTable->data),
                static_cast<const int32_t *>(lengths->data),
                static_cast<const int32_t *>(drafted->data),
                static_cast<const int32_t *>(path->data)};
    return finish(ex, kCache->data, workspaceSize, executor);
}

int mhcCacheKeep(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kKeep, workspace, workspaceSize, executor, stream);
}

int mhcCacheBoundsGetWorkspaceSize(const mhcStridedTensor *kCache, const mhcTensor *pageTable, const mhcTensor *lengths,
                                   const mhcTensor *counts, int64_t tokens, const mhcStridedTensor *lo,
                                   const mhcStridedTensor *hi, uint64_t *workspaceSize, mhcServeExecutor **executor)
{
    if (lo == nullptr || hi == nullptr || workspaceSize == nullptr || executor == nullptr) {
        return MHC_STATUS_NULL_ARGUMENT;
    }
    int st = cache_limits(kCache);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t pages = kCache->dims[0], pageSize = kCache->dims[1], kvHeads = kCache->dims[2], d = kCache->dims[3];
    if (kCache->dtype != MHC_DTYPE_FLOAT16 && kCache->dtype != MHC_DTYPE_BF16) {
        return MHC_STATUS_INVALID_DTYPE;
    }
    if ((st = table_limits(pageTable, lengths, pages, pageSize)) != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t B = pageTable->dims[0];
    if (tokens < 0) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (!mhc::paged_attention_head_size(d) || kvHeads > 65536) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    st = first_of({check_strided(kCache, kCache->dtype, {pages, pageSize, kvHeads, d}, 16),
                   check_strided(lo, kCache->dtype, {pages, kvHeads, d}, 16),
                   check_strided(hi, kCache->dtype, {pages, kvHeads, d}, 16),
                   check_dense(counts, {MHC_DTYPE_INT32}, {B})});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kBounds;
    ex->empty = B == 0 || tokens == 0;
    ex->bounds = mhc::CacheBoundsArgs{};
    mhc::CacheBoundsArgs &a = ex->bounds;
    a.isBf16 = kCache->dtype == MHC_DTYPE_BF16;
    a.B = static_cast<int>(B);
    a.kvHeads = static_cast<int>(kvHeads);
    a.d = static_cast<int>(d);
    a.k = cache_rows(kCache);
    a.lo = head_rows(lo);
    a.hi = head_rows(hi);
    a.pages = pages;
    a.pageSize = static_cast<int>(pageSize);
    a.width = static_cast<int>(pageTable->dims[1]);
    a.tokens = static_cast<int>(tokens < kMaxCount ? tokens : kMaxCount);
    a.table = static_cast<const int32_t *>(pageTable->data);
    a.lengths = static_cast<const int32_t *>(lengths->data);
    a.counts = static_cast<const int32_t *>(counts->data);
    return finish(ex, kCache->data, workspaceSize, executor);
}

int mhcCacheBounds(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kBounds, workspace, workspaceSize, executor, stream);
}

int mhcSparseAttentionGetWorkspaceSize(const mhcStridedTensor *q, const mhcStridedTensor *kCache,
                                       const mhcStridedTensor *vCache, const mhcStridedTensor *lo,
                                       const mhcStridedTensor *hi, const mhcTensor *pageTable,
                                       const mhcTensor *lengths, int64_t top, int64_t first, int64_t last, float scale,
                                       const mhcStridedTensor *out, const mhcTensor *lse, const mhcTensor *columns,
                                       uint64_t *workspaceSize, mhcServeExecutor **executor)
{
    mhc::SparseAttentionArgs s{};
    int st = attention_args(q, kCache, vCache, pageTable, lengths, scale, 0, out, lse, workspaceSize, executor,
                            s.attention);
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    const int64_t pages = kCache->dims[0], kvHeads = kCache->dims[2], d = kCache->dims[3], B = q->dims[0];
    if (first < 0 || last < 0 || top < 1 || first > top || last > top - first) {
        return MHC_STATUS_INVALID_SHAPE;
    }
    if (top > kMaxCount / kCache->dims[1]) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    st = first_of({check_strided(lo, q->dtype, {pages, kvHeads, d}, 16), check_strided(hi, q->dtype, {pages, kvHeads, d}, 16),
                   check_dense(columns, {MHC_DTYPE_INT32}, {B, kvHeads, top})});
    if (st != MHC_STATUS_SUCCESS) {
        return st;
    }
    s.lo = head_rows(lo);
    s.hi = head_rows(hi);
    s.top = static_cast<int>(top);
    s.first = static_cast<int>(first);
    s.last = static_cast<int>(last);
    s.columns = static_cast<int32_t *>(columns->data);
    if (!mhc::sparse_attention_fits(s)) {
        return MHC_STATUS_UNSUPPORTED_SHAPE;
    }
    mhcServeExecutor *ex = new (std::nothrow) mhcServeExecutor;
    if (ex == nullptr) {
        return MHC_STATUS_HIP_ERROR;
    }
    ex->op = Op::kSparse;
    ex->empty = B == 0;
    ex->sparse = s;
    return finish(ex, q->data, workspaceSize, executor);
}

int mhcSparseAttention(void *workspace, uint64_t workspaceSize, mhcServeExecutor *executor, hipStream_t stream)
{
    return launch(Op::kSparse, workspace, workspaceSize, executor, stream);
}

}  // extern "C"
