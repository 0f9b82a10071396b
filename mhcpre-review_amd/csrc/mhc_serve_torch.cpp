// PyTorch operators over the serving operators' C ABI (include/mhc_serve.h):
//   torch.ops.mhcpre.qk_norm_rope, qk_norm_rope_append, paged_attention,
//   cache_update, cache_compact, cache_copy_pages
//
// Each call runs phase 1 on the given tensors, takes outputs and workspace
// from PyTorch's caching allocator and launches on the current stream.  The
// library's status codes come back as errors naming the status.  Only device
// tensors have a kernel; the shape-only implementations for tracing are
// registered from Python.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <cmath>

#include "mhc_serve.h"

namespace {

int32_t dtype_code(at::ScalarType t)
{
    switch (t) {
    case at::kFloat:
        return MHC_DTYPE_FLOAT;
    case at::kHalf:
        return MHC_DTYPE_FLOAT16;
    case at::kBFloat16:
        return MHC_DTYPE_BF16;
    case at::kInt:
        return MHC_DTYPE_INT32;
    case at::kLong:
        return MHC_DTYPE_INT64;
    case at::kDouble:
        return MHC_DTYPE_DOUBLE;
    default:
        return -1;  // the library rejects it with MHC_STATUS_INVALID_DTYPE
    }
}

mhcTensor dense(const at::Tensor &t)
{
    mhcTensor d{};
    d.data = t.data_ptr();
    d.dtype = dtype_code(t.scalar_type());
    TORCH_CHECK(t.dim() <= MHC_MAX_DIMS, "mhcpre: tensor of rank ", t.dim());
    d.ndim = static_cast<int32_t>(t.dim());
    for (int64_t i = 0; i < t.dim(); ++i) {
        d.dims[i] = t.size(i);
    }
    return d;
}

mhcStridedTensor strided(const at::Tensor &t)
{
    mhcStridedTensor d{};
    d.data = t.data_ptr();
    d.dtype = dtype_code(t.scalar_type());
    TORCH_CHECK(t.dim() <= MHC_MAX_DIMS, "mhcpre: tensor of rank ", t.dim());
    d.ndim = static_cast<int32_t>(t.dim());
    for (int64_t i = 0; i < t.dim(); ++i) {
        d.dims[i] = t.size(i);
        d.strides[i] = t.stride(i);
    }
    return d;
}

[[noreturn]] void fail(const char *where, int status)
{
    TORCH_CHECK(false, where, " failed: ", mhcPreStatusString(status), " (", status, ")");
}

struct ExecutorOwner {
    mhcServeExecutor *exe = nullptr;
    ~ExecutorOwner()
    {
        if (exe != nullptr) {
            mhcServeExecutorDestroy(exe);
        }
    }
};

using Launch = int (*)(void *, uint64_t, mhcServeExecutor *, hipStream_t);

// Phase 2 on the current stream of `like`'s device.  The workspace goes back to
// the caching allocator in that stream's order.
void enqueue(const char *phase1, int status, const char *phase2, Launch launch, const ExecutorOwner &owner,
             uint64_t bytes, const at::Tensor &like)
{
    if (status != MHC_STATUS_SUCCESS) {
        fail(phase1, status);
    }
    at::Tensor ws;
    if (bytes > 0) {
        ws = at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
    }
    hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(like.device().index()).stream();
    const int rc = launch(bytes > 0 ? ws.data_ptr() : nullptr, bytes, owner.exe, stream);
    if (rc != MHC_STATUS_SUCCESS) {
        fail(phase2, rc);
    }
}

void same_device(const at::Tensor &like, std::initializer_list<const at::Tensor *> others)
{
    TORCH_CHECK(like.is_cuda(), "mhcpre: tensors must be on a device");
    for (const at::Tensor *t : others) {
        TORCH_CHECK(t->device() == like.device(), "mhcpre: tensors on ", t->device(), " and ", like.device());
    }
}

// x [..., heads, d] as [rows, heads, d]: a view where the leading dimensions
// are one, d is contiguous, and (align > 1) rows and heads start at multiples
// of `align` elements; else a copy.
at::Tensor head_rows(const at::Tensor &x, const char *name, int64_t align = 1)
{
    TORCH_CHECK(x.dim() >= 2, "mhcpre: ", name, " must be [..., heads, d]");
    int64_t rows = 1;
    for (int64_t i = 0; i < x.dim() - 2; ++i) {
        rows *= x.size(i);
    }
    at::Tensor t = x.dim() == 3 ? x : x.reshape({rows, x.size(-2), x.size(-1)});
    const auto fits = [&](int64_t i) { return t.size(i) <= 1 || (t.stride(i) >= 0 && t.stride(i) % align == 0); };
    const bool whole = (t.size(2) <= 1 || t.stride(2) == 1) && fits(0) && fits(1) &&
                       reinterpret_cast<uintptr_t>(t.data_ptr()) % (align * t.element_size()) == 0;
    return whole ? t : t.clone(at::MemoryFormat::Contiguous);
}

at::Tensor flat(const at::Tensor &t) { return t.dim() == 1 ? t.contiguous() : t.reshape({t.numel()}).contiguous(); }

struct Rotary {
    at::Tensor positions, invFreq, qWeight, kWeight;
    mhcTensor dPositions{}, dFreq{}, dq{}, dk{};

    Rotary(const at::Tensor &q, const at::Tensor &positions_, const std::optional<at::Tensor> &invFreq_,
           const std::optional<at::Tensor> &qWeight_, const std::optional<at::Tensor> &kWeight_)
        : positions(flat(positions_))
    {
        same_device(q, {&positions});
        dPositions = dense(positions);
        take(q, invFreq_, invFreq, dFreq);
        take(q, qWeight_, qWeight, dq);
        take(q, kWeight_, kWeight, dk);
    }
    static void take(const at::Tensor &q, const std::optional<at::Tensor> &from, at::Tensor &to, mhcTensor &desc)
    {
        if (from.has_value() && from->defined()) {
            same_device(q, {&*from});
            to = flat(*from);
            desc = dense(to);
        }
    }
    const mhcTensor *freq() const { return invFreq.defined() ? &dFreq : nullptr; }
    const mhcTensor *wq() const { return qWeight.defined() ? &dq : nullptr; }
    const mhcTensor *wk() const { return kWeight.defined() ? &dk : nullptr; }
};

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor &q_, const at::Tensor &k_, const at::Tensor &positions,
                                                const std::optional<at::Tensor> &invFreq,
                                                const std::optional<at::Tensor> &qWeight,
                                                const std::optional<at::Tensor> &kWeight, double eps, bool interleaved,
                                                double amplitude)
{
    same_device(q_, {&k_});
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(q_.device());
    const at::Tensor q = head_rows(q_, "q"), k = head_rows(k_, "k");
    const Rotary rot(q, positions, invFreq, qWeight, kWeight);
    at::Tensor qOut = at::empty(q.sizes(), q.options()), kOut = at::empty(k.sizes(), k.options());
    const mhcStridedTensor dq = strided(q), dk = strided(k), dqo = strided(qOut), dko = strided(kOut);
    uint64_t bytes = 0;
    ExecutorOwner owner;
    const int st = mhcQkNormRopeGetWorkspaceSize(
        &dq, &dk, nullptr, &rot.dPositions, rot.freq(), rot.wq(), rot.wk(), static_cast<float>(eps), interleaved,
        static_cast<float>(amplitude), nullptr, &dqo, &dko, nullptr, nullptr, &bytes, &owner.exe);
    enqueue("mhcQkNormRopeGetWorkspaceSize", st, "mhcQkNormRope", mhcQkNormRope, owner, bytes, q);
    return {q_.dim() == 3 ? qOut : qOut.view(q_.sizes()), k_.dim() == 3 ? kOut : kOut.view(k_.sizes())};
}

at::Tensor qk_norm_rope_append(const at::Tensor &q_, const at::Tensor &k_, const at::Tensor &v_,
                               const at::Tensor &positions, const std::optional<at::Tensor> &invFreq,
                               const at::Tensor &slots_, const at::Tensor &kCache, const at::Tensor &vCache,
                               const std::optional<at::Tensor> &qWeight, const std::optional<at::Tensor> &kWeight,
                               double eps, bool interleaved, double amplitude)
{
    same_device(q_, {&k_, &v_, &slots_, &kCache, &vCache});
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(q_.device());
    const at::Tensor q = head_rows(q_, "q"), k = head_rows(k_, "k"), v = head_rows(v_, "v"), slots = flat(slots_);
    const Rotary rot(q, positions, invFreq, qWeight, kWeight);
    at::Tensor qOut = at::empty(q.sizes(), q.options());
    const mhcStridedTensor dq = strided(q), dk = strided(k), dv = strided(v), dqo = strided(qOut),
                           dkc = strided(kCache), dvc = strided(vCache);
    const mhcTensor ds = dense(slots);
    uint64_t bytes = 0;
    ExecutorOwner owner;
    const int st = mhcQkNormRopeGetWorkspaceSize(
        &dq, &dk, &dv, &rot.dPositions, rot.freq(), rot.wq(), rot.wk(), static_cast<float>(eps), interleaved,
        static_cast<float>(amplitude), &ds, &dqo, nullptr, &dkc, &dvc, &bytes, &owner.exe);
    enqueue("mhcQkNormRopeGetWorkspaceSize", st, "mhcQkNormRope", mhcQkNormRope, owner, bytes, q);
    return q_.dim() == 3 ? qOut : qOut.view(q_.sizes());
}

std::tuple<at::Tensor, at::Tensor> paged_attention(const at::Tensor &q_, const at::Tensor &kCache,
                                                   const at::Tensor &vCache, const at::Tensor &pageTable_,
                                                   const at::Tensor &lengths_, std::optional<double> scale,
                                                   int64_t window)
{
    same_device(q_, {&kCache, &vCache, &pageTable_, &lengths_});
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(q_.device());
    const at::Tensor q = head_rows(q_, "q", 8), pageTable = pageTable_.contiguous(), lengths = flat(lengths_);
    at::Tensor out = at::empty(q.sizes(), q.options());
    at::Tensor lse = at::empty(q.sizes().slice(0, 2), q.options().dtype(at::kFloat));
    const mhcStridedTensor dq = strided(q), dkc = strided(kCache), dvc = strided(vCache), dout = strided(out);
    const mhcTensor dt = dense(pageTable), dl = dense(lengths), dlse = dense(lse);
    const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2)));
    uint64_t bytes = 0;
    ExecutorOwner owner;
    const int st = mhcPagedAttentionGetWorkspaceSize(&dq, &dkc, &dvc, &dt, &dl, static_cast<float>(s), window, &dout,
                                                     &dlse, &bytes, &owner.exe);
    enqueue("mhcPagedAttentionGetWorkspaceSize", st, "mhcPagedAttention", mhcPagedAttention, owner, bytes, q);
    if (q_.dim() == 3) {
        return {out, lse};
    }
    return {out.view(q_.sizes()), lse.view(q_.sizes().slice(0, q_.dim() - 1))};
}

using Six = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

Six cache_update(const at::Tensor &pageTable_, const at::Tensor &lengths_, const at::Tensor &parents_,
                 const at::Tensor &counts_, int64_t pages, int64_t pageSize, int64_t tokens)
{
    same_device(pageTable_, {&lengths_, &parents_, &counts_});
    TORCH_CHECK(pageTable_.dim() == 2, "mhcpre: page_table must be [rows, width]");
    TORCH_CHECK(tokens >= 0, "mhcpre: tokens ", tokens);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(pageTable_.device());
    const at::Tensor pageTable = pageTable_.contiguous(), lengths = flat(lengths_), parents = flat(parents_),
                     counts = flat(counts_);
    const auto i32 = pageTable.options().dtype(at::kInt);
    const int64_t rows = pageTable.size(0);
    at::Tensor newTable = at::empty(pageTable.sizes(), i32), newLengths = at::empty({rows}, i32),
               slots = at::empty({rows, tokens}, i32.dtype(at::kLong)), granted = at::empty({rows}, i32),
               src = at::empty({rows}, i32), dst = at::empty({rows}, i32);
    const mhcTensor dt = dense(pageTable), dl = dense(lengths), dp = dense(parents), dc = dense(counts),
                    dnt = dense(newTable), dnl = dense(newLengths), dsl = dense(slots), dg = dense(granted),
                    dsrc = dense(src), ddst = dense(dst);
    uint64_t bytes = 0;
    ExecutorOwner owner;
    const int st = mhcCacheUpdateGetWorkspaceSize(&dt, &dl, &dp, &dc, pages, pageSize, &dnt, &dnl, &dsl, &dg, &dsrc,
                                                  &ddst, &bytes, &owner.exe);
    enqueue("mhcCacheUpdateGetWorkspaceSize", st, "mhcCacheUpdate", mhcCacheUpdate, owner, bytes, pageTable);
    return {newTable, newLengths, slots, granted, src, dst};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> cache_compact(const at::Tensor &pageTable_,
                                                                         const at::Tensor &lengths_, int64_t pages,
                                                                         int64_t pageSize)
{
    same_device(pageTable_, {&lengths_});
    TORCH_CHECK(pages >= 1, "mhcpre: pages ", pages);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(pageTable_.device());
    const at::Tensor pageTable = pageTable_.contiguous(), lengths = flat(lengths_);
    const auto i32 = pageTable.options().dtype(at::kInt);
    at::Tensor newTable = at::empty(pageTable.sizes(), i32), src = at::empty({pages / 2}, i32),
               dst = at::empty({pages / 2}, i32), used = at::empty({1}, i32);
    const mhcTensor dt = dense(pageTable), dl = dense(lengths), dnt = dense(newTable), dsrc = dense(src),
                    ddst = dense(dst), du = dense(used);
    uint64_t bytes = 0;
    ExecutorOwner owner;
    const int st = mhcCacheCompactGetWorkspaceSize(&dt, &dl, pages, pageSize, &dnt, &dsrc, &ddst, &du, &bytes,
                                                   &owner.exe);
    enqueue("mhcCacheCompactGetWorkspaceSize", st, "mhcCacheCompact", mhcCacheCompact, owner, bytes, pageTable);
    return {newTable, src, dst, used};
}

void cache_copy_pages(const at::Tensor &kCache, const at::Tensor &vCache, const at::Tensor &src_,
                      const at::Tensor &dst_)
{
    same_device(kCache, {&vCache, &src_, &dst_});
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(kCache.device());
    const at::Tensor src = flat(src_), dst = flat(dst_);
    const mhcStridedTensor dk = strided(kCache), dv = strided(vCache);
    const mhcTensor ds = dense(src), dd = dense(dst);
    uint64_t bytes = 0;
    ExecutorOwner owner;
    const int st = mhcCacheCopyPagesGetWorkspaceSize(&dk, &dv, &ds, &dd, &bytes, &owner.exe);
    enqueue("mhcCacheCopyPagesGetWorkspaceSize", st, "mhcCacheCopyPages", mhcCacheCopyPages, owner, bytes, kCache);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mhcpre, m)
{
    m.def("qk_norm_rope(Tensor q, Tensor k, Tensor positions, Tensor? inv_freq, Tensor? q_weight=None, "
          "Tensor? k_weight=None, float eps=1e-06, bool interleaved=False, float amplitude=1.0) "
          "-> (Tensor, Tensor)");
    m.def("qk_norm_rope_append(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor? inv_freq, Tensor slots, "
          "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor? q_weight=None, Tensor? k_weight=None, "
          "float eps=1e-06, bool interleaved=False, float amplitude=1.0) -> Tensor");
    m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor lengths, "
          "float? scale=None, int window=0) -> (Tensor, Tensor)");
    m.def("cache_update(Tensor page_table, Tensor lengths, Tensor parents, Tensor counts, int pages, "
          "int page_size, int tokens=1) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("cache_compact(Tensor page_table, Tensor lengths, int pages, int page_size) "
          "-> (Tensor, Tensor, Tensor, Tensor)");
    m.def("cache_copy_pages(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor src, Tensor dst) -> ()");
}

TORCH_LIBRARY_IMPL(mhcpre, CUDA, m)
{
    m.impl("qk_norm_rope", &qk_norm_rope);
    m.impl("qk_norm_rope_append", &qk_norm_rope_append);
    m.impl("paged_attention", &paged_attention);
    m.impl("cache_update", &cache_update);
    m.impl("cache_compact", &cache_compact);
    m.impl("cache_copy_pages", &cache_copy_pages);
}
