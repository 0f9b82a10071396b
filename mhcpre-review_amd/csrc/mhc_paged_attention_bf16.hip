// mhcPagedAttention in bf16, and its host side.

#include "mhc_paged_attention.h"

namespace mhc {
namespace attention {

hipError_t launch_bf16(const Args &args, bool wide, hipStream_t stream)
{
    return wide ? launch_heads<true, 2>(args, stream) : launch_heads<true, 1>(args, stream);
}

namespace {

Args plan(const PagedAttentionArgs &a, int cus, bool &wide)
{
    Args p{};
    p.a = a;
    p.group = a.heads / a.kvHeads;
    // 32 query heads at a time where the registers hold them: d = 256 spills, and reading the
    // cache once for each 16 heads is faster (64 rows of 8192, 32 heads to one: 285 us
    // against 166).
    wide = p.group > 16 && a.d <= kWideMost;
    p.blocks = (p.group + (wide ? 31 : 15)) / (wide ? 32 : 16);
    p.most = cus * workgroups_per_cu(a.d, wide);
    p.most = p.most < kMaxExchangeGrid ? p.most : kMaxExchangeGrid;
    return p;
}

}  // namespace
}  // namespace attention

bool paged_attention_head_size(int64_t d)
{
    return d == 32 || d == 64 || d == 80 || d == 96 || d == 112 || d == 128 || d == 160 || d == 192 || d == 256;
}

bool paged_attention_units_fit(const PagedAttentionArgs &a)
{
    bool wide;
    const attention::Args p = attention::plan(a, 1, wide);
    const int64_t units = (int64_t)a.width * a.pageSize / attention::kUnit + 2;
    int64_t all;
    return !__builtin_mul_overflow(units, (int64_t)a.B * a.kvHeads * p.blocks, &all) && all < INT32_MAX;
}

size_t paged_attention_workspace(const PagedAttentionArgs &a, int cus)
{
    bool wide;
    const attention::Args p = attention::plan(a, cus, wide);
    return kWsHeaderBytes + (size_t)2 * p.most * ((wide ? 32 : 16) * (a.d + 2) * 4 + 8);
}

hipError_t launch_paged_attention(const PagedAttentionArgs &a, void *workspace, int device, int cus,
                                  hipStream_t stream)
{
    bool wide;
    attention::Args p = attention::plan(a, cus, wide);
    p.parts = static_cast<char *>(workspace) + kWsHeaderBytes;
    const hipError_t err = make_launch_tag(next_launch_id(), device, p.most, workspace, stream, p.tag);
    if (err != hipSuccess) {
        return err;
    }
    return a.isBf16 ? attention::launch_bf16(p, wide, stream) : attention::launch_f16(p, wide, stream);
}

}  // namespace mhc
