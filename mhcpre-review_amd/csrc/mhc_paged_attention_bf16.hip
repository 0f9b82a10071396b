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
    // 32 query heads at a time where there are as many and the registers hold them.
    wide = p.group > 16 && a.d <= kWideMost;
    p.blocks = (p.group + (wide ? 31 : 15)) / (wide ? 32 : 16);
    p.most = cus * workgroups_per_cu(a.d, wide);
    p.most = p.most < kMaxExchangeGrid ? p.most : kMaxExchangeGrid;
    return p;
}

// Whether no row has more than kShortKeys keys and there are enough (row, kv head,
// block)s for half of the waves: then each wave does its own.  us, workgroups / waves
// (8 kv heads of 128): 256 rows of 16 keys 20.9 / 8.7, 64 22.1 / 14.7, 256 57.2 / 51.6,
// 512 101.5 / 97.2, of 1 to 256 36.2 / 34.9, with a window of 128 32.1 / 27.9; 1024 rows
// of 32 72.3 / 34.5; but 64 rows (512 of them, a quarter of the waves) of 128 10.6 / 11.7,
// of 512 27.8 / 41.8.  The lengths are on the device, so the rule goes by the table: short
// rows in a table of a long context's width are shared out in units like long ones (256 rows
// of 16 keys, width 1 / 512 pages of 16: 7.8 / 20.4).
constexpr int64_t kShortKeys = 512;
bool short_rows(const PagedAttentionArgs &a, const Args &p, bool wide)
{
    int64_t keys = (int64_t)a.width * a.pageSize;
    keys = a.window > 0 && a.window < keys ? a.window : keys;
    return !wide && keys <= kShortKeys && (int64_t)a.B * a.kvHeads * p.blocks >= 2 * (int64_t)p.most;
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
    if (attention::short_rows(a, p, wide)) {
        return 0;
    }
    return kWsHeaderBytes + (size_t)2 * p.most * ((wide ? 32 : 16) * (a.d + 4) * 4 + 16);
}

hipError_t launch_paged_attention(const PagedAttentionArgs &a, void *workspace, int device, int cus,
                                  hipStream_t stream)
{
    bool wide;
    attention::Args p = attention::plan(a, cus, wide);
    if (attention::short_rows(a, p, wide)) {
        return a.isBf16 ? attention::launch_bf16(p, wide, stream) : attention::launch_f16(p, wide, stream);
    }
    p.parts = static_cast<char *>(workspace) + kWsHeaderBytes;
    const hipError_t err = make_launch_tag(next_launch_id(), device, p.most, workspace, stream, p.tag);
    if (err != hipSuccess) {
        return err;
    }
    return a.isBf16 ? attention::launch_bf16(p, wide, stream) : attention::launch_f16(p, wide, stream);
}

}  // namespace mhc
