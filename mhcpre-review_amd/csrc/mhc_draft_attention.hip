// mhcDraftAttention's host side.

#include "mhc_draft_attention.h"

namespace mhc {
namespace draft {
namespace {

// The layout for rows of a (sequence, kv head): blocks that hold them, for smaller ones read the
// cache again and larger ones multiply rows that are not there.  us, 32 / 64 / 128 rows a block,
// 8 kv heads of 128: 32 rows, 32 sequences of 8192 212 / 219 / 274, 2 of 65536 82 / 86 / 92; 64
// rows, the same 355 / 222 / 259 and 124 / 90 / 95; 128 rows, 32 of 8192 608 / 349 / 287.  Blocks
// of 256 rows have one workgroup a CU; 128 / 256: 512 rows, 2 of 65536 322 / 297, 32 of up to 8192
// 321 / 317; 256 rows, 2 of 65536 178 / 167, 32 of up to 8192 with trees of different sizes 196 /
// 207.
Kind kind_of(const DraftAttentionArgs &a)
{
    const int64_t rows = (int64_t)a.S * (a.heads / a.kvHeads);
    const bool eight = rows > 256 && (padded(a.d) == 64 || padded(a.d) == 128);
    return rows <= 32 ? Kind::kOne : rows <= 64 ? Kind::kTwo : eight ? Kind::kEight : Kind::kFour;
}

template <Kind kKind>
void plan_kind(Args &p, int cus)
{
    with_size<kKind>(p.a.d, [&](auto l) {
        using L = decltype(l);
        p.rows = L::kBlock;
        p.unit = L::kUnit;
        p.most = cus * L::kPerCu;
        // (A page's rows by 32-bit offsets from a group's first one; d as wide as the layout, for
        // what lies behind a narrower row is not read.)
        const DraftAttentionArgs &a = p.a;
        p.grouped = a.pageSize % L::kGroupRows == 0 && a.d == L::D && a.kCache.page == a.vCache.page &&
                    a.kCache.slot == a.vCache.slot && a.kCache.slot < (1 << 24);
        return 0;
    });
}

Args plan(const DraftAttentionArgs &a, int cus)
{
    Args p{};
    p.a = a;
    p.group = a.heads / a.kvHeads;
    switch (kind_of(a)) {
    case Kind::kOne: plan_kind<Kind::kOne>(p, cus); break;
    case Kind::kTwo: plan_kind<Kind::kTwo>(p, cus); break;
    case Kind::kFour: plan_kind<Kind::kFour>(p, cus); break;
    case Kind::kEight: plan_kind<Kind::kEight>(p, cus); break;
    }
    p.blocks = (int)(((int64_t)a.S * p.group + p.rows - 1) / p.rows);
    return p;
}

}  // namespace
}  // namespace draft

bool draft_attention_units_fit(const DraftAttentionArgs &a)
{
    const int64_t blocks = ((int64_t)a.S * (a.heads / a.kvHeads) + draft::kRows - 1) / draft::kRows;
    const int64_t units = (int64_t)a.width * a.pageSize / 32 + 2 + draft::kItemUnits;
    int64_t all;
    return blocks <= (1 << 25) && !__builtin_mul_overflow(units, blocks, &all) && !__builtin_mul_overflow(all, (int64_t)a.B * a.kvHeads, &all) &&
           all < INT32_MAX;
}

size_t draft_attention_workspace(const DraftAttentionArgs &a, int cus)
{
    const draft::Args p = draft::plan(a, cus);
    return (size_t)2 * p.most * p.rows * (draft::padded(a.d) + 2) * 4 + p.most * sizeof(draft::Open);
}

hipError_t launch_draft_attention(const DraftAttentionArgs &a, void *workspace, int cus, hipStream_t stream)
{
    draft::Args p = draft::plan(a, cus);
    p.outs = static_cast<float *>(workspace);
    p.ends = p.outs + (size_t)2 * p.most * p.rows * draft::padded(a.d);
    p.open = reinterpret_cast<draft::Open *>(p.ends + (size_t)2 * p.most * p.rows * 2);
    switch (draft::kind_of(a)) {
    case draft::Kind::kOne:
        return a.isBf16 ? draft::launch_kind<true, draft::Kind::kOne>(p, stream)
                        : draft::launch_kind<false, draft::Kind::kOne>(p, stream);
    case draft::Kind::kTwo:
        return a.isBf16 ? draft::launch_kind<true, draft::Kind::kTwo>(p, stream)
                        : draft::launch_kind<false, draft::Kind::kTwo>(p, stream);
    case draft::Kind::kFour:
        return a.isBf16 ? draft::launch_kind<true, draft::Kind::kFour>(p, stream)
                        : draft::launch_kind<false, draft::Kind::kFour>(p, stream);
    default:
        return a.isBf16 ? draft::launch_kind<true, draft::Kind::kEight>(p, stream)
                        : draft::launch_kind<false, draft::Kind::kEight>(p, stream);
    }
}

}  // namespace mhc
