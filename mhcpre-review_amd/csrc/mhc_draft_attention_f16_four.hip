#include "mhc_draft_attention.h"

namespace mhc {
namespace draft {

template <>
hipError_t launch_kind<false, Kind::kFour>(const Args &args, hipStream_t stream)
{
    return with_size<Kind::kFour>(args.a.d, [&](auto l) { return launch_layout<false, decltype(l)>(args, stream); });
}

}  // namespace draft
}  // namespace mhc
