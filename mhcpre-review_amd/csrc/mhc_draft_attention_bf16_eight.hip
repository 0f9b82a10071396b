#include "mhc_draft_attention.h"

namespace mhc {
namespace draft {

template <>
hipError_t launch_kind<true, Kind::kEight>(const Args &args, hipStream_t stream)
{
    return with_size<Kind::kEight>(args.a.d, [&](auto l) { return launch_layout<true, decltype(l)>(args, stream); });
}

}  // namespace draft
}  // namespace mhc
