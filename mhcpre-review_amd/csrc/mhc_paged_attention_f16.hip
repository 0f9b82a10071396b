// mhcPagedAttention in fp16.

#include "mhc_paged_attention.h"

namespace mhc {
namespace attention {

hipError_t launch_f16(const Args &args, bool wide, hipStream_t stream)
{
    return wide ? launch_heads<false, 2>(args, stream) : launch_heads<false, 1>(args, stream);
}

}  // namespace attention
}  // namespace mhc
