// Attention over selected pages in bf16: the kernels of mhc_paged_attention.h with a
// page table and a length for each kv head of a sequence.

#include "mhc_paged_attention.h"

namespace mhc {
namespace attention {

hipError_t launch_each_bf16(const Args &args, bool wide, hipStream_t stream)
{
    return wide ? launch_heads<true, 2, true>(args, stream) : launch_heads<true, 1, true>(args, stream);
}

}  // namespace attention
}  // namespace mhc
