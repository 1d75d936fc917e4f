// cbq_q4_attn.h's kernels for f16 queries.
#include "cbq_q4_attn.h"

namespace cbq_q4 {

int launch_f16(const AttnArgs &a, int hd, hipStream_t stream)
{
    return launch_hd<_Float16>(a, hd, stream);
}

}  // namespace cbq_q4
