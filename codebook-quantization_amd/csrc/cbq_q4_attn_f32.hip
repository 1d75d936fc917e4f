// cbq_q4_attn.h's kernels for f32 queries.
#include "cbq_q4_attn.h"

namespace cbq_q4 {

int launch_f32(const AttnArgs &a, int hd, hipStream_t stream)
{
    return launch_hd<float>(a, hd, stream);
}

}  // namespace cbq_q4
