// cbq_prefix_attn.h's kernels for bf16 caches.
#include "cbq_prefix_attn.h"

namespace cbq_attn {

int launch_bf16(const AttnArgs &a, const Plan &p, bool prompt, hipStream_t stream)
{
    return launch_hd<__bf16>(a, p, prompt, stream);
}

}  // namespace cbq_attn
