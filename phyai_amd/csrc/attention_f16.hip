// Attention over 16-bit pages with half precision queries: prompts, shared keys, with and without a cap (attention.h).
#include "attention.h"

namespace phyai {

hipError_t launch_attention_f16(const PagedAttention& p, const AttentionPlan& plan, hipStream_t stream) {
    constexpr int MODE = MODE_MORE;
    if (p.cap > kWideCap) return launch_d<HEAD_F16, MODE | MODE_WIDE>(p, plan, stream);
    return p.cap > 0.f ? launch_d<HEAD_F16, MODE | MODE_CAP>(p, plan, stream) : launch_d<HEAD_F16, MODE>(p, plan, stream);
}

}  // namespace phyai
