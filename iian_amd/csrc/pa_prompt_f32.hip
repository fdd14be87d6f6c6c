// pa_prompt_f32.hip - whole-prompt attention: F32 rows, as pairs of f16 terms (pa_prompt.h).
#include "pa_prompt.h"

namespace iian_pa {

hipError_t launch_prompt_f32(const PromptParams &p, hipStream_t stream) {
    const bool vec = prompt_vec<0>(p);
    const int d = std::max(p.D, p.Dv);
    if (d <= 64) return launch_prompt_d<0, 64, 64, true, true>(p, vec, stream);
    if (d <= 128) return launch_prompt_d<0, 128, 128, false, true>(p, vec, stream);
    return launch_prompt_d<0, 256, 256, false, false>(p, vec, stream);
}

}  // namespace iian_pa
