// pa_prompt.hip - whole-prompt attention: F16 rows, and the choice of the kernel (pa_prompt.h).
#include "pa_prompt.h"

namespace iian_pa {

hipError_t launch_prompt_f16(const PromptParams &p, hipStream_t stream) {
    const bool vec = prompt_vec<1>(p);
    const int d = std::max(p.D, p.Dv);
    if (d <= 64) return launch_prompt_d<1, 64, 64, true, true>(p, vec, stream);
    if (d <= 96 && p.D <= 80) return launch_prompt_d<1, 80, 96, false, true>(p, vec, stream);
    if (d <= 96) return launch_prompt_d<1, 96, 96, false, true>(p, vec, stream);
    if (d <= 128) return launch_prompt_d<1, 128, 128, false, true>(p, vec, stream);
    return launch_prompt_d<1, 256, 256, false, true, true>(p, vec, stream);
}

hipError_t launch_prompt(const PromptParams &p, int type, hipStream_t stream) {
    // (millions of tiny prompts would pass a launch's size)
    if (std::max(p.D, p.Dv) > 256 || prompt_blocks(p, 128) > kPromptMaxBlocks)
        return launch_prompt_rows(p, type, stream);
    switch (type) {
        case 0: return launch_prompt_f32(p, stream);
        case 1: return launch_prompt_f16(p, stream);
        case 30: return launch_prompt_bf16(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace iian_pa
