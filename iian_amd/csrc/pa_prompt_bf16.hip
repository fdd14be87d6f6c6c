// pa_prompt_bf16.hip - whole-prompt attention: BF16 rows (pa_prompt.h).
#include "pa_prompt.h"

namespace iian_pa {

hipError_t launch_prompt_bf16(const PromptParams &p, hipStream_t stream) {
    const bool vec = prompt_vec<30>(p);
    const int d = std::max(p.D, p.Dv);
    if (d <= 64) return launch_prompt_d<30, 64, 64, true, true>(p, vec, stream);
    // (a fifth fewer products of Q and K than at 96: 6 images of 563 to 2100 tokens, H16/D80, 74 us, 76)
    if (d <= 96 && p.D <= 80) return launch_prompt_d<30, 80, 96, false, true>(p, vec, stream);
    if (d <= 96) return launch_prompt_d<30, 96, 96, false, true>(p, vec, stream);
    if (d <= 128) return launch_prompt_d<30, 128, 128, false, true>(p, vec, stream);
    return launch_prompt_d<30, 256, 256, false, true, true>(p, vec, stream);
}

}  // namespace iian_pa
