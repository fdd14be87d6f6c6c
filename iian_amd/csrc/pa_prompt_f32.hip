// pa_prompt_f32.hip - whole-prompt attention: F32 rows, as pairs of f16 terms (pa_prompt.h).
#include "pa_prompt.h"

namespace iian_pa {

hipError_t launch_prompt_f32(const PromptParams &p, hipStream_t stream) {
    const bool vec = prompt_vec<0>(p);
    const int d = std::max(p.D, p.Dv);
    // Small calls: 8 waves, which share a tile's conversion into f16 terms, KW of them their rows (one 700-token prompt,
    // H32/Hkv8/D128, 50 us, 61 with 4 waves that share by two); others two workgroups of 4 per CU, which do not wait for
    // each other (one of 1500 128 us, 137 with 8 waves).
    if (vec && d <= 64) {
        if (prompt_blocks(p, 64) <= kPromptCus) return launch_prompt_k<0, 64, 64, true, 4, 8>(p, stream);
        return launch_prompt_k<0, 64, 64, true, 1, 4>(p, stream);
    }
    if (vec && d <= 128) {
        if (prompt_blocks(p, 128) <= kPromptCus) return launch_prompt_k<0, 128, 128, true, 2, 8>(p, stream);
        return launch_prompt_k<0, 128, 128, true, 1, 4>(p, stream);
    }
    if (vec) return launch_prompt_k<0, 256, 256, true, 1, 4>(p, stream);
    if (d <= 64) return launch_prompt_k<0, 64, 64, false, 1, 4>(p, stream);
    if (d <= 128) return launch_prompt_k<0, 128, 128, false, 1, 4>(p, stream);
    return launch_prompt_k<0, 256, 256, false, 1, 4>(p, stream);
}

}  // namespace iian_pa
