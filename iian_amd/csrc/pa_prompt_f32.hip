// pa_prompt_f32.hip - whole-prompt attention: F32 rows, as pairs of f16 terms (pa_prompt.h).
#include "pa_prompt.h"

namespace iian_pa {

hipError_t launch_prompt_f32(const PromptParams &p, hipStream_t stream) {
    const bool vec = prompt_vec<0>(p);
    const int d = std::max(p.D, p.Dv);
    // Small calls: 8 waves, which share a tile's conversion into f16 terms, KW of them their rows (one 700-token prompt,
    // H32/Hkv8/D128, 50 us, 61 with 4 waves that share by two); others two workgroups of 4 per CU, which do not wait for
    // each other, also up to 64 tokens, where joining costs more than the second tile (4 of 16 tokens 9 us, 11 with 8
    // waves).  Causal calls of longer prompts stay small up to twice as many workgroups as CUs, and three times for the
    // longest at head size 64: their last row blocks see the most tokens and are the call's critical path (H32/Hkv8/D128:
    // prompts of 1100 and 300 tokens 71 us, 91 with 4 waves, one of 2048 135 and 166; beyond, 3 of 1000 122 and 103; shorter,
    // 6 of 300 42 and 35; H14/Hkv2/D64: one of 3000 113 and 147, 3 of 1000 55 and 55).
    const bool causal = p.causal || p.row_end, joined = !prompt_short(p);
    if (vec && d <= 64) {
        if (joined && prompt_blocks(p, 64) <= kPromptCus * (!causal || p.max_q < 500 ? 1 : p.max_q < 1500 ? 2 : 3))
            return launch_prompt_k<0, 64, 64, true, 4, 8>(p, stream);
        return launch_prompt_k<0, 64, 64, true, 1, 4>(p, stream);
    }
    if (vec && d <= 128) {
        if (joined && prompt_blocks(p, 128) <= kPromptCus * (!causal || p.max_q < 500 ? 1 : 2))
            return launch_prompt_k<0, 128, 128, true, 2, 8>(p, stream);
        return launch_prompt_k<0, 128, 128, true, 1, 4>(p, stream);
    }
    if (vec) return launch_prompt_k<0, 256, 256, true, 1, 4>(p, stream);
    if (d <= 64) return launch_prompt_k<0, 64, 64, false, 1, 4>(p, stream);
    if (d <= 128) return launch_prompt_k<0, 128, 128, false, 1, 4>(p, stream);
    return launch_prompt_k<0, 256, 256, false, 1, 4>(p, stream);
}

}  // namespace iian_pa
