// k_attn_masked_wide.hip — attention under masks for heads of 80 to 128 features (k_attn_masked.h)
#include "k_attn_masked.h"

namespace mgh {

hipError_t launch_attn_masked_wide(const MaskedAttnArgs& a, const MaskedPlan& p, hipStream_t s) {
    return a.D <= 96 ? launch_masked_d<6>(a, p, s) : launch_masked_d<8>(a, p, s);
}

}  // namespace mgh
