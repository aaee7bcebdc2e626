// draws from rows of __hip_bfloat16 logits
#include "kernels_draw.h"

namespace bn_draw {

hipError_t launch_bf16(const Draws& a, hipStream_t s) { return launch<__hip_bfloat16>(a, s); }

}  // namespace bn_draw
