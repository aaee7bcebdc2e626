// draws from rows of float logits
#include "kernels_draw.h"

namespace bn_draw {

hipError_t launch_f32(const Draws& a, hipStream_t s) { return launch<float>(a, s); }

}  // namespace bn_draw
