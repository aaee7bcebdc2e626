// draws from rows of __half logits
#include "kernels_draw.h"

namespace bn_draw {

hipError_t launch_f16(const Draws& a, hipStream_t s) { return launch<__half>(a, s); }

}  // namespace bn_draw
