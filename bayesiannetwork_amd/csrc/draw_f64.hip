// draws from rows of double logits
#include "kernels_draw.h"

namespace bn_draw {

hipError_t launch_f64(const Draws& a, hipStream_t s) { return launch<double>(a, s); }

}  // namespace bn_draw
