// gsr_linear_bf16.hip -- the bfloat16 products of gsr_linear.hip (gsr_product.h, gsr_strip.h).
#include "gsr_strip.h"

namespace gsr {
GSR_PRODUCTS(__hip_bfloat16)
}
