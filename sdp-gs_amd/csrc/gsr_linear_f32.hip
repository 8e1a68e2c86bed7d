// gsr_linear_f32.hip -- the 32-bit products of gsr_linear.hip (gsr_product.h, gsr_strip.h).
#include "gsr_strip.h"

namespace gsr {
GSR_PRODUCTS(float)
}
