// gsr_linear_f16.hip -- the 16-bit-float products of gsr_linear.hip (gsr_product.h, gsr_strip.h).
#include "gsr_strip.h"

namespace gsr {
GSR_PRODUCTS(__half)
}
