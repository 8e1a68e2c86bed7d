// gsr_linear_f32.hip -- the 32-bit products of gsr_linear.hip (gsr_product.h).
#include "gsr_product.h"

namespace gsr {
GSR_PRODUCTS(float)
}
