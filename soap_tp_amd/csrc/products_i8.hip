// The grouped products' kernels for 8-bit integer operands.
#include "products_launch.hpp"

namespace soapmi {
template int row_products<ElemI8, KC>(hipStream_t, const RowProblem&, bool);
}  // namespace soapmi
