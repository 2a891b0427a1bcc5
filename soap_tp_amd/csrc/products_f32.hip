// The grouped products' kernels for fp32 operands.
#include "products_launch.hpp"

namespace soapmi {
template int row_products<ElemF32, KC>(hipStream_t, const RowProblem&, bool);
template int row_products<ElemF32, XC>(hipStream_t, const RowProblem&, bool);
template int sum_products<ElemF32>(hipStream_t, const SumProblem&, bool);
}  // namespace soapmi
