// The grouped products' kernels for fp16 operands.
#include "products_launch.hpp"

namespace soapmi {
template int row_products<ElemF16, KC>(hipStream_t, const RowProblem&, bool);
template int row_products<ElemF16, XC>(hipStream_t, const RowProblem&, bool);
template int sum_products<ElemF16>(hipStream_t, const SumProblem&, bool);
}  // namespace soapmi
