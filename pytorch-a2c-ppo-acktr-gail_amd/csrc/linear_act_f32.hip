// linear_act.hip's products on fp32 operands.
#include "linear_act_kernels.hpp"

namespace acktr {
template int linear_product<float>(LinKind, const LinArgs&, float*, hipStream_t);
template int linear_gradients<float>(LinArgs, LinArgs, float*, hipStream_t);
template int linear_bias<float>(const LinArgs&, hipStream_t);
}
