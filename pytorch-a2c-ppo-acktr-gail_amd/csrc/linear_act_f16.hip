// linear_act.hip's products on fp16 operands.
#include "linear_act_kernels.hpp"

namespace acktr {
template int linear_product<_Float16>(LinKind, const LinArgs&, float*, hipStream_t);
template int linear_gradients<_Float16>(LinArgs, LinArgs, float*, hipStream_t);
template int linear_bias<_Float16>(const LinArgs&, hipStream_t);
}
