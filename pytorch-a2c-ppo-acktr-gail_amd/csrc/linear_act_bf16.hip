// linear_act.hip's products on bf16 operands.
#include "linear_act_kernels.hpp"

namespace acktr {
template int linear_product<__bf16>(LinKind, const LinArgs&, float*, hipStream_t);
template int linear_gradients<__bf16>(LinArgs, LinArgs, float*, hipStream_t);
template int linear_bias<__bf16>(const LinArgs&, hipStream_t);
}
