// linear_bf16.hip -- the dense layers' kernels for bf16.
#include "linear_kernels.hpp"

namespace tg {

TG_LINEAR_OF(bf16)

}  // namespace tg
