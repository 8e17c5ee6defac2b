// linear_f16.hip -- the dense layers' kernels for f16.
#include "linear_kernels.hpp"

namespace tg {

TG_LINEAR_OF(f16)

}  // namespace tg
