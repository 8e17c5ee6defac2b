// linear_f32.hip -- the dense layers' kernels for float.
#include "linear_kernels.hpp"

namespace tg {

TG_LINEAR_OF(float)

}  // namespace tg
