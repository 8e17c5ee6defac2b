// losses_f32.hip -- the losses' kernels for float.
#include "losses_kernels.hpp"

namespace tg {

TG_LOSSES_OF(float)

}  // namespace tg
