// losses_f16.hip -- the losses' kernels for f16.
#include "losses_kernels.hpp"

namespace tg {

TG_LOSSES_OF(f16)

}  // namespace tg
