// losses_bf16.hip -- the losses' kernels for bf16.
#include "losses_kernels.hpp"

namespace tg {

TG_LOSSES_OF(bf16)

}  // namespace tg
