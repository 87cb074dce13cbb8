// The forward kernels of group norm (mz_norm_dev.h) for f16 states.
#include "mz_norm_dev.h"

namespace mz_norm {
template void forward<mz::f16>(const Plan&, hipStream_t);
}  // namespace mz_norm
