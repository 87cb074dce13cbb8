// The forward kernels of group norm (mz_norm_dev.h) for f32 states.
#include "mz_norm_dev.h"

namespace mz_norm {
template void forward<float>(const Plan&, hipStream_t);
}  // namespace mz_norm
