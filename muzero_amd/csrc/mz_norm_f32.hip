// The group norm kernels (mz_norm_dev.h) of float.
#include "mz_norm_dev.h"

namespace mz_norm {
template void forward<float>(const Plan&, int, hipStream_t);
template void backward<float>(const Plan&, int, hipStream_t);
}  // namespace mz_norm
