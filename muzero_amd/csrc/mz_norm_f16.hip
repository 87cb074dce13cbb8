// The group norm kernels (mz_norm_dev.h) of f16.
#include "mz_norm_dev.h"

namespace mz_norm {
template void forward<mz::f16>(const Plan&, int, hipStream_t);
template void backward<mz::f16>(const Plan&, int, hipStream_t);
}  // namespace mz_norm
