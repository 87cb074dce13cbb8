// The group norm kernels (mz_norm_dev.h) of bf16.
#include "mz_norm_dev.h"

namespace mz_norm {
template void forward<mz::bf16>(const Plan&, int, hipStream_t);
template void backward<mz::bf16>(const Plan&, int, hipStream_t);
}  // namespace mz_norm
