// The backward kernels of group norm (mz_norm_dev.h) for bf16 states.
#include "mz_norm_dev.h"

namespace mz_norm {
template void backward<mz::bf16>(const Plan&, hipStream_t);
}  // namespace mz_norm
