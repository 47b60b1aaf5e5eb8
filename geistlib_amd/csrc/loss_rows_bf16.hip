/* The kernels of the losses over bf16 logit rows. */
#include "loss_rows_kernels.h"

namespace gs {
template void launch_loss<GEIST_HIP_TYPE_BF16>(LossStage, int, int, const LossArgs &, size_t, int, int, hipStream_t);
} // namespace gs
