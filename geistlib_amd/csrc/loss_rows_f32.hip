/* The kernels of the losses over f32 logit rows. */
#include "loss_rows_kernels.h"

namespace gs {
template void launch_loss<GEIST_HIP_TYPE_F32>(LossStage, int, int, const LossArgs &, size_t, int, int, hipStream_t);
} // namespace gs
