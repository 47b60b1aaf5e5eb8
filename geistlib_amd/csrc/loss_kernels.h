/* Launchers of the losses over logit rows (loss_rows.hip, include/geist_loss_hip.h). */
#ifndef GEIST_LOSS_KERNELS_H
#define GEIST_LOSS_KERNELS_H

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "loss_checks.h"

namespace gs {

void launch_distill(const geist_hip_loss_rows &r, const geist_hip_teacher &t, float *loss, void *ws,
                    hipStream_t stream);
void launch_policy(const geist_hip_loss_rows &r, const geist_hip_policy &p, float *loss,
                   float *logprob, float *entropy, void *ws, hipStream_t stream);
void launch_preference(const geist_hip_loss_rows &r, const geist_hip_preference &p, float *loss,
                       float *ratios, float *logprob, void *ws, hipStream_t stream);

} // namespace gs
#endif /* GEIST_LOSS_KERNELS_H */
