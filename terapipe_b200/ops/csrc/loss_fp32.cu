// The kernels of loss.cuh for fp32 logits (a file per type: they compile side by side).
#include "loss.cuh"

namespace tp {
int loss_launch_fp32(const LossArgs& a, int mode, cudaStream_t s) { return loss_launch<float>(a, mode, s); }
}  // namespace tp

TP_DEFINE_WAIT_LIMIT_SETTER(tp_set_wait_limit_ns_loss_fp32)
