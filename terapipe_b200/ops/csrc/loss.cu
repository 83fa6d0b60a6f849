// Entry point of the losses over a vocabulary (loss.cuh).
#include "loss.cuh"

using namespace tp;

// mode: 1 loss and stats, 2 gradient from stats, 3 loss and gradient.  dtype, tlog_dtype: 0 fp16, 1 bf16, 2 fp32.  Outer
// index i of an array lies at (i / cols) * s0 + (i % cols) * s1.  dlogits may be logits.
extern "C" int tp_loss(int mode, int dtype, const void* logits, long long ld, int rows, int V, const void* labels,
                       int labels64, int label_cols, long long label_s0, long long label_s1, long long ignore,
                       const void* tid, int tid64, int tid_cols, long long tid_s0, long long tid_s1, const void* tlog,
                       int tlog_dtype, int tlog_cols, long long tlog_s0, long long tlog_s1, int top, float temperature,
                       float weight, float* loss, float* stats, void* dlogits, long long ldd, const float* grad_loss,
                       long long ldg, float grad_scale, int* status, void* stream) {
  if (mode < 1 || mode > 3 || dtype < 0 || dtype > 2 || tlog_dtype < 0 || tlog_dtype > 2 || rows < 0 || V < 0 || top < 0 ||
      label_cols < 1 || tid_cols < 1 || tlog_cols < 1 || !(temperature >= 0x1p-10f && temperature <= 0x1p10f) || (top > 0 && (!tid || !tlog)))
    return kErrBadArgument;
  if (top > kMaxTop) return kErrTooLarge;
  if (rows == 0) return kOk;
  if (((mode & kLossFwd) && !loss) || (mode == kLossBwd && !stats) || ((mode & kLossBwd) && V > 0 && !dlogits))
    return kErrBadArgument;
  LossArgs a{logits, ld, rows, V, labels, OuterIndex{label_s0, label_s1, label_cols}, ignore, labels64, tid, tlog,
             OuterIndex{tid_s0, tid_s1, tid_cols}, OuterIndex{tlog_s0, tlog_s1, tlog_cols}, top, tid64, tlog_dtype,
             temperature, weight, loss, stats, dlogits, ldd, grad_loss, ldg, grad_scale, status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return loss_launch_fp16(a, mode, s);
  if (dtype == 1) return loss_launch_bf16(a, mode, s);
  return loss_launch_fp32(a, mode, s);
}
