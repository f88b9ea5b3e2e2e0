// Torch-free launchers of the top-logit distillation loss (csrc/xentropy/topk_distill.hip), the
// kernels behind apex.contrib.xentropy.SoftmaxTopKDistillationLoss.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace apex_amd {

constexpr int kDistillMaxTop = 1024;  // teacher entries of a row

struct TopkDistillArgs {
  const void* logits;           // [rows][classes], rows `pitch` elements apart
  int64_t pitch;
  int64_t rows;
  int classes, top;
  const float* teacher_logits;  // [rows][top]
  const void* teacher_indices;  // [rows][top], int64 or int32; negative = no entry
  bool index64;
  float temperature;
  int dtype;                    // logits and gradient
};

// fp32 workspace of a forward whose rows are split over workgroups (0: not split)
int64_t topk_distill_part_floats(const TopkDistillArgs& a, int cus);
// losses [rows] and stats [rows][2]: the row's maximum m and its sum of exp((x - m) / temperature),
// kept for the backward
void topk_distill_fwd(const TopkDistillArgs& a, float* losses, float* stats, float* parts, int cus, hipStream_t s);
// grad [rows][classes] contiguous, in the logits' dtype
void topk_distill_bwd(const TopkDistillArgs& a, const float* grad_loss, int64_t grad_loss_stride, const float* stats,
                      void* grad, int cus, hipStream_t s);

}  // namespace apex_amd
