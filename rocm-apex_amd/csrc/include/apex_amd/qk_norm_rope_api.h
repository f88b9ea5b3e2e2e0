// Torch-free launchers of the per-head RMS norm + rotary rotation of queries and keys
// (csrc/transformer/qk_norm_rope.hip), the kernels behind
// apex.transformer.functional.fused_qk_norm_rope.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace apex_amd {

constexpr int kQkRopeMaxDim = 512;  // largest head size

// One [n0][n1][heads][d] operand, d contiguous, the other strides in elements.
struct QkRopeView {
  void* p;
  int64_t s0, s1, sh;
};

struct QkRopeArgs {
  int64_t n0, n1;               // token axes
  int hq, hk, d, rot;           // heads of q and k, head size, rotated part (even, <= d)
  QkRopeView q, k;              // inputs
  QkRopeView qo, ko;            // forward: outputs; backward: dq, dk
  QkRopeView gq, gk;            // backward: gradients of the outputs
  const void* qw;               // [d] norm weights or null
  const void* kw;
  const float* cos;             // [table][rot / 2]
  const float* sin;
  int64_t table;
  const int64_t* pos;           // positions, strides below (0 = broadcast)
  int64_t ps0, ps1;
  float eps;
  bool interleaved;             // pairs (2i, 2i + 1) instead of (i, i + rot / 2)
  int dtype, wdtype;            // q / k / outputs; weights
  float* part;                  // backward with weights: qk_norm_rope_part_floats()
  void* dqw;                    // backward with weights: [d] each, in wdtype
  void* dkw;
};

int64_t qk_norm_rope_part_floats(const QkRopeArgs& a, int cus);
void qk_norm_rope_fwd(const QkRopeArgs& a, int cus, hipStream_t s);
void qk_norm_rope_bwd(const QkRopeArgs& a, int cus, hipStream_t s);

}  // namespace apex_amd
