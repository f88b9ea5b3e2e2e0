// Torch-free launchers of the gated feed-forward block (csrc/gemm/gated_ffn.hip), the kernels behind
// apex.fused_dense.fused_dense_gated_dense_function / FusedDenseGatedDense:
//   a = x Wg^T + bg,  u = x Wu^T + bu,  h = act(a) * u,  y = h W2^T + b2
// weight1 [2F][K] holds Wg's rows, then Wu's; `au` [M][2F] holds a, then u, of a row, as the upper 24 bits
// of fp32 in a 16-bit and an 8-bit plane.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace apex_amd {

enum GatedAct : int { kGateSilu = 0, kGateGelu = 1 };
enum FfnOp : int {
  kFfnPlain = 0,   // C[M][N] = A B (+ bias)
  kFfnGated = 1,   // A = x (k-major), B = weight1 (k-major), N = F: C = h; au written or null
  kFfnDGated = 2,  // A = dy, B = weight2 (n-major), N = F: dh = A B; C = [da | du] (ldc = 2F) from au
};

// Operand layouts as in gemm_api.h: k-major A[m * lda + k] / B[n * ldb + k], else A[k * lda + m] /
// B[k * ldb + n].
struct FfnArgs {
  const void* a;
  const void* b;
  void* c;
  int64_t lda, ldb, ldc;
  int m, n, k;
  bool a_kmajor, b_kmajor;
  int dtype;  // kF16 / kBF16
  int op, act;
  const void* bias;    // [N], gated: [2F]; or null
  uint16_t* au_hi;     // kFfnDGated: read; kFfnGated: written unless null
  uint8_t* au_lo;
  float* ws;           // ffn_workspace_floats(), or null for none
};

// the kernels' conditions: sizes, strides and bases in 16-byte vectors
bool ffn_supported(const FfnArgs& g);
// the kernels that a product takes: tile width (0: the few-row kernel) and splits of K, from op, sizes and layouts
struct FfnPlan { int bn, splits; };
FfnPlan ffn_plan(const FfnArgs& g, int cus);
int64_t ffn_workspace_floats(const FfnArgs& g, int cus);
void ffn_gemm(const FfnArgs& g, int cus, hipStream_t s);

}  // namespace apex_amd
