// Softmax cross entropy of a linear layer over few classes (ce_few.cu): both passes in one launch each.
#pragma once
#include <cuda_runtime.h>

namespace tfk {

// What shared memory holds of fp32 operands: the weight and two tiles of x, two slopes, two planes of each.  120 001 rows, loss and gradients,
// fp32 and bf16: 64 classes of 256 columns 170 and 115 us here; 65 classes 349 and 178, 264 columns 378 and 215 by way of plane_gemm.cu.
constexpr int kFewClasses = 64, kFewCols = 256;

struct CeFewCall {
  const void *x = nullptr, *w = nullptr;
  long long ld_x = 0, ld_w = 0;
  int dtype = 0, rows = 0, cols = 0, vocab = 0;
  const long long *target = nullptr;
  long long ignore = 0;
  int *error = nullptr;
  int wait_limit = 0;
  // forward
  float *lse2 = nullptr, *row_loss = nullptr;    // row_loss or, for each CTA, the sum of its rows' losses and their number
  double *cta_loss = nullptr;
  int *cta_count = nullptr;
  // backward
  const float *row_scale = nullptr, *unscale = nullptr;
  void *dx = nullptr;                            // null: not asked for
  float *dw_parts = nullptr;                     // [CTA][vocab][cols], times 1 / *unscale; null: not asked for
};

bool ce_few_supported(int cols, int vocab);
int ce_few_ctas(int rows);
cudaError_t ce_few_forward(const CeFewCall &c, cudaStream_t s);
cudaError_t ce_few_backward(const CeFewCall &c, cudaStream_t s);

}  // namespace tfk
