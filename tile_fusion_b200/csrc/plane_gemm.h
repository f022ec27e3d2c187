// D = A * B^T on the tensor cores from operands that lie in memory as 16-bit planes: one plane for bf16 and fp16 data, two
// (x = 2^-e (hi + lo), both fp16) for fp32 data.  What becomes of a tile of D is the caller's epilogue.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace tfk {

enum PlaneEpilogue { kPlaneStore = 0, kPlaneSoftmaxSums = 1, kPlaneSoftmaxSlope = 2 };

// One operand: rows x depth logically.  `along_rows` false: memory holds rows of `depth` values (depth contiguous), true: it
// holds `depth` rows of `rows` values.  ld: values from one memory row to the next, a multiple of 8; bases 16-byte aligned.
struct PlaneOperand {
  const void *hi = nullptr, *lo = nullptr;  // lo: second plane or null
  long long ld = 0;
  bool along_rows = false;
};

struct PlaneGemmCall {
  PlaneOperand a, b;
  int m = 0, n = 0, k = 0;
  bool f16 = false;        // planes are fp16 (else bf16); the same for both operands
  int chain = 0;           // slices of 64 whose products stay in tensor memory before they are added up in registers
  PlaneEpilogue epilogue = kPlaneStore;
  // D is multiplied by the powers of two at these addresses (device; null: 1)
  const float *scale_a = nullptr, *scale_b = nullptr;
  // kPlaneStore: out[m][ld_out] of out_dtype; sum_in: fp32 [m][ld_sum] added before scaling; sum_out: the unscaled sums go there
  // instead of `out` (ld_sum a multiple of 8, 32-byte aligned).  split_slices > 0: K is cut every so many slices of 64, and cut s
  // has the sums at s * m * ld_sum.
  void *out = nullptr;
  int out_dtype = 0;
  long long ld_out = 0;
  const float *sum_in = nullptr;
  float *sum_out = nullptr;
  long long ld_sum = 0;
  int split_slices = 0;
  // softmax: D holds logits of columns col0 .. col0 + n
  const long long *target = nullptr;
  int col0 = 0;
  // kPlaneSoftmaxSums: sums[part][m] = (largest logit, sum of exp) of a part of the columns, in units of log2; target_logit[m]
  float2 *sums = nullptr;
  float *target_logit = nullptr;
  // kPlaneSoftmaxSlope: slope[m][ld_slope] = (exp(l - lse) - (column == target)) * row_scale[m] as planes
  const float *lse2 = nullptr, *row_scale = nullptr;
  void *slope_hi = nullptr, *slope_lo = nullptr;
  long long ld_slope = 0;
};

int plane_gemm_width(int m, int n, bool b_along_rows);  // columns of a tile
int plane_gemm_parts(int m, int n);                     // parts that kPlaneSoftmaxSums writes for a row
int plane_gemm_splits(int k, int split_slices);  // cuts of a sum of k terms
int plane_gemm(const PlaneGemmCall &c, int *error, int wait_limit, int sm_count, cudaStream_t s);

}  // namespace tfk
