// Softmax cross entropy of a linear layer, loss_i = log sum_v exp(x_i . w_v) - x_i . w_t(i), without the logits in memory.
//
//   forward    logits tile by tile in tensor memory (plane_gemm.cu); a tile leaves the largest logit and the sum of
//              exponentials of each row, in units of log2, and the target's logit.  A second kernel joins the parts.
//   backward   the vocabulary in pieces: logits again, the slope P = exp(l - lse) - (column == target) of a piece as 16-bit
//              planes (at most kCeSlopeBytes of them, or 256 classes' where rows are many), then dx += P W_piece and
//              dW_piece = P^T x.  Four products of 2 n d V operations in all where kept logits would need three.
//
//   Bound by the products: 4 096 rows, 2 048 columns, 50 021 classes in bf16, loss and gradients, 2 343 us, of which 2 285 are products
//   (1 433 TFLOP/s over all).
//   Up to 64 classes and 256 columns have kernels of their own (ce_few.cu), which read x once a pass; beyond, fp32 rows are read for their
//   largest value, written as planes, and those read, in both passes.
//
// Types.  bf16 and fp16 operands are multiplied as they are.  The slope is rounded to their type before its products, one
// rounding of at most 2^-8 (bf16) or 2^-11 (fp16) of each summand; the sums are fp32.  fp32 operands are split into two fp16
// planes behind a power of two that brings the operand's largest finite value to [2^14, 2^15): 22 bits of every value down to 2^-17 of
// that value, where the second plane becomes subnormal; below, an absolute error of 2^-39 of it (at 2^-27 twelve bits are left).
// An infinity's second plane is zero, and what it is multiplied with may make it a NaN.  The slope of fp32 operands is two planes too.
// A slope lies in [-1, 1]; in fp16 it is held times 2^14: a first plane has its eleven bits down to 2^-28, both together (fp32) are off by 2^-39.
// Rows that do not count (target == ignore_index) have a slope of zero, and the rows of x that dW is summed over are a copy in
// which they are zero, so that what such rows hold -- padding, infinities, NaN -- reaches nothing.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <string>

#include "ce_few.h"
#include "plane_gemm.h"
#include "tf_internal.h"
#include "values.cuh"

namespace tfk {

namespace {

constexpr long long kCeSlopeBytes = 256ll << 20;
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kSlopeUnit = 16384.f;  // of fp16 slopes: 2^14

struct CeHeader {            // at the start of the workspace, zeroed by every call
  unsigned top_grad;         // bits of the largest finite |gradient of a row's loss|
  int counted;               // rows that count
  int error;                 // a bounded wait ran out
  int joined;                // blocks whose losses are written
  float unscale_x, unscale_w, unscale_slope;
  int pad[25];
};
constexpr int kCeGrid = 148 * 8;       // blocks of a pass over the operands
constexpr int kCeFewRows = 8192;       // rows up to which one block does what needs all of them, and a launch less is worth more

struct CeOperand {
  const void *src; long long ld; int rows;
  unsigned short *hi, *lo;   // null: multiplied where they lie
  unsigned *tops; float *unscale;  // tops: bits of the largest finite |value| that each block of ce_top_kernel saw (fp32 operands)
  const long long *target;   // rows whose target is `ignore` become zero; null: none
};

// The largest finite |value| of one operand (blockIdx.y chooses it) among a block's; `zero`: the header, if this is the first launch of a call.
__global__ void __launch_bounds__(256) ce_top_kernel(CeOperand a, CeOperand b, int cols, long long ignore, CeHeader *zero) {
  __shared__ unsigned seen[8];
  const CeOperand o = blockIdx.y ? b : a;
  if (zero && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < sizeof(CeHeader) / 4) reinterpret_cast<int *>(zero)[threadIdx.x] = 0;
  const int quads = (cols + 3) / 4;
  const bool whole = cols % 4 == 0 && o.ld % 4 == 0 && (reinterpret_cast<uintptr_t>(o.src) & 15) == 0;
  const long long total = (long long)o.rows * quads, step = (long long)gridDim.x * blockDim.x;
  unsigned top = 0;
  auto see = [&](float v) {
    const unsigned u = __float_as_uint(v) & 0x7fffffffu;
    if (u < 0x7f800000u) top = max(top, u);
  };
#pragma unroll 4
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += step) {
    const long long r = i / quads;
    const int c = (int)(i - r * quads) * 4;
    if (o.target && __ldg(o.target + r) == ignore) continue;
    const float *x = static_cast<const float *>(o.src) + r * o.ld + c;
    if (whole) {
      const float4 q = __ldg(reinterpret_cast<const float4 *>(x));
      see(q.x); see(q.y); see(q.z); see(q.w);
    } else
      for (int k = 0; k < 4 && c + k < cols; ++k) see(__ldg(x + k));
  }
  for (int k = 16; k; k >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, k));
  if ((threadIdx.x & 31) == 0) seen[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, seen[k]);
  o.tops[blockIdx.x] = top;
}

// 2^(14 - floor(log2 top)), at most 2^126
__device__ __forceinline__ int ce_exponent(unsigned top) { return top ? min(126, 14 - ((int)(top >> 23) - 127)) : 0; }
__device__ __forceinline__ float ce_power(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// Planes [rows][ldp] of an operand: fp32 split, 16-bit values copied; zeros from `cols` on and in rows that do not count.
__global__ void __launch_bounds__(256) ce_planes_kernel(CeOperand a, CeOperand b, int dtype, int cols, int ldp, long long ignore) {
  const CeOperand o = blockIdx.y ? b : a;
  if (!o.hi) return;  // (all threads of the block)
  const int eights = ldp / 8;
  const long long total = (long long)o.rows * eights, step = (long long)gridDim.x * blockDim.x;
  const bool whole = cols % 8 == 0 && o.ld * value_bytes(dtype) % 16 == 0 && (reinterpret_cast<uintptr_t>(o.src) & 15) == 0;
  float by = 1.f;
  if (dtype == TF_F32) {
    __shared__ unsigned seen[8];
    unsigned top = 0;
    for (int i = threadIdx.x; i < gridDim.x; i += blockDim.x) top = max(top, o.tops[i]);
    for (int k = 16; k; k >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, k));
    if ((threadIdx.x & 31) == 0) seen[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, seen[k]);
    const int e = ce_exponent(top);
    by = ce_power(max(e, -126));  // (e is at least -113)
    if (blockIdx.x == 0 && threadIdx.x == 0) *o.unscale = ce_power(-e);
  }
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += step) {
    const long long r = i / eights;
    const int c = (int)(i - r * eights) * 8;
    const bool none = o.target && __ldg(o.target + r) == ignore;
    uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
    if (!none && dtype == TF_F32) {
      const float *x = static_cast<const float *>(o.src) + r * o.ld + c;
      float v[8];
      if (whole) {
        const float4 p = __ldg(reinterpret_cast<const float4 *>(x)), q = __ldg(reinterpret_cast<const float4 *>(x) + 1);
        v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = q.x; v[5] = q.y; v[6] = q.z; v[7] = q.w;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? __ldg(x + k) : 0.f;
      }
      unsigned *h = &hi.x, *l = &lo.x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float p = v[2 * k] * by, q = v[2 * k + 1] * by;
        h[k] = pack_pair(p, q, true);
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[k]));
        l[k] = pack_pair(isinf(f.x) ? 0.f : p - f.x, isinf(f.y) ? 0.f : q - f.y, true);
      }
    } else if (!none) {
      const unsigned short *x = static_cast<const unsigned short *>(o.src) + r * o.ld + c;
      if (whole) hi = __ldg(reinterpret_cast<const uint4 *>(x));
      else {
        unsigned *h = &hi.x;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < cols) h[k / 2] |= (unsigned)__ldg(x + k) << (k & 1) * 16;
      }
    }
    *reinterpret_cast<uint4 *>(o.hi + r * ldp + c) = hi;
    if (o.lo) *reinterpret_cast<uint4 *>(o.lo + r * ldp + c) = lo;
  }
}

// Joins a row's parts: lse2 = log2 sum exp, and the row's loss.  Eight threads to a row, 32 rows to a block.
__global__ void __launch_bounds__(256) ce_join_kernel(const float2 *__restrict__ sums, int parts, int rows, const float *__restrict__ target_logit,
                                                      const long long *__restrict__ target, long long ignore, int vocab, float *__restrict__ lse2,
                                                      float *__restrict__ row_loss, double *block_loss, int *block_count, CeHeader *h, int mean,
                                                      float *total) {
  __shared__ float2 part[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f;
  auto add = [&](float2 p) {
    const float top = max3(m, p.x, p.x);  // (a NaN stays one)
    if (top == -INFINITY) return;  // nothing yet
    s = s * exp2f(m - top) + p.y * exp2f(p.x - top);
    m = top;
  };
  if (row < rows)
    for (int k = w; k < parts; k += 8) add(__ldg(sums + (size_t)k * rows + row));
  part[w][lane] = make_float2(m, s);
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) add(part[k][lane]);
  double loss = 0.;
  int counts = 0;
  if (row < rows) {
    const float l2 = h->error ? __int_as_float(0x7fc00000) : m + log2f(s);  // (a wait ran out: the gradients are lost with the loss)
    lse2[row] = l2;
    const long long t = target[row];
    float l = 0.f;
    if (t != ignore) {
      counts = 1;
      l = t < 0 || t >= vocab ? __int_as_float(0x7fc00000) : l2 * kLn2 - target_logit[row];
    }
    if (row_loss) row_loss[row] = l;
    loss = l;
  }
  if (!block_loss) return;
  for (int k = 16; k; k >>= 1) {
    loss += __shfl_xor_sync(0xffffffffu, loss, k);
    counts += __shfl_xor_sync(0xffffffffu, counts, k);
  }
  if (lane == 0) { block_loss[blockIdx.x] = loss; block_count[blockIdx.x] = counts; }
  if (!total) return;
  // few blocks: the last one adds them up, in their order
  int last = 0;
  if (lane == 0) {
    __threadfence();
    last = atomicAdd(&h->joined, 1) == (int)gridDim.x - 1;
  }
  if (!__shfl_sync(0xffffffffu, last, 0)) return;
  __threadfence();
  loss = 0.;
  counts = 0;
  for (int i = lane; i < (int)gridDim.x; i += 32) {
    loss += *reinterpret_cast<volatile double *>(block_loss + i);
    counts += *reinterpret_cast<volatile int *>(block_count + i);
  }
  for (int k = 16; k; k >>= 1) {
    loss += __shfl_xor_sync(0xffffffffu, loss, k);
    counts += __shfl_xor_sync(0xffffffffu, counts, k);
  }
  if (lane == 0) *total = (float)(mean ? loss / max(counts, 1) : loss);
}

// The blocks' losses in a fixed order, in 64 bits.
__global__ void __launch_bounds__(1024) ce_total_kernel(const double *__restrict__ loss, const int *__restrict__ count, int blocks, int mean, float *out) {
  __shared__ double ls[32];
  __shared__ int cs[32];
  double l = 0.;
  int c = 0;
  for (int i = threadIdx.x; i < blocks; i += blockDim.x) { l += loss[i]; c += count[i]; }
  for (int pass = 0; pass < 2; ++pass) {
    for (int k = 16; k; k >>= 1) { l += __shfl_xor_sync(0xffffffffu, l, k); c += __shfl_xor_sync(0xffffffffu, c, k); }
    if (pass) break;
    if ((threadIdx.x & 31) == 0) { ls[threadIdx.x >> 5] = l; cs[threadIdx.x >> 5] = c; }
    __syncthreads();
    if (threadIdx.x >= 32) return;
    l = threadIdx.x < blockDim.x / 32 ? ls[threadIdx.x] : 0.;
    c = threadIdx.x < blockDim.x / 32 ? cs[threadIdx.x] : 0;
  }
  if (threadIdx.x == 0) *out = (float)(mean ? l / max(c, 1) : l);
}

// How many rows count, and (a gradient to each row) the largest of them.
__global__ void __launch_bounds__(256) ce_count_kernel(const long long *__restrict__ target, const float *__restrict__ grad, int rows, long long ignore,
                                                       CeHeader *h) {
  int c = 0;
  unsigned top = 0;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < rows; i += gridDim.x * blockDim.x) {
    if (target[i] == ignore) continue;
    ++c;
    if (grad) {
      const unsigned u = __float_as_uint(grad[i]) & 0x7fffffffu;
      if (u < 0x7f800000u) top = max(top, u);
    }
  }
  for (int k = 16; k; k >>= 1) { c += __shfl_xor_sync(0xffffffffu, c, k); top = max(top, __shfl_xor_sync(0xffffffffu, top, k)); }
  if ((threadIdx.x & 31) == 0) {
    if (c) atomicAdd(&h->counted, c);
    if (top) atomicMax(&h->top_grad, top);
  }
}

// What a row's slope is multiplied by before it is rounded, and what the sums of slopes are multiplied by.  reduction 0: a gradient to
// each row, brought to at most one by a power of two; 1, 2: one gradient, which the sums take.
__device__ __forceinline__ float2 ce_scales(int reduction, float unit, unsigned top_grad, int counted, const float *grad) {
  float by = unit, back = 1.f / unit;
  if (reduction == 0) {
    // (unit * 2^e stays a number, or rows of zero gradients would become NaN)
    const int e = top_grad ? min(unit == 1.f ? 126 : 112, max(-126, -((int)(top_grad >> 23) - 126))) : 0;
    by *= ce_power(e);
    back *= ce_power(-e);
  } else back *= grad[0] / (reduction == 1 ? (float)max(counted, 1) : 1.f);
  return make_float2(by, back);
}
__device__ __forceinline__ float ce_row_scale(long long t, long long ignore, int vocab, int reduction, const float *grad, int i, float by) {
  if (t == ignore) return 0.f;
  return t < 0 || t >= vocab ? __int_as_float(0x7fc00000) : reduction == 0 ? grad[i] * by : by;
}
__global__ void __launch_bounds__(256) ce_scale_kernel(const long long *__restrict__ target, const float *__restrict__ grad, int rows, long long ignore,
                                                       int vocab, int reduction, float unit, float *__restrict__ row_scale, CeHeader *h) {
  const float2 scale = ce_scales(reduction, unit, h->top_grad, h->counted, grad);
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i == 0) h->unscale_slope = scale.y;
  if (i < rows) row_scale[i] = ce_row_scale(target[i], ignore, vocab, reduction, grad, i, scale.x);
}

// Both of these in one block, behind the zeroed header.
__global__ void __launch_bounds__(1024) ce_prepare_kernel(const long long *__restrict__ target, const float *__restrict__ grad, int rows, long long ignore,
                                                          int vocab, int reduction, float unit, float *__restrict__ row_scale, CeHeader *h) {
  __shared__ int cs[32];
  __shared__ unsigned ts[32];
  if (threadIdx.x < sizeof(CeHeader) / 4) reinterpret_cast<int *>(h)[threadIdx.x] = 0;
  int c = 0;
  unsigned top = 0;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    if (target[i] == ignore) continue;
    ++c;
    if (reduction == 0) {
      const unsigned u = __float_as_uint(grad[i]) & 0x7fffffffu;
      if (u < 0x7f800000u) top = max(top, u);
    }
  }
  for (int k = 16; k; k >>= 1) { c += __shfl_xor_sync(0xffffffffu, c, k); top = max(top, __shfl_xor_sync(0xffffffffu, top, k)); }
  if ((threadIdx.x & 31) == 0) { cs[threadIdx.x >> 5] = c; ts[threadIdx.x >> 5] = top; }
  __syncthreads();
  c = 0;
  top = 0;
  for (int k = 0; k < 32; ++k) { c += cs[k]; top = max(top, ts[k]); }
  const float2 scale = ce_scales(reduction, unit, top, c, grad);
  if (threadIdx.x == 0) h->unscale_slope = scale.y;
  for (int i = threadIdx.x; i < rows; i += 1024) row_scale[i] = ce_row_scale(target[i], ignore, vocab, reduction, grad, i, scale.x);
}

// out = (part[0] + part[1] + ...) * scales, parts [splits][rows][ld]
__global__ void __launch_bounds__(256) ce_parts_kernel(const float *__restrict__ part, int splits, int rows, int cols, int ld, const float *scale_a,
                                                       const float *scale_b, void *__restrict__ out, int dtype) {
  const float sa = scale_a ? *scale_a : 1.f, sb = scale_b ? *scale_b : 1.f;
  const long long total = (long long)rows * ld / 4, each = (long long)rows * ld;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const float *p = part + i * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      const float4 q = __ldg(reinterpret_cast<const float4 *>(p + k * each));
      s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
    }
    const long long r = i * 4 / ld;
    const int c = (int)(i * 4 - r * ld);
    const float v[4] = {s.x * sa * sb, s.y * sa * sb, s.z * sa * sb, s.w * sa * sb};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < cols) store_value(out, dtype, r * cols + c + k, v[k]);
  }
}

// out[i] = (part[0][i] + part[1][i] + ...) * *scale, in order; eight threads share an element's parts.
__global__ void __launch_bounds__(256) ce_few_sum_kernel(const float *__restrict__ part, int parts, int n, const float *scale, void *__restrict__ out, int dtype) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, l = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (i < n)
#pragma unroll 4
    for (int k = l; k < parts; k += 8) v += __ldg(part + (size_t)k * n + i);
  s[l][lane] = v;
  __syncthreads();
  if (l || i >= n) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += s[k][lane];
  store_value(out, dtype, i, v * *scale);
}

// Gradients of a call one of whose bounded waits ran out: NaN, as the forward's loss.
__global__ void __launch_bounds__(256) ce_lost_kernel(const CeHeader *h, void *__restrict__ dx, long long nx, void *__restrict__ dw, long long nw, int dtype) {
  if (!h->error) return;
  const float nan = __int_as_float(0x7fc00000);
  const long long i0 = blockIdx.x * (long long)blockDim.x + threadIdx.x, step = (long long)gridDim.x * blockDim.x;
  if (dx)
    for (long long i = i0; i < nx; i += step) store_value(dx, dtype, i, nan);
  if (dw)
    for (long long i = i0; i < nw; i += step) store_value(dw, dtype, i, nan);
}

long long up(long long v, long long to) { return (v + to - 1) / to * to; }

// What the workspace holds, for the sizes of a call; `base` null: sizes only.
struct CeSpace {
  CeHeader *h;
  unsigned *tops = nullptr;  // [2][kCeGrid]
  unsigned short *x_hi = nullptr, *x_lo = nullptr, *w_hi = nullptr, *w_lo = nullptr;
  float2 *sums = nullptr; float *target_logit = nullptr; double *block_loss = nullptr; int *block_count = nullptr;
  float *row_scale = nullptr; unsigned short *slope_hi = nullptr, *slope_lo = nullptr; float *parts_x = nullptr, *parts_w = nullptr;
  int ldp, ld_slope = 0, piece = 0, cut_x = 0, cut_w = 0;  // cut_: slices of a cut of the sum, 0: not cut
  long long bytes;
  bool few, copy_x, copy_w;
};

// Slices of a cut of the long sum of a gradient product (0: not cut), so that few tiles still fill the pairs of the device.  Where tiles
// nearly do, a cut has at least 32 slices (2 048 terms), so that reading the parts back stays small beside the products; where
// they leave most pairs idle, at least four.
int ce_cut(int m, int n, int k, bool along_rows) {
  const int bn = plane_gemm_width(m, n, along_rows), pairs = 74;
  const long long tiles = (long long)((m + 255) / 256) * ((n + bn - 1) / bn);
  const int slices = (k + 63) / 64, most = std::max(1, slices / (4 * tiles <= pairs ? 4 : 32));
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= std::min(most, pairs); ++s) {
    const double waves = (double)((tiles * s + pairs - 1) / pairs) / s;  // rounds of the device, in whole products
    if (waves < 0.93 * cost) { cost = waves; best = s; }
  }
  return best > 1 ? (slices + best - 1) / best : 0;
}

CeSpace ce_space(char *base, int rows, int cols, int vocab, int dtype, bool backward, bool whole_x, bool whole_w) {
  CeSpace s;
  long long at = 0;
  auto take = [&](long long bytes) {
    char *p = base + at;
    at += up(bytes, 256);
    return p;
  };
  const bool f32 = dtype == TF_F32;
  s.h = (CeHeader *)take(sizeof(CeHeader));
  s.few = ce_few_supported(cols, vocab);
  if (s.few) {
    const int ctas = ce_few_ctas(rows);
    s.block_loss = (double *)take(8ll * ctas);
    s.block_count = (int *)take(4ll * ctas);
    if (backward) {
      s.row_scale = (float *)take(4ll * rows);
      s.parts_w = (float *)take(4ll * ctas * vocab * cols);
    }
    s.bytes = at;
    return s;
  }
  s.ldp = (int)up(cols, 8);
  if (f32) s.tops = (unsigned *)take(8ll * kCeGrid);
  s.copy_x = f32 || backward || !whole_x;
  s.copy_w = f32 || !whole_w;
  if (s.copy_x) s.x_hi = (unsigned short *)take(2ll * rows * s.ldp);
  if (f32) s.x_lo = (unsigned short *)take(2ll * rows * s.ldp);
  if (s.copy_w) s.w_hi = (unsigned short *)take(2ll * vocab * s.ldp);
  if (f32) s.w_lo = (unsigned short *)take(2ll * vocab * s.ldp);
  if (!backward) {
    s.sums = (float2 *)take(8ll * rows * plane_gemm_parts(rows, vocab));
    s.target_logit = (float *)take(4ll * rows);
    s.block_loss = (double *)take(8ll * ((rows + 31) / 32));
    s.block_count = (int *)take(4ll * ((rows + 31) / 32));
  } else {
    s.row_scale = (float *)take(4ll * rows);
    // pieces of equal width, whole tiles of columns
    const long long most = std::max<long long>(256, kCeSlopeBytes / (rows * (f32 ? 4ll : 2ll)) / 256 * 256);
    const long long pieces = (vocab + most - 1) / most;
    s.piece = (int)std::min<long long>(vocab, up((vocab + pieces - 1) / pieces, 256));
    s.ld_slope = (int)up(s.piece, 8);
    s.slope_hi = (unsigned short *)take(2ll * rows * s.ld_slope);
    if (f32) s.slope_lo = (unsigned short *)take(2ll * rows * s.ld_slope);
    s.cut_x = ce_cut(rows, cols, s.piece, true);
    s.cut_w = ce_cut(s.piece, cols, rows, true);
    const long long ld_sum = up(cols, 8);
    if (s.cut_x || pieces > 1) s.parts_x = (float *)take(4ll * plane_gemm_splits(s.piece, s.cut_x) * rows * ld_sum);
    if (s.cut_w) s.parts_w = (float *)take(4ll * plane_gemm_splits(rows, s.cut_w) * s.piece * ld_sum);
  }
  s.bytes = at;
  return s;
}

bool ce_whole(const void *p, long long ld, int dtype) { return dtype != TF_F32 && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int ce_check(const char *who, const void *x, long long ld_x, const void *w, long long ld_w, int dtype, const long long *target, int rows, int cols,
             int vocab, int reduction, const void *work) {
  auto bad = [&](const char *what) { return tf::fail(TF_ERR_ARG, std::string(who) + ": " + what); };
  if (!known_dtype(dtype)) return bad("unknown type");
  if (rows < 0 || cols <= 0 || vocab <= 0 || rows > kMaxRows || cols > kMaxRows || vocab > kMaxRows) return bad("bad size");
  if (rows > 0 && (!x || !target)) return bad("null argument");
  if (!w || !work) return bad("null argument");
  if (ld_x < cols || ld_w < cols) return bad("rows overlap");
  if (reduction < 0 || reduction > 2) return bad("unknown reduction");
  if ((reinterpret_cast<uintptr_t>(work) & 255) != 0) return bad("the work space must be 256-byte aligned");
  return TF_OK;
}

int ce_fail(const char *who, cudaError_t e) { return tf::fail(TF_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e)); }

cudaError_t ce_lost(const CeHeader *h, void *dx, long long nx, void *dw, long long nw, int dtype, cudaStream_t s) {
  ce_lost_kernel<<<(unsigned)std::min<long long>((std::max(nx, nw) + 1023) / 1024, 148 * 4), 256, 0, s>>>(h, dx, nx, dw, nw, dtype);
  return cudaGetLastError();
}

std::atomic<int> wait_limit{1 << 22};

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

CeFewCall few_call(const CeSpace &sp, const void *x, long long ld_x, const void *w, long long ld_w, int dtype, const long long *target, int rows, int cols,
                   int vocab, long long ignore) {
  CeFewCall c;
  c.x = x; c.w = w; c.ld_x = ld_x; c.ld_w = ld_w; c.dtype = dtype; c.rows = rows; c.cols = cols; c.vocab = vocab;
  c.target = target; c.ignore = ignore;
  c.error = &sp.h->error;
  c.wait_limit = dense_wait_limit();
  return c;
}

// Planes of both operands, where they are not multiplied as they lie.
cudaError_t ce_planes(const CeSpace &sp, const void *x, long long ld_x, const void *w, long long ld_w, int dtype, int rows, int cols, int vocab,
                      const long long *target, long long ignore, CeHeader *zero, cudaStream_t s) {
  CeOperand ox = {x, ld_x, rows, sp.x_hi, sp.x_lo, sp.tops, &sp.h->unscale_x, target};
  CeOperand ow = {w, ld_w, vocab, sp.w_hi, sp.w_lo, sp.tops + kCeGrid, &sp.h->unscale_w, nullptr};
  if (!sp.copy_x && !sp.copy_w) return cudaSuccess;
  const long long most = (long long)std::max(sp.copy_x ? rows : 0, sp.copy_w ? vocab : 0) * sp.ldp / 8;
  const dim3 grid((unsigned)std::min<long long>((most + 255) / 256, kCeGrid), 2);
  if (dtype == TF_F32) ce_top_kernel<<<grid, 256, 0, s>>>(ox, ow, cols, ignore, zero);
  ce_planes_kernel<<<grid, 256, 0, s>>>(ox, ow, dtype, cols, sp.ldp, ignore);
  return cudaGetLastError();
}

}  // namespace

int dense_wait_limit() { return wait_limit.load(std::memory_order_relaxed); }

}  // namespace tfk

using namespace tfk;

extern "C" long long tf_linear_ce_work_bytes(int rows, int cols, int vocab, int dtype, int backward) {
  if (rows < 0 || cols <= 0 || vocab <= 0 || rows > kMaxRows || cols > kMaxRows || vocab > kMaxRows || !known_dtype(dtype)) return 0;
  return ce_space(nullptr, std::max(rows, 1), cols, vocab, dtype, backward != 0, false, false).bytes;
}

extern "C" long long tf_linear_ce_work_bytes_for(const void *x, long long ld_x, const void *w, long long ld_w, int rows, int cols, int vocab, int dtype,
                                                 int backward) {
  if (rows < 0 || cols <= 0 || vocab <= 0 || rows > kMaxRows || cols > kMaxRows || vocab > kMaxRows || !known_dtype(dtype)) return 0;
  return ce_space(nullptr, std::max(rows, 1), cols, vocab, dtype, backward != 0, ce_whole(x, ld_x, dtype), ce_whole(w, ld_w, dtype)).bytes;
}

extern "C" int tf_linear_ce_fwd(const void *x, long long ld_x, const void *w, long long ld_w, int dtype, const long long *target, int rows,
                                int cols, int vocab, long long ignore_index, int reduction, float *loss, float *lse2, void *work,
                                long long work_bytes, void *stream) {
  const char *who = "tf_linear_ce_fwd";
  int rc = ce_check(who, x, ld_x, w, ld_w, dtype, target, rows, cols, vocab, reduction, work);
  if (rc != TF_OK) return rc;
  if ((!loss && (reduction || rows)) || (!lse2 && rows)) return tf::fail(TF_ERR_ARG, "tf_linear_ce_fwd: null argument");
  if (work_bytes < tf_linear_ce_work_bytes_for(x, ld_x, w, ld_w, rows, cols, vocab, dtype, 0)) return tf::fail(TF_ERR_ARG, "tf_linear_ce_fwd: work space too small");
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    cudaError_t e = cudaMemsetAsync(work, 0, sizeof(CeHeader), s);
    if (e == cudaSuccess && reduction) e = cudaMemsetAsync(loss, 0, 4, s);
    return e == cudaSuccess ? TF_OK : ce_fail(who, e);
  }
  const CeSpace sp = ce_space((char *)work, rows, cols, vocab, dtype, false, ce_whole(x, ld_x, dtype), ce_whole(w, ld_w, dtype));
  // (fp32: the first pass over the operands zeroes the header)
  const bool zeroes = dtype == TF_F32 && !sp.few;
  cudaError_t e = zeroes ? cudaSuccess : cudaMemsetAsync(sp.h, 0, sizeof(CeHeader), s);
  if (sp.few) {
    CeFewCall c = few_call(sp, x, ld_x, w, ld_w, dtype, target, rows, cols, vocab, ignore_index);
    c.lse2 = lse2;
    c.row_loss = reduction ? nullptr : loss;
    if (reduction) { c.cta_loss = sp.block_loss; c.cta_count = sp.block_count; }
    if (e == cudaSuccess) e = ce_few_forward(c, s);
    if (e == cudaSuccess && reduction) {
      ce_total_kernel<<<1, 1024, 0, s>>>(sp.block_loss, sp.block_count, ce_few_ctas(rows), reduction == 1, loss);
      e = cudaGetLastError();
    }
    return e == cudaSuccess ? TF_OK : ce_fail(who, e);
  }
  if (e == cudaSuccess) e = ce_planes(sp, x, ld_x, w, ld_w, dtype, rows, cols, vocab, target, ignore_index, zeroes ? sp.h : nullptr, s);
  if (e != cudaSuccess) return ce_fail(who, e);
  const bool f32 = dtype == TF_F32;
  PlaneGemmCall c;
  c.a = {sp.copy_x ? sp.x_hi : x, sp.x_lo, sp.copy_x ? sp.ldp : ld_x, false};
  c.b = {sp.copy_w ? sp.w_hi : w, sp.w_lo, sp.copy_w ? sp.ldp : ld_w, false};
  c.m = rows; c.n = vocab; c.k = cols;
  c.f16 = dtype != TF_BF16;
  c.chain = f32 ? 2 : 8;  // (16 bits, 4 096 x 2 048 x 50 021: loss off by 6e-8 with 4, 4e-7 with 16; 562 and 529 us)
  c.epilogue = kPlaneSoftmaxSums;
  if (f32) { c.scale_a = &sp.h->unscale_x; c.scale_b = &sp.h->unscale_w; }
  c.target = target;
  c.sums = sp.sums; c.target_logit = sp.target_logit;
  rc = plane_gemm(c, &sp.h->error, dense_wait_limit(), sm_count(), s);
  if (rc != TF_OK) return rc;
  const int blocks = (rows + 31) / 32;
  ce_join_kernel<<<blocks, 256, 0, s>>>(sp.sums, plane_gemm_parts(rows, vocab), rows, sp.target_logit, target, ignore_index, vocab, lse2,
                                        reduction ? nullptr : loss, reduction ? sp.block_loss : nullptr, sp.block_count, sp.h, reduction == 1,
                                        reduction && rows <= kCeFewRows ? loss : nullptr);
  if (reduction && rows > kCeFewRows) ce_total_kernel<<<1, 1024, 0, s>>>(sp.block_loss, sp.block_count, blocks, reduction == 1, loss);
  e = cudaGetLastError();
  return e == cudaSuccess ? TF_OK : ce_fail(who, e);
}

extern "C" int tf_linear_ce_bwd(const void *x, long long ld_x, const void *w, long long ld_w, int dtype, const long long *target, int rows,
                                int cols, int vocab, long long ignore_index, int reduction, const float *lse2, const float *grad, void *dx,
                                void *dw, void *work, long long work_bytes, void *stream) {
  const char *who = "tf_linear_ce_bwd";
  int rc = ce_check(who, x, ld_x, w, ld_w, dtype, target, rows, cols, vocab, reduction, work);
  if (rc != TF_OK) return rc;
  if (rows > 0 && (!lse2 || !grad)) return tf::fail(TF_ERR_ARG, "tf_linear_ce_bwd: null argument");
  if (work_bytes < tf_linear_ce_work_bytes_for(x, ld_x, w, ld_w, rows, cols, vocab, dtype, 1)) return tf::fail(TF_ERR_ARG, "tf_linear_ce_bwd: work space too small");
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    cudaError_t e = cudaMemsetAsync(work, 0, sizeof(CeHeader), s);
    if (e == cudaSuccess && dw) e = cudaMemsetAsync(dw, 0, (size_t)vocab * cols * value_bytes(dtype), s);
    return e == cudaSuccess ? TF_OK : ce_fail(who, e);
  }
  if (!dx && !dw) return TF_OK;
  const CeSpace sp = ce_space((char *)work, rows, cols, vocab, dtype, true, ce_whole(x, ld_x, dtype), ce_whole(w, ld_w, dtype));
  const bool f32 = dtype == TF_F32;
  const float unit = dtype == TF_BF16 ? 1.f : kSlopeUnit;
  cudaError_t e = cudaSuccess;
  if (rows <= kCeFewRows)
    ce_prepare_kernel<<<1, 1024, 0, s>>>(target, grad, rows, ignore_index, vocab, reduction, unit, sp.row_scale, sp.h);
  else {
    e = cudaMemsetAsync(sp.h, 0, sizeof(CeHeader), s);
    if (e != cudaSuccess) return ce_fail(who, e);
    if (reduction != 2)
      ce_count_kernel<<<std::min((rows + 255) / 256, 148 * 4), 256, 0, s>>>(target, reduction ? nullptr : grad, rows, ignore_index, sp.h);
    ce_scale_kernel<<<(rows + 255) / 256, 256, 0, s>>>(target, grad, rows, ignore_index, vocab, reduction, unit, sp.row_scale, sp.h);
  }
  if (sp.few) {
    CeFewCall c = few_call(sp, x, ld_x, w, ld_w, dtype, target, rows, cols, vocab, ignore_index);
    c.lse2 = const_cast<float *>(lse2);
    c.row_scale = sp.row_scale; c.unscale = &sp.h->unscale_slope;
    c.dx = dx; c.dw_parts = dw ? sp.parts_w : nullptr;
    e = ce_few_backward(c, s);
    if (e == cudaSuccess && dw) {
      ce_few_sum_kernel<<<(vocab * cols + 31) / 32, 256, 0, s>>>(sp.parts_w, ce_few_ctas(rows), vocab * cols, &sp.h->unscale_slope, dw, dtype);
      e = cudaGetLastError();
    }
    return e == cudaSuccess ? TF_OK : ce_fail(who, e);
  }
  e = ce_planes(sp, x, ld_x, w, ld_w, dtype, rows, cols, vocab, target, ignore_index, nullptr, s);
  if (e != cudaSuccess) return ce_fail(who, e);
  const int sms = sm_count();
  const long long ld_sum = up(cols, 8), ld_w16 = sp.copy_w ? sp.ldp : ld_w;
  const unsigned short *w_hi = sp.copy_w ? sp.w_hi : (const unsigned short *)w;
  for (int v0 = 0; v0 < vocab; v0 += sp.piece) {
    const int nv = std::min(sp.piece, vocab - v0);
    const unsigned short *wp_hi = w_hi + v0 * ld_w16, *wp_lo = f32 ? sp.w_lo + v0 * ld_w16 : nullptr;
    PlaneGemmCall c;  // the slope
    c.a = {sp.x_hi, sp.x_lo, sp.ldp, false};
    c.b = {wp_hi, wp_lo, ld_w16, false};
    c.m = rows; c.n = nv; c.k = cols;
    c.f16 = dtype != TF_BF16;
    c.chain = f32 ? 2 : 16;
    c.epilogue = kPlaneSoftmaxSlope;
    if (f32) { c.scale_a = &sp.h->unscale_x; c.scale_b = &sp.h->unscale_w; }
    c.target = target; c.col0 = v0;
    c.lse2 = lse2; c.row_scale = sp.row_scale;
    c.slope_hi = sp.slope_hi; c.slope_lo = sp.slope_lo; c.ld_slope = sp.ld_slope;
    rc = plane_gemm(c, &sp.h->error, dense_wait_limit(), sms, s);
    if (rc != TF_OK) return rc;
    const bool last = v0 + nv == vocab;
    if (dx) {
      PlaneGemmCall g;
      g.a = {sp.slope_hi, sp.slope_lo, sp.ld_slope, false};
      g.b = {wp_hi, wp_lo, ld_w16, true};
      g.m = rows; g.n = cols; g.k = nv;
      g.f16 = c.f16;
      g.chain = f32 ? 2 : 16;
      g.scale_a = &sp.h->unscale_slope;
      g.scale_b = f32 ? &sp.h->unscale_w : nullptr;
      g.split_slices = sp.cut_x;
      g.ld_sum = ld_sum;
      if (v0) g.sum_in = sp.parts_x;
      if (!last || sp.cut_x) g.sum_out = sp.parts_x;
      g.out = dx; g.out_dtype = dtype; g.ld_out = cols;
      rc = plane_gemm(g, &sp.h->error, dense_wait_limit(), sms, s);
      if (rc != TF_OK) return rc;
    }
    if (dw) {
      PlaneGemmCall g;
      g.a = {sp.slope_hi, sp.slope_lo, sp.ld_slope, true};
      g.b = {sp.x_hi, sp.x_lo, sp.ldp, true};
      g.m = nv; g.n = cols; g.k = rows;
      g.f16 = c.f16;
      g.chain = f32 ? 2 : 16;
      g.scale_a = &sp.h->unscale_slope;
      g.scale_b = f32 ? &sp.h->unscale_x : nullptr;
      g.split_slices = sp.cut_w;
      g.ld_sum = ld_sum;
      if (sp.cut_w) g.sum_out = sp.parts_w;
      char *to = (char *)dw + (size_t)v0 * cols * value_bytes(dtype);
      g.out = to; g.out_dtype = dtype; g.ld_out = cols;
      rc = plane_gemm(g, &sp.h->error, dense_wait_limit(), sms, s);
      if (rc != TF_OK) return rc;
      if (sp.cut_w) {
        const long long q = (long long)nv * ld_sum / 4;
        ce_parts_kernel<<<(unsigned)std::min<long long>((q + 255) / 256, 148 * 16), 256, 0, s>>>(sp.parts_w, plane_gemm_splits(rows, sp.cut_w), nv, cols,
                                                                                                 (int)ld_sum, g.scale_a, g.scale_b, to, dtype);
      }
    }
  }
  if (dx && sp.cut_x) {
    const long long q = (long long)rows * ld_sum / 4;
    ce_parts_kernel<<<(unsigned)std::min<long long>((q + 255) / 256, 148 * 16), 256, 0, s>>>(sp.parts_x, plane_gemm_splits(sp.piece, sp.cut_x), rows, cols, (int)ld_sum,
                                                                                             &sp.h->unscale_slope, f32 ? &sp.h->unscale_w : nullptr, dx, dtype);
  }
  e = cudaGetLastError();
  if (e == cudaSuccess) e = ce_lost(sp.h, dx, (long long)rows * cols, dw, (long long)vocab * cols, dtype, s);
  return e == cudaSuccess ? TF_OK : ce_fail(who, e);
}

extern "C" int tf_dense_set_wait_limit(int polls) {
  if (polls != 0 && polls < kInFlightPolls) return tf::fail(TF_ERR_ARG, "tf_dense_set_wait_limit: 0, or 65 536 polls at least");
  wait_limit.store(polls, std::memory_order_relaxed);
  return TF_OK;
}

extern "C" int tf_linear_ce_status(const void *work, void *stream) {
  if (!work) return tf::fail(TF_ERR_ARG, "tf_linear_ce_status: null argument");
  CeHeader h;
  cudaError_t e = cudaStreamSynchronize((cudaStream_t)stream);
  if (e == cudaSuccess) e = cudaMemcpy(&h, work, sizeof(h), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return ce_fail("tf_linear_ce_status", e);
  return h.error ? tf::fail(TF_ERR_TIMEOUT, "linear cross entropy: a bounded wait on a copy or on the tensor core ran out") : TF_OK;
}
