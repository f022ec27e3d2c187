// Layer norm over the last dimension, y = (x - mean) rstd w + b, and its gradients.
//
//   dx = rstd (h - mean(h) - xh mean(h xh)),   h = dy w,  xh = (x - mean) rstd;   dw = sum_rows dy xh;   db = sum_rows dy
//
// Both passes are bound by the rows that they read and write (two and three of them).  A row stays in registers between its
// sums and its use, so it is read once: eight lanes, a warp or a whole CTA to a row, at most 16 values to a thread; the variance is
// that of the centred values.  Threads walk the rows with the grid's stride, so that a thread's columns stay the same: the weight is
// read once, and the sums of dw and db over rows stay in registers until the end, where they are joined in shared memory; a second
// launch adds the CTAs' sums in order, so results don't depend on scheduling.  The next row's loads are issued before the sums
// of the row at hand.  Statistics and sums are fp32 whatever the values' type.
//   The forward pass can leave its input in 8 bits on the way (pack8.cuh), which the backward pass then reads in its place.
#include <algorithm>
#include <string>

#include "pack8.cuh"
#include "tf_internal.h"

namespace tfk {

namespace {

constexpr int kLnValues = 16;                  // of a thread
constexpr int kLnMaxThreads = 1024;
constexpr int kLnMaxCols = kLnValues * kLnMaxThreads;
constexpr int kLnWarpThreads = 256;            // CTAs whose rows have a warp or less
constexpr int kLnRowThreads = 512;             // the largest CTA that has 128 registers a thread
// LANES of a row: 8, 32, kLnRow (the CTA), kLnWideRow (a CTA of up to kLnMaxThreads: 64 registers, some values spill)
constexpr int kLnRow = 0, kLnWideRow = -1;
constexpr int ln_most_threads(int lanes) { return lanes > 0 ? kLnWarpThreads : lanes == kLnRow ? kLnRowThreads : kLnMaxThreads; }

struct LnParams {
  const void *x; long long ld_x;
  const void *w, *b; int w_dtype;
  int rows, cols; float eps;
  void *y; long long ld_y;
  float *mean, *rstd;
  signed char *codes; int ld_codes; unsigned char *exps;   // forward: written (null: not); backward: read instead of x
  const void *dy; long long ld_dy;
  void *dx; long long ld_dx;
  float *part;                                             // [CTA][2][cols]
};

// Sum over the LANES lanes of a row, or (LANES <= 0) over the CTA; `slot` alternates between two scratch arrays.
template <int LANES, int K> __device__ __forceinline__ void ln_sum(float (&v)[K], float (*scratch)[32][2], int &slot) {
#pragma unroll
  for (int k = (LANES > 0 ? LANES : 32) / 2; k; k >>= 1)
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], k);
  if (LANES <= 0 && blockDim.x > 32) {
    const int warps = blockDim.x / 32, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < K; ++i) scratch[slot][threadIdx.x >> 5][i] = v[i];
    __syncthreads();  // (one to a sum: the scratch array of the sum before last has been read by then)
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] = lane < warps ? scratch[slot][lane][i] : 0.f;
#pragma unroll
    for (int k = 16; k; k >>= 1)
#pragma unroll
      for (int i = 0; i < K; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], k);
    slot ^= 1;
  }
}

// Where a thread's columns are, and its rows: N values at a time, NV times.
template <int N, int NV, int LANES> struct LnPlace {
  int t, lanes;
  long long row, step;
  __device__ LnPlace() {
    constexpr int L = LANES > 0 ? LANES : 32;
    if (LANES > 0) {
      t = threadIdx.x % L; lanes = L;
      row = blockIdx.x * (long long)(blockDim.x / L) + threadIdx.x / L;
      step = (long long)gridDim.x * (blockDim.x / L);
    } else { t = threadIdx.x; lanes = blockDim.x; row = blockIdx.x; step = gridDim.x; }
  }
  __device__ int col(int i) const { return (i * lanes + t) * N; }
  // rows of a warp's lanes end at different times: it goes on as one
  __device__ bool more(int rows) const { return LANES > 0 && LANES < 32 ? __any_sync(0xffffffffu, row < rows) : row < rows; }
};

template <int N> __device__ __forceinline__ void ln_weight(const void *w, int dtype, int col, int cols, float none, float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = w && col + k < cols ? load_value(w, dtype, col + k) : none;
}

template <class T, int N, int NV, int LANES, bool KEEP8>
__global__ void __launch_bounds__(ln_most_threads(LANES), 1)
ln_forward_kernel(const LnParams P) {
  __shared__ float scratch[2][32][2];
  LnPlace<N, NV, LANES> at;
  int slot = 0;
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    ln_weight<N>(P.w, P.w_dtype, at.col(i), P.cols, 1.f, w[i]);
    ln_weight<N>(P.b, P.w_dtype, at.col(i), P.cols, 0.f, b[i]);
  }
  const float over = 1.f / (float)P.cols;
  Pack<T, N> next[NV];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (row < P.rows && at.col(i) < P.cols) next[i] = *reinterpret_cast<const Pack<T, N> *>(static_cast<const T *>(P.x) + row * P.ld_x + at.col(i));
  };
  fetch(at.row);
  for (; at.more(P.rows); at.row += at.step) {
    const bool in = at.row < P.rows;
    float x[NV][N], sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        x[i][k] = in && at.col(i) < P.cols ? to_float(next[i].v[k]) : 0.f;
        sum[0] += x[i][k];
      }
    fetch(at.row + at.step);
    ln_sum<LANES, 1>(sum, scratch, slot);
    const float mean = sum[0] * over;
    float var[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float c = at.col(i) < P.cols ? x[i][k] - mean : 0.f;
        var[0] = fmaf(c, c, var[0]);
      }
    ln_sum<LANES, 1>(var, scratch, slot);
    const float rstd = 1.f / sqrtf(var[0] * over + P.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (KEEP8) {
        int code[N];
        const int e = pack8_lanes<N, false>(x[i], code);
        if (in && at.col(i) < P.ld_codes) {
          store_codes<N>(P.codes + at.row * P.ld_codes + at.col(i), code);
          if (at.col(i) % kPackGroup == 0) P.exps[at.row * (P.ld_codes / kPackGroup) + at.col(i) / kPackGroup] = (unsigned char)(e + 127);
        }
      }
      float y[N];
#pragma unroll
      for (int k = 0; k < N; ++k) y[k] = fmaf((x[i][k] - mean) * rstd, w[i][k], b[i][k]);
      if (in && at.col(i) < P.cols) store_pack<T, N>(static_cast<T *>(P.y) + at.row * P.ld_y + at.col(i), y);
    }
    if (in && at.t == 0) {
      if (P.mean) P.mean[at.row] = mean;
      if (P.rstd) P.rstd[at.row] = rstd;
    }
  }
}

template <class T, int N, int NV, int LANES, bool KEEP8>
__global__ void __launch_bounds__(ln_most_threads(LANES), 1)
ln_backward_kernel(const LnParams P) {
  extern __shared__ float joined[];  // [warps][2][cols] (LANES > 0)
  __shared__ float scratch[2][32][2];
  LnPlace<N, NV, LANES> at;
  int slot = 0;
  float w[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    ln_weight<N>(P.w, P.w_dtype, at.col(i), P.cols, 1.f, w[i]);
#pragma unroll
    for (int k = 0; k < N; ++k) dw[i][k] = db[i][k] = 0.f;
  }
  const float over = 1.f / (float)P.cols;
  Pack<T, N> next_x[NV], next_g[NV];
  Pack<signed char, N> next_c[NV];
  unsigned char next_e[NV];
  float next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](long long row) {
    if (row >= P.rows) return;
    next_mean = __ldg(P.mean + row);
    next_rstd = __ldg(P.rstd + row);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = at.col(i);
      if (c >= P.cols) continue;
      if (KEEP8) {
        next_c[i] = *reinterpret_cast<const Pack<signed char, N> *>(P.codes + row * P.ld_codes + c);
        next_e[i] = __ldg(P.exps + row * (P.ld_codes / kPackGroup) + c / kPackGroup);
      } else next_x[i] = *reinterpret_cast<const Pack<T, N> *>(static_cast<const T *>(P.x) + row * P.ld_x + c);
      next_g[i] = *reinterpret_cast<const Pack<T, N> *>(static_cast<const T *>(P.dy) + row * P.ld_dy + c);
    }
  };
  fetch(at.row);
  for (; at.more(P.rows); at.row += at.step) {
    const bool in = at.row < P.rows;
    const float mean = next_mean, rstd = next_rstd;
    float xh[NV][N], h[NV][N], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool here = in && at.col(i) < P.cols;
      float step = 0.f;
      if (KEEP8) step = here ? unpack8_step(next_e[i]) : 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float x = KEEP8 ? unpack8_value(next_c[i].v[k], step) : to_float(next_x[i].v[k]);
        const float g = here ? to_float(next_g[i].v[k]) : 0.f;
        xh[i][k] = here ? (x - mean) * rstd : 0.f;
        dw[i][k] = fmaf(g, xh[i][k], dw[i][k]);
        db[i][k] += g;
        h[i][k] = g * w[i][k];
        sum[0] += h[i][k];
        sum[1] = fmaf(h[i][k], xh[i][k], sum[1]);
      }
    }
    fetch(at.row + at.step);
    ln_sum<LANES, 2>(sum, scratch, slot);
    const float m0 = sum[0] * over, m1 = sum[1] * over;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!P.dx || !in || at.col(i) >= P.cols) continue;
      float d[N];
#pragma unroll
      for (int k = 0; k < N; ++k) d[k] = rstd * (h[i][k] - m0 - xh[i][k] * m1);
      store_pack<T, N>(static_cast<T *>(P.dx) + at.row * P.ld_dx + at.col(i), d);
    }
  }
  if (!P.part) return;
  float *part = P.part + (size_t)blockIdx.x * 2 * P.cols;
  if (LANES <= 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int c = at.col(i) + k;
        if (c < P.cols) { part[c] = dw[i][k]; part[P.cols + c] = db[i][k]; }
      }
    return;
  }
  // rows of one warp, then the warps of the CTA in order
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
      for (int o = LANES > 0 ? LANES : 32; o < 32; o <<= 1) {
        dw[i][k] += __shfl_xor_sync(0xffffffffu, dw[i][k], o);
        db[i][k] += __shfl_xor_sync(0xffffffffu, db[i][k], o);
      }
      const int c = at.col(i) + k;
      if (lane < (LANES > 0 ? LANES : 32) && c < P.cols) {
        joined[(warp * 2) * P.cols + c] = dw[i][k];
        joined[(warp * 2 + 1) * P.cols + c] = db[i][k];
      }
    }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * P.cols; c += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < (int)blockDim.x / 32; ++k) s += joined[k * 2 * P.cols + c];
    part[c] = s;
  }
}

// dw[c], db[c]: the CTAs' sums; 32 columns x 32 to a block, each of the 32 adds every 32nd part, and they are joined in order.
__global__ void __launch_bounds__(1024) ln_join_kernel(const float *__restrict__ part, int parts, int cols, void *dw, void *db, int dtype) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < 2 * cols)
#pragma unroll 4
    for (int k = w; k < parts; k += 32) v += __ldg(part + (size_t)k * 2 * cols + c);
  s[w][lane] = v;
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) v += s[k][lane];
  if (c < cols) {
    if (dw) store_value(dw, dtype, c, v);
  } else if (c < 2 * cols && db) store_value(db, dtype, c - cols, v);
}

struct LnShape { int n, nv, lanes, threads; };  // lanes 0: a CTA to a row

// N: 16 bytes of values where every row starts on such a boundary, else two values, else one.  Eight lanes to a row where they hold
// it and a group of 32 columns; a warp up to 512 columns; a CTA of as many warps as leave the fewest threads idle beyond.
LnShape ln_shape(int n, int cols, bool keep8) {
  const int vecs = (cols + n - 1) / n, most = kLnValues / n;
  LnShape s = {n, 1, 0, 0};
  const int padded = keep8 ? (cols + kPackGroup - 1) / kPackGroup * kPackGroup / n : vecs;  // (codes are written to the end of the group)
  auto least = [&](int lanes) { int nv = 1; while (nv < most && lanes * nv < padded) nv *= 2; return nv; };
  if (n >= 4 && padded <= 8 * most) { s.lanes = 8; s.nv = least(8); s.threads = kLnWarpThreads; return s; }
  if (padded <= 32 * most) { s.lanes = 32; s.nv = least(32); s.threads = kLnWarpThreads; return s; }
  int best = 1 << 30;
  for (int nv = most; nv >= 1; nv /= 2) {
    const int threads = ((padded + nv - 1) / nv + 31) & ~31;
    if (threads <= (nv == most ? kLnMaxThreads : kLnRowThreads) && threads * nv < best) { best = threads * nv; s.nv = nv; s.threads = threads; }
  }
  return s;
}

int ln_ctas(const LnShape &s, int rows) {
  const int rows_cta = s.lanes ? s.threads / s.lanes : 1;
  // a few CTAs to an SM: as many threads as the registers of the backward pass leave
  const int each = s.lanes ? 4 : std::max(1, std::min(8, 768 / s.threads));
  return std::max(1, std::min((rows + rows_cta - 1) / rows_cta, 148 * each));
}

template <class T, int N, int NV, bool KEEP8> cudaError_t ln_launch(const LnShape &s, const LnParams &P, bool backward, int ctas, cudaStream_t st) {
  auto go = [&](auto fwd, auto bwd, size_t smem) {
    if (backward) {
      if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute((const void *)bwd, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
        if (e != cudaSuccess) return e;
      }
      bwd<<<ctas, s.threads, smem, st>>>(P);
    } else fwd<<<ctas, s.threads, 0, st>>>(P);
    return cudaGetLastError();
  };
  const size_t joined = (size_t)kLnWarpThreads / 32 * 2 * P.cols * 4;
  if constexpr (N >= 4)
    if (s.lanes == 8) return go(ln_forward_kernel<T, N, NV, 8, KEEP8>, ln_backward_kernel<T, N, NV, 8, KEEP8>, joined);
  if (s.lanes == 32) return go(ln_forward_kernel<T, N, NV, 32, KEEP8>, ln_backward_kernel<T, N, NV, 32, KEEP8>, joined);
  if constexpr (N * NV == kLnValues)
    if (s.threads > kLnRowThreads) return go(ln_forward_kernel<T, N, NV, kLnWideRow, KEEP8>, ln_backward_kernel<T, N, NV, kLnWideRow, KEEP8>, 0);
  return go(ln_forward_kernel<T, N, NV, kLnRow, KEEP8>, ln_backward_kernel<T, N, NV, kLnRow, KEEP8>, 0);
}
template <class T, int N, bool KEEP8> cudaError_t ln_by_nv(const LnShape &s, const LnParams &P, bool backward, int ctas, cudaStream_t st) {
  constexpr int M = kLnValues / N;
  if (s.nv == 1) return ln_launch<T, N, 1, KEEP8>(s, P, backward, ctas, st);
  if (s.nv == 2) return ln_launch<T, N, 2, KEEP8>(s, P, backward, ctas, st);
  if constexpr (M >= 4) if (s.nv == 4) return ln_launch<T, N, 4, KEEP8>(s, P, backward, ctas, st);
  if constexpr (M >= 8) if (s.nv == 8) return ln_launch<T, N, 8, KEEP8>(s, P, backward, ctas, st);
  if constexpr (M >= 16) if (s.nv == 16) return ln_launch<T, N, 16, KEEP8>(s, P, backward, ctas, st);
  return cudaErrorInvalidValue;
}
template <class T, int N> cudaError_t ln_by_keep(const LnShape &s, const LnParams &P, bool backward, int ctas, cudaStream_t st) {
  return P.codes ? ln_by_nv<T, N, true>(s, P, backward, ctas, st) : ln_by_nv<T, N, false>(s, P, backward, ctas, st);
}
template <class T> cudaError_t ln_by_n(const LnShape &s, const LnParams &P, bool backward, int ctas, cudaStream_t st) {
  constexpr int W = 16 / sizeof(T);
  if (s.n == W) return ln_by_keep<T, W>(s, P, backward, ctas, st);
  if (s.n == 2) return ln_by_keep<T, 2>(s, P, backward, ctas, st);
  return ln_by_keep<T, 1>(s, P, backward, ctas, st);
}
cudaError_t ln_by_type(int dtype, const LnShape &s, const LnParams &P, bool backward, int ctas, cudaStream_t st) {
  if (dtype == TF_F32) return ln_by_n<float>(s, P, backward, ctas, st);
  if (dtype == TF_BF16) return ln_by_n<__nv_bfloat16>(s, P, backward, ctas, st);
  return ln_by_n<__half>(s, P, backward, ctas, st);
}

bool whole(const void *p, long long ld, int n, int bytes) { return ld % n == 0 && reinterpret_cast<uintptr_t>(p) % (n * bytes) == 0; }

int ln_check(const char *who, int rows, int cols, int dtype, int w_dtype, const void *codes, int ld_codes, const void *exps) {
  auto bad = [&](const char *what) { return tf::fail(TF_ERR_ARG, std::string(who) + ": " + what); };
  if (!known_dtype(dtype) || !known_dtype(w_dtype)) return bad("unknown type");
  if (rows < 0 || cols <= 0) return bad("bad size");
  if (cols > kLnMaxCols) return tf::fail(TF_ERR_UNSUPPORTED, std::string(who) + ": at most " + std::to_string(kLnMaxCols) + " columns");
  if (codes && (!exps || ld_codes < cols || ld_codes % kPackGroup != 0 || (reinterpret_cast<uintptr_t>(codes) & 31) != 0))
    return bad("codes need exponents, rows of whole groups of 32 and 32-byte alignment");
  return TF_OK;
}

}  // namespace

}  // namespace tfk

using namespace tfk;

extern "C" int tf_layer_norm_fwd(const void *x, long long ld_x, int dtype, const void *weight, const void *bias, int w_dtype, int rows, int cols,
                                 float eps, void *y, long long ld_y, float *mean, float *rstd, signed char *codes, int ld_codes,
                                 unsigned char *exponents, void *stream) {
  int rc = ln_check("tf_layer_norm_fwd", rows, cols, dtype, w_dtype, codes, ld_codes, exponents);
  if (rc != TF_OK || rows == 0) return rc;
  if (!x || !y) return tf::fail(TF_ERR_ARG, "tf_layer_norm_fwd: null argument");
  if (ld_x < cols || ld_y < cols) return tf::fail(TF_ERR_ARG, "tf_layer_norm_fwd: rows overlap");
  const int bytes = value_bytes(dtype);
  int n = 1;
  for (int k : {2, 16 / bytes})
    if (cols % k == 0 && whole(x, ld_x, k, bytes) && whole(y, ld_y, k, bytes)) n = k;
  LnParams P = {};
  P.x = x; P.ld_x = ld_x; P.w = weight; P.b = bias; P.w_dtype = w_dtype;
  P.rows = rows; P.cols = cols; P.eps = eps; P.y = y; P.ld_y = ld_y; P.mean = mean; P.rstd = rstd;
  P.codes = codes; P.ld_codes = codes ? (cols + kPackGroup - 1) / kPackGroup * kPackGroup : 0; P.exps = exponents;
  if (codes && ld_codes != P.ld_codes) return tf::fail(TF_ERR_ARG, "tf_layer_norm_fwd: codes need rows as long as the columns' groups");
  const LnShape s = ln_shape(n, cols, codes != nullptr);
  const cudaError_t e = ln_by_type(dtype, s, P, false, ln_ctas(s, rows), (cudaStream_t)stream);
  return e == cudaSuccess ? TF_OK : tf::fail(TF_ERR_CUDA, std::string("tf_layer_norm_fwd: ") + cudaGetErrorString(e));
}

extern "C" long long tf_layer_norm_work_floats(int rows, int cols) {
  if (rows < 0 || cols <= 0 || cols > kLnMaxCols) return 0;
  return 148ll * 8 * 2 * cols < 2ll * std::max(rows, 1) * cols ? 148ll * 8 * 2 * cols : 2ll * std::max(rows, 1) * cols;
}

extern "C" int tf_layer_norm_bwd(const void *x, long long ld_x, const signed char *codes, int ld_codes, const unsigned char *exponents, int dtype,
                                 const void *weight, int w_dtype, int rows, int cols, const float *mean, const float *rstd, const void *dy,
                                 long long ld_dy, void *dx, long long ld_dx, void *dweight, void *dbias, float *work, long long work_floats,
                                 void *stream) {
  int rc = ln_check("tf_layer_norm_bwd", rows, cols, dtype, w_dtype, codes, ld_codes, exponents);
  if (rc != TF_OK) return rc;
  const bool sums = dweight || dbias;
  if ((rows > 0 && ((!x && !codes) || !mean || !rstd || !dy)) || (sums && !work)) return tf::fail(TF_ERR_ARG, "tf_layer_norm_bwd: null argument");
  if ((!codes && ld_x < cols) || ld_dy < cols || (dx && ld_dx < cols)) return tf::fail(TF_ERR_ARG, "tf_layer_norm_bwd: rows overlap");
  if (sums && work_floats < tf_layer_norm_work_floats(rows, cols)) return tf::fail(TF_ERR_ARG, "tf_layer_norm_bwd: work space too small");
  const int bytes = value_bytes(dtype);
  int n = 1;
  for (int k : {2, 16 / bytes})
    if (cols % k == 0 && (codes || whole(x, ld_x, k, bytes)) && whole(dy, ld_dy, k, bytes) && (!dx || whole(dx, ld_dx, k, bytes))) n = k;
  LnParams P = {};
  P.x = x; P.ld_x = ld_x; P.w = weight; P.w_dtype = w_dtype; P.rows = rows; P.cols = cols;
  P.mean = const_cast<float *>(mean); P.rstd = const_cast<float *>(rstd);
  P.codes = const_cast<signed char *>(codes); P.ld_codes = ld_codes; P.exps = const_cast<unsigned char *>(exponents);
  P.dy = dy; P.ld_dy = ld_dy; P.dx = dx; P.ld_dx = ld_dx; P.part = sums ? work : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  const LnShape s = ln_shape(n, cols, false);
  const int ctas = ln_ctas(s, rows);
  cudaError_t e = cudaSuccess;
  if (rows > 0) e = ln_by_type(dtype, s, P, true, ctas, st);
  if (e == cudaSuccess && sums) {
    ln_join_kernel<<<(2 * cols + 31) / 32, 1024, 0, st>>>(work, rows > 0 ? ctas : 0, cols, dweight, dbias, w_dtype);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? TF_OK : tf::fail(TF_ERR_CUDA, std::string("tf_layer_norm_bwd: ") + cudaGetErrorString(e));
}
