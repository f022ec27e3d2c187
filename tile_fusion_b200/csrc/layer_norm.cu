// Layer norm over the last dimension, y = (x - mean) rstd w + b: the forward pass (layer_norm_grad.cu has the gradients).
//
// Bound by the row read and the row written.  A row stays in registers or in shared memory between its sums and its use, so it is
// read once; the variance is that of the centred values.  Threads walk the rows with the grid's stride and keep their columns'
// weights.  Up to 1 024 columns (768 with codes) a row belongs to eight lanes or a warp, and the next row is on its way in registers (50 021
// x 602 fp32: 39 us, 64 with a CTA to a row; 60 000 x 1 024 bf16 51 and 65; 30 000 x 1 024 fp32 with codes 75 and 58); wider ones to a CTA,
// R rows a turn so that a barrier serves them all, and the rows of two turns ahead are on their way into shared memory; a thread
// copies what it alone reads, so copies need no barrier.  Statistics are fp32 whatever the values' type.
//   120 001 x 256 fp32: 36 us (6.8 TB/s, part of it into L2); 16 384 x 4 096 bf16: 60 (4.5 TB/s; 0.63 instructions a cycle
//   and scheduler, with two barriers a turn: nothing is at its limit).
//   The pass can leave its input in 8 bits on the way (pack8.cuh), which the backward pass then reads in its place.
#include <algorithm>
#include <initializer_list>
#include <string>
#include <utility>

#include "layer_norm.cuh"

namespace tfk {

namespace {

// One row whose statistics are known.
template <class T, int AL, int PIECE, int NV, bool KEEP8, class Value, class Weights>
__device__ __forceinline__ void ln_write(const LnParams &P, Value x, long long row, bool in, float mean, float rstd, LnCols<T, PIECE> col, Weights weights) {
  constexpr int N = kLnN<T>;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Pack<T, N> raw = x(i);
    float v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = to_float(raw.v[k]);
    if (KEEP8) {
      unsigned code[N];
      const int e = pack8_lanes<N, false>(v, code), c = col(i, 0);
      if (in && c < P.ld_codes) {
        store_codes<N>(P.codes + row * P.ld_codes + c, code);
        if (c % kPackGroup == 0) P.exps[row * (P.ld_codes / kPackGroup) + c / kPackGroup] = (unsigned char)(e + 127);
      }
    }
    if (!in || col(i, 0) >= P.cols) continue;
    weights(i, [&](int k, float w, float b) { v[k] = fmaf((v[k] - mean) * rstd, w, b); });
    ln_store<T, AL, PIECE>(static_cast<T *>(P.y) + row * P.ld_y, col, i, P.cols, v);
  }
}

template <class T, int NV, class Value> __device__ __forceinline__ float ln_total(Value x) {
  float s = 0.f;  // (columns that do not exist are zero)
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Pack<T, kLnN<T>> v = x(i);
#pragma unroll
    for (int k = 0; k < kLnN<T>; ++k) s += to_float(v.v[k]);
  }
  return s;
}
template <class T, int NV, int PIECE, class Value> __device__ __forceinline__ float ln_spread(Value x, float mean, int cols, LnCols<T, PIECE> col) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Pack<T, kLnN<T>> v = x(i);
    if (col(i, kLnN<T> - 1) < cols) {
#pragma unroll
      for (int k = 0; k < kLnN<T>; ++k) {
        const float c = to_float(v.v[k]) - mean;
        s = fmaf(c, c, s);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kLnN<T>; ++k) {
        const float c = col(i, k) < cols ? to_float(v.v[k]) - mean : 0.f;
        s = fmaf(c, c, s);
      }
    }
  }
  return s;
}

// Weights of more than 16 values of a thread would take the registers of rows in flight where values are packed or make codes: they
// lie in shared memory, and CTAs of 128 threads are held to 102 registers (80 000 x 768 bf16: 48 us, 58 with weights in registers;
// 128 where every value is an access of its own, 50 021 x 999 bf16: 52 and 66).
template <class T, int NV, bool KEEP8> __host__ __device__ constexpr bool ln_shares() { return NV * kLnN<T> > 16 && (KEEP8 || sizeof(T) == 2); }
// A read that stays where it is: hoisted out of the loop over rows it would take the registers it is there to save.
__device__ __forceinline__ float4 ln_shared4(const float4 *p) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"((unsigned)__cvta_generic_to_shared(p)));
  return v;
}

// Eight lanes or a warp to a row.
template <class T, int AL, int PIECE, int NV, int LANES, bool KEEP8>
__global__ void __launch_bounds__(NV * kLnN<T> > 16 ? kLnWarpThreads / 2 : kLnWarpThreads, ln_shares<T, NV, KEEP8>() ? (PIECE > 1 ? 5 : 4) : 0) ln_forward_kernel(const LnParams P) {
  constexpr int N = kLnN<T>;
  LnPlace<T, LANES> at;
  const int t = at.t;
  const LnCols<T, PIECE> col = {t, LANES};
  constexpr bool SHARED = ln_shares<T, NV, KEEP8>();
  __shared__ float4 sw[SHARED ? NV * N / 4 : 1][SHARED ? 32 : 1], sb[SHARED ? NV * N / 4 : 1][SHARED ? 32 : 1];
  float w[SHARED ? 1 : NV][N], b[SHARED ? 1 : NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float(&wi)[N] = w[SHARED ? 0 : i], (&bi)[N] = b[SHARED ? 0 : i];
    if (SHARED && threadIdx.x >= 32) break;
    ln_weight<T, PIECE>(P.w, P, col, i, 1.f, wi);
    ln_weight<T, PIECE>(P.b, P, col, i, 0.f, bi);
    if constexpr (SHARED)
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        sw[(i * N + k) / 4][t] = make_float4(wi[k], wi[k + 1], wi[k + 2], wi[k + 3]);
        sb[(i * N + k) / 4][t] = make_float4(bi[k], bi[k + 1], bi[k + 2], bi[k + 3]);
      }
  }
  if (SHARED) __syncthreads();
  auto weights = [&](int i, auto f) {
    if constexpr (SHARED) {
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const float4 p = ln_shared4(&sw[(i * N + k) / 4][t]), q = ln_shared4(&sb[(i * N + k) / 4][t]);
        f(k, p.x, q.x); f(k + 1, p.y, q.y); f(k + 2, p.z, q.z); f(k + 3, p.w, q.w);
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) f(k, w[i][k], b[i][k]);
    }
  };
  const float over = 1.f / (float)P.cols;
  Pack<T, N> next[NV];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) next[i] = ln_load<T, AL, PIECE>(static_cast<const T *>(P.x) + row * P.ld_x, col, i, P.cols, row < P.rows);
  };
  fetch(at.row);
  for (; at.more(P.rows); at.row += at.step) {
    const bool in = at.row < P.rows;
    Pack<T, N> now[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) now[i] = next[i];
    fetch(at.row + at.step);
    auto x = [&](int i) { return now[i]; };
    float sum[1] = {ln_total<T, NV>(x)};
    ln_sum<LANES, 1>(sum);
    const float mean = sum[0] * over;
    float var[1] = {ln_spread<T, NV, PIECE>(x, mean, P.cols, col)};
    ln_sum<LANES, 1>(var);
    const float rstd = rsqrtf(var[0] * over + P.eps);
    ln_write<T, AL, PIECE, NV, KEEP8>(P, x, at.row, in, mean, rstd, col, weights);
    if (in && t == 0) {
      if (P.mean) P.mean[at.row] = mean;
      if (P.rstd) P.rstd[at.row] = rstd;
    }
  }
}

// A CTA to a row, R rows a turn.  Shared memory: [turn][row][NV][thread].
template <class T, int NV> __host__ __device__ constexpr int ln_turn_bytes(int threads) { return ln_rows_at_once<NV>() * NV * threads * 16; }
template <class T, int AL, int PIECE, int NV, bool KEEP8>
__global__ void __launch_bounds__(kLnRowThreads, 1) ln_forward_rows_kernel(const LnParams P) {
  constexpr int N = kLnN<T>, R = ln_rows_at_once<NV>(), AHEAD = ln_ahead<NV>();
  extern __shared__ float4 rows_smem[];
  __shared__ float scratch[2][kLnRowThreads / 32 * R];
  const int t = threadIdx.x, lanes = blockDim.x;
  Pack<T, N> *sx = reinterpret_cast<Pack<T, N> *>(rows_smem);
  const LnCols<T, PIECE> col = {t, lanes};
  auto at = [&](int turn, int r, int i) { return ((turn * R + r) * NV + i) * lanes + t; };
  int slot = 0;
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    ln_weight<T, PIECE>(P.w, P, col, i, 1.f, w[i]);
    ln_weight<T, PIECE>(P.b, P, col, i, 0.f, b[i]);
  }
  auto weights = [&](int i, auto f) {
#pragma unroll
    for (int k = 0; k < N; ++k) f(k, w[i][k], b[i][k]);
  };
  const float over = 1.f / (float)P.cols;
  const long long step = gridDim.x * (long long)R;
  auto fetch = [&](long long row, int turn) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = row + r < P.rows;
#pragma unroll
      for (int i = 0; i < NV; ++i) ln_copy<T, AL, PIECE>(sx + at(turn, r, i), static_cast<const T *>(P.x) + (in ? row + r : 0) * P.ld_x, col, i, P.cols, in);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  long long row = blockIdx.x * (long long)R;
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) fetch(row + k * step, k);
  int turn = 0;
  for (; row < P.rows; row += step) {
    fetch(row + AHEAD * step, turn == 0 ? AHEAD : turn - 1);  // (a thread has read its part of that turn)
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
    float sum[R], var[R];
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] = ln_total<T, NV>([&](int i) { return sx[at(turn, r, i)]; });
    ln_sum_cta<R>(sum, scratch, slot);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum[r] *= over;  // the mean
      var[r] = ln_spread<T, NV, PIECE>([&](int i) { return sx[at(turn, r, i)]; }, sum[r], P.cols, col);
    }
    ln_sum_cta<R>(var, scratch, slot);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = row + r < P.rows;
      const float rstd = rsqrtf(var[r] * over + P.eps);
      ln_write<T, AL, PIECE, NV, KEEP8>(P, [&](int i) { return sx[at(turn, r, i)]; }, row + r, in, sum[r], rstd, col, weights);
      if (in && t == 0) {
        if (P.mean) P.mean[row + r] = sum[r];
        if (P.rstd) P.rstd[row + r] = rstd;
      }
    }
    turn = turn == AHEAD ? 0 : turn + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <class T, int AL, int PIECE, bool KEEP8> cudaError_t ln_by_nv(const LnShape &s, const LnParams &P, cudaStream_t st) {
  int ctas;
#define TF_LN(NV)                                                                                                                              \
  if (s.nv == NV) {                                                                                                                            \
    if constexpr ((NV & (NV - 1)) == 0 && (NV > 1 || KEEP8 || sizeof(T) == 2)) if (s.lanes == 0)                                                                                                                          \
      return ln_go(ln_forward_rows_kernel<T, AL, PIECE, NV, KEEP8>, s, P, ln_rows_at_once<NV>(), (ln_ahead<NV>() + 1) * ln_turn_bytes<T, NV>(s.threads), ctas, st); \
    if constexpr (NV * kLnN<T> < 32 || !KEEP8) if (s.lanes == 32) return ln_go(ln_forward_kernel<T, AL, PIECE, NV, 32, KEEP8>, s, P, s.threads / 32, 0, ctas, st);                         \
    if constexpr (NV <= 16 / kLnN<T>) {                                                                                                        \
      return ln_go(ln_forward_kernel<T, AL, PIECE, NV, 8, KEEP8>, s, P, kLnWarpThreads / 8, 0, ctas, st);                                             \
    }                                                                                                                                          \
  }
  TF_LN(1) TF_LN(2) TF_LN(4)
  if constexpr (sizeof(T) == 4) { TF_LN(5) TF_LN(6) TF_LN(8) } else { TF_LN(3) }
#undef TF_LN
  return cudaErrorInvalidValue;
}
template <class T> cudaError_t ln_by_align(const LnShape &s, const LnParams &P, cudaStream_t st) {
  constexpr int N = kLnN<T>;
  if (P.codes) return s.al == N ? ln_by_nv<T, N, N, true>(s, P, st) : s.al == 2 ? ln_by_nv<T, 2, N, true>(s, P, st) : ln_by_nv<T, 1, N, true>(s, P, st);
  if (s.piece == N) return s.al == N ? ln_by_nv<T, N, N, false>(s, P, st) : ln_by_nv<T, 1, N, false>(s, P, st);
  if (s.piece == 2) return s.al == 2 ? ln_by_nv<T, 2, 2, false>(s, P, st) : ln_by_nv<T, 1, 2, false>(s, P, st);
  return ln_by_nv<T, 1, 1, false>(s, P, st);
}

}  // namespace

int ln_check(const char *who, int rows, int cols, int dtype, int w_dtype, const void *codes, int ld_codes, const void *exps) {
  auto bad = [&](const char *what) { return tf::fail(TF_ERR_ARG, std::string(who) + ": " + what); };
  if (!known_dtype(dtype) || !known_dtype(w_dtype)) return bad("unknown type");
  if (rows < 0 || rows > kMaxRows || cols <= 0) return bad("bad size");
  if (cols > kLnMaxCols) return tf::fail(TF_ERR_UNSUPPORTED, std::string(who) + ": at most " + std::to_string(kLnMaxCols) + " columns");
  if (codes && (!exps || ld_codes != (cols + kPackGroup - 1) / kPackGroup * kPackGroup || (reinterpret_cast<uintptr_t>(codes) & 31) != 0))
    return bad("codes need exponents, rows as long as the columns' groups of 32, and 32-byte alignment");
  return TF_OK;
}

}  // namespace tfk

using namespace tfk;

extern "C" int tf_layer_norm_fwd(const void *x, long long ld_x, int dtype, const void *weight, const void *bias, int w_dtype, int rows, int cols,
                                 float eps, void *y, long long ld_y, float *mean, float *rstd, signed char *codes, int ld_codes,
                                 unsigned char *exponents, void *stream) {
  const int rc = ln_check("tf_layer_norm_fwd", rows, cols, dtype, w_dtype, codes, ld_codes, exponents);
  if (rc != TF_OK || rows == 0) return rc;
  if (!x || !y) return tf::fail(TF_ERR_ARG, "tf_layer_norm_fwd: null argument");
  if (ld_x < cols || ld_y < cols) return tf::fail(TF_ERR_ARG, "tf_layer_norm_fwd: rows overlap");
  const int bytes = value_bytes(dtype);
  LnParams P = {};
  P.x = x; P.ld_x = ld_x; P.w = weight; P.b = bias; P.w_dtype = w_dtype;
  P.w_whole = ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(bias)) & 15) == 0;
  P.rows = rows; P.cols = cols; P.eps = eps; P.y = y; P.ld_y = ld_y; P.mean = mean; P.rstd = rstd;
  P.codes = codes; P.ld_codes = ld_codes; P.exps = exponents;
  // (codes reach to the end of the columns' group)
  const LnShape s = ln_shape(ln_pieces(cols, bytes, codes != nullptr, {{x, ld_x}, {y, ld_y}}), codes ? ld_codes : cols, bytes, codes ? 768 : 1024);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == TF_F32 ? ln_by_align<float>(s, P, st) : dtype == TF_BF16 ? ln_by_align<__nv_bfloat16>(s, P, st) : ln_by_align<__half>(s, P, st);
  return e == cudaSuccess ? TF_OK : tf::fail(TF_ERR_CUDA, std::string("tf_layer_norm_fwd: ") + cudaGetErrorString(e));
}
