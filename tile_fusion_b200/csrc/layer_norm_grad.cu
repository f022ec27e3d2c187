// The gradients of the layer norm (layer_norm.cu):
//
//   dx = rstd (h - mean(h) - xh mean(h xh)),   h = dy w,  xh = (x - mean) rstd;   dw = sum_rows dy xh;   db = sum_rows dy
//
// Bound by two rows read and one written; x may come in 8 bits (pack8.cuh).  Threads walk the rows with the grid's stride, so that a
// thread's columns stay the same: the weight is read once, and the sums over rows of dw and db stay in registers until the end,
// where they are joined in shared memory; a second launch adds the CTAs' sums in order, so results don't depend on scheduling.
//   Up to 512 columns a row belongs to eight lanes or a warp, and the next row is on its way in registers.
// Wider rows belong to a CTA (two sums to each column take the registers: 60 000 x 640 bf16 53 us, 130 with a warp to a row), R at a
// time so that a barrier serves them all, and come through shared memory with asynchronous copies two turns ahead; a thread copies what
// it alone reads, so copies need no barrier.
// Sums are fp32 whatever the values' type.
//   120 001 x 256 fp32: 66 us (5.6 TB/s); 16 384 x 4 096 bf16: 85 (4.7 TB/s at 0.65 instructions a cycle and scheduler); 50 021 x 602 fp32 from 8 bits: 66 (4.1).
#include <algorithm>
#include <initializer_list>
#include <string>
#include <utility>

#include "layer_norm.cuh"

namespace tfk {

namespace {

// Eight lanes or a warp to a row.
template <class T, int AL, int PIECE, int NV, int LANES, bool KEEP8>
__global__ void __launch_bounds__(kLnWarpThreads) ln_backward_kernel(const LnParams P) {
  constexpr int N = kLnN<T>;
  extern __shared__ float joined[];  // [warps][2][cols]
  LnPlace<T, LANES> at;
  const LnCols<T, PIECE> col = {at.t, LANES};
  float w[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    ln_weight<T, PIECE>(P.w, P, col, i, 1.f, w[i]);
#pragma unroll
    for (int k = 0; k < N; ++k) dw[i][k] = db[i][k] = 0.f;
  }
  const float over = 1.f / (float)P.cols;
  Pack<T, N> next_x[NV], next_g[NV];
  Pack<signed char, N> next_c[NV];
  unsigned char next_e[NV];
  float next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](long long row) {
    const bool in = row < P.rows;
    if (in) { next_mean = __ldg(P.mean + row); next_rstd = __ldg(P.rstd + row); }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i, 0);
      if (!KEEP8) next_x[i] = ln_load<T, AL, PIECE>(static_cast<const T *>(P.x) + row * P.ld_x, col, i, P.cols, in);
      else if (in && c < P.cols) {
        next_c[i] = *reinterpret_cast<const Pack<signed char, N> *>(P.codes + row * P.ld_codes + c);
        next_e[i] = __ldg(P.exps + row * (P.ld_codes / kPackGroup) + c / kPackGroup);
      }
      next_g[i] = ln_load<T, AL, PIECE>(static_cast<const T *>(P.dy) + row * P.ld_dy, col, i, P.cols, in);
    }
  };
  fetch(at.row);
  for (; at.more(P.rows); at.row += at.step) {
    const bool in = at.row < P.rows;
    const float mean = next_mean, rstd = next_rstd;
    float xh[NV][N], h[NV][N], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[N];
      if (KEEP8) unpack8_values<N>(next_c[i], unpack8_step(next_e[i]), x);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const bool here = in && col(i, k) < P.cols;
        const float g = here ? to_float(next_g[i].v[k]) : 0.f;
        xh[i][k] = here ? ((KEEP8 ? x[k] : to_float(next_x[i].v[k])) - mean) * rstd : 0.f;
        dw[i][k] = fmaf(g, xh[i][k], dw[i][k]);
        db[i][k] += g;
        h[i][k] = g * w[i][k];
        sum[0] += h[i][k];
        sum[1] = fmaf(h[i][k], xh[i][k], sum[1]);
      }
    }
    fetch(at.row + at.step);
    ln_sum<LANES, 2>(sum);
    const float m0 = sum[0] * over, m1 = sum[1] * over;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!P.dx || !in || col(i, 0) >= P.cols) continue;
      float d[N];
#pragma unroll
      for (int k = 0; k < N; ++k) d[k] = rstd * (h[i][k] - m0 - xh[i][k] * m1);
      ln_store<T, AL, PIECE>(static_cast<T *>(P.dx) + at.row * P.ld_dx, col, i, P.cols, d);
    }
  }
  if (!P.part) return;
  float *part = P.part + (size_t)blockIdx.x * 2 * P.cols;
  // rows of one warp, then the warps of the CTA in order
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) {
        dw[i][k] += __shfl_xor_sync(0xffffffffu, dw[i][k], o);
        db[i][k] += __shfl_xor_sync(0xffffffffu, db[i][k], o);
      }
      const int c = col(i, k);
      if (lane < LANES && c < P.cols) {
        joined[(warp * 2) * P.cols + c] = dw[i][k];
        joined[(warp * 2 + 1) * P.cols + c] = db[i][k];
      }
    }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * P.cols; c += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < blockDim.x / 32; ++k) s += joined[k * 2 * P.cols + c];
    part[c] = s;
  }
}

// A CTA to a row, R rows a turn.  Shared memory: [turn][row][NV][thread] of (x or codes), then of dy.
template <int NV> __host__ __device__ constexpr int ln_grad_rows() { return NV >= 4 ? 1 : 2; }
template <class T, int NV, bool KEEP8> __host__ __device__ constexpr int ln_turn_bytes(int threads) {
  return ln_grad_rows<NV>() * NV * threads * (16 + (KEEP8 ? kLnN<T> : 16));
}
template <class T, int AL, int PIECE, int NV, bool KEEP8>
__global__ void __launch_bounds__(kLnRowThreads, 1) ln_backward_rows_kernel(const LnParams P) {
  constexpr int N = kLnN<T>, R = ln_grad_rows<NV>(), AHEAD = ln_ahead<NV>(), TURNS = AHEAD + 1;
  extern __shared__ float4 rows_smem[];
  __shared__ float scratch[2][kLnRowThreads / 32 * 2 * R];
  using Kept = Pack<signed char, N>;
  const int t = threadIdx.x, lanes = blockDim.x;
  Pack<T, N> *sg = reinterpret_cast<Pack<T, N> *>(rows_smem);
  Pack<T, N> *sx = sg + (KEEP8 ? 0 : TURNS * R * NV * lanes);
  Kept *sc = reinterpret_cast<Kept *>(sg + TURNS * R * NV * lanes);
  const LnCols<T, PIECE> col = {t, lanes};
  auto at = [&](int turn, int r, int i) { return ((turn * R + r) * NV + i) * lanes + t; };
  int slot = 0;
  float w[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    ln_weight<T, PIECE>(P.w, P, col, i, 1.f, w[i]);
#pragma unroll
    for (int k = 0; k < N; ++k) dw[i][k] = db[i][k] = 0.f;
  }
  const float over = 1.f / (float)P.cols;
  const long long step = gridDim.x * (long long)R;
  auto fetch = [&](long long row, int turn) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = row + r < P.rows;
      const long long q = in ? row + r : 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (KEEP8) {
          const unsigned dst = (unsigned)__cvta_generic_to_shared(sc + at(turn, r, i));
          const bool here = in && col(i, 0) < P.cols;
          asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(P.codes + q * P.ld_codes + (here ? col(i, 0) : 0)), "n"(N),
                       "r"(here ? N : 0) : "memory");
        } else ln_copy<T, AL, PIECE>(sx + at(turn, r, i), static_cast<const T *>(P.x) + q * P.ld_x, col, i, P.cols, in);
        ln_copy<T, AL, PIECE>(sg + at(turn, r, i), static_cast<const T *>(P.dy) + q * P.ld_dy, col, i, P.cols, in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  long long row = blockIdx.x * (long long)R;
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) fetch(row + k * step, k);
  int turn = 0;
  // what a row has besides its values comes a turn ahead too
  float next_mean[R], next_rstd[R];
  unsigned char next_e[KEEP8 ? R : 1][NV];
  auto fetch_stats = [&](long long row) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = row + r < P.rows;
      next_mean[r] = in ? __ldg(P.mean + row + r) : 0.f;
      next_rstd[r] = in ? __ldg(P.rstd + row + r) : 0.f;
      if (KEEP8)
#pragma unroll
        for (int i = 0; i < NV; ++i)
          next_e[r][i] = in && col(i, 0) < P.cols ? __ldg(P.exps + (row + r) * (P.ld_codes / kPackGroup) + col(i, 0) / kPackGroup) : 127;
    }
  };
  fetch_stats(row);
  for (; row < P.rows; row += step) {
    float mean[R], rstd[R], unit[KEEP8 ? R : 1][NV], sum[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = next_mean[r];
      rstd[r] = next_rstd[r];
      if (KEEP8)
#pragma unroll
        for (int i = 0; i < NV; ++i) unit[r][i] = unpack8_step(next_e[r][i]);
    }
    constexpr bool KEEP = NV == 1;
    Pack<T, N> kept_g[KEEP ? R : 1];
    float kept_x[KEEP ? R : 1][N];
    fetch_stats(row + step);
    fetch(row + AHEAD * step, turn == 0 ? AHEAD : turn - 1);  // (a thread has read its part of that turn)
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
    auto hats = [&](int r, int i, float (&xh)[N]) {
      if (KEEP8) unpack8_values<N>(sc[at(turn, r, i)], unit[KEEP8 ? r : 0][i], xh);
      else {
        const Pack<T, N> x = sx[at(turn, r, i)];
#pragma unroll
        for (int k = 0; k < N; ++k) xh[k] = to_float(x.v[k]);
      }
#pragma unroll
      for (int k = 0; k < N; ++k) xh[k] = (xh[k] - mean[r]) * rstd[r];
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum[2 * r] = sum[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float xh[N];
        hats(r, i, xh);
        const Pack<T, N> g = sg[at(turn, r, i)];
        if (KEEP) {
          kept_g[r] = g;
#pragma unroll
          for (int k = 0; k < N; ++k) kept_x[r][k] = xh[k];
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {  // (dy is zero where there is no value, and xh finite)
          const float gk = to_float(g.v[k]), h = gk * w[i][k];
          dw[i][k] = fmaf(gk, xh[k], dw[i][k]);
          db[i][k] += gk;
          sum[2 * r] += h;
          sum[2 * r + 1] = fmaf(h, xh[k], sum[2 * r + 1]);
        }
      }
    }
    if (P.dx) {
      // (with more than one access a thread its values are read and converted again rather than kept: registers bound the rows in flight)
      ln_sum_cta<2 * R>(sum, scratch, slot);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float m0 = sum[2 * r] * over, m1 = sum[2 * r + 1] * over;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (row + r >= P.rows || col(i, 0) >= P.cols) continue;
          float xh[N], d[N];
          Pack<T, N> g;
          if (KEEP) {
            g = kept_g[r];
#pragma unroll
            for (int k = 0; k < N; ++k) xh[k] = kept_x[r][k];
          } else {
            hats(r, i, xh);
            g = sg[at(turn, r, i)];
          }
#pragma unroll
          for (int k = 0; k < N; ++k) d[k] = rstd[r] * (to_float(g.v[k]) * w[i][k] - m0 - xh[k] * m1);
          ln_store<T, AL, PIECE>(static_cast<T *>(P.dx) + (row + r) * P.ld_dx, col, i, P.cols, d);
        }
      }
    }
    turn = turn == AHEAD ? 0 : turn + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!P.part) return;
  float *part = P.part + (size_t)blockIdx.x * 2 * P.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = col(i, k);
      if (c < P.cols) { part[c] = dw[i][k]; part[P.cols + c] = db[i][k]; }
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

template <class T, int AL, int PIECE, bool KEEP8> cudaError_t ln_by_nv(const LnShape &s, const LnParams &P, int &ctas, cudaStream_t st) {
  const size_t joined = (size_t)s.threads / 32 * 2 * P.cols * 4;
#define TF_LN(NV)                                                                                                                                  \
  if (s.nv == NV) {                                                                                                                                \
    if (s.lanes == 0)                                                                                                                              \
      return ln_go(ln_backward_rows_kernel<T, AL, PIECE, NV, KEEP8>, s, P, ln_grad_rows<NV>(), (ln_ahead<NV>() + 1) * ln_turn_bytes<T, NV, KEEP8>(s.threads), ctas, st); \
    if constexpr (NV <= 16 / kLnN<T>) {                                                                                                            \
      if (s.lanes == 32) return ln_go(ln_backward_kernel<T, AL, PIECE, NV, 32, KEEP8>, s, P, s.threads / 32, joined, ctas, st);                    \
      return ln_go(ln_backward_kernel<T, AL, PIECE, NV, 8, KEEP8>, s, P, kLnWarpThreads / 8, joined, ctas, st);                                           \
    }                                                                                                                                              \
  }
  TF_LN(1) TF_LN(2) TF_LN(4)
  if constexpr (sizeof(T) == 4) { TF_LN(8) }
#undef TF_LN
  return cudaErrorInvalidValue;
}
template <class T> cudaError_t ln_by_align(const LnShape &s, const LnParams &P, int &ctas, cudaStream_t st) {
  constexpr int N = kLnN<T>;
  if (P.codes) return s.al == N ? ln_by_nv<T, N, N, true>(s, P, ctas, st) : s.al == 2 ? ln_by_nv<T, 2, N, true>(s, P, ctas, st) : ln_by_nv<T, 1, N, true>(s, P, ctas, st);
  if (s.piece == N) return s.al == N ? ln_by_nv<T, N, N, false>(s, P, ctas, st) : ln_by_nv<T, 1, N, false>(s, P, ctas, st);
  if (s.piece == 2) return s.al == 2 ? ln_by_nv<T, 2, 2, false>(s, P, ctas, st) : ln_by_nv<T, 1, 2, false>(s, P, ctas, st);
  return ln_by_nv<T, 1, 1, false>(s, P, ctas, st);
}

}  // namespace

}  // namespace tfk

using namespace tfk;

extern "C" long long tf_layer_norm_work_floats(int rows, int cols) {
  if (rows < 0 || cols <= 0 || cols > kLnMaxCols) return 0;
  return 2ll * cols * std::min(kLnMaxCtas, std::max(rows, 1));
}

extern "C" int tf_layer_norm_bwd(const void *x, long long ld_x, const signed char *codes, int ld_codes, const unsigned char *exponents, int dtype,
                                 const void *weight, int w_dtype, int rows, int cols, const float *mean, const float *rstd, const void *dy,
                                 long long ld_dy, void *dx, long long ld_dx, void *dweight, void *dbias, float *work, long long work_floats,
                                 void *stream) {
  const int rc = ln_check("tf_layer_norm_bwd", rows, cols, dtype, w_dtype, codes, ld_codes, exponents);
  if (rc != TF_OK) return rc;
  const bool sums = dweight || dbias;
  if ((rows > 0 && ((!x && !codes) || !mean || !rstd || !dy)) || (sums && !work)) return tf::fail(TF_ERR_ARG, "tf_layer_norm_bwd: null argument");
  if ((!codes && ld_x < cols) || ld_dy < cols || (dx && ld_dx < cols)) return tf::fail(TF_ERR_ARG, "tf_layer_norm_bwd: rows overlap");
  if (sums && work_floats < tf_layer_norm_work_floats(rows, cols)) return tf::fail(TF_ERR_ARG, "tf_layer_norm_bwd: work space too small");
  const int bytes = value_bytes(dtype);
  LnParams P = {};
  P.x = x; P.ld_x = ld_x; P.w = weight; P.w_dtype = w_dtype; P.w_whole = (reinterpret_cast<uintptr_t>(weight) & 15) == 0;
  P.rows = rows; P.cols = cols;
  P.mean = const_cast<float *>(mean); P.rstd = const_cast<float *>(rstd);
  P.codes = const_cast<signed char *>(codes); P.ld_codes = ld_codes; P.exps = const_cast<unsigned char *>(exponents);
  P.dy = dy; P.ld_dy = ld_dy; P.dx = dx; P.ld_dx = ld_dx; P.part = sums ? work : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  const LnShape s = ln_shape(ln_pieces(cols, bytes, codes != nullptr, {{codes ? nullptr : x, ld_x}, {dy, ld_dy}, {dx, ld_dx}}), cols, bytes, 512);
  int ctas = 0;
  cudaError_t e = cudaSuccess;
  if (rows > 0)
    e = dtype == TF_F32 ? ln_by_align<float>(s, P, ctas, st) : dtype == TF_BF16 ? ln_by_align<__nv_bfloat16>(s, P, ctas, st) : ln_by_align<__half>(s, P, ctas, st);
  if (e == cudaSuccess && sums) {
    ln_join_kernel<<<(2 * cols + 31) / 32, 1024, 0, st>>>(work, ctas, cols, dweight, dbias, w_dtype);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? TF_OK : tf::fail(TF_ERR_CUDA, std::string("tf_layer_norm_bwd: ") + cudaGetErrorString(e));
}
