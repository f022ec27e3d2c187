// What the two passes of the layer norm share (layer_norm.cu, layer_norm_grad.cu): how a row lies over threads.
//
// A thread holds N columns (16 bytes of values) NV times, in pieces of PIECE neighbours: all N, two or one, whichever divides the
// width, so that rows one behind the other start on whole pieces.  A warp's pieces lie side by side, and its accesses are whole
// sectors.  (With the 8 bits always N: a group of 32 belongs to few lanes.)  Accesses are of AL values, a piece or, where operands
// are aligned otherwise, less.  Which columns a thread adds up depends on the width alone, so results do not depend on alignment.
#pragma once
#include "pack8.cuh"
#include "tf_internal.h"

namespace tfk {

constexpr int kLnWarpThreads = 256;            // CTAs whose rows have a warp or less
constexpr int kLnRowThreads = 512;             // the largest CTA of a row: 128 registers a thread
constexpr int kLnMaxCols = 16384;              // 32 values to each of them
constexpr int kLnMaxCtas = 148 * 8;

struct LnParams {
  const void *x; long long ld_x;
  const void *w, *b; int w_dtype; bool w_whole;  // w_whole: both start on 16 bytes
  int rows, cols; float eps;
  void *y; long long ld_y;
  float *mean, *rstd;
  signed char *codes; int ld_codes; unsigned char *exps;   // forward: written (null: not); backward: read instead of x
  const void *dy; long long ld_dy;
  void *dx; long long ld_dx;
  float *part;                                             // [CTA][2][cols]
};

template <class T> constexpr int kLnN = 16 / (int)sizeof(T);

// The column of value k of a thread's i-th access; PIECE neighbouring columns of a thread.
template <class T, int PIECE> struct LnCols {
  int t, lanes;
  __device__ int operator()(int i, int k) const { return ((i * (kLnN<T> / PIECE) + k / PIECE) * lanes + t) * PIECE + k % PIECE; }
};

template <class T, int AL, int PIECE> __device__ __forceinline__ Pack<T, kLnN<T>> ln_load(const T *row, LnCols<T, PIECE> col, int i, int cols, bool in) {
  constexpr int N = kLnN<T>;
  Pack<T, N> v;
#pragma unroll
  for (int p = 0; p < N; p += AL) {
    Pack<T, AL> a;
#pragma unroll
    for (int k = 0; k < AL; ++k) a.v[k] = from_float<T>(0.f);
    if (in && col(i, p) < cols) a = *reinterpret_cast<const Pack<T, AL> *>(row + col(i, p));
#pragma unroll
    for (int k = 0; k < AL; ++k) v.v[p + k] = a.v[k];
  }
  return v;
}
template <class T, int AL, int PIECE> __device__ __forceinline__ void ln_store(T *row, LnCols<T, PIECE> col, int i, int cols, const float (&v)[kLnN<T>]) {
  constexpr int N = kLnN<T>;
#pragma unroll
  for (int p = 0; p < N; p += AL) {
    if (col(i, p) >= cols) break;
    float a[AL];
#pragma unroll
    for (int k = 0; k < AL; ++k) a[k] = v[p + k];
    store_pack<T, AL>(row + col(i, p), a);
  }
}
// A thread's weights of its i-th access, `none` where there are none.
template <class T, int PIECE> __device__ __forceinline__ void ln_weight(const void *w, const LnParams &P, LnCols<T, PIECE> cols_, int i, float none, float (&v)[kLnN<T>]) {
  constexpr int N = kLnN<T>;
  const int col = cols_(i, 0);
  if (PIECE == N && w && P.w_whole && col + N <= P.cols) {
    if (P.w_dtype == TF_F32) {
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(w) + col + k));
        v[k] = q.x; v[k + 1] = q.y; v[k + 2] = q.z; v[k + 3] = q.w;
      }
      return;
    }
    const unsigned *u = reinterpret_cast<const unsigned *>(static_cast<const unsigned short *>(w) + col);
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const unsigned q = __ldg(u + k / 2);
      if (P.w_dtype == TF_BF16) { v[k] = __uint_as_float(q << 16); v[k + 1] = __uint_as_float(q & 0xffff0000u); }
      else { const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&q)); v[k] = f.x; v[k + 1] = f.y; }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = w && cols_(i, k) < P.cols ? load_value(w, P.w_dtype, cols_(i, k)) : none;
}

// K sums over LANES lanes.
template <int LANES, int K> __device__ __forceinline__ void ln_sum(float (&v)[K]) {
#pragma unroll
  for (int k = LANES / 2; k; k >>= 1)
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], k);
}
// K sums (a power of two) over the CTA; `slot` alternates between two scratch arrays.  A lane hands on half of its sums and adds
// up the other half until it has one: 6 shuffles for four sums where one at a time would take 20.  Behind the barrier the lanes
// of each warp add up the warps' sums in the same order.
template <int K> __device__ __forceinline__ void ln_sum_cta(float (&v)[K], float (*scratch)[kLnRowThreads / 32 * K], int &slot) {
  const int lane = threadIdx.x & 31, warps = blockDim.x / 32;
  if (warps == 1) return ln_sum<32, K>(v);
#pragma unroll
  for (int k = K / 2, o = 16; k; k >>= 1, o >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < k; ++i) {
      const float given = upper ? v[i] : v[i + k], kept = upper ? v[i + k] : v[i];
      v[i] = kept + __shfl_xor_sync(0xffffffffu, given, o);
    }
  }
#pragma unroll
  for (int o = 16 / K; o; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  if (lane % (32 / K) == 0) scratch[slot][(threadIdx.x >> 5) * K + lane / (32 / K)] = v[0];
  __syncthreads();  // (one to a sum: the scratch array of the sum before last has been read by then)
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < kLnRowThreads / 32 * K; i += 32)
    if (i + lane < warps * K) total += scratch[slot][i + lane];
#pragma unroll
  for (int o = 16; o >= K; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
#pragma unroll
  for (int i = 0; i < K; ++i) v[i] = K == 1 ? total : __shfl_sync(0xffffffffu, total, i);
  slot ^= 1;
}

// ---- a CTA to a row, several rows a turn, the rows of later turns on their way into shared memory ----
template <int NV> __host__ __device__ constexpr int ln_rows_at_once() { return NV >= 4 ? 1 : NV == 2 ? 2 : 4; }
// turns of rows in flight behind the one at hand (rows of 8 accesses a thread fill the shared memory)
template <int NV> __host__ __device__ constexpr int ln_ahead() { return NV >= 8 ? 0 : 2; }

// Copies of AL values of a thread into its own shared memory, zeros where there are none.  Below four bytes there is no asynchronous copy.
template <class T, int AL, int PIECE> __device__ __forceinline__ void ln_copy(Pack<T, kLnN<T>> *to, const T *row, LnCols<T, PIECE> col, int i, int cols, bool in) {
  constexpr int N = kLnN<T>, BYTES = AL * (int)sizeof(T);
  if constexpr (BYTES < 4) *to = ln_load<T, AL, PIECE>(row, col, i, cols, in);
  else {
    const unsigned dst = (unsigned)__cvta_generic_to_shared(to);
#pragma unroll
    for (int p = 0; p < N; p += AL) {
      const bool here = in && col(i, p) < cols;
      const T *src = here ? row + col(i, p) : row;  // (nothing is read for a size of zero)
      if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(here ? 16 : 0) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst + p * (int)sizeof(T)), "l"(src), "n"(BYTES), "r"(here ? BYTES : 0) : "memory");
    }
  }
}

// The rows of a thread that has a warp or less of company, and its columns.
template <class T, int LANES> struct LnPlace {
  int t;
  long long row, step;
  __device__ LnPlace() {
    t = threadIdx.x % LANES;
    row = blockIdx.x * (long long)(blockDim.x / LANES) + threadIdx.x / LANES;
    step = (long long)gridDim.x * (blockDim.x / LANES);
  }
  // rows of a warp's lanes end at different times: it goes on as one
  __device__ bool more(int rows) const { return LANES < 32 ? __any_sync(0xffffffffu, row < rows) : row < rows; }
};

struct LnShape { int al, piece, nv, lanes, threads; };  // lanes 0: a CTA to a row

// al and piece of a shape
inline LnShape ln_pieces(int cols, int bytes, bool keep8, std::initializer_list<std::pair<const void *, long long>> operands) {
  const int n = 16 / bytes, piece = keep8 || cols % n == 0 ? n : cols % 2 == 0 ? 2 : 1;
  int al = 1;
  for (int k : {2, n}) {
    bool whole = cols % k == 0 && k <= piece && (keep8 || k == piece);
    for (const auto &o : operands) whole = whole && (!o.first || (o.second % k == 0 && reinterpret_cast<uintptr_t>(o.first) % (k * bytes) == 0));
    if (whole) al = k;
  }
  return {al, piece, 1, 0, 0};
}
// Eight lanes to a row where they hold it with 16 values each; a warp up to `warp_cols` columns, of as many accesses as it takes; a CTA
// beyond: of as many threads as hold it with one access each up to 256, with two, four or (fp32) eight up to 512 (16 384 x 4 096 bf16,
// forward and backward: 256 threads with two 67 and 98 us, 512 with one 74 and 108).
inline LnShape ln_shape(LnShape s, int cols, int bytes, int warp_cols) {
  const int n = 16 / bytes, vecs = (cols + n - 1) / n, most = 16 / n;
  auto least = [&](int lanes, int nv) { while (lanes * nv < vecs) nv += nv < most ? nv : 1; return nv == 7 ? 8 : nv; };
  if (vecs <= 8 * most) return {s.al, s.piece, least(8, 1), 8, kLnWarpThreads};
  if (cols <= warp_cols) { const int nv = least(32, 1); return {s.al, s.piece, nv, 32, nv <= most ? kLnWarpThreads : kLnWarpThreads / 2}; }
  int nv = 1;
  while ((vecs + nv - 1) / nv > (nv == 1 ? 256 : kLnRowThreads)) nv *= 2;
  return {s.al, s.piece, nv, 0, ((vecs + nv - 1) / nv + 31) / 32 * 32};
}
// What the runtime says of a kernel's resident CTAs, asked once (it takes 2 us to say so).
inline cudaError_t ln_occupancy(const void *f, int threads, size_t smem, int &each) {
  struct Entry { const void *f; int threads; size_t smem; int each; };
  thread_local Entry last[16] = {};
  Entry &e = last[(reinterpret_cast<uintptr_t>(f) >> 4 ^ (uintptr_t)threads) & 15];
  if (e.f != f || e.threads != threads || e.smem != smem) {
    const cudaError_t rc = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, f, threads, smem);
    if (rc != cudaSuccess) return rc;
    e = {f, threads, smem, each};
  }
  each = e.each;
  return cudaSuccess;
}
// CTAs of a launch: as many as fit the device at one time, or as have rows.
template <class F> cudaError_t ln_ctas(F f, int threads, size_t smem, int rows, int rows_cta, int &ctas) {
  int each = 1;
  const cudaError_t e = ln_occupancy((const void *)f, threads, smem, each);
  ctas = std::max(1, std::min((rows + rows_cta - 1) / rows_cta, std::min(kLnMaxCtas, 148 * std::max(1, each))));
  return e;
}

// Launches f with as many CTAs as fit the device at one time, or as have rows.
template <class F> cudaError_t ln_go(F f, const LnShape &s, const LnParams &P, int rows_cta, size_t smem, int &ctas, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (smem > 32 * 1024) e = cudaFuncSetAttribute((const void *)f, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  if (e == cudaSuccess) e = ln_ctas(f, s.threads, smem, P.rows, rows_cta, ctas);
  if (e != cudaSuccess) return e;
  f<<<ctas, s.threads, smem, st>>>(P);
  return cudaGetLastError();
}

int ln_check(const char *who, int rows, int cols, int dtype, int w_dtype, const void *codes, int ld_codes, const void *exps);

}  // namespace tfk
