// Activations into 8 bits and back (pack8.cuh), and the ReLU's gradient from the codes.  One pass each, bound by what it reads
// and writes: a thread takes up to 32 bytes of values at a time, four such in flight.  1 048 576 x 128 fp32: 110 us there (6.1 TB/s),
// 126 back (5.3); 500 009 x 256 bf16 with ReLU 87 (4.4 TB/s at 0.61 instructions a cycle and
// scheduler; the code of a positive zero is a comparison and a selection more).  The mask, in place, 1 048 576 x 128 fp32: 236 (5.1).
#include <algorithm>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "pack8.cuh"
#include "tf_internal.h"

namespace tfk {

namespace {

constexpr int kPackThreads = 256, kPackUnroll = 4;

// The places of a thread in [rows][quads] walked with one stride, without a division at each step.  FLAT: one long row.
template <bool FLAT> struct Walk {
  using Int = typename std::conditional<FLAT, long long, int>::type;  // (rows and a step beyond them fit 32 bits)
  Int row, quad, quads, d_row, d_quad;
  __device__ Walk(long long quads_) : quads((Int)quads_) {
    const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x, step = (long long)gridDim.x * blockDim.x;
    if (FLAT) { row = 0; quad = (Int)i; d_row = 0; d_quad = (Int)step; return; }
    row = (Int)(i / quads_); quad = (Int)(i % quads_);
    d_row = (Int)(step / quads_); d_quad = (Int)(step % quads_);
  }
  __device__ bool in(int rows) const { return FLAT ? quad < quads : row < rows; }
  __device__ void next() {
    quad += d_quad;
    if (FLAT) return;
    row += d_row;
    if (quad >= quads) { quad -= quads; ++row; }
  }
};

// N values a thread, in pieces of AL; codes [rows][ld_codes], exponents [rows][ld_codes / 32]; columns from `cols` on become zero.
// FLAT: rows of whole groups with nothing between them, one row of rows * cols values.
template <class T, int N, int AL, bool RELU, bool FLAT>
__global__ void __launch_bounds__(kPackThreads)
pack8_kernel(const T *__restrict__ x, long long ld, int rows, long long cols, signed char *__restrict__ codes, long long ld_codes,
             unsigned char *__restrict__ exps) {
  Walk<FLAT> w(ld_codes / N);
  // (a warp leaves as one: the lanes of a group are in one row)
  while (__any_sync(0xffffffffu, w.in(rows))) {
    long long to[kPackUnroll];  // where the codes go, or -1
    Pack<T, N> v[kPackUnroll];
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u, w.next()) {
      const bool in = w.in(rows);
      const auto col = w.quad * N;
      to[u] = in ? (FLAT ? (long long)col : w.row * ld_codes + col) : -1;
#pragma unroll
      for (int i = 0; i < N; ++i) v[u].v[i] = from_float<T>(0.f);
      if constexpr (AL == N) {
        if (in && (FLAT || col < cols)) v[u] = load_raw<T, N>(x + (FLAT ? col : w.row * ld + col));
      } else if (in) {
        const T *p = x + w.row * ld + col;
#pragma unroll
        for (int i = 0; i < N; i += AL) {
          if (col + i >= cols) continue;
          const Pack<T, AL> a = *reinterpret_cast<const Pack<T, AL> *>(p + i);
#pragma unroll
          for (int k = 0; k < AL; ++k) v[u].v[i + k] = a.v[k];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u) {
      float f[N];
      unsigned code[N];
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = to_float(v[u].v[i]);
      const int e = pack8_lanes<N, RELU>(f, code);
      if (to[u] < 0) continue;
      store_codes<N>(codes + to[u], code);
      if (to[u] % kPackGroup == 0) exps[to[u] / kPackGroup] = (unsigned char)(e + 127);  // (rows of codes are whole groups)
    }
  }
}

template <class T, int N, bool FLAT>
__global__ void __launch_bounds__(kPackThreads)
unpack8_kernel(const signed char *__restrict__ codes, long long ld_codes, const unsigned char *__restrict__ exps, int rows, long long cols,
               T *__restrict__ out, long long ld) {
  for (Walk<FLAT> w(cols / N); w.in(rows);) {
    long long to[kPackUnroll];
    Pack<signed char, N> c[kPackUnroll];
    unsigned e[kPackUnroll];
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u, w.next()) {
      const long long col = w.quad * N, at = FLAT ? col : w.row * ld_codes + col;
      to[u] = w.in(rows) ? (FLAT ? col : w.row * ld + col) : -1;
      if (to[u] < 0) continue;
      c[u] = *reinterpret_cast<const Pack<signed char, N> *>(codes + at);
      e[u] = __ldg(exps + at / kPackGroup);
    }
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u) {
      if (to[u] < 0) continue;
      float v[N];
      unpack8_values<N>(c[u], unpack8_step(e[u]), v);
      Pack<T, N> a;
#pragma unroll
      for (int i = 0; i < N; ++i) a.v[i] = from_float<T>(v[i]);
      store_raw<T, N>(out + to[u], a);
    }
  }
}

// Rows that start anywhere, but one behind the other: 16 bytes of values a thread as the whole array has them, across the ends of
// rows, so that what is written are whole sectors; the codes come byte by byte, from L1.
template <class T>
__global__ void __launch_bounds__(kPackThreads)
unpack8_flat_kernel(const signed char *__restrict__ codes, int ld_codes, const unsigned char *__restrict__ exps, long long all, int cols, T *__restrict__ out) {
  constexpr int N = 16 / (int)sizeof(T);
  const long long step = (long long)gridDim.x * blockDim.x * N, d_row = step / cols;
  const int d_col = (int)(step - d_row * cols), ld_e = ld_codes / kPackGroup;
  long long at = (blockIdx.x * (long long)blockDim.x + threadIdx.x) * N, row = at / cols;
  int col = (int)(at - row * cols);
  for (; at < all; at += step, row += d_row, col += d_col) {
    if (col >= cols) { col -= cols; ++row; }
    const signed char *c = codes + row * ld_codes;
    const unsigned char *e = exps + row * ld_e;
    int q = col;
    float v[N];
    int code[N];
    unsigned exp[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = at + i < all;
      code[i] = in ? __ldg(c + q) : 0;
      exp[i] = in ? __ldg(e + q / kPackGroup) : 127;
      if (++q == cols) { q = 0; c += ld_codes; e += ld_e; }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = unpack8_value(code[i], unpack8_step(exp[i]));
    if (at + N <= all) store_pack<T, N>(out + at, v);
    else
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at + i < all) out[at + i] = from_float<T>(v[i]);
  }
}

// grad (in place) where the packed value was positive, zero elsewhere.
template <class T, int N>
__global__ void __launch_bounds__(kPackThreads)
mask8_kernel(const signed char *__restrict__ codes, long long ld_codes, int rows, int cols, T *__restrict__ grad, long long ld) {
  for (Walk<false> w(cols / N); w.in(rows);) {
    long long to[kPackUnroll];
    Pack<signed char, N> c[kPackUnroll];
    Pack<T, N> g[kPackUnroll];
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u, w.next()) {
      to[u] = w.in(rows) ? w.row * ld + w.quad * N : -1;
      if (to[u] < 0) continue;
      c[u] = *reinterpret_cast<const Pack<signed char, N> *>(codes + w.row * ld_codes + w.quad * N);
      g[u] = *reinterpret_cast<const Pack<T, N> *>(grad + to[u]);
    }
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u) {
      if (to[u] < 0) continue;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c[u].v[i] == 0) g[u].v[i] = from_float<T>(0.f);
      *reinterpret_cast<Pack<T, N> *>(grad + to[u]) = g[u];
    }
  }
}

// Values that one access of a thread takes: as many as fill 32 or 16 bytes where rows and widths are whole multiples of that, two, or one.
int pack_width(const void *p, long long ld, int cols, int bytes) {
  for (int n : {32 / bytes, 16 / bytes, 2})
    if (cols % n == 0 && ld % n == 0 && reinterpret_cast<uintptr_t>(p) % (n * bytes) == 0) return n;
  return 1;
}
unsigned pack_grid(long long places) {
  return (unsigned)std::max<long long>(1, std::min<long long>((places + kPackThreads * kPackUnroll - 1) / (kPackThreads * kPackUnroll), 148 * 8));
}
int done(const char *who) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TF_OK : tf::fail(TF_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}
int check(const char *who, const void *values, long long ld, int dtype, int rows, int cols, const void *codes, int ld_codes, const void *exps) {
  auto bad = [&](const char *what) { return tf::fail(TF_ERR_ARG, std::string(who) + ": " + what); };
  if (!known_dtype(dtype)) return bad("unknown type");
  if (rows < 0 || rows > kMaxRows || cols <= 0 || cols > (1 << 30)) return bad("bad size");
  if (ld < cols || ld_codes < cols) return bad("rows overlap");
  if (ld_codes % kPackGroup != 0 || (reinterpret_cast<uintptr_t>(codes) & 31) != 0) return bad("codes need rows of whole groups of 32 and 32-byte alignment");
  if (rows > 0 && (!values || !codes || !exps)) return bad("null argument");
  return TF_OK;
}

template <class T, int N, int AL> void launch_pack_as(const void *x, long long ld, int rows, int cols, signed char *codes, int ld_codes, unsigned char *exps,
                                                     bool relu, cudaStream_t s) {
  const unsigned grid = pack_grid((long long)rows * (ld_codes / N));
  if constexpr (AL == N)
    if (ld == cols && cols == ld_codes) {
      const long long all = (long long)rows * cols;
      if (relu) pack8_kernel<T, N, N, true, true><<<grid, kPackThreads, 0, s>>>((const T *)x, all, 1, all, codes, all, exps);
      else pack8_kernel<T, N, N, false, true><<<grid, kPackThreads, 0, s>>>((const T *)x, all, 1, all, codes, all, exps);
      return;
    }
  if (relu) pack8_kernel<T, N, AL, true, false><<<grid, kPackThreads, 0, s>>>((const T *)x, ld, rows, cols, codes, ld_codes, exps);
  else pack8_kernel<T, N, AL, false, false><<<grid, kPackThreads, 0, s>>>((const T *)x, ld, rows, cols, codes, ld_codes, exps);
}
// n: values that one access takes; eight to a thread where it takes fewer (2 449 029 x 100 fp32: 203 us, 279 with four; 300 000 x 1 000
// bf16: 189, 256 with sixteen)
template <class T, int N> void launch_pack(const void *x, long long ld, int rows, int cols, signed char *codes, int ld_codes, unsigned char *exps, bool relu,
                                           cudaStream_t s) {
  constexpr int M = 8;
  launch_pack_as<T, (N < M ? M : N), N>(x, ld, rows, cols, codes, ld_codes, exps, relu, s);
}
template <class T, int N> void launch_unpack(const signed char *codes, int ld_codes, const unsigned char *exps, int rows, int cols, void *out, long long ld,
                                             cudaStream_t s) {
  const unsigned grid = pack_grid((long long)rows * (cols / N));
  const long long all = (long long)rows * cols;
  constexpr int M = 16 / (int)sizeof(T);
  if (N >= M && ld == cols && cols == ld_codes) unpack8_kernel<T, N, true><<<grid, kPackThreads, 0, s>>>(codes, all, exps, 1, all, (T *)out, all);
  else if (N < M && ld == cols && (reinterpret_cast<uintptr_t>(out) & 15) == 0)
    unpack8_flat_kernel<T><<<pack_grid(4 * (all / M + 1)), kPackThreads, 0, s>>>(codes, ld_codes, exps, all, cols, (T *)out);
  else unpack8_kernel<T, N, false><<<grid, kPackThreads, 0, s>>>(codes, ld_codes, exps, rows, cols, (T *)out, ld);
}
template <class T, int N> void launch_mask(const signed char *codes, int ld_codes, int rows, int cols, void *grad, long long ld, cudaStream_t s) {
  mask8_kernel<T, N><<<pack_grid((long long)rows * (cols / N)), kPackThreads, 0, s>>>(codes, ld_codes, rows, cols, (T *)grad, ld);
}

}  // namespace

}  // namespace tfk

using namespace tfk;

// f<type, values of a thread>(arguments) for the operand's type and width
#define TF_BY_TYPE(f, dtype, n, ...)                                                                              \
  do {                                                                                                            \
    if (dtype == TF_F32) n == 8 ? f<float, 8>(__VA_ARGS__) : n == 4 ? f<float, 4>(__VA_ARGS__) : n == 2 ? f<float, 2>(__VA_ARGS__) : f<float, 1>(__VA_ARGS__); \
    else if (dtype == TF_BF16)                                                                                    \
      n == 16 ? f<__nv_bfloat16, 16>(__VA_ARGS__) : n == 8 ? f<__nv_bfloat16, 8>(__VA_ARGS__) : n == 2 ? f<__nv_bfloat16, 2>(__VA_ARGS__) : f<__nv_bfloat16, 1>(__VA_ARGS__); \
    else n == 16 ? f<__half, 16>(__VA_ARGS__) : n == 8 ? f<__half, 8>(__VA_ARGS__) : n == 2 ? f<__half, 2>(__VA_ARGS__) : f<__half, 1>(__VA_ARGS__);       \
  } while (0)

extern "C" int tf_pack8(const void *x, long long ld, int dtype, int rows, int cols, int relu, signed char *codes, int ld_codes,
                        unsigned char *exponents, void *stream) {
  const int rc = check("tf_pack8", x, ld, dtype, rows, cols, codes, ld_codes, exponents);
  if (rc != TF_OK || rows == 0) return rc;
  const int n = pack_width(x, ld, cols, value_bytes(dtype));
  TF_BY_TYPE(launch_pack, dtype, n, x, ld, rows, cols, codes, ld_codes, exponents, relu != 0, (cudaStream_t)stream);
  return done("tf_pack8");
}

extern "C" int tf_unpack8(const signed char *codes, int ld_codes, const unsigned char *exponents, int dtype, int rows, int cols, void *out,
                          long long ld, void *stream) {
  const int rc = check("tf_unpack8", out, ld, dtype, rows, cols, codes, ld_codes, exponents);
  if (rc != TF_OK || rows == 0) return rc;
  const int n = pack_width(out, ld, cols, value_bytes(dtype));
  TF_BY_TYPE(launch_unpack, dtype, n, codes, ld_codes, exponents, rows, cols, out, ld, (cudaStream_t)stream);
  return done("tf_unpack8");
}

extern "C" int tf_relu_grad8(const signed char *codes, int ld_codes, int dtype, int rows, int cols, void *grad, long long ld, void *stream) {
  const int rc = check("tf_relu_grad8", grad, ld, dtype, rows, cols, codes, ld_codes, codes);
  if (rc != TF_OK || rows == 0) return rc;
  const int n = pack_width(grad, ld, cols, value_bytes(dtype));
  TF_BY_TYPE(launch_mask, dtype, n, codes, ld_codes, rows, cols, grad, ld, (cudaStream_t)stream);
  return done("tf_relu_grad8");
}
