// Activations into 8 bits and back (pack8.cuh), and the ReLU's gradient from the codes.  One pass each, bound by what it reads
// and writes: a thread takes up to 16 bytes of values at a time, four such in flight.
#include <algorithm>
#include <string>

#include "pack8.cuh"
#include "tf_internal.h"

namespace tfk {

namespace {

constexpr int kPackThreads = 256, kPackUnroll = 4;

// The places of a thread in [rows][quads] walked with one stride, without a division at each step.
struct Walk {
  long long row;
  int quad, quads, d_row, d_quad;
  __device__ Walk(int quads_) : quads(quads_) {
    const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x, step = (long long)gridDim.x * blockDim.x;
    row = i / quads; quad = (int)(i - row * quads);
    d_row = (int)(step / quads); d_quad = (int)(step - (long long)d_row * quads);
  }
  __device__ void next() {
    row += d_row; quad += d_quad;
    if (quad >= quads) { quad -= quads; ++row; }
  }
};

// N values a thread; codes [rows][ld_codes], exponents [rows][ld_codes / 32]; columns from `cols` on become zero.
template <class T, int N, bool RELU>
__global__ void __launch_bounds__(kPackThreads)
pack8_kernel(const T *__restrict__ x, long long ld, int rows, int cols, signed char *__restrict__ codes, int ld_codes, unsigned char *__restrict__ exps) {
  Walk w(ld_codes / N);
  // (a warp leaves as one: the lanes of a group are in one row)
  while (__any_sync(0xffffffffu, w.row < rows)) {
    long long row[kPackUnroll];
    int col[kPackUnroll];
    float v[kPackUnroll][N];
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u, w.next()) {
      row[u] = w.row; col[u] = w.quad * N;
#pragma unroll
      for (int i = 0; i < N; ++i) v[u][i] = 0.f;
      if (row[u] < rows && col[u] < cols) load_pack<T, N>(x + row[u] * ld + col[u], v[u]);
    }
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u) {
      int code[N];
      const int e = pack8_lanes<N, RELU>(v[u], code);
      if (row[u] >= rows) continue;
      store_codes<N>(codes + row[u] * ld_codes + col[u], code);
      if (col[u] % kPackGroup == 0) exps[row[u] * (ld_codes / kPackGroup) + col[u] / kPackGroup] = (unsigned char)(e + 127);
    }
  }
}

template <class T, int N>
__global__ void __launch_bounds__(kPackThreads)
unpack8_kernel(const signed char *__restrict__ codes, int ld_codes, const unsigned char *__restrict__ exps, int rows, int cols, T *__restrict__ out,
               long long ld) {
  for (Walk w((cols + N - 1) / N); w.row < rows;) {
    long long row[kPackUnroll];
    int col[kPackUnroll];
    Pack<signed char, N> c[kPackUnroll];
    unsigned e[kPackUnroll];
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u, w.next()) {
      row[u] = w.row; col[u] = w.quad * N;
      if (row[u] >= rows) continue;
      c[u] = *reinterpret_cast<const Pack<signed char, N> *>(codes + row[u] * ld_codes + col[u]);
      e[u] = __ldg(exps + row[u] * (ld_codes / kPackGroup) + col[u] / kPackGroup);
    }
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u) {
      if (row[u] >= rows) continue;
      const float step = unpack8_step(e[u]);
      float v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = unpack8_value(c[u].v[i], step);
      store_pack<T, N>(out + row[u] * ld + col[u], v);
    }
  }
}

// grad (in place) where the packed value was positive, zero elsewhere.
template <class T, int N>
__global__ void __launch_bounds__(kPackThreads)
mask8_kernel(const signed char *__restrict__ codes, int ld_codes, int rows, int cols, T *__restrict__ grad, long long ld) {
  for (Walk w((cols + N - 1) / N); w.row < rows;) {
    long long row[kPackUnroll];
    int col[kPackUnroll];
    Pack<signed char, N> c[kPackUnroll];
    Pack<T, N> g[kPackUnroll];
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u, w.next()) {
      row[u] = w.row; col[u] = w.quad * N;
      if (row[u] >= rows) continue;
      c[u] = *reinterpret_cast<const Pack<signed char, N> *>(codes + row[u] * ld_codes + col[u]);
      g[u] = *reinterpret_cast<const Pack<T, N> *>(grad + row[u] * ld + col[u]);
    }
#pragma unroll
    for (int u = 0; u < kPackUnroll; ++u) {
      if (row[u] >= rows) continue;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c[u].v[i] == 0) g[u].v[i] = from_float<T>(0.f);
      *reinterpret_cast<Pack<T, N> *>(grad + row[u] * ld + col[u]) = g[u];
    }
  }
}

// Values that one access of a thread takes: as many as fill 16 bytes where rows and widths are whole multiples of that, two, or one.
int pack_width(const void *p, long long ld, int cols, int bytes) {
  for (int n = 16 / bytes; n > 1; n = n > 2 ? 2 : 1)
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
  if (rows < 0 || cols <= 0 || cols > (1 << 30)) return bad("bad size");
  if (ld < cols || ld_codes < cols) return bad("rows overlap");
  if (ld_codes % kPackGroup != 0 || (reinterpret_cast<uintptr_t>(codes) & 31) != 0) return bad("codes need rows of whole groups of 32 and 32-byte alignment");
  if (rows > 0 && (!values || !codes || !exps)) return bad("null argument");
  return TF_OK;
}

template <class T, int N> void launch_pack(const void *x, long long ld, int rows, int cols, signed char *codes, int ld_codes, unsigned char *exps, bool relu,
                                           cudaStream_t s) {
  const unsigned grid = pack_grid((long long)rows * (ld_codes / N));
  if (relu) pack8_kernel<T, N, true><<<grid, kPackThreads, 0, s>>>((const T *)x, ld, rows, cols, codes, ld_codes, exps);
  else pack8_kernel<T, N, false><<<grid, kPackThreads, 0, s>>>((const T *)x, ld, rows, cols, codes, ld_codes, exps);
}
template <class T, int N> void launch_unpack(const signed char *codes, int ld_codes, const unsigned char *exps, int rows, int cols, void *out, long long ld,
                                             cudaStream_t s) {
  unpack8_kernel<T, N><<<pack_grid((long long)rows * ((cols + N - 1) / N)), kPackThreads, 0, s>>>(codes, ld_codes, exps, rows, cols, (T *)out, ld);
}
template <class T, int N> void launch_mask(const signed char *codes, int ld_codes, int rows, int cols, void *grad, long long ld, cudaStream_t s) {
  mask8_kernel<T, N><<<pack_grid((long long)rows * ((cols + N - 1) / N)), kPackThreads, 0, s>>>(codes, ld_codes, rows, cols, (T *)grad, ld);
}

}  // namespace

}  // namespace tfk

using namespace tfk;

// f<type, values of a thread>(arguments) for the operand's type and width
#define TF_BY_TYPE(f, dtype, n, ...)                                                                              \
  do {                                                                                                            \
    if (dtype == TF_F32) n == 4 ? f<float, 4>(__VA_ARGS__) : n == 2 ? f<float, 2>(__VA_ARGS__) : f<float, 1>(__VA_ARGS__); \
    else if (dtype == TF_BF16)                                                                                    \
      n == 8 ? f<__nv_bfloat16, 8>(__VA_ARGS__) : n == 2 ? f<__nv_bfloat16, 2>(__VA_ARGS__) : f<__nv_bfloat16, 1>(__VA_ARGS__); \
    else n == 8 ? f<__half, 8>(__VA_ARGS__) : n == 2 ? f<__half, 2>(__VA_ARGS__) : f<__half, 1>(__VA_ARGS__);       \
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
