// dW = G^T X for a tall gradient G (fp32, bf16 or fp16) and an X kept in 8 bits (pack8.cuh): the weight gradient of a layer that
// keeps its input in 8 bits.  A sum over all rows with a small result, bound by reading G and the codes once.
//
//   * The rows are cut into as many ranges as the device holds CTAs; each adds up a tile of 128 x 256 or 256 x 128 sums (which of
//     the two: whatever reads less), and a second launch adds the ranges' tiles in order.
//   * Sixteen warps bring 32 rows at a time from memory through registers into shared memory as 16-bit operands, row by row as they
//     lie (MN-major, 128-byte swizzle: nothing is transposed), the next 32 rows on their way meanwhile; one warp issues
//     tcgen05.mma.  A value of X is seven bits and a power of two, exact in bf16.  G in fp32 is three bf16 planes (24 bits, exact), in
//     fp16 two (exact), in bf16 one.  So products lose nothing.
//   * The tensor core cuts off what it adds to an accumulator, 2e-8 of the sum each time: after 128 rows (at most 24 additions)
//     the accumulator, one of two, is read and added in registers, where sums round.
// All waits are bounded: where one runs out the CTA's sums, and with them the result, become NaN.
#include <algorithm>
#include <string>

#include "pack8.cuh"
#include "pair_mma.cuh"
#include "tf_internal.h"

namespace tfk {

namespace {

constexpr int kWgWarps = 16, kWgThreads = 32 * (kWgWarps + 1);
constexpr int kWgRows = 32;                    // of a slice: two K steps of 16
constexpr int kWgChain = 4;                    // slices added up in tensor memory
constexpr int kWgBlock = kWgRows * 128;        // bytes of 64 columns of a slice
constexpr int kWgMaxStages = 5;
constexpr int kWgSmem = 224 * 1024;
constexpr int kWgWaitLimit = 1 << 22;

__host__ __device__ constexpr int wg_stage_bytes(int planes, int mt) { return planes * mt * 2 * kWgBlock + (mt == 1 ? 4 : 2) * kWgBlock; }
__host__ __device__ constexpr int wg_stages(int planes, int mt) {
  return kWgSmem / wg_stage_bytes(planes, mt) < kWgMaxStages ? kWgSmem / wg_stage_bytes(planes, mt) : kWgMaxStages;
}

struct WgParams {
  const void *g; long long ld_g; int na;
  const signed char *codes; int ld_codes, nb; const unsigned char *exps;
  int m, rows;  // rows of a range
  bool whole_g;
  float *part;  // [range][na][nb]
};

struct WgShared {
  unsigned long long full[kWgMaxStages], empty[kWgMaxStages], acc_full[2], acc_empty[2];
  unsigned tmem_base;
  int dead;
};

// MN-major, 128-byte swizzle: blocks of 64 columns kWgBlock apart, groups of eight rows 1 KB apart.
__device__ __forceinline__ unsigned long long wg_desc(unsigned addr) {
  return (umma_desc_sw128(addr) & ~((unsigned long long)0x3fff << 16)) | (unsigned long long)(kWgBlock >> 4) << 16;
}
__device__ __forceinline__ void wg_mma(unsigned d, unsigned long long da, unsigned long long db, unsigned idesc, unsigned acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}

// Eight neighbouring values of a gradient's row, zeros where there are none.
template <class T> __device__ __forceinline__ void wg_load(const T *row, int col, int cols, bool whole, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (whole) {
    if (col < cols) {
      constexpr int W = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < 8; i += W) {
        const Pack<T, W> a = *reinterpret_cast<const Pack<T, W> *>(row + col + i);
#pragma unroll
        for (int k = 0; k < W; ++k) v[i + k] = to_float(a.v[k]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < cols) v[i] = to_float(row[col + i]);
  }
}

template <class T, int PLANES, int MT>
__global__ void __launch_bounds__(kWgThreads, 1) weight_grad8_kernel(const WgParams P) {
  constexpr int NT = MT == 1 ? 256 : 128, kPlane = MT * 2 * kWgBlock, kStage = wg_stage_bytes(PLANES, MT), kStages = wg_stages(PLANES, MT);
  constexpr int QG = MT, QX = NT / 128;  // chunks of eight columns of a thread
  extern __shared__ char dyn[];
  __shared__ WgShared s;
  char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  const int a0 = blockIdx.y * MT * 128, b0 = blockIdx.z * NT;
  const int n_pad = (min(NT, P.nb - b0) + 15) / 16 * 16;
  const long long r0 = (long long)blockIdx.x * P.rows;
  const long long r1 = min((long long)P.m, r0 + P.rows);
  const int slices = (int)((r1 - r0 + kWgRows - 1) / kWgRows);

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&s.full[i], kWgWarps); mbar_init(&s.empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s.acc_full[i], 1); mbar_init(&s.acc_empty[i], kWgWarps); }
    s.dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem_base)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");

  if (warp == kWgWarps) {
    // ---- products ----
    const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((unsigned)(n_pad >> 3) << 17) | ((unsigned)(128 >> 4) << 24);
    int st = 0;
    unsigned ph = 0;
    bool ok = true;
    auto wait = [&](unsigned long long *bar, unsigned parity) { return ok = __all_sync(kFull, pair_wait(bar, parity, s.dead, kWgWaitLimit)); };
    for (int sl = 0; sl < slices; ++sl) {
      const int chain = sl / kWgChain, buf = chain & 1, in = sl % kWgChain;
      if (in == 0 && chain >= 2 && !wait(&s.acc_empty[buf], (unsigned)(chain / 2 - 1) & 1u)) break;
      if (!wait(&s.full[st], ph)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned base = smem_u32(smem + st * kStage);
      const unsigned long long a = wg_desc(base), b = wg_desc(base + PLANES * kPlane);
      const unsigned d = s.tmem_base + (unsigned)(buf * 256);
      const bool last = in == kWgChain - 1 || sl == slices - 1;
      if (elect_one()) {
#pragma unroll
        for (int p = PLANES - 1; p >= 0; --p)  // the small products first
#pragma unroll
          for (int k = 0; k < kWgRows / 16; ++k)
#pragma unroll
            for (int t = 0; t < MT; ++t)
              wg_mma(d + (unsigned)(t * NT), a + (unsigned)((p * kPlane + t * 2 * kWgBlock + k * 2048) >> 4), b + (unsigned)(k * 2048 >> 4), idesc,
                     in || p != PLANES - 1 || k ? 1u : 0u);
        umma_commit(&s.empty[st]);
        if (last) umma_commit(&s.acc_full[buf]);
      }
      __syncwarp();
      if (++st == kStages) { st = 0; ph ^= 1u; }
    }
  } else {
    // ---- rows into operands; and every fourth slice the sums of the four before out of tensor memory ----
    const int quadrant = warp & 3, cols0 = (warp >> 2) * 64;  // this thread's row and columns of the accumulator
    float acc[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) acc[i] = 0.f;
    bool ok = true;
    auto wait = [&](unsigned long long *bar, unsigned parity) { return ok = __all_sync(kFull, pair_wait(bar, parity, s.dead, kWgWaitLimit)); };
    auto drain = [&](int chain) {
      const int buf = chain & 1;
      if (!wait(&s.acc_full[buf], (unsigned)(chain / 2) & 1u)) return;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (MT == 2 ? (cols0 & 127) < n_pad : cols0 < n_pad) {
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          float v[16];
          tmem_load16(v, s.tmem_base + ((unsigned)(quadrant * 32) << 16) + (unsigned)(buf * 256 + cols0 + c));
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[c + q] += v[q];
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&s.acc_empty[buf])) : "memory");
    };
    float g[QG][8];
    uint2 x[QX];
    unsigned e[QX];
    auto fetch = [&](int sl) {
#pragma unroll
      for (int i = 0; i < QG; ++i) {
        const int q = tid + i * 512, c = q % (MT * 16) * 8;
        const long long row = r0 + sl * kWgRows + q / (MT * 16);
        if (row < r1) wg_load<T>(static_cast<const T *>(P.g) + row * P.ld_g, a0 + c, P.na, P.whole_g, g[i]);
        else
#pragma unroll
          for (int k = 0; k < 8; ++k) g[i][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < QX; ++i) {
        const int q = tid + i * 512, c = b0 + q % (NT / 8) * 8;
        const long long row = r0 + sl * kWgRows + q / (NT / 8);
        x[i] = make_uint2(0, 0);
        e[i] = 127;
        if (row < r1 && c < P.ld_codes) {
          x[i] = __ldg(reinterpret_cast<const uint2 *>(P.codes + row * P.ld_codes + c));
          e[i] = __ldg(P.exps + row * (P.ld_codes / kPackGroup) + c / kPackGroup);
        }
      }
    };
    int st = 0;
    unsigned ph = 0;
    if (slices > 0) fetch(0);
    for (int sl = 0; sl < slices && ok; ++sl) {
      if (sl >= kStages && !wait(&s.empty[st], ph ^ 1u)) break;
      char *base = smem + st * kStage;
#pragma unroll
      for (int i = 0; i < QG; ++i) {
        const int q = tid + i * 512, r = q / (MT * 16), chunk = q % (MT * 16);
        char *to = base + chunk / 8 * kWgBlock + r * 128 + ((chunk & 7) ^ (r & 7)) * 16;
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
          unsigned u[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            u[k] = pack_pair(g[i][2 * k], g[i][2 * k + 1], false);
            if (p < PLANES - 1) {
              g[i][2 * k] -= __uint_as_float(u[k] << 16);
              g[i][2 * k + 1] -= __uint_as_float(u[k] & 0xffff0000u);
            }
          }
          *reinterpret_cast<uint4 *>(to + p * kPlane) = make_uint4(u[0], u[1], u[2], u[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < QX; ++i) {
        const int q = tid + i * 512, r = q / (NT / 8), chunk = q % (NT / 8);
        const float step = unpack8_step(e[i]);
        float v[8];
        unpack8_word(x[i].x, step, v);
        unpack8_word(x[i].y, step, v + 4);
        unsigned u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = pack_pair(v[2 * k], v[2 * k + 1], false);
        *reinterpret_cast<uint4 *>(base + PLANES * kPlane + chunk / 8 * kWgBlock + r * 128 + ((chunk & 7) ^ (r & 7)) * 16) =
            make_uint4(u[0], u[1], u[2], u[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read next by the tensor core
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&s.full[st])) : "memory");
      if (sl + 1 < slices) fetch(sl + 1);
      if (sl % kWgChain == kWgChain - 1 && sl / kWgChain >= 1) drain(sl / kWgChain - 1);
      if (++st == kStages) { st = 0; ph ^= 1u; }
    }
    const int chains = (slices + kWgChain - 1) / kWgChain;
    if (ok && chains >= 2 && slices % kWgChain != 0) drain(chains - 2);
    if (ok && chains >= 1) drain(chains - 1);
    const int t = MT == 2 ? cols0 / 128 : 0, col = b0 + (MT == 2 ? cols0 % 128 : cols0), row = a0 + t * 128 + quadrant * 32 + lane;
    const bool lost = !ok || *reinterpret_cast<volatile int *>(&s.dead);
    if (row < P.na) {
      float *to = P.part + ((size_t)blockIdx.x * P.na + row) * P.nb + col;
      const bool quads = P.nb % 4 == 0;
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        if (lost) acc[c] = acc[c + 1] = acc[c + 2] = acc[c + 3] = __int_as_float(0x7fc00000);
        if (quads && col + c < P.nb) *reinterpret_cast<float4 *>(to + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (col + c + k < P.nb) to[c + k] = acc[c + k];
        }
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem_base), "n"(512) : "memory");
  }
}

// out[i] = part[0][i] + part[1][i] + ..., in order; eight lanes share an element's parts and are added pairwise.
__global__ void __launch_bounds__(256) wg_sum_kernel(const float *__restrict__ part, int parts, int n, void *__restrict__ out, int dtype) {
  const int i = blockIdx.x * 32 + (threadIdx.x & 31), l = threadIdx.x >> 5;
  __shared__ float s[8][32];
  float v = 0.f;
  if (i < n)
#pragma unroll 4
    for (int k = l; k < parts; k += 8) v += __ldg(part + (size_t)k * n + i);
  s[l][threadIdx.x & 31] = v;
  __syncthreads();
  if (l || i >= n) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += s[k][threadIdx.x];
  store_value(out, dtype, i, v);
}

struct WgPlan { int mt, tiles_a, tiles_b, parts, rows; };
WgPlan wg_plan(int m, int na, int nb, int dtype) {
  auto tiles = [&](int mt) {
    WgPlan p;
    p.mt = mt;
    p.tiles_a = (na + mt * 128 - 1) / (mt * 128);
    p.tiles_b = mt == 1 ? (nb + 255) / 256 : (nb + 127) / 128;
    return p;
  };
  const WgPlan wide = tiles(1), tall = tiles(2);
  auto read = [&](const WgPlan &p) { return (double)p.tiles_b * na * value_bytes(dtype) + (double)p.tiles_a * nb; };
  // (a row of 256 x 128 sums takes as many products as one of 128 x 256)
  WgPlan p = wide.tiles_a * wide.tiles_b < tall.tiles_a * tall.tiles_b                                  ? wide
             : wide.tiles_a * wide.tiles_b > tall.tiles_a * tall.tiles_b || read(tall) < read(wide) ? tall
                                                                                                       : wide;
  // one CTA to an SM; a range of fewer than 128 rows spends its time on the result
  const int parts = std::max(1, std::min(148 / (p.tiles_a * p.tiles_b), (m + 127) / 128));
  p.rows = ((m + parts - 1) / parts + kWgRows - 1) / kWgRows * kWgRows;
  p.parts = std::max(1, (m + p.rows - 1) / std::max(1, p.rows));
  return p;
}

template <class T, int PLANES, int MT> cudaError_t wg_launch(const WgPlan &p, const WgParams &P, cudaStream_t s) {
  auto f = weight_grad8_kernel<T, PLANES, MT>;
  const int smem = wg_stages(PLANES, MT) * wg_stage_bytes(PLANES, MT) + 1024;
  const cudaError_t e = cudaFuncSetAttribute((const void *)f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  f<<<dim3(p.parts, p.tiles_a, p.tiles_b), kWgThreads, smem, s>>>(P);
  return cudaGetLastError();
}

}  // namespace

}  // namespace tfk

using namespace tfk;

extern "C" long long tf_weight_grad8_work_floats(int m, int na, int nb, int dtype) {
  if (m < 0 || na <= 0 || nb <= 0 || !known_dtype(dtype)) return 0;
  return (long long)wg_plan(m, na, nb, dtype).parts * na * nb;
}

extern "C" int tf_weight_grad8(const void *g, long long ld_g, int dtype, int na, const signed char *codes, int ld_codes,
                               const unsigned char *exponents, int nb, int m, void *out, float *work, long long work_floats, void *stream) {
  auto bad = [&](const char *what) { return tf::fail(TF_ERR_ARG, std::string("tf_weight_grad8: ") + what); };
  if (!known_dtype(dtype)) return bad("unknown type");
  if (m < 0 || na <= 0 || nb <= 0) return bad("bad size");
  if ((long long)na * nb > (1 << 26)) return tf::fail(TF_ERR_UNSUPPORTED, "tf_weight_grad8: at most 2^26 entries");
  if (!out || !work || (m > 0 && (!g || !codes || !exponents))) return bad("null argument");
  if (ld_g < na || ld_codes < nb) return bad("rows overlap");
  if (ld_codes % kPackGroup != 0 || (reinterpret_cast<uintptr_t>(codes) & 31) != 0) return bad("codes need rows of whole groups of 32 and 32-byte alignment");
  if ((reinterpret_cast<uintptr_t>(work) & 15) != 0) return bad("the work space must be 16-byte aligned");
  if (work_floats < tf_weight_grad8_work_floats(m, na, nb, dtype)) return bad("work space too small");
  const WgPlan p = wg_plan(m, na, nb, dtype);
  WgParams P;
  P.g = g; P.ld_g = ld_g; P.na = na; P.codes = codes; P.ld_codes = ld_codes; P.nb = nb; P.exps = exponents; P.m = m; P.rows = p.rows;
  P.whole_g = na % 8 == 0 && ld_g * value_bytes(dtype) % 16 == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  P.part = work;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  if (m > 0) {
    if (dtype == TF_F32) e = p.mt == 1 ? wg_launch<float, 3, 1>(p, P, s) : wg_launch<float, 3, 2>(p, P, s);
    else if (dtype == TF_F16) e = p.mt == 1 ? wg_launch<__half, 2, 1>(p, P, s) : wg_launch<__half, 2, 2>(p, P, s);
    else e = p.mt == 1 ? wg_launch<__nv_bfloat16, 1, 1>(p, P, s) : wg_launch<__nv_bfloat16, 1, 2>(p, P, s);
  }
  if (e == cudaSuccess) {
    const int n = na * nb;
    wg_sum_kernel<<<(n + 31) / 32, 256, 0, s>>>(work, m > 0 ? p.parts : 0, n, out, dtype);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? TF_OK : tf::fail(TF_ERR_CUDA, std::string("tf_weight_grad8: ") + cudaGetErrorString(e));
}
