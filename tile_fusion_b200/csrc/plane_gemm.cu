// D = A * B^T from 16-bit planes on CTA pairs (tcgen05.mma.cta_group::2, kind::f16, fp32 accumulators in tensor memory).
//
//   * A tile is 256 rows x BN columns (64, 128 or 256).  Each CTA of the pair holds 128 rows of A and half of the columns of B:
//     per slice of 64 terms 16 KB of A and up to 16 KB of B a plane, so an operand crosses from L2 once per pair.
//   * One warp keeps TMA loads running ahead through a ring of stages (192 KB); those of the odd CTA complete on the even CTA's
//     barrier, so that the one warp that issues the products of both waits once a slice.  Eight warps drain.
//   * Operands come with either index contiguous: K-major tiles of 64 terms x rows, or MN-major tiles of 64 rows x 64 terms,
//     both with the 128-byte swizzle.  The gradient products read the slope both ways without a transposition.
//   * fp32 operands are two fp16 planes of a power-of-two multiple of the value: x = 2^-e (hi + lo), and
//     hi hi + hi lo + lo hi leaves out 2^-22 of a product; that is three products at the 16-bit rate, where the same number of
//     TF32 products take twice as long.
//   * The tensor core cuts off what it adds to an accumulator.  A chain of sums drifts by about 2e-8 of the sum an addition, so
//     chains are kept short: after `chain` slices the accumulator (one of two, 256 columns each) is read and added in registers,
//     where sums round; the products of the next chain run meanwhile.
// Bound by the tensor cores, 74 to 81 % of whose cycles are products: 4 096 x 2 048 x 50 021 bf16 is 541 us with the softmax's sums
// (1 553 TFLOP/s), 581 with the slope or as a gradient (1 444).
// All waits are bounded: the one that runs out sets the error flag, and every role leaves.
#include "plane_gemm.h"

#include <algorithm>
#include <string>

#include "gemm_tc_host.h"
#include "pair_mma.cuh"
#include "tf_internal.h"
#include "values.cuh"

namespace tfk {

namespace {

constexpr int kPgDrainWarps = 8, kPgThreads = 32 * (kPgDrainWarps + 2);
constexpr int kPgSlice = 64;                     // terms: 128 bytes, a swizzle row
constexpr int kPgABytes = 128 * 128;             // a CTA's rows of A, one slice
constexpr int kPgMaxStages = 8;
constexpr int kPgRingBytes = 192 * 1024;
__host__ __device__ constexpr int pg_b_bytes(int bn) { return bn / 2 * 128; }

struct PlaneGemmParams {
  int m, n, slices, chain, planes, stages;
  int tiles_m, tiles_n, group, splits, split_slices;
  int a_rows, b_rows, f16;
  const float *scale_a, *scale_b;
  void *out; int out_dtype; long long ld_out;
  const float *sum_in; float *sum_out; long long ld_sum;
  const long long *target; int col0;
  float2 *sums; float *target_logit;
  const float *lse2, *row_scale;
  unsigned short *slope_hi, *slope_lo; long long ld_slope;
  int *error, wait_limit;
};

// kPlaneStore by way of shared memory.  Rows of a result lie apart: a lane stores whole sectors of 32 bytes of its row where rows start on
// them; where they don't, neighbouring columns go to neighbouring lanes first (100 000 x 300 fp32 from 100 terms: 72 us, 236 value by
// value; a kernel of its own, since one with both has fewer registers for the sums: 4 096 x 2 048 x 50 021 bf16 3 % slower).
constexpr int kPgTurned = 3;
constexpr int kPgTurn = 17;  // words of a row on its way through shared memory, 16 and one so that columns lie in different banks

struct PgShared {
  unsigned long long full[kPgMaxStages], empty[kPgMaxStages];
  unsigned long long acc_full[2], acc_empty[2], drained;
  unsigned tmem_base;
  int dead;
};

// K-major tile: as umma_desc_sw128.  MN-major tile: blocks of 64 rows (128 bytes) x 64 terms, 8 KB from one to the next (leading
// offset), groups of eight terms 1 KB apart (stride offset).
__device__ __forceinline__ unsigned long long pg_desc(unsigned addr) {
  return (umma_desc_sw128(addr) & ~((unsigned long long)0x3fff << 16)) | (unsigned long long)(8192 >> 4) << 16;
}
__device__ __forceinline__ void pg_mma(unsigned d, unsigned long long da, unsigned long long db, unsigned idesc, unsigned acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
// A box of a 2-D tensor into this CTA's shared memory; its bytes count on the barrier at `bar`, an address in the cluster.
__device__ __forceinline__ void pg_load(unsigned dst, const CUtensorMap *tm, int c0, int c1, unsigned bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"((unsigned long long)tm), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct PgTile { int m0, n0, split; };
// Tiles of `group` row blocks go through all columns before the next group's: what runs at one time shares rows and columns.
__device__ __forceinline__ PgTile pg_tile(const PlaneGemmParams &P, int t, int bn) {
  const int per = P.tiles_m * P.tiles_n, split = t / per;
  t -= split * per;
  const int band = P.group * P.tiles_n, g = t / band, rows = min(P.group, P.tiles_m - g * P.group);
  t -= g * band;
  return {(g * P.group + t % rows) * 256, t / rows * bn, split};
}

constexpr float kLog2e = 1.4426950408889634f;

template <int BN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPgThreads, 1)
plane_gemm_kernel(const __grid_constant__ CUtensorMap tm_ahi, const __grid_constant__ CUtensorMap tm_alo,
                  const __grid_constant__ CUtensorMap tm_bhi, const __grid_constant__ CUtensorMap tm_blo,
                  const __grid_constant__ PlaneGemmParams P) {
  constexpr int kCols = BN / 2;  // columns of a draining warp
  extern __shared__ char dyn[];
  __shared__ PgShared s;
  __shared__ unsigned turned[EPI == kPgTurned ? kPgDrainWarps : 1][EPI == kPgTurned ? 32 * kPgTurn : 1];
  char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  const unsigned rank = pair_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = P.tiles_m * P.tiles_n * P.splits;
  constexpr int plane_bytes = kPgABytes + pg_b_bytes(BN);
  const int stage_bytes = plane_bytes * P.planes;

  if (tid == 0) {
    for (int i = 0; i < P.stages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], 2 * kPgDrainWarps);
    }
    mbar_init(&s.drained, 1);
    s.dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem_base)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  pair_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");

  if (warp == kPgDrainWarps) {
    // ---- loads ----
    int st = 0, issued = 0;
    unsigned ph = 0;
    bool ok = true;
    auto wait = [&](unsigned long long *bar, unsigned parity) {
      return ok = __all_sync(kFull, pair_wait(bar, parity, s.dead, P.wait_limit));
    };
    for (int t = pair; t < tiles && ok; t += pairs) {
      const PgTile tile = pg_tile(P, t, BN);
      const int row = tile.m0 + (int)rank * 128, col = tile.n0 + (int)rank * kCols;
      const int sl1 = min(P.slices, (tile.split + 1) * P.split_slices);
      for (int sl = tile.split * P.split_slices; sl < sl1; ++sl) {
        if (issued >= P.stages && !wait(&s.empty[st], ph ^ 1u)) break;
        const unsigned base = smem_u32(smem + st * stage_bytes);
        unsigned bar;  // the even CTA's barrier
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(bar) : "r"(smem_u32(&s.full[st])));
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(&s.full[st], (unsigned)(2 * stage_bytes));
          const int k0 = sl * kPgSlice;
          for (int p = 0; p < P.planes; ++p) {
            const CUtensorMap *ta = p ? &tm_alo : &tm_ahi, *tb = p ? &tm_blo : &tm_bhi;
            const unsigned a = base + p * plane_bytes, b = a + kPgABytes;
            if (P.a_rows) {
              pg_load(a, ta, row, k0, bar);
              pg_load(a + 8192, ta, row + 64, k0, bar);
            } else pg_load(a, ta, k0, row, bar);
            if (BN >= 128 && P.b_rows) {
#pragma unroll
              for (int i = 0; i < kCols / 64; ++i) pg_load(b + i * 8192, tb, col + i * 64, k0, bar);
            } else pg_load(b, tb, k0, col, bar);
          }
        }
        __syncwarp();
        if (issued < P.stages) ++issued;
        if (++st == P.stages) { st = 0; ph ^= 1u; }
      }
    }
    // the tensor core's arrivals on this CTA's barriers come from the even CTA: the last of them must be in before the CTA ends
    for (int i = 0; ok && i < issued; ++i) wait(&s.empty[i], i < st ? ph : ph ^ 1u);
    // a copy still in flight must not outlive the pair (only after a wait ran out is one possible)
    if ((!ok || s.dead) && rank == 0)
      for (int i = 0; i < issued; ++i)
        mbar_wait(&s.full[i], i < st ? ph : ph ^ 1u, kInFlightPolls);
  } else if (warp == kPgDrainWarps + 1) {
    // ---- products (even CTA) ----
    if (rank == 0) {
      // fp32 accumulators, M = 256, N = BN; operands' type and which index of theirs is contiguous
      const unsigned type = P.f16 ? 0u : 1u;
      const unsigned idesc = (1u << 4) | (type << 7) | (type << 10) | ((unsigned)P.a_rows << 15) | ((unsigned)P.b_rows << 16) |
                             ((unsigned)(BN >> 3) << 17) | ((unsigned)(256 >> 4) << 24);
      const int step_a = P.a_rows ? 2048 >> 4 : 32 >> 4, step_b = P.b_rows ? 2048 >> 4 : 32 >> 4;  // 16 terms on, in descriptors
      int st = 0, buf = 0, uses = 0;
      unsigned ph = 0, acc_ph = 0;
      bool ok = true;
      auto wait = [&](unsigned long long *bar, unsigned parity) {
        return ok = __all_sync(kFull, pair_wait<true>(bar, parity, s.dead, P.wait_limit));
      };
      const unsigned tmem = s.tmem_base;
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int split = t / (P.tiles_m * P.tiles_n), sl0 = split * P.split_slices, sl1 = min(P.slices, sl0 + P.split_slices);
        int in_chain = 0;
        for (int sl = sl0; sl < sl1; ++sl) {
          if (in_chain == 0) {  // the accumulator has been read
            if (uses >= 2 && !wait(&s.acc_empty[buf], acc_ph ^ 1u)) break;
            if (uses < 2) ++uses;
          }
          if (!wait(&s.full[st], ph)) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const unsigned d = tmem + (unsigned)(buf * 256), a = smem_u32(smem + st * stage_bytes), b = a + kPgABytes;
          const unsigned long long ah = pg_desc(a), bh = pg_desc(b), al = pg_desc(a + plane_bytes), bl = pg_desc(b + plane_bytes);
          const bool last = sl == sl1 - 1 || in_chain == P.chain - 1;
          if (elect_one()) {
            if (P.planes == 2) {  // the small products first
#pragma unroll
              for (int j = 0; j < 4; ++j) pg_mma(d, al + j * step_a, bh + j * step_b, idesc, (in_chain | j) ? 1u : 0u);
#pragma unroll
              for (int j = 0; j < 4; ++j) pg_mma(d, ah + j * step_a, bl + j * step_b, idesc, 1u);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) pg_mma(d, ah + j * step_a, bh + j * step_b, idesc, P.planes == 2 || (in_chain | j) ? 1u : 0u);
            pair_commit(&s.empty[st]);
            if (last) pair_commit(&s.acc_full[buf]);
          }
          __syncwarp();
          if (last) {
            in_chain = 0;
            buf ^= 1;
            if (buf == 0) acc_ph ^= 1u;
          } else ++in_chain;
          if (++st == P.stages) { st = 0; ph ^= 1u; }
        }
      }
      if (!ok) {  // products still running read shared memory of both CTAs
        if (elect_one()) pair_commit_own(&s.drained);
        mbar_wait(&s.drained, 0, kInFlightPolls);
      }
    }
  } else {
    // ---- drain: warp w holds 32 rows and half of the columns ----
    const int quadrant = warp & 3, side = warp >> 2;
    int buf = 0;
    unsigned acc_ph = 0;
    bool ok = true;
    const unsigned lanes = s.tmem_base + ((unsigned)(quadrant * 32) << 16) + (unsigned)(side * kCols);
    float scale_a = 1.f, scale_b = 1.f;
    if (P.scale_a) scale_a = __ldg(P.scale_a);
    if (P.scale_b) scale_b = __ldg(P.scale_b);
    for (int t = pair; t < tiles && ok; t += pairs) {
      const PgTile tile = pg_tile(P, t, BN);
      const int sl0 = tile.split * P.split_slices, sl1 = min(P.slices, sl0 + P.split_slices);
      float acc[kCols];
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[c] = 0.f;
      for (int sl = sl0; sl < sl1; sl += P.chain) {
        if (!(ok = __all_sync(kFull, pair_wait(&s.acc_full[buf], acc_ph, s.dead, P.wait_limit)))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
          float v[16];
          tmem_load16(v, lanes + (unsigned)(buf * 256 + c));
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[c + q] += v[q];
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) pair_arrive_leader(&s.acc_empty[buf]);
        buf ^= 1;
        if (buf == 0) acc_ph ^= 1u;
      }
      if (!ok) break;
      const int row = tile.m0 + (int)rank * 128 + quadrant * 32 + lane, col = tile.n0 + side * kCols;
      if (row >= P.m && EPI != kPgTurned) continue;
      if (EPI == kPlaneStore || EPI == kPgTurned) {
        if (P.sum_in && row < P.m) {
          const float *x = P.sum_in + ((size_t)tile.split * P.m + row) * P.ld_sum + col;
#pragma unroll
          for (int c = 0; c < kCols; c += 4)
            if (col + c < P.n) {  // (sums have rows of whole eights)
              const float4 q = *reinterpret_cast<const float4 *>(x + c);
              acc[c] += q.x; acc[c + 1] += q.y; acc[c + 2] += q.z; acc[c + 3] += q.w;
            }
        }
        if (EPI != kPgTurned && P.sum_out) {
          float *x = P.sum_out + ((size_t)tile.split * P.m + row) * P.ld_sum + col;
#pragma unroll
          for (int c = 0; c < kCols; c += 8)
            if (col + c < P.n) {
              Pack<float, 8> q;
#pragma unroll
              for (int k = 0; k < 8; ++k) q.v[k] = acc[c + k];
              store_raw<float, 8>(x + c, q);
            }
        } else {
#pragma unroll
          for (int c = 0; c < kCols; ++c) acc[c] = acc[c] * scale_a * scale_b;
          const long long at = (long long)row * P.ld_out + col;
          const bool f16 = P.out_dtype == TF_F16;
          if (EPI == kPgTurned) {
            unsigned *words = turned[EPI == kPgTurned ? warp : 0];
            const int row0 = row - lane, rows = min(32, P.m - row0);
            if (P.out_dtype == TF_F32) {
              const int in = lane & 15;
#pragma unroll
              for (int c = 0; c < kCols; c += 16) {
                if (col + c >= P.n) break;
#pragma unroll
                for (int q = 0; q < 16; ++q) words[lane * kPgTurn + q] = __float_as_uint(acc[c + q]);
                __syncwarp();
                float *x = static_cast<float *>(P.out) + (long long)row0 * P.ld_out + col + c + in;
                if (col + c + in < P.n)
                  for (int r = lane >> 4; r < rows; r += 2) x[r * P.ld_out] = __uint_as_float(words[r * kPgTurn + in]);
                __syncwarp();
              }
            } else {
#pragma unroll
              for (int c = 0; c < kCols; c += 32) {
                if (col + c >= P.n) break;
#pragma unroll
                for (int q = 0; q < 16; ++q) words[lane * kPgTurn + q] = pack_pair(acc[c + 2 * q], acc[c + 2 * q + 1], f16);
                __syncwarp();
                unsigned short *x = static_cast<unsigned short *>(P.out) + (long long)row0 * P.ld_out + col + c + lane;
                if (col + c + lane < P.n)
                  for (int r = 0; r < rows; ++r) x[r * P.ld_out] = (unsigned short)(words[r * kPgTurn + lane / 2] >> (lane & 1) * 16);
                __syncwarp();
              }
            }
          } else if (P.out_dtype == TF_F32) {
            float *x = static_cast<float *>(P.out) + at;
#pragma unroll
            for (int c = 0; c < kCols; c += 8) {
              if (col + c + 7 < P.n) {
                Pack<float, 8> a;
#pragma unroll
                for (int q = 0; q < 8; ++q) a.v[q] = acc[c + q];
                store_raw<float, 8>(x + c, a);
              } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                  if (col + c + q < P.n) x[c + q] = acc[c + q];
              }
            }
          } else {
            unsigned short *x = static_cast<unsigned short *>(P.out) + at;
#pragma unroll
            for (int c = 0; c < kCols; c += 16) {
              Pack<unsigned, 8> a;
#pragma unroll
              for (int q = 0; q < 8; ++q) a.v[q] = pack_pair(acc[c + 2 * q], acc[c + 2 * q + 1], f16);
              if (col + c + 15 < P.n) store_raw<unsigned, 8>(reinterpret_cast<unsigned *>(x + c), a);
              else {
#pragma unroll
                for (int q = 0; q < 16; ++q)
                  if (col + c + q < P.n) x[c + q] = (unsigned short)(a.v[q / 2] >> (q & 1) * 16);
              }
            }
          }
        }
      } else {
        const float to_logit = scale_a, more = scale_b;
        const long long place = P.target[row] - P.col0 - col;
        const int want = place >= 0 && place < kCols && col + place < P.n ? (int)place : -1;  // the target among this thread's columns
        if (EPI == kPlaneSoftmaxSums) {
          float top = -INFINITY;
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            acc[c] = acc[c] * to_logit * more;
            if (col + c >= P.n) acc[c] = -INFINITY;
          }
#pragma unroll
          for (int c = 0; c < kCols; c += 2) top = max3(top, acc[c], acc[c + 1]);  // (a NaN if one of them is: a part of NaN alone is not an empty one)
          if (want >= 0) {
            float l = 0.f;
#pragma unroll
            for (int c = 0; c < kCols; ++c)
              if (c == want) l = acc[c];
            P.target_logit[row] = l;
          }
          const float top2 = top * kLog2e;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          if (top != -INFINITY) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) sum[c & 3] += ex2(fmaf(acc[c], kLog2e, -top2));
          }
          P.sums[(size_t)(tile.n0 / kCols + side) * P.m + row] = make_float2(top2, (sum[0] + sum[1]) + (sum[2] + sum[3]));
        } else {
          const float lse2 = __ldg(P.lse2 + row), by = __ldg(P.row_scale + row);
          const float in2 = to_logit * kLog2e;  // (a power of two: exact)
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            const float p = ex2(fmaf(acc[c] * more, in2, -lse2)) - (c == want ? 1.f : 0.f);
            acc[c] = by == 0.f ? 0.f : p * by;  // (a row that does not count stays zero whatever it holds)
          }
          unsigned short *hi = P.slope_hi + (size_t)row * P.ld_slope + col;
          unsigned short *lo = P.slope_lo ? P.slope_lo + (size_t)row * P.ld_slope + col : nullptr;
#pragma unroll
          for (int c = 0; c < kCols; c += 8) {
            if (col + c >= P.ld_slope) break;
            unsigned u[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) u[q] = pack_pair(acc[c + 2 * q], acc[c + 2 * q + 1], P.f16);
            *reinterpret_cast<uint4 *>(hi + c) = make_uint4(u[0], u[1], u[2], u[3]);
            if (lo) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&u[q]));
                u[q] = pack_pair(acc[c + 2 * q] - h.x, acc[c + 2 * q + 1] - h.y, true);
              }
              *reinterpret_cast<uint4 *>(lo + c) = make_uint4(u[0], u[1], u[2], u[3]);
            }
          }
        }
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (tid == 0 && s.dead) atomicExch(P.error, 1);
  pair_sync();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(s.tmem_base), "n"(512) : "memory");
  }
}

// 16-bit planes: boxes of 64 contiguous values (128 bytes, swizzled) x box_rows, zero outside.
int pg_map(CUtensorMap *out, const void *base, long long inner, long long rows, long long ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return tf::fail(TF_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t gdim[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t gstride[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {(cuuint32_t)kPgSlice, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), gdim, gstride, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TF_OK : tf::fail(TF_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
}

template <int BN, int EPI>
cudaError_t pg_launch(const CUtensorMap *maps, const PlaneGemmParams &P, int pairs, cudaStream_t s) {
  auto f = plane_gemm_kernel<BN, EPI>;
  const int smem = kPgRingBytes + 1024;
  const cudaError_t e = cudaFuncSetAttribute((const void *)f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  f<<<2 * pairs, kPgThreads, smem, s>>>(maps[0], maps[1], maps[2], maps[3], P);
  return cudaGetLastError();
}

}  // namespace

// As narrow as keeps every pair of SMs at a tile at most: few rows leave few tiles, whose sums then take as long as their width.
int plane_gemm_width(int m, int n, bool b_along_rows) {
  const long long tiles_m = (m + 255) / 256;
  for (int bn = b_along_rows ? 128 : 64; bn < 256; bn *= 2)
    if (n <= bn || tiles_m * ((n + bn - 1) / bn) <= 74) return bn;
  return 256;
}
int plane_gemm_parts(int m, int n) { const int bn = plane_gemm_width(m, n, false); return 2 * ((n + bn - 1) / bn); }

int plane_gemm_splits(int k, int split_slices) {
  const int slices = (k + kPgSlice - 1) / kPgSlice;
  return split_slices > 0 ? (slices + split_slices - 1) / split_slices : 1;
}

int plane_gemm(const PlaneGemmCall &c, int *error, int wait_limit, int sm_count, cudaStream_t s) {
  const int bn = plane_gemm_width(c.m, c.n, c.b.along_rows);
  PlaneGemmParams P = {};
  P.m = c.m; P.n = c.n;
  P.slices = (c.k + kPgSlice - 1) / kPgSlice;
  P.chain = std::max(1, c.chain);
  P.planes = c.a.lo ? 2 : 1;
  P.stages = std::min(kPgMaxStages, kPgRingBytes / ((kPgABytes + pg_b_bytes(bn)) * P.planes));
  P.tiles_m = (c.m + 255) / 256; P.tiles_n = (c.n + bn - 1) / bn;
  P.group = std::min(P.tiles_m, 16);
  P.split_slices = c.split_slices > 0 ? c.split_slices : P.slices;
  P.splits = plane_gemm_splits(c.k, c.split_slices);
  P.a_rows = c.a.along_rows; P.b_rows = c.b.along_rows; P.f16 = c.f16;
  P.scale_a = c.scale_a; P.scale_b = c.scale_b;
  P.out = c.out; P.out_dtype = c.out_dtype; P.ld_out = c.ld_out;
  P.sum_in = c.sum_in; P.sum_out = c.sum_out; P.ld_sum = c.ld_sum;
  P.target = c.target; P.col0 = c.col0;
  P.sums = c.sums; P.target_logit = c.target_logit;
  P.lse2 = c.lse2; P.row_scale = c.row_scale;
  P.slope_hi = (unsigned short *)c.slope_hi; P.slope_lo = (unsigned short *)c.slope_lo; P.ld_slope = c.ld_slope;
  P.error = error; P.wait_limit = wait_limit;
  CUtensorMap maps[4];
  auto map = [&](CUtensorMap *to, const PlaneOperand &o, const void *plane, int rows, int box) {
    return o.along_rows ? pg_map(to, plane, rows, c.k, o.ld, kPgSlice) : pg_map(to, plane, c.k, rows, o.ld, box);
  };
  int rc = map(&maps[0], c.a, c.a.hi, c.m, 128);
  if (rc == TF_OK) rc = map(&maps[1], c.a, c.a.lo ? c.a.lo : c.a.hi, c.m, 128);
  if (rc == TF_OK) rc = map(&maps[2], c.b, c.b.hi, c.n, bn / 2);
  if (rc == TF_OK) rc = map(&maps[3], c.b, c.b.lo ? c.b.lo : c.b.hi, c.n, bn / 2);
  if (rc != TF_OK) return rc;
  const long long tiles = (long long)P.tiles_m * P.tiles_n * P.splits;
  if (tiles > (1 << 30)) return tf::fail(TF_ERR_UNSUPPORTED, "dense product: too many tiles");
  const int pairs = (int)std::max<long long>(1, std::min<long long>(tiles, sm_count / 2));
  const bool whole = c.sum_out || (c.ld_out * value_bytes(c.out_dtype) % 32 == 0 && (reinterpret_cast<uintptr_t>(c.out) & 31) == 0);
  cudaError_t e;
#define TF_PG(BN)                                                                                  \
  (c.epilogue == kPlaneStore         ? (whole ? pg_launch<BN, kPlaneStore> : pg_launch<BN, kPgTurned>)(maps, P, pairs, s) \
   : c.epilogue == kPlaneSoftmaxSums ? pg_launch<BN, kPlaneSoftmaxSums>(maps, P, pairs, s)         \
                                     : pg_launch<BN, kPlaneSoftmaxSlope>(maps, P, pairs, s))
  e = bn == 64 ? TF_PG(64) : bn == 128 ? TF_PG(128) : TF_PG(256);
#undef TF_PG
  if (e != cudaSuccess) return tf::fail(TF_ERR_CUDA, std::string("dense product: ") + cudaGetErrorString(e));
  return TF_OK;
}

}  // namespace tfk
