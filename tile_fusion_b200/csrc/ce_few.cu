// Softmax cross entropy of a linear layer over at most 64 classes and 256 columns: node classification, many rows and little work
// to each.  Bound by x, which the forward pass reads once, and by x and dx, which the backward pass reads and writes once.
//
//   * A CTA walks tiles of 64 rows.  Seven warps (forward thirteen) bring the next tile from memory, all of it in flight at once, and
//     leave it in shared memory as 16-bit operands (two buffers); the weight is there from the start, in the same form.  fp32 values
//     become two fp16 planes behind a power of two, x = 2^-e (hi + lo), of which a tile has one of its own: products hi hi + hi lo +
//     lo hi.
//   * One warp issues the products of a tile (tcgen05.mma, M = 128 of which 64 rows count): logits L = X W^T, one tile ahead;
//     then, 128 columns at a time through three accumulators, dX = P W and dW += P^T X.  X, W and P lie in shared memory once and
//     are read along either index (K-major or MN-major, both with the 128-byte swizzle).
//   * Eight warps (forward two) turn logits into losses, or into the slope P = (exp(l - lse) - (class == target)) * row_scale as operand planes,
//     write dX, and add up dW in registers: 24 additions in tensor memory, which cuts off, then one that rounds.
//   * The CTAs' dW are added by a second launch, in order.
// 120 001 rows, 256 columns, 47 classes: the forward pass 55 us in fp32 and 33 in bf16, the backward pass 111 and 78, small launches before and
// behind included, bound by a tile's way through these stages: neither memory (2.4 TB/s in fp32) nor the tensor cores (25 and 35 % of the time)
// nor the schedulers (0.36 and 0.26 instructions a cycle) are busy for long.
// All waits are bounded: the one that runs out sets the error flag, and every role leaves.
#include "ce_few.h"

#include <algorithm>
#include <type_traits>

#include "pair_mma.cuh"
#include "values.cuh"

namespace tfk {

namespace {

constexpr int kFewRows = 64, kFewThreads = 512;
constexpr int kFewBlock = kFewRows * 128;  // bytes of 64 columns of a tile
// Warps of the backward pass: those that may read the accumulators' lanes of 64 rows (of four two), one that issues the products, and
// seven for the tiles; forward two of the former are enough, and thirteen bring tiles.
constexpr int kFewMmaWarp = 15;
__host__ __device__ constexpr int few_drains(bool back) { return back ? 8 : 2; }
__host__ __device__ constexpr int few_loaders(bool back) { return 15 - few_drains(back); }
constexpr int kFewRegions = 3;             // accumulators of 128 columns behind two of 64 for the logits
constexpr float kFewLog2e = 1.4426950408889634f, kFewLn2 = 0.69314718055994531f;

struct FewShared {
  unsigned long long x_full[2], x_empty[2], w_full, log_full[2], log_empty[2], p_full[2], job_full[kFewRegions], job_empty[kFewRegions], drained;
  unsigned top[2][few_loaders(false)];
  float unscale_x[2], unscale_w;
  double loss[2];
  int count[2];
  unsigned tmem_base;
  int dead;
};

__device__ __forceinline__ unsigned long long few_desc(unsigned addr) {  // MN-major: blocks of 64 columns kFewBlock apart
  return (umma_desc_sw128(addr) & ~((unsigned long long)0x3fff << 16)) | (unsigned long long)(kFewBlock >> 4) << 16;
}
__device__ __forceinline__ unsigned few_idesc(bool f16, int a_rows, int b_rows, int n) {
  const unsigned type = f16 ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | ((unsigned)a_rows << 15) | ((unsigned)b_rows << 16) | ((unsigned)(n >> 3) << 17) | ((unsigned)(128 >> 4) << 24);
}
__device__ __forceinline__ void few_mma(unsigned d, unsigned long long da, unsigned long long db, unsigned idesc, unsigned acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ float few_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void few_arrive(unsigned long long *bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Whether a phase has completed, without waiting for it (a try_wait may be put to sleep).
__device__ __forceinline__ bool few_done(unsigned long long *bar, unsigned parity) {
  unsigned done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return __all_sync(kFull, done != 0);
}

// DT: tf_dtype of x, w and dx.  BLOCKS: blocks of 64 columns; known, so that the issuing warp's descriptors are one register and
// constants.
template <int DT, int BLOCKS, bool BACK>
__global__ void __launch_bounds__(kFewThreads, 1) ce_few_kernel(const CeFewCall P) {
  constexpr int PLANES = DT == TF_F32 ? 2 : 1;
  constexpr bool F16 = DT != TF_BF16;
  constexpr int kFewLoaders = few_loaders(BACK), kDrains = few_drains(BACK);
  extern __shared__ char dyn[];
  __shared__ FewShared s;
  char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  constexpr int plane = BLOCKS * kFewBlock, tile_bytes = PLANES * plane;
  // two slopes, two tiles of x, the weight: an operand of 128 rows of which 64 count reads into what lies behind it
  constexpr int slope_bytes = PLANES * kFewBlock;
  const unsigned at_p = smem_u32(smem), at_x = at_p + 2 * slope_bytes, at_w = at_x + 2 * tile_bytes;
  const int tiles_all = (P.rows + kFewRows - 1) / kFewRows;
  const int tiles = tiles_all > (int)blockIdx.x ? (tiles_all - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x : 0;
  constexpr int halves = (BLOCKS + 1) / 2;  // of 128 columns

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.x_full[i], kFewLoaders); mbar_init(&s.x_empty[i], BACK ? 1 : 1 + kDrains);
      mbar_init(&s.log_full[i], 1); mbar_init(&s.log_empty[i], kDrains);
      mbar_init(&s.p_full[i], kDrains);
    }
    mbar_init(&s.w_full, kFewLoaders);
    mbar_init(&s.drained, 1);
    for (int i = 0; i < kFewRegions; ++i) { mbar_init(&s.job_full[i], 1); mbar_init(&s.job_empty[i], kDrains); }
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
  bool ok = true;
  auto wait = [&](unsigned long long *bar, unsigned parity) { return ok = __all_sync(kFull, pair_wait(bar, parity, s.dead, P.wait_limit)); };

  if (warp == kFewMmaWarp) {
    // ---- products ----
    const unsigned tmem = s.tmem_base;
    int job = 0;  // accumulators of 128 columns handed out so far
    // D = sum of BL products of planes, the small ones (lo hi, hi lo) before all hi hi; of four steps of 16 terms each
    auto product = [&](auto bl, unsigned d, unsigned a, unsigned b, auto plane_a, auto plane_b, auto step_a, auto step_b, unsigned idesc) {
      const unsigned long long da = few_desc(a), db = few_desc(b);
#pragma unroll
      for (int q = PLANES == 2 ? 0 : 2; q < 3; ++q)
#pragma unroll
        for (int c = 0; c < decltype(bl)::value; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            few_mma(d, da + (unsigned)(((q == 0 ? decltype(plane_a)::value : 0) + c * kFewBlock + k * decltype(step_a)::value) >> 4),
                    db + (unsigned)(((q == 1 ? decltype(plane_b)::value : 0) + c * kFewBlock + k * decltype(step_b)::value) >> 4), idesc,
                    q == (PLANES == 2 ? 0 : 2) && c == 0 && k == 0 ? 0u : 1u);
    };
    using One = std::integral_constant<int, 1>;
    using Plane = std::integral_constant<int, plane>;
    using Slope = std::integral_constant<int, kFewBlock>;
    using Along = std::integral_constant<int, 32>;     // 16 terms on where they are contiguous
    using Across = std::integral_constant<int, 2048>;  // and where they are rows
    static_assert(kFewRows / 16 == 4 && kFewClasses / 16 == 4, "steps of a product");
    auto logits = [&](int t) {
      const int b = t & 1;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (elect_one()) {  // (a block of 64 columns is a K-major tile of its own)
        product(std::integral_constant<int, BLOCKS>(), tmem + b * 64, at_x + b * tile_bytes, at_w, Plane(), Plane(), Along(), Along(), few_idesc(F16, 0, 0, 64));
        umma_commit(&s.log_full[b]);
        if (!BACK) umma_commit(&s.x_empty[b]);
      }
      __syncwarp();
    };
    // One of the products of a tile's gradients: 128 columns of dW, which the tile's place is free after, or of dX.
    const int jobs_w = P.dw_parts ? halves : 0, jobs = jobs_w + (P.dx ? halves : 0);
    auto gradient = [&](int t, int j) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned x = at_x + (t & 1) * tile_bytes, slope = at_p + (t & 1) * slope_bytes;
      const bool to_w = j < jobs_w;
      const int h = to_w ? j : j - jobs_w, n = min(128, BLOCKS * 64 - h * 128), r = job % kFewRegions;
      if (elect_one()) {
        const unsigned d = tmem + 128 + r * 128;
        if (to_w) product(One(), d, slope, x + h * 2 * kFewBlock, Slope(), Plane(), Across(), Across(), few_idesc(F16, 1, 1, n));
        else product(One(), d, slope, at_w + h * 2 * kFewBlock, Slope(), Plane(), Along(), Across(), few_idesc(F16, 0, 1, n));
        umma_commit(&s.job_full[r]);
        if (j == max(jobs_w, 1) - 1) umma_commit(&s.x_empty[t & 1]);
      }
      __syncwarp();
    };
    // Whatever can run: logits of the next tile whose rows and accumulator are ready, else a product of the gradients of the next whose
    // slope is, into the next accumulator that has been read.  Nothing is waited for: the warps that read accumulators wait for the
    // logits of the next tile before they read this one's gradients.
    if (tiles > 0) wait(&s.w_full, 0);
    int next = 0, done = BACK ? 0 : tiles, step = 0;
    for (long long idle = 0; ok && (next < tiles || done < tiles);) {
      if (next < tiles && few_done(&s.x_full[next & 1], (unsigned)(next / 2) & 1u) &&
          (next < 2 || few_done(&s.log_empty[next & 1], (unsigned)(next / 2 - 1) & 1u))) {
        logits(next++);
        idle = 0;
      } else if (BACK && done < next && (step > 0 || few_done(&s.p_full[done & 1], (unsigned)(done / 2) & 1u)) &&
                 (job < kFewRegions || few_done(&s.job_empty[job % kFewRegions], (unsigned)(job / kFewRegions - 1) & 1u))) {
        gradient(done, step);
        ++job;
        if (++step == jobs) { step = 0; ++done; }
        idle = 0;
      } else {
        __nanosleep(20);  // (the loop would take the issue slots of the warps that bring tiles)
        if (++idle <= 64ll * P.wait_limit && !*reinterpret_cast<volatile int *>(&s.dead)) continue;
        s.dead = 1;
        ok = false;
      }
    }
    // the last arrivals on barriers that nobody waits for must be in before the CTA ends
    if (ok)
      for (int t = max(0, tiles - 2); t < tiles; ++t) wait(&s.x_empty[t & 1], (unsigned)(t / 2) & 1u);
    if (!ok) {  // products still running read shared memory and write tensor memory
      if (elect_one()) umma_commit(&s.drained);
      mbar_wait(&s.drained, 0, kInFlightPolls);
    }
  } else if (BACK ? (warp & 3) < 2 : warp < 2) {
    // ---- rows 32 (warp & 3) .. + 31 of a tile, and (backward) a quarter of the columns ----
    const int quadrant = warp & 3, side = warp >> 2, in_tile = quadrant * 32 + lane;
    const unsigned lanes = s.tmem_base + ((unsigned)(quadrant * 32) << 16);
    float dw[BACK ? 64 : 1];
    if (BACK)
#pragma unroll
      for (int i = 0; i < 64; ++i) dw[BACK ? i : 0] = 0.f;
    double loss = 0.;
    int count = 0, job = 0;
    float unscale_w = 1.f, unscale_p = 1.f;
    const bool whole_dx = P.cols % 8 == 0 && (reinterpret_cast<uintptr_t>(P.dx) & (DT == TF_F32 ? 31 : 15)) == 0;  // (32 or 16 bytes a store)
    if (tiles > 0 && wait(&s.w_full, 0)) unscale_w = s.unscale_w;
    if (BACK) unscale_p = __ldg(P.unscale);
    float scale_of[2];
    // logits of a tile into losses, or into its slope
    auto softmax = [&](int t) {
      const int b = t & 1;
      const long long row = ((long long)blockIdx.x + (long long)t * gridDim.x) * kFewRows + in_tile;
      const bool in = row < P.rows;
      const long long target = in ? __ldg(P.target + row) : -1;
      float lse2 = 0.f, by = 0.f;
      if (BACK && in) { lse2 = __ldg(P.lse2 + row); by = __ldg(P.row_scale + row); }
      if (!wait(&s.x_full[b], (unsigned)(t / 2) & 1u) || !wait(&s.log_full[b], (unsigned)(t / 2) & 1u)) return;
      const float unscale_x = scale_of[b] = s.unscale_x[b];  // (backward: before P, after which the tile may be replaced)
      if (!BACK) few_arrive(&s.x_empty[b]);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (!BACK) {
        {  // all classes of a row are one thread's
          float top = -INFINITY, own = 0.f, sum = 0.f, l[64];
#pragma unroll
          for (int c = 0; c < 64; c += 16) {
            float v[16];
            tmem_load16(v, lanes + b * 64 + c);
#pragma unroll
            for (int q = 0; q < 16; ++q) {
              l[c + q] = c + q < P.vocab ? v[q] * unscale_x * unscale_w : -INFINITY;
              top = fmaxf(top, l[c + q]);
              if (c + q == target) own = l[c + q];
            }
          }
          const float top2 = top * kFewLog2e;
#pragma unroll
          for (int c = 0; c < 64; ++c) sum += few_ex2(fmaf(l[c], kFewLog2e, -top2));
          const float out = top2 + log2f(sum);
          if (in) {
            P.lse2[row] = out;
            float r = 0.f;
            if (target != P.ignore) {
              ++count;
              r = target < 0 || target >= P.vocab ? __int_as_float(0x7fc00000) : out * kFewLn2 - own;
            }
            if (P.row_loss) P.row_loss[row] = r;
            loss += r;
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        few_arrive(&s.log_empty[b]);
        return;
      }
      {
        float v[16];
        tmem_load16(v, lanes + b * 64 + side * 16);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        few_arrive(&s.log_empty[b]);
        const float in2 = unscale_w * kFewLog2e;  // (one power of two at a time: a logit of zero stays zero where their product leaves the range)
        const int mine = in && target >= side * 16 && target < side * 16 + 16 ? (int)target - side * 16 : -1;
        const unsigned to = at_p + b * slope_bytes + in_tile * 128;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float e = few_ex2(fmaf(PLANES == 2 ? v[c] * unscale_x : v[c], in2, -lse2)) - (c == mine ? 1.f : 0.f);
          v[c] = by == 0.f || side * 16 + c >= P.vocab ? 0.f : e * by;  // (a row that does not count stays zero whatever it holds)
        }
#pragma unroll
        for (int c = 0; c < 16; c += 8) {
          unsigned hi[4], lo[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            hi[q] = pack_pair(v[c + 2 * q], v[c + 2 * q + 1], F16);
            if (PLANES == 2) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[q]));
              lo[q] = pack_pair(v[c + 2 * q] - f.x, v[c + 2 * q + 1] - f.y, true);
            }
          }
          const unsigned a = to + (unsigned)(((side * 2 + c / 8) ^ (in_tile & 7)) * 16);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
          if (PLANES == 2)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a + kFewBlock), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        few_arrive(&s.p_full[b]);
      }
    };
    // a tile's gradients out of tensor memory
    auto drain = [&](int t) {
      const long long row = ((long long)blockIdx.x + (long long)t * gridDim.x) * kFewRows + in_tile;
      const bool in = row < P.rows;
      const float unscale_x = t & 1 ? scale_of[1] : scale_of[0];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool to_w = j < 2;
        const int h = j & 1;
        if (h >= halves || (to_w ? !P.dw_parts : !P.dx)) continue;
        const int r = job % kFewRegions;
        if (!wait(&s.job_full[r], (unsigned)(job / kFewRegions) & 1u)) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int col = h * 128 + side * 32;
        float v[32];
        tmem_load32(v, lanes + 128 + r * 128 + side * 32);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        tmem_loaded(v);
        if (to_w) {
          if (col < BLOCKS * 64) {
#pragma unroll
            for (int c = 0; c < 32; ++c) dw[BACK ? h * 32 + c : 0] = fmaf(v[c], unscale_x, dw[BACK ? h * 32 + c : 0]);
          }
        } else if (in) {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = v[c] * unscale_p * unscale_w;
          const long long at = row * P.cols + col;
          if (whole_dx) {  // whole sectors at a time
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
              if (col + c >= P.cols) break;
              if constexpr (DT == TF_F32) {
                Pack<float, 8> a;
#pragma unroll
                for (int k = 0; k < 8; ++k) a.v[k] = v[c + k];
                store_raw<float, 8>(static_cast<float *>(P.dx) + at + c, a);
              } else
                *reinterpret_cast<uint4 *>(static_cast<unsigned short *>(P.dx) + at + c) =
                    make_uint4(pack_pair(v[c], v[c + 1], F16), pack_pair(v[c + 2], v[c + 3], F16), pack_pair(v[c + 4], v[c + 5], F16), pack_pair(v[c + 6], v[c + 7], F16));
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (col + c < P.cols) store_value(P.dx, DT, at + c, v[c]);
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        few_arrive(&s.job_empty[r]);
        ++job;
      }
    };
    // The slope of the next tile first, so that its products follow this one's.
    if (tiles > 0) softmax(0);
    for (int t = 0; t < tiles && ok; ++t) {
      if (t + 1 < tiles) softmax(t + 1);
      if (BACK && ok) drain(t);
    }
    const bool lost = !ok || *reinterpret_cast<volatile int *>(&s.dead);
    if (BACK && P.dw_parts && in_tile < P.vocab) {
      float *to = P.dw_parts + ((size_t)blockIdx.x * P.vocab + in_tile) * P.cols;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const int col = h * 128 + side * 32 + c;
          if (col < P.cols) to[col] = lost ? __int_as_float(0x7fc00000) : dw[BACK ? h * 32 + c : 0];
        }
    }
    if (!BACK) {
      if (lost) loss = __longlong_as_double(0x7ff8000000000000ll);
      for (int k = 16; k; k >>= 1) {
        loss += __shfl_xor_sync(kFull, loss, k);
        count += __shfl_xor_sync(kFull, count, k);
      }
      if (lane == 0) { s.loss[quadrant] = loss; s.count[quadrant] = count; }
    }
  } else if (warp < kFewMmaWarp) {
    // ---- tiles of 64 rows into operands ----
    const int loader = BACK ? (warp >> 2) * 2 + (warp & 3) - 2 : warp - 2;
    constexpr int kMine = (kFewRows + kFewLoaders - 1) / kFewLoaders;  // rows of a warp: eight columns a lane
    const int col = lane * 8;
    using Raw = unsigned[kMine][PLANES * 4];  // rows as they lie in memory
    auto fetch = [&](Raw &raw, const void *src, long long ld, long long row0, unsigned wanted) {
      constexpr int BYTES = DT == TF_F32 ? 4 : 2;
      const bool whole = P.cols % 8 == 0 && ld * BYTES % 16 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
      const char *p = static_cast<const char *>(src) + ((row0 + loader) * ld + col) * BYTES;
#pragma unroll
      for (int i = 0; i < kMine; ++i, p += kFewLoaders * ld * BYTES) {
#pragma unroll
        for (int k = 0; k < PLANES * 4; ++k) raw[i][k] = 0;
        const bool in = (wanted >> i & 1u) && col < P.cols;
        if (whole) {
          if (in) {
#pragma unroll
            for (int k = 0; k < PLANES; ++k) {
              // (volatile: issued here, a tile ahead, not where the values are used)
              asm volatile("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(raw[i][4 * k]), "=r"(raw[i][4 * k + 1]), "=r"(raw[i][4 * k + 2]), "=r"(raw[i][4 * k + 3]) : "l"(p + k * 16));
            }
          }
        } else if (DT == TF_F32) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (in && col + k < P.cols) raw[i][k & (PLANES * 4 - 1)] = __ldg(reinterpret_cast<const unsigned *>(p) + k);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (in && col + k < P.cols) raw[i][k / 2] |= (unsigned)__ldg(reinterpret_cast<const unsigned short *>(p) + k) << (k & 1) * 16;
        }
      }
    };
    int turn = 0;
    auto put = [&](const Raw &raw, unsigned to, float *unscale) {
      float by = 1.f;
      if (DT == TF_F32) {  // the power of two that brings the tile's largest finite value to [2^14, 2^15)
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
#pragma unroll
          for (int k = 0; k < PLANES * 4; k += 2) m = max3_abs_numbers(m, __uint_as_float(raw[i][k]), __uint_as_float(raw[i][k + 1]));
        if (m == INFINITY) {
          m = 0.f;
#pragma unroll
          for (int i = 0; i < kMine; ++i)
#pragma unroll
            for (int k = 0; k < PLANES * 4; ++k) {
              const float a = fabsf(__uint_as_float(raw[i][k]));
              if (a < INFINITY) m = fmaxf(m, a);
            }
        }
        unsigned top = __float_as_uint(m);
        for (int k = 16; k; k >>= 1) top = max(top, __shfl_xor_sync(kFull, top, k));
        if (lane == 0) s.top[turn & 1][loader] = top;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kFewLoaders) : "memory");
#pragma unroll
        for (int k = 0; k < kFewLoaders; ++k) top = max(top, *reinterpret_cast<volatile unsigned *>(&s.top[turn & 1][k]));
        const int e = top ? min(126, 14 - ((int)(top >> 23) - 127)) : 0;
        by = __uint_as_float((unsigned)(e + 127) << 23);
        if (loader == 0 && lane == 0) *unscale = __uint_as_float((unsigned)(127 - e) << 23);
      } else if (loader == 0 && lane == 0) *unscale = 1.f;
      ++turn;
      if (col < BLOCKS * 64) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int r = i * kFewLoaders + loader;
          if (r >= kFewRows) continue;
          const unsigned a = to + (unsigned)(lane / 8 * kFewBlock + r * 128 + ((lane & 7) ^ (r & 7)) * 16);
          if (DT == TF_F32) {
            unsigned hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // (an infinity becomes a NaN in the sums: infinity and its rest, infinity - infinity)
              const float p = __uint_as_float(raw[i][(2 * k) & (PLANES * 4 - 1)]) * by, q = __uint_as_float(raw[i][(2 * k + 1) & (PLANES * 4 - 1)]) * by;
              hi[k] = pack_pair(p, q, true);
              const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[k]));
              lo[k] = pack_pair(p - f.x, q - f.y, true);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a + plane), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
          } else
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(raw[i][0]), "r"(raw[i][1]), "r"(raw[i][2]), "r"(raw[i][3]) : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read next by the tensor core
    };
    // Which of this warp's rows exist and count: lane i asks for the i-th, a tile before the rows themselves.
    auto row_of = [&](int t) { return ((long long)blockIdx.x + (long long)t * gridDim.x) * kFewRows; };
    const int mine = lane * kFewLoaders + loader;
    bool there = false;
    long long asked = 0;
    auto ask = [&](int t) {
      there = lane < kMine && mine < kFewRows && row_of(t) + mine < P.rows;
      if (there) asm volatile("ld.global.nc.b64 %0, [%1];" : "=l"(asked) : "l"(P.target + row_of(t) + mine));
    };
    auto fetch_tile = [&](Raw &raw, int t) {
      const unsigned wanted = __ballot_sync(kFull, there && asked != P.ignore);
      fetch(raw, P.x, P.ld_x, row_of(t), wanted);
      if (t + 1 < tiles) ask(t + 1);
    };
    auto put_tile = [&](const Raw &raw, int t) {
      // (where a wait has run out the waits end at once; no warp leaves, for the others would stay at the barrier in put())
      if (t >= 2) wait(&s.x_empty[t & 1], (unsigned)(t / 2 - 1) & 1u);
      put(raw, at_x + (t & 1) * tile_bytes, &s.unscale_x[t & 1]);
      few_arrive(&s.x_full[t & 1]);
    };
    Raw raw;
    if (tiles > 0) {
      ask(0);
      fetch(raw, P.w, P.ld_w, 0, __ballot_sync(kFull, lane < kMine && mine < kFewRows && mine < P.vocab));
      put(raw, at_w, &s.unscale_w);
      few_arrive(&s.w_full);
      fetch_tile(raw, 0);
    }
    if constexpr (BACK) {
      for (int t = 0; t < tiles; ++t) {
        put_tile(raw, t);
        if (t + 1 < tiles) fetch_tile(raw, t + 1);
      }
    } else {  // (five rows of a warp leave registers for the next tile's)
      Raw more;
      for (int t = 0; t < tiles; t += 2) {
        if (t + 1 < tiles) fetch_tile(more, t + 1);
        put_tile(raw, t);
        if (t + 1 >= tiles) break;
        if (t + 2 < tiles) fetch_tile(raw, t + 2);
        put_tile(more, t + 1);
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    if (s.dead) atomicExch(P.error, 1);
    if (!BACK && P.cta_loss) {
      P.cta_loss[blockIdx.x] = tiles > 0 ? s.loss[0] + s.loss[1] : 0.;
      P.cta_count[blockIdx.x] = tiles > 0 ? s.count[0] + s.count[1] : 0;
    }
  }
  // (a wait ran out: the losses of this CTA's rows are NaN, or their gradients, as its part of dW)
  if (!BACK && s.dead)
    for (int t = 0; t < tiles; ++t) {
      const long long row = ((long long)blockIdx.x + (long long)t * gridDim.x) * kFewRows + tid;
      if (tid >= kFewRows || row >= P.rows) continue;
      P.lse2[row] = __int_as_float(0x7fc00000);
      if (P.row_loss) P.row_loss[row] = P.target[row] == P.ignore ? 0.f : __int_as_float(0x7fc00000);
    }
  if (BACK && s.dead && P.dx)
    for (int t = 0; t < tiles; ++t) {
      const long long row0 = ((long long)blockIdx.x + (long long)t * gridDim.x) * kFewRows, at = row0 * P.cols;
      const int n = (int)min((long long)kFewRows, P.rows - row0) * P.cols;
      for (int i = tid; i < n; i += kFewThreads) store_value(P.dx, DT, at + i, __int_as_float(0x7fc00000));
    }
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem_base), "n"(512) : "memory");
  }
}

template <int DT, int BLOCKS, bool BACK> cudaError_t few_launch(const CeFewCall &c, cudaStream_t s) {
  auto f = ce_few_kernel<DT, BLOCKS, BACK>;
  constexpr int smem = (DT == TF_F32 ? 2 : 1) * (3 * BLOCKS + 2) * kFewBlock + 1024;
  const cudaError_t e = cudaFuncSetAttribute((const void *)f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  f<<<ce_few_ctas(c.rows), kFewThreads, smem, s>>>(c);
  return cudaGetLastError();
}
template <int DT, bool BACK> cudaError_t few_by_width(const CeFewCall &c, cudaStream_t s) {
  return c.cols <= 64 ? few_launch<DT, 1, BACK>(c, s) : c.cols <= 128 ? few_launch<DT, 2, BACK>(c, s) : few_launch<DT, 4, BACK>(c, s);
}
template <bool BACK> cudaError_t few_by_type(const CeFewCall &c, cudaStream_t s) {
  return c.dtype == TF_F32 ? few_by_width<TF_F32, BACK>(c, s) : c.dtype == TF_BF16 ? few_by_width<TF_BF16, BACK>(c, s) : few_by_width<TF_F16, BACK>(c, s);
}

}  // namespace

bool ce_few_supported(int cols, int vocab) { return vocab <= kFewClasses && cols <= kFewCols; }
int ce_few_ctas(int rows) { return std::max(1, std::min(148, (rows + kFewRows - 1) / kFewRows)); }
cudaError_t ce_few_forward(const CeFewCall &c, cudaStream_t s) { return few_by_type<false>(c, s); }
cudaError_t ce_few_backward(const CeFewCall &c, cudaStream_t s) { return few_by_type<true>(c, s); }

}  // namespace tfk
