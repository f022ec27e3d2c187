// dW = G^T X for a tall gradient G (fp32, bf16 or fp16) and an X kept in 8 bits (pack8.cuh): the weight gradient of a layer that
// keeps its input in 8 bits.  A sum over all rows with a small result, bound by reading G and the codes once.
//
//   * The rows are cut into as many ranges as the device holds CTAs; each adds up a tile of 128 x 256 or 256 x 128 sums (which of
//     the two: whatever reads less), and a second launch adds the ranges' tiles in order.
//   * Four teams of four warps (six for gradients in 16 bits) each turn 16 rows at a time into 16-bit operands in shared memory, row by
//     row as they lie (MN-major, 128-byte swizzle: nothing is transposed), while further rows are on their way; one warp issues
//     tcgen05.mma.  (All warps on the same 32 rows wait for one another in every step: 500 009 rows, 47 x 256 bf16: 127 us.)
//   * A value of X is seven bits and a power of two, exact in bf16.  G in fp32 is three bf16 planes (24 bits, exact), in fp16 two
//     (exact), in bf16 one.  So products lose nothing.
//   * The tensor core cuts off what it adds to an accumulator, 2e-8 of the sum each time: for fp32 after 128 rows (24 additions)
//     the accumulator, one of two, is read and added in registers, where sums round.
// Bound by the warps that make the operands: a scheduler issues 0.70 (bf16) and 0.55 (fp32) instructions a cycle, the tensor pipe is busy for
// 22 and 28 % of the time.  500 009 rows, 47 x 256 bf16: 75 us, 2.4 TB/s; 2 449 029 rows, 256 x 100 fp32: 663 us, 4.2 TB/s (three planes of G
// to make, and a look at each value for infinities: 22 us of them).
// All waits are bounded: where one runs out the CTA's sums, and with them the result, become NaN.
#include <algorithm>
#include <string>
#include <type_traits>

#include "pack8.cuh"
#include "pair_mma.cuh"
#include "tf_internal.h"

namespace tfk {

namespace {

// Teams of four warps.  Gradients in 16 bits (one or two planes) leave their sums in tensor memory to the end: 2e-8 of the sum for each
// of at most 4 096 additions (kWgStayRows) is 1e-4, where the result is rounded to 2^-8 or 2^-11 = 5e-4, and warps that hold no sums
// are small enough for six teams.
constexpr int kWgStayRows = 32768;
constexpr int kWgTeam = 128, kWgMaxTeams = 6;
__host__ __device__ constexpr int wg_teams(int planes) { return planes == 3 ? 4 : 6; }
__host__ __device__ constexpr int wg_threads(int planes, bool ring) { return kWgTeam * wg_teams(planes) + 32 * (ring ? 2 : 1); }
constexpr int kWgRows = 16;                    // of a slice: a K step
constexpr int kWgChain = 8;                    // (fp32) slices added up in tensor memory, a multiple of the teams
constexpr int kWgBlock = kWgRows * 128;        // bytes of 64 columns of a slice
constexpr int kWgMaxRing = 16;
constexpr int kWgSmem = 224 * 1024;

__host__ __device__ constexpr int wg_stage_bytes(int planes, int mt) { return planes * mt * 2 * kWgBlock + (mt == 1 ? 4 : 2) * kWgBlock; }
static_assert(wg_teams(3) * wg_stage_bytes(3, 2) <= kWgSmem && wg_teams(2) * wg_stage_bytes(2, 2) <= kWgSmem, "a stage to each team");

struct WgParams {
  const void *g; long long ld_g; int na;
  const signed char *codes; int ld_codes, nb; const unsigned char *exps;
  int m, rows;  // rows of a range
  bool whole_g;
  int wait_limit;
  int ring, g_bytes, ring_bytes;  // slices as they lie in memory that are on their way, bytes of G and of all of one
  float *part;  // [range][na][nb]
};

struct WgShared {
  unsigned long long raw_full[kWgMaxRing], raw_empty[kWgMaxRing];
  unsigned long long full[kWgMaxTeams], empty[kWgMaxTeams], tail[kWgMaxTeams], acc_full[2], acc_empty[2], drained;
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

// Where rows are read from: global memory (a pointer), or places of the ring in shared memory (an address).  Nothing is written there
// while they are read, but the compiler cannot know: these loads say nothing of memory, so that those of several rows are issued
// together and not each behind the stores of the row before.  (A place of the ring is read between two barriers; ring_place orders
// the address itself behind the first.)
template <class V> __device__ __forceinline__ V wg_read(const char *p) { return __ldg(reinterpret_cast<const V *>(p)); }
template <class V> __device__ __forceinline__ V wg_read(unsigned a) {
  V v;
  if constexpr (sizeof(V) == 16) asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  else if constexpr (sizeof(V) == 8) asm("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  else if constexpr (sizeof(V) == 4) asm("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  else if constexpr (sizeof(V) == 2) asm("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(a));
  else {
    unsigned short u;
    asm("ld.shared.u8 %0, [%1];" : "=h"(u) : "r"(a));
    v = (V)u;
  }
  return v;
}
__device__ __forceinline__ unsigned ring_place(unsigned a) {
  asm volatile("" : "+r"(a) :: "memory");
  return a;
}
// 16 bytes of neighbouring values of a gradient; WHOLE: all exist, and start on 16 bytes; else zeros from the n-th on.
template <class T, bool WHOLE, class At> __device__ __forceinline__ void wg_load(At at, int n, float (&v)[16 / sizeof(T)]) {
  constexpr int W = 16 / sizeof(T);
  using U = typename std::conditional<sizeof(T) == 4, unsigned, unsigned short>::type;
  Pack<U, W> a;
  if constexpr (WHOLE) {
    const uint4 q = wg_read<uint4>(at);
    a = reinterpret_cast<const Pack<U, W> &>(q);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) {  // (what does not exist is read again from the start: no branches)
      const U u = wg_read<U>(at + (i < n ? i : 0) * (int)sizeof(T));
      a.v[i] = i < n ? u : (U)0;
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] = to_float(reinterpret_cast<const T &>(a.v[i]));
}
// They as bf16 operands, one plane after the other (each what the planes before leave).  FAR: some may be infinite or beyond bf16's largest
// number: what the first plane keeps is cut off, not rounded, so that a number does not become an infinity, and an infinity leaves nothing.
constexpr float kWgFar = 0x1.fep127f;
template <int PLANES, int W, bool FAR = false> __device__ __forceinline__ void wg_planes(float (&g)[W], unsigned to, int plane) {
#pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    unsigned u[W / 2];
#pragma unroll
    for (int k = 0; k < W / 2; ++k) {
      float a = g[2 * k], b = g[2 * k + 1];
      if (FAR && p == 0) {
        if (a == a) a = __uint_as_float(__float_as_uint(a) & 0xffff0000u);  // (a NaN stays one)
        if (b == b) b = __uint_as_float(__float_as_uint(b) & 0xffff0000u);
      }
      u[k] = pack_pair(a, b, false);
      if (p < PLANES - 1) {
        g[2 * k] -= __uint_as_float(u[k] << 16);
        g[2 * k + 1] -= __uint_as_float(u[k] & 0xffff0000u);
        if (FAR && p == 0) {
          if (isinf(a)) g[2 * k] = 0.f;
          if (isinf(b)) g[2 * k + 1] = 0.f;
        }
      }
    }
    if constexpr (W == 8) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + p * plane), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]));
    else asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + p * plane), "r"(u[0]), "r"(u[1]));
  }
}

// A chunk's rows of a slice, some of them infinite or beyond bf16's largest number, as planes.
template <class T, int PLANES, bool WHOLE, class At, class Ld>
__device__ __noinline__ void wg_far_rows(At at, Ld ld, int rows, int first, int step, int n, unsigned to, int chunk, int plane) {
#pragma unroll 1
  for (int r = first; r < rows; r += step) {
    float g[16 / sizeof(T)];
    wg_load<T, WHOLE>(at + r * ld, n, g);
    wg_planes<PLANES, 16 / (int)sizeof(T), true>(g, to + (unsigned)(r * 128 + ((chunk ^ r) & 7) * 16), plane);
  }
}

// RING: G and the codes have nothing between their rows, so that 16 rows are one run of bytes each (a multiple of 16, whatever the
// width): one warp keeps bulk copies of them running ahead through a ring, and what the copies brought is read from shared memory.
// (Whole rows, of which a tile may use a part: 528 846 rows, 191 x 224 bf16.)  Else (strided rows, or a ring that does not fit four
// slices) the teams read rows from memory themselves.
template <class T, int PLANES, int MT, bool RING>
__global__ void __launch_bounds__(wg_threads(PLANES, RING), 1) weight_grad8_kernel(const WgParams P) {
  constexpr int NT = MT == 1 ? 256 : 128, kPlane = MT * 2 * kWgBlock, kStage = wg_stage_bytes(PLANES, MT);
  constexpr int kTeams = wg_teams(PLANES), kWarps = 4 * kTeams, kTeamWarps = kWgTeam / 32;
  constexpr bool STAY = PLANES < 3;  // sums stay in tensor memory
  constexpr int W = 16 / sizeof(T);  // values of G that a thread takes at a time; of X eight
  extern __shared__ char dyn[];
  __shared__ WgShared s;
  char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
  const int a0 = blockIdx.y * MT * 128, b0 = blockIdx.z * NT;
  const int n_pad = (min(NT, P.nb - b0) + 15) / 16 * 16;
  const long long r0 = (long long)blockIdx.x * P.rows;
  const long long r1 = min((long long)P.m, r0 + P.rows);
  const int slices = (int)((r1 - r0 + kWgRows - 1) / kWgRows);

  // columns beyond the operands' stay zero
  for (int i = tid; i < kTeams * kStage / 16; i += wg_threads(PLANES, RING)) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < kTeams; ++i) { mbar_init(&s.full[i], kTeamWarps); mbar_init(&s.empty[i], 1); mbar_init(&s.tail[i], kTeamWarps); }
    if (RING)
      for (int i = 0; i < P.ring; ++i) { mbar_init(&s.raw_full[i], 1); mbar_init(&s.raw_empty[i], kTeamWarps); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s.acc_full[i], 1); mbar_init(&s.acc_empty[i], kWarps); }
    mbar_init(&s.drained, 1);
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

  const int whole = RING ? (int)((r1 - r0) / kWgRows) : 0;  // slices of the ring: those with all their rows
  char *raw = smem + kTeams * kStage;
  if (RING && warp == kWarps + 1) {
    // ---- copies ----
    int rs = 0, issued = 0;
    unsigned ph = 0;
    bool ok = true;
    for (int sl = 0; sl < whole; ++sl) {
      if (sl >= P.ring && !(ok = __all_sync(kFull, pair_wait(&s.raw_empty[rs], ph ^ 1u, s.dead, P.wait_limit)))) break;
      if (elect_one()) {
        const long long row = r0 + (long long)sl * kWgRows;
        const unsigned to = smem_u32(raw + rs * P.ring_bytes), bar = smem_u32(&s.raw_full[rs]);
        mbar_expect_tx(&s.raw_full[rs], (unsigned)P.ring_bytes);
        auto copy = [&](unsigned dst, const void *src, int bytes) {
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                       : "memory");
        };
        copy(to, static_cast<const T *>(P.g) + row * P.na, P.g_bytes);
        copy(to + P.g_bytes, P.codes + row * P.ld_codes, kWgRows * P.ld_codes);
        copy(to + P.g_bytes + kWgRows * P.ld_codes, P.exps + row * (P.ld_codes / kPackGroup), kWgRows * P.ld_codes / kPackGroup);
      }
      __syncwarp();
      if (issued < P.ring) ++issued;
      if (++rs == P.ring) { rs = 0; ph ^= 1u; }
    }
    // no copy may outlive the CTA (where a wait has run out some may be in flight)
    for (int i = 0; i < issued; ++i) mbar_wait(&s.raw_full[i], i < rs ? ph : ph ^ 1u, kInFlightPolls);
  } else if (warp == kWarps) {
    // ---- products ----
    const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((unsigned)(n_pad >> 3) << 17) | ((unsigned)(128 >> 4) << 24);
    bool ok = true;
    auto wait = [&](unsigned long long *bar, unsigned parity) { return ok = __all_sync(kFull, pair_wait(bar, parity, s.dead, P.wait_limit)); };
    for (int sl = 0; sl < slices; ++sl) {
      const int st = sl % kTeams;
      const int chain = STAY ? 0 : sl / kWgChain, buf = chain & 1, in = STAY ? sl : sl % kWgChain;
      if (!STAY && in == 0 && chain >= 2 && !wait(&s.acc_empty[buf], (unsigned)(chain / 2 - 1) & 1u)) break;
      if (!wait(&s.full[st], (unsigned)(sl / kTeams) & 1u)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned base = smem_u32(smem + st * kStage);
      const unsigned long long a = wg_desc(base), b = wg_desc(base + PLANES * kPlane);
      const unsigned d = s.tmem_base + (unsigned)(buf * 256);
      const bool last = (!STAY && in == kWgChain - 1) || sl == slices - 1;
      if (elect_one()) {
#pragma unroll
        for (int p = PLANES - 1; p >= 0; --p)  // the small products first
#pragma unroll
          for (int t = 0; t < MT; ++t)
            wg_mma(d + (unsigned)(t * NT), a + (unsigned)((p * kPlane + t * 2 * kWgBlock) >> 4), b, idesc, in || p != PLANES - 1 ? 1u : 0u);
        umma_commit(&s.empty[st]);
        if (last) umma_commit(&s.acc_full[buf]);
      }
      __syncwarp();
    }
    if (!ok) {  // products still running read shared memory and write tensor memory
      if (elect_one()) umma_commit(&s.drained);
      mbar_wait(&s.drained, 0, kInFlightPolls);
    }
  } else {
    // ---- rows into operands, each team every so many slices; and (fp32) the sums of the chain before out of tensor memory ----
    const int team = warp / kTeamWarps, in_team = tid % kWgTeam;
    const int quadrant = warp & 3, cols0 = (warp >> 2) * 64;  // this thread's row and columns of the accumulator
    float acc[STAY ? 1 : 64];
    if (!STAY)
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[STAY ? 0 : i] = 0.f;
    bool ok = true;
    auto wait = [&](unsigned long long *bar, unsigned parity) { return ok = __all_sync(kFull, pair_wait(bar, parity, s.dead, P.wait_limit)); };
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
          for (int q = 0; q < 16; ++q) acc[STAY ? 0 : c + q] += v[q];
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&s.acc_empty[buf])) : "memory");
    };
    // A thread takes one column chunk of every few rows: a power of two of threads to a row, at least as many as it has chunks.
    const int chunks_g = (min(MT * 128, P.na - a0) + W - 1) / W, chunks_x = (min(NT, P.ld_codes - b0) + 7) / 8;
    const int lg = 32 - __clz(chunks_g - 1), lx = 32 - __clz(chunks_x - 1);
    const int chunk_g = in_team & ((1 << lg) - 1), chunk_x = in_team & ((1 << lx) - 1);
    const int first_g = chunk_g < chunks_g ? in_team >> lg : kWgRows, first_x = chunk_x < chunks_x ? in_team >> lx : kWgRows;
    const int step_g = kWgTeam >> lg, step_x = kWgTeam >> lx;
    const int at_g = chunk_g * W / 8;  // (half a chunk of 16 bytes where a value has four)
    const int to_g = at_g / 8 * kWgBlock + (W == 4 ? (chunk_g & 1) * 8 : 0), to_x = PLANES * kPlane + chunk_x / 8 * kWgBlock;
    const int n_g = min(W, P.na - a0 - chunk_g * W), from_x = b0 + chunk_x * 8, from_e = from_x / kPackGroup, ld_e = P.ld_codes / kPackGroup;
    // Rows of G, codes and exponents that start at the given places, `ld` bytes of G from one to the next, as operands at `base`.  From
    // memory only `rows` of them are there; the others are read as the first and count as zero.
    auto convert = [&](unsigned base, auto pg, auto ld, auto pc, auto pe, int rows) {
      pg += (a0 + chunk_g * W) * (int)sizeof(T);
      auto gradient = [&](auto whole) {
        float top = 0.f;
#pragma unroll 4
        for (int r = first_g; r < kWgRows; r += step_g) {
          const bool here = RING || r < rows;
          const unsigned to = base + (unsigned)(to_g + r * 128 + ((at_g ^ r) & 7) * 16);
          if constexpr (std::is_same<T, __nv_bfloat16>::value && decltype(whole)::value) {  // the operand as it lies in memory
            uint4 q = wg_read<uint4>(pg + (here ? r : 0) * ld);
            if (!here) q = make_uint4(0, 0, 0, 0);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w));
            continue;
          }
          float g[W];
          wg_load<T, decltype(whole)::value>(pg + (here ? r : 0) * ld, n_g, g);
          if (!here)
#pragma unroll
            for (int k = 0; k < W; ++k) g[k] = 0.f;
          if constexpr (PLANES > 1)
#pragma unroll
            for (int k = 0; k < W; k += 2) top = max3_abs_numbers(top, g[k], g[k + 1]);
          wg_planes<PLANES, W>(g, to, kPlane);
        }
        // (rare: the rows again, in a call of its own, so that what they need takes no registers above)
        if constexpr (PLANES > 1)
          if (top > kWgFar) wg_far_rows<T, PLANES, decltype(whole)::value>(pg, ld, RING ? kWgRows : min(rows, kWgRows), first_g, step_g, n_g, base + to_g, at_g, kPlane);
      };
      if (P.whole_g) gradient(std::true_type());
      else gradient(std::false_type());
      pc += from_x;
      pe += from_e;
#pragma unroll 4
      for (int r = first_x; r < kWgRows; r += step_x) {
        const bool here = RING || r < rows;
        uint2 x = wg_read<uint2>(pc + (here ? r : 0) * P.ld_codes);
        const unsigned e = wg_read<unsigned char>(pe + (here ? r : 0) * ld_e);
        if (!here) x = make_uint2(0, 0);
        float v[8];
        unpack8_values<8>(reinterpret_cast<const Pack<signed char, 8> &>(x), here ? unpack8_step(e) : 0.f, v);
        unsigned u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = pack_pair(v[2 * k], v[2 * k + 1], false);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + (unsigned)(to_x + r * 128 + ((chunk_x ^ r) & 7) * 16)), "r"(u[0]), "r"(u[1]),
                     "r"(u[2]), "r"(u[3]));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read next by the tensor core
    };
    auto arrive = [&](unsigned long long *bar) {
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
    };
    // (a team keeps to its stage and, the ring being a multiple of the teams, to its places in the ring: no other team's phase passes it by)
    const int chains = (slices + kWgChain - 1) / kWgChain;
    int drained = 0, turn = 0, rs = team;
    unsigned raw_ph = 0;
    const unsigned stage = smem_u32(smem + team * kStage);
    for (int sl = team; sl < slices && ok; sl += kTeams, ++turn) {
      if (turn && !wait(&s.empty[team], (unsigned)(turn - 1) & 1u)) break;
      const long long row = r0 + (long long)sl * kWgRows;
      if constexpr (RING) {
        char *at = raw + rs * P.ring_bytes;
        const bool all = sl < whole;
        if (all && !wait(&s.raw_full[rs], raw_ph)) break;
        if (!all) {  // the last rows: the team copies them itself, and zeros behind them (what was there it has read, once its warps have met)
          const int rows = (int)(r1 - row), per = P.ld_codes / kPackGroup;
          // (its warps meet in bounded waits: one whose wait has run out does not come)
          arrive(&s.tail[team]);
          if (!wait(&s.tail[team], 0)) break;
          T *to = reinterpret_cast<T *>(at);
          for (int i = in_team; i < kWgRows * P.na; i += kWgTeam) to[i] = i < rows * P.na ? static_cast<const T *>(P.g)[row * P.na + i] : from_float<T>(0.f);
          for (int i = in_team; i < kWgRows * P.ld_codes; i += kWgTeam) at[P.g_bytes + i] = i < rows * P.ld_codes ? P.codes[row * P.ld_codes + i] : 0;
          for (int i = in_team; i < kWgRows * per; i += kWgTeam)
            at[P.g_bytes + kWgRows * P.ld_codes + i] = (char)(i < rows * per ? P.exps[row * per + i] : 127);
          arrive(&s.tail[team]);
          if (!wait(&s.tail[team], 1)) break;
        }
        const unsigned place = ring_place(smem_u32(at));
        convert(stage, place, (unsigned)(P.na * sizeof(T)), place + P.g_bytes, place + P.g_bytes + kWgRows * P.ld_codes, kWgRows);
        arrive(&s.raw_empty[rs]);
        if ((rs += kTeams) >= P.ring) { rs = team; raw_ph ^= 1u; }
      } else
        convert(stage, static_cast<const char *>(P.g) + row * P.ld_g * (long long)sizeof(T), P.ld_g * (long long)sizeof(T),
                reinterpret_cast<const char *>(P.codes) + row * P.ld_codes, reinterpret_cast<const char *>(P.exps) + row * ld_e,
                (int)min((long long)kWgRows, r1 - row));
      arrive(&s.full[team]);
      // this team's last slice of a chain: the chain before has been computed, or is about to be
      const int chain = sl / kWgChain;
      if (!STAY && sl % kWgChain >= kWgChain - kTeams && chain >= 1) { drain(chain - 1); ++drained; }
    }
    while (!STAY && ok && drained < chains) drain(drained++);
    if (STAY && wait(&s.acc_full[0], 0)) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int t = MT == 2 ? cols0 / 128 : 0, col = b0 + (MT == 2 ? cols0 % 128 : cols0), row = a0 + t * 128 + quadrant * 32 + lane;
    const bool lost = __any_sync(kFull, !ok || *reinterpret_cast<volatile int *>(&s.dead));
    float *to = P.part + ((size_t)blockIdx.x * P.na + row) * P.nb + col;
    const bool quads = P.nb % 4 == 0;
    if (cols0 < 256) {  // (six teams: the first four have a part of the sums each)
#pragma unroll
      for (int c = 0; c < 64; c += 16) {
        float v[16];
        if (STAY) {
          if (!lost && (MT == 2 ? (cols0 & 127) < n_pad : cols0 < n_pad)) tmem_load16(v, s.tmem_base + ((unsigned)(quadrant * 32) << 16) + (unsigned)(cols0 + c));
        } else
#pragma unroll
          for (int q = 0; q < 16; ++q) v[q] = acc[STAY ? 0 : c + q];
        if (row < P.na) {
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            if (lost) v[k] = v[k + 1] = v[k + 2] = v[k + 3] = __int_as_float(0x7fc00000);
            if (quads && col + c + k < P.nb) *reinterpret_cast<float4 *>(to + c + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
            else {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (col + c + k + q < P.nb) to[c + k + q] = v[k + q];
            }
          }
        }
        __syncwarp();
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

// out[i] = part[0][i] + part[1][i] + ..., in order; eight lanes share an element's parts and are added pairwise.  before: the sums of the
// launches before this one, added last; after: where they go if more follow, instead of out.
__global__ void __launch_bounds__(256) wg_sum_kernel(const float *__restrict__ part, int parts, int n, const float *before, float *after, void *__restrict__ out,
                                                     int dtype) {
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
  if (before) v += before[i];
  if (after) after[i] = v;
  else store_value(out, dtype, i, v);
}

// parts: ranges of rows, `group` of them a launch.  Ranges of 32 768 rows at most (gradients in 16 bits) are more than fill the device where
// there are many rows; those of a launch together hold 256 MB of sums at most, or as many as fill it.
struct WgPlan { int mt, tiles_a, tiles_b, parts, rows, group; };
constexpr long long kWgMaxFloats = 64ll << 20;
int wg_ranges(int m, int rows) { return (int)std::max(1ll, ((long long)m + rows - 1) / std::max(1, rows)); }
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
  int parts = std::max(1, std::min(148 / (p.tiles_a * p.tiles_b), (m + 127) / 128));
  if (dtype != TF_F32) parts = std::max(parts, (m + kWgStayRows - 1) / kWgStayRows);
  p.rows = (int)(((long long)m + parts - 1) / parts + kWgRows - 1) / kWgRows * kWgRows;
  p.parts = wg_ranges(m, p.rows);
  p.group = (int)std::min<long long>(p.parts, std::max<long long>(std::max(1, 148 / (p.tiles_a * p.tiles_b)), kWgMaxFloats / ((long long)na * nb)));
  return p;
}

template <class T, int PLANES, int MT, bool RING> cudaError_t wg_launch(const WgPlan &p, const WgParams &P, cudaStream_t s) {
  auto f = weight_grad8_kernel<T, PLANES, MT, RING>;
  const int smem = wg_teams(PLANES) * wg_stage_bytes(PLANES, MT) + P.ring * P.ring_bytes + 1024;
  const cudaError_t e = cudaFuncSetAttribute((const void *)f, cudaFuncAttributeMaxDynamicSharedMemorySize, kWgSmem + 2048);
  if (e != cudaSuccess) return e;
  f<<<dim3(wg_ranges(P.m, p.rows), p.tiles_a, p.tiles_b), wg_threads(PLANES, RING), smem, s>>>(P);
  return cudaGetLastError();
}
template <class T, int PLANES> cudaError_t wg_run(const WgPlan &p, WgParams P, cudaStream_t s) {
  auto whole = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  P.ring = 0;
  P.g_bytes = kWgRows * P.na * (int)sizeof(T);
  P.ring_bytes = P.g_bytes + kWgRows * P.ld_codes + kWgRows * P.ld_codes / kPackGroup;
  if (P.ld_g == P.na && whole(P.g) && whole(P.exps))
    P.ring = std::min(kWgMaxRing, (kWgSmem - wg_teams(PLANES) * wg_stage_bytes(PLANES, p.mt)) / P.ring_bytes) / wg_teams(PLANES) * wg_teams(PLANES);
  if (P.ring > 0) return p.mt == 1 ? wg_launch<T, PLANES, 1, true>(p, P, s) : wg_launch<T, PLANES, 2, true>(p, P, s);
  P.ring = 0;
  return p.mt == 1 ? wg_launch<T, PLANES, 1, false>(p, P, s) : wg_launch<T, PLANES, 2, false>(p, P, s);
}

// (the tiles of a side are a dimension of the grid, 65 535 at most, and a slice's bytes are counted in 32 bits)
bool wg_fits(int na, int nb) { return (long long)na * nb <= (1 << 26) && na <= (1 << 20) && nb <= (1 << 20); }
constexpr int kWgMaxLdCodes = 1 << 26;

}  // namespace

}  // namespace tfk

using namespace tfk;

extern "C" long long tf_weight_grad8_work_floats(int m, int na, int nb, int dtype) {
  if (m < 0 || m > kMaxRows || na <= 0 || nb <= 0 || !wg_fits(na, nb) || !known_dtype(dtype)) return 0;
  const WgPlan p = wg_plan(m, na, nb, dtype);
  return (p.group + (p.group < p.parts ? 1ll : 0ll)) * na * nb;
}

extern "C" int tf_weight_grad8(const void *g, long long ld_g, int dtype, int na, const signed char *codes, int ld_codes,
                               const unsigned char *exponents, int nb, int m, void *out, float *work, long long work_floats, void *stream) {
  auto bad = [&](const char *what) { return tf::fail(TF_ERR_ARG, std::string("tf_weight_grad8: ") + what); };
  if (!known_dtype(dtype)) return bad("unknown type");
  if (m < 0 || m > kMaxRows || na <= 0 || nb <= 0) return bad("bad size");
  if (!wg_fits(na, nb)) return tf::fail(TF_ERR_UNSUPPORTED, "tf_weight_grad8: at most 2^26 entries, 2^20 to a side");
  if (ld_codes > kWgMaxLdCodes) return tf::fail(TF_ERR_UNSUPPORTED, "tf_weight_grad8: rows of codes at most 2^26 bytes apart");
  if (!out || !work || (m > 0 && (!g || !codes || !exponents))) return bad("null argument");
  if (ld_g < na || ld_codes < nb) return bad("rows overlap");
  if (ld_codes % kPackGroup != 0 || (reinterpret_cast<uintptr_t>(codes) & 31) != 0) return bad("codes need rows of whole groups of 32 and 32-byte alignment");
  if ((reinterpret_cast<uintptr_t>(work) & 15) != 0) return bad("the work space must be 16-byte aligned");
  if (work_floats < tf_weight_grad8_work_floats(m, na, nb, dtype)) return bad("work space too small");
  const WgPlan p = wg_plan(m, na, nb, dtype);
  WgParams P;
  P.g = g; P.ld_g = ld_g; P.na = na; P.codes = codes; P.ld_codes = ld_codes; P.nb = nb; P.exps = exponents; P.m = m; P.rows = p.rows;
  P.whole_g = na % (16 / value_bytes(dtype)) == 0 && ld_g * value_bytes(dtype) % 16 == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  P.part = work;
  P.wait_limit = dense_wait_limit();
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  const int n = na * nb;
  float *sums = work + (size_t)p.group * n;  // of the launches before (there is room where there are several)
  long long row = 0;
  do {
    P.g = static_cast<const char *>(g) + row * ld_g * value_bytes(dtype);
    P.codes = codes + row * ld_codes;
    P.exps = exponents + row * (ld_codes / kPackGroup);
    P.m = (int)std::min<long long>(m - row, (long long)p.group * p.rows);
    if (m > 0) e = dtype == TF_F32 ? wg_run<float, 3>(p, P, s) : dtype == TF_F16 ? wg_run<__half, 2>(p, P, s) : wg_run<__nv_bfloat16, 1>(p, P, s);
    if (e != cudaSuccess) break;
    wg_sum_kernel<<<(n + 31) / 32, 256, 0, s>>>(work, m > 0 ? wg_ranges(P.m, p.rows) : 0, n, row ? sums : nullptr, row + P.m < m ? sums : nullptr, out, dtype);
    e = cudaGetLastError();
    row += P.m;
  } while (e == cudaSuccess && row < m);
  return e == cudaSuccess ? TF_OK : tf::fail(TF_ERR_CUDA, std::string("tf_weight_grad8: ") + cudaGetErrorString(e));
}
