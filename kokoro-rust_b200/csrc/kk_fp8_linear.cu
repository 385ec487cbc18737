// The 8-bit linear layer, y = act(x W^T + bias) + residual, on the 5th-generation tensor cores
// (layout of the operands in kk_fp8.h).
//
// x [m][k] has a scale for each 128 columns of a row, W [n][k] one for each 128 x 128 block, both powers
// of two: the block-scaled MMA (kind::mxf8f6f4, one scale for each 32 columns, the same for the four of a
// block) applies them inside the tensor core, so a whole row of K is accumulated in TMEM in 32 bits and
// nothing is rescaled in registers.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <atomic>
#include <type_traits>

#include "kk_fp8.h"
#include "kk_fp8_math.cuh"
#include "kk_tc_ptx.cuh"

namespace kk {

// Blocks of the stand-alone operators that gave up a bounded pipeline wait, since the process began; one per device. It
// only grows, so that nobody who reads it takes a failure from another.
__device__ unsigned g_fp8_wait_failures;

// One thread of a block, once all its warps are through, if one of them gave up: raises the caller's flag, or counts.
__device__ __forceinline__ void report_failure(int* err, const volatile int* abort_flag) {
  if (*abort_flag == 0) return;
  if (err)
    atomicExch(err, 2);
  else
    atomicAdd(&g_fp8_wait_failures, 1u);
}

// ---- PTX of the block-scaled MMA

// Shared-memory matrix descriptor, K-major, 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1024 bytes
// apart (SBO); version 1; swizzle mode 2 in bits 61..63.
__device__ __forceinline__ uint64_t sdesc_sw128(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor, kind::mxf8f6f4: A and B e4m3 (format 0), scales E8M0 (bit 23), both K-major, M x N;
// sf selects the byte (0..3) of the scale words that this MMA applies.
__host__ __device__ constexpr uint32_t idesc_mxf8(int M, int N, int sf) {
  return ((uint32_t)sf << 4) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24) | ((uint32_t)sf << 29);
}
__device__ __forceinline__ void mma_mxf8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                         uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 lanes x 16 bytes of shared memory (512 contiguous bytes) to four TMEM columns, in all four lane quarters:
// word w of lane l is the scale word of row 32 w + l.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// ---- the same over a pair of CTAs (cta_group::2): the MMA is issued by the pair's first CTA and reads both
// CTAs' shared memory at the same offsets; each CTA holds its own 128 rows of the accumulator
__device__ __forceinline__ void mma_mxf8_pair(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                              uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_cp_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// true on one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// arrives on the barrier at this offset in both CTAs once the pair's MMAs so far are done
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((unsigned short)3)
      : "memory");
}
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// the address of this CTA's shared-memory location in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The same where no memory is handed over, only TMEM columns, whose reads are complete (tcgen05.wait::ld and the
// fence before): a release would wait for every load the warp has on its way, 1000 to 3000 cycles here.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// a load into this CTA's shared memory whose bytes complete on a barrier of either CTA of the pair
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// whether a phase of a barrier that the other CTA of the cluster arrives on is complete
__device__ __forceinline__ bool mbar_try_cluster(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// the same, asleep until it is or about 0.5 ms have passed
__device__ __forceinline__ bool mbar_sleep_cluster(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(parity), "r"(500000u)
      : "memory");
  return ok != 0;
}
// mbar_wait on such a barrier
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* b, uint32_t parity, volatile int* abort_flag, int* err,
                                                  unsigned long long limit_ns = KK_WAIT_TIMEOUT_NS) {
  if (mbar_sleep_cluster(b, parity)) return true;
  const unsigned long long t0 = tc_now();
  while (true) {
    if (mbar_sleep_cluster(b, parity)) return true;
    if (*abort_flag) return false;
    if (tc_now() - t0 > limit_ns) {
      *abort_flag = 1;
      atomicExch(err, 2);
      return false;
    }
  }
}
// Waits, at most KK_WAIT_TIMEOUT_NS, for a phase that work already in flight completes.
__device__ __forceinline__ void mbar_drain(uint64_t* b, uint32_t parity) {
  const unsigned long long t0 = tc_now();
  while (!mbar_try_sleep(b, parity) && tc_now() - t0 < KK_WAIT_TIMEOUT_NS) {
  }
}
// Waits of a whole warp. The lanes meet after each: one that fell behind the lane that issues by a whole ring of
// stages would wait for a phase whose parity has come round, and what a wait says has to be the same for all.
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity, volatile int* abort_flag, int* err) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(b, parity, abort_flag, err));
}
__device__ __forceinline__ bool warp_wait_cluster(uint64_t* b, uint32_t parity, volatile int* abort_flag, int* err) {
  return __all_sync(0xFFFFFFFFu, mbar_wait_cluster(b, parity, abort_flag, err));
}

__device__ __forceinline__ void pause_1ms() {
  const unsigned long long t0 = tc_now();
  while (tc_now() - t0 < 1000000ull) __nanosleep(1000);
}

constexpr int SF_RING = 4;  // scale groups (4 blocks of K each) of a pair, in shared memory and TMEM

// Waits until what used a ring's places last is done, from place s on, with the parity of its loop's next wait (which a place
// that was never used passes). The commits of a pair's MMAs arrive on barriers of both CTAs, the second CTA's from the
// first: none may still be on its way there when its shared memory goes.
template <int RING>
__device__ __forceinline__ void last_uses(uint64_t* done, uint32_t s, uint32_t ph, volatile int* abort_flag, int* err) {
#pragma unroll 1
  for (int i = 0; i < RING; i++) {
    if (!warp_wait(done + s, ph, abort_flag, err)) return;
    if (++s == RING) s = 0, ph ^= 1;
  }
}

// ---- scales
// One warp brings the scales of a CTA's tiles, a group (four blocks of K: a word for each row of x and of W) at a
// time, into a ring of shared-memory slots in the layout of the TMEM copy. A word waits behind the TMA's boxes on its
// way from L2 (about 2000 cycles, as long as the MMAs of two or three groups), so the words of the next AHEAD groups
// are always on their way, in registers; waiting for each group in turn held the MMAs up by half.
template <int RING, int ROWS_W, bool PAIR>
struct ScaleFeed {
  static constexpr int NB = (ROWS_W + 127) / 128, BYTES = 512 * (1 + NB), AHEAD = 4;
  const Fp8Linear& a;
  uint32_t ring;  // shared-memory address of the slots
  uint64_t *full, *empty;
  volatile int* abort_flag;
  int* err;
  int lane;

  // start(t, &m0, &n0): rows and columns of a CTA's tile t; its groups are the blocks b_lo, b_lo + 4, .. below b_hi
  // (b_lo a multiple of 4). Tiles first, first + step, .. below tiles.
  template <class F>
  __device__ __forceinline__ void run(int first, int step, int tiles, int b_lo, int b_hi, F&& start) {
    uint32_t w[AHEAD][4 + 4 * NB];
    const uint8_t *px[4], *pw[4 * NB];
    int t = first, b = b_lo;  // of the next group to load
    auto open = [&] {
      if (t >= tiles) return;
      long m0, n0;
      start(t, &m0, &n0);
      // (rows past the last take the last one's scales: what they scale is zero, and is not stored)
#pragma unroll
      for (int i = 0; i < 4; i++) px[i] = a.x.e + min(m0 + 32 * i + lane, a.m - 1) * a.x.lde;
#pragma unroll
      for (int i = 0; i < 4 * NB; i++)  // (a tile may begin inside a block of W's rows)
        pw[i] = a.w.e + (min(n0 + 32 * i, a.n - 1) >> 7) * a.w.lde;
    };
    auto load = [&](uint32_t(&d)[4 + 4 * NB]) {
      if (t >= tiles) return;
#pragma unroll
      for (int i = 0; i < 4; i++) d[i] = __ldg(reinterpret_cast<const uint32_t*>(px[i] + b));
#pragma unroll
      for (int i = 0; i < 4 * NB; i++) d[4 + i] = __ldg(reinterpret_cast<const uint32_t*>(pw[i] + b));
      b += 4;
      if (b >= b_hi) b = b_lo, t += step, open();
    };
    open();
#pragma unroll
    for (int i = 0; i < AHEAD; i++) load(w[i]);
    long left = first < tiles ? (long)((tiles - first + step - 1) / step) * ((b_hi - b_lo + 3) / 4) : 0;
    uint32_t slot = 0, ph = 1;
    bool used = false;  // the ring has gone round once
    while (true) {
#pragma unroll
      for (int i = 0; i < AHEAD; i++) {
        if (left-- == 0) {
          if (PAIR) last_uses<RING>(empty, slot, ph, abort_flag, err);
          return;
        }
        if (used && !warp_wait(empty + slot, ph, abort_flag, err)) return;
        const uint32_t dst = ring + slot * BYTES + lane * 16;
#pragma unroll
        for (int j = 0; j < 1 + NB; j++)
          sts_u4(dst + 512 * j, make_uint4(w[i][4 * j], w[i][4 * j + 1], w[i][4 * j + 2], w[i][4 * j + 3]));
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(full + slot);
        if (++slot == RING) slot = 0, ph ^= 1, used = true;
        load(w[i]);
      }
    }
  }
};

// What the MMA warp waits for: stages and scale groups. Asking a barrier takes about 130 cycles, so the next one is asked
// while the MMAs before it are issued.
struct MmaFeed {
  uint64_t *full, *sf_full;
  int stages;
  volatile int* abort_flag;
  int* err;
  uint32_t s = 0, ph = 0, slot = 0, sph = 0;
  uint32_t last = 0, last_ph = 0;  // the stage of the last MMAs issued
  bool any = false, stage_in = false, scales_in = false;

  __device__ __forceinline__ bool stage() {
    if (!__all_sync(0xFFFFFFFFu, stage_in) && !warp_wait_cluster(full + s, ph, abort_flag, err)) return false;
    tc_fence_after();
    last = s, last_ph = ph, any = true;
    const bool wrap = (int)s + 1 == stages;
    stage_in = mbar_try_cluster(full + (wrap ? 0 : s + 1), wrap ? ph ^ 1 : ph);
    return true;
  }
  __device__ __forceinline__ void next_stage() {
    if ((int)++s == stages) s = 0, ph ^= 1;
  }
  __device__ __forceinline__ bool scales() {
    if (!__all_sync(0xFFFFFFFFu, scales_in) && !warp_wait_cluster(sf_full + slot, sph, abort_flag, err)) return false;
    const bool wrap = slot + 1 == SF_RING;
    scales_in = mbar_try_cluster(sf_full + (wrap ? 0 : slot + 1), wrap ? sph ^ 1 : sph);
    return true;
  }
  __device__ __forceinline__ void next_scales() {
    if (++slot == SF_RING) slot = 0, sph ^= 1;
  }
};

// In the pair's second CTA: hands each of its groups on to the first CTA, whose MMA warp takes both. (The loading warp
// could arrive there itself, but a release to the cluster waits for the loads that it has on its way.)
template <int RING>
__device__ __forceinline__ void forward_scales(long groups, uint64_t* full, int lane, volatile int* abort_flag, int* err) {
  uint32_t slot = 0, ph = 0;
  for (long g = 0; g < groups; g++) {
    if (!warp_wait(full + slot, ph, abort_flag, err)) return;
    if (lane == 0) mbar_arrive_cluster(map_rank(full + slot, 0));
    if (++slot == RING) slot = 0, ph ^= 1;
  }
}

struct TcFp8Args {
  Fp8Linear a;
  int* err;
  int kb;              // blocks of 128 columns of K
  int m_tiles, n_tiles;
  int tma_y;           // y (and the residual) can be stored (loaded) by TMA: 16-byte aligned rows
  int tma_edge;        // so can their last columns: TMA writes whole 16-byte units, so n has to end on one
};

// ---- large layers: persistent pairs of CTAs, a tile of 256 rows x 256 columns at a time
//
// Bound by the tensor cores from about K = 1000 on, by HBM below. One CTA with a 128 x 256 tile reads 96 bytes of
// L2 per SM and clock at the full MMA rate, more than L2 gives; a pair shares the 256 rows of W (each CTA loads
// and holds half of them), which takes 64.
constexpr int TM = 128, TN = 256;  // a CTA's rows, the pair's columns
constexpr int CTRL_WARPS = 3;      // loads, MMAs, scales
constexpr int BOX = 4096;          // 32 rows of 128 bytes: what an epilogue warp stores (or loads) at once

template <int OUT>
struct PairShape {
  static constexpr bool Q = OUT == FP8_E4M3;
  // Epilogue warps: two for each TMEM lane quarter, 128 columns each (with four, f32 and bf16 results are 15% slower:
  // the warps of the main loop get fewer of the issue slots); four with 64 columns each for an e4m3 result, whose
  // thread holds all of its columns until their maximum is known (with 128, too few registers are left to work on
  // several at once: 10% slower with GELU)
  static constexpr int EPI = Q ? 16 : 8, COLS = Q ? 64 : 128;
  static constexpr int THREADS = 32 * (CTRL_WARPS + EPI);
  static constexpr int N = TN, STAGES = 5;
  static constexpr int A_BYTES = TM * 128, B_BYTES = N / 2 * 128;
  static constexpr int NB = N / 128, SF_BYTES = 512 * (1 + NB);
  // TMEM columns: the two accumulators share columns 192..255 (see the epilogue), so one barrier each way goes for
  // both; scales behind them
  static constexpr int D1 = 192, ACC = 1, SF_COL = D1 + N, SF_COLS = 4 * (1 + NB);
  static constexpr int BOXES = 8;  // e4m3: two warps share one
  static constexpr int OFF_B = STAGES * A_BYTES, OFF_BOX = OFF_B + STAGES * B_BYTES;
  static constexpr int OFF_SF = OFF_BOX + BOXES * BOX, OFF_BIAS = OFF_SF + SF_RING * SF_BYTES;
  static constexpr int OFF_MAX = OFF_BIAS + EPI * COLS * 4, OFF_BAR = OFF_MAX + (Q ? 2 * EPI * 32 * 4 : 0);
  static constexpr int SMEM = OFF_BAR + 512 + 1024;  // 1024: alignment of the first stage
  static_assert(SF_COL + SF_RING * SF_COLS <= 512, "TMEM columns");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// Rows at strides or offsets that TMA does not take: a warp's box of 32 rows (the thread's row at row_s, written as for
// TMA) leaves row by row, its columns side by side, so that a store instruction still fills whole sectors. What it takes
// is instructions, so whole boxes have loops of their own without a test in them: 33,104 x 768 -> 2306 bf16 69 us
// (119 with a test at each row, 58 for 2304 by TMA), 768 -> 769 f32 44 (31 for 768), with a residual 69 (46; 224 with
// the residual's rows loaded one after the other).
//
// 32 columns in 32 bits, one a lane: residual columns of the 32 rows from r0, all on their way at once (as raw bits:
// widened here, they would be waited for here)...
template <typename T>
__device__ __forceinline__ void load_rows(const Fp8Linear& a, long r0, long c, int lane, uint32_t* res) {
  using U = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
  const U* r = (const U*)a.res + r0 * a.ldr + c + lane;
  const bool in = c + lane < a.n;
  if (r0 + 32 <= a.m) {
#pragma unroll
    for (int j = 0; j < 32; j++, r += a.ldr) res[j] = in ? *r : 0;
  } else {
#pragma unroll
    for (int j = 0; j < 32; j++, r += a.ldr) res[j] = in && r0 + j < a.m ? *r : 0;
  }
}
__device__ __forceinline__ void stage_rows(const float* v, uint32_t row_s, int lane) {
#pragma unroll
  for (int q = 0; q < 8; q++)
    sts_u4(row_s + ((q ^ (lane & 7)) << 4),
           make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]),
                      __float_as_uint(v[4 * q + 3])));
}
// ...and the staged rows, the residual added, into y.
template <typename T, bool RES>
__device__ __forceinline__ void store_rows(const Fp8Linear& a, const uint8_t* box, long r0, long c, int lane,
                                           const uint32_t* res) {
  __syncwarp();
  T* y = (T*)a.y + r0 * a.ldy + c + lane;
  auto row = [&](int j) {
    float o = *reinterpret_cast<const float*>(box + j * 128 + ((((lane >> 2) ^ (j & 7)) << 4) | ((lane & 3) << 2)));
    if (RES) o += __uint_as_float(sizeof(T) == 4 ? res[j] : res[j] << 16);
    return (T)o;
  };
  if (c + lane < a.n) {
    if (r0 + 32 <= a.m) {
#pragma unroll
      for (int j = 0; j < 32; j++, y += a.ldy) *y = row(j);
    } else {
#pragma unroll
      for (int j = 0; j < 32; j++, y += a.ldy)
        if (r0 + j < a.m) *y = row(j);
    }
  }
  __syncwarp();  // the box is free
}
// 64 bf16 columns: two a lane where the row is 4-byte aligned, else one in each half.
__device__ __forceinline__ void store_rows_bf16(const Fp8Linear& a, const uint8_t* box, long r0, long c, int lane) {
  __syncwarp();
  uint16_t* const y = (uint16_t*)a.y + r0 * a.ldy + c;
  const int in = (lane & 7) << 1, unit = lane >> 3;
  auto pair = [&](int j) {
    return *reinterpret_cast<const uint32_t*>(box + j * 128 + ((((lane >> 2) ^ (j & 7)) << 4) | ((lane & 3) << 2)));
  };
  auto one = [&](int j, int half) {
    return *reinterpret_cast<const uint16_t*>(box + j * 128 + ((((unit + 4 * half) ^ (j & 7)) << 4) | in));
  };
  if (r0 + 32 <= a.m && c + 64 <= a.n) {
#pragma unroll
    for (int i = 0; i < 2; i++) {  // every other row: all of one alignment
      uint16_t* r = y + i * a.ldy;
      if (((uintptr_t)r & 3) == 0) {
        r += 2 * lane;
#pragma unroll
        for (int j = i; j < 32; j += 2, r += 2 * a.ldy) *reinterpret_cast<uint32_t*>(r) = pair(j);
      } else {
        r += lane;
#pragma unroll
        for (int j = i; j < 32; j += 2, r += 2 * a.ldy) r[0] = one(j, 0), r[32] = one(j, 1);
      }
    }
  } else {
    uint16_t* r = y + lane;
    const bool in0 = c + lane < a.n, in1 = c + lane + 32 < a.n;
#pragma unroll 8
    for (int j = 0; j < 32; j++, r += a.ldy) {
      if (r0 + j >= a.m) break;
      if (in0) r[0] = one(j, 0);
      if (in1) r[32] = one(j, 1);
    }
  }
  __syncwarp();
}

// The largest finite magnitude of a thread's 64 columns, as bits; *infinite: one of them is infinite.
__device__ __forceinline__ uint32_t finite_max64(const float* v, bool* infinite) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 64; i++) m = fmaxf(m, fabsf(v[i]));  // (a NaN is passed over)
  uint32_t b = __float_as_uint(m);
  *infinite = b == 0x7F800000u;
  if (*infinite) {
    b = 0;
#pragma unroll
    for (int i = 0; i < 64; i++) b = max(b, finite_bits(v[i]));
  }
  return b;
}
__device__ __forceinline__ void quantize64(const float* v, float inv, bool infinite, uint32_t* u) {
  if (!infinite) {
#pragma unroll
    for (int i = 0; i < 16; i++) u[i] = e4m3x4_finite(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv);
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++) u[i] = e4m3x4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv);
  }
}

// bias of columns c and c + 1, zero past the last
__device__ __forceinline__ float2 load_bias2(const Fp8Linear& a, long c) {
  float2 b = make_float2(0.0f, 0.0f);
  if (!a.bias) return b;
  if (c < a.n) b.x = a.bias[c];
  if (c + 1 < a.n) b.y = a.bias[c + 1];
  return b;
}
// ...into a warp's row of biases, once it is there
__device__ __forceinline__ void stage_bias2(const Fp8Linear& a, float* bias_s, float2 b) {
  if (a.gelu) b.x = gelu_bias(b.x), b.y = gelu_bias(b.y);
  *reinterpret_cast<float2*>(bias_s) = b;
}

__device__ __forceinline__ void add_bias32(float* v, const float* bias_s) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 b = *reinterpret_cast<const float4*>(bias_s + j);
    add2(v[j], v[j + 1], b.x, b.y);
    add2(v[j + 2], v[j + 3], b.z, b.w);
  }
}

// Tiles in the order in which the pairs take them: columns fastest within groups of 8 row tiles (down the group
// first), so that the tiles of a wave share few rows of x and of W in L2.
__device__ __forceinline__ void tile_at(const TcFp8Args& p, int t, int* mt, int* nt) {
  constexpr int G = 8;
  const unsigned per = G * p.n_tiles, g = (unsigned)t / per, r = t - g * per;
  const unsigned h = min(G, p.m_tiles - (int)g * G);
  *nt = h == G ? r / G : r / h;
  *mt = g * G + (r - *nt * h);
}

// ---- the main loop of a pair
//
// In each CTA warp 0 loads its boxes of x and W (128 bytes x 128 rows, or half the tile's columns; 128-byte swizzle)
// into a ring of stages, and warp 2 brings the scales, four blocks of K at a time; warp 1 of the first CTA issues the
// pair's MMAs, that of the second hands its CTA's scales on. Barriers that the MMA warp waits on live in the first
// CTA; those it commits to, in both.
template <class S>
struct PairLoop {
  const TcFp8Args& p;
  uint8_t* smem;
  uint64_t *full, *empty, *sf_full, *sf_empty, *acc_full, *acc_free, *more;  // more: the first barrier behind these
  volatile int* abort_flag;
  int* err;
  uint32_t *tmem_slot, tmem, rank;
  int warp, lane, tiles, first, step;

  __device__ __forceinline__ PairLoop(const TcFp8Args& args, uint8_t* raw) : p(args) {
    smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    tmem_slot = (uint32_t*)(smem + S::OFF_BAR);
    abort_flag = (volatile int*)(tmem_slot + 1);
    full = (uint64_t*)(tmem_slot + 2);
    empty = full + S::STAGES, sf_full = empty + S::STAGES, sf_empty = sf_full + SF_RING;
    acc_full = sf_empty + SF_RING, acc_free = acc_full + S::ACC, more = acc_free + S::ACC;
    err = (int*)abort_flag;  // (raised outside at the end)
    warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    rank = cta_rank();
    tiles = p.m_tiles * p.n_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
  }
  // one thread; the kernel's own barriers come with it
  __device__ __forceinline__ void init_barriers() {
    for (int i = 0; i < S::STAGES; i++) mbar_init(full + i, 1), mbar_init(empty + i, 1);
    for (int i = 0; i < SF_RING; i++) mbar_init(sf_full + i, rank == 0 ? 2 : 1), mbar_init(sf_empty + i, 1);
    for (int i = 0; i < S::ACC; i++) mbar_init(acc_full + i, 1), mbar_init(acc_free + i, 2 * S::EPI);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __device__ __forceinline__ void begin() {
    if (warp == 0) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    tmem = *tmem_slot;
  }
  __device__ __forceinline__ void end() {
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) report_failure(p.err, abort_flag);
    __syncwarp();
    cluster_sync();
    if (warp == 0) {
      tc_fence_after();
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
  }

  __device__ __forceinline__ void loads(const CUtensorMap* xmap, const CUtensorMap* wmap) {
    const bool lead = elect_one();
    uint32_t it = 0, s = 0, ph = 1;  // ph: of the wait for the stage's last use
    bool ok = true;
    for (int t = first; ok && t < tiles; t += step) {
      int mt, nt;
      tile_at(p, t, &mt, &nt);
      const int m0 = mt * 2 * TM + (int)rank * TM, n0 = nt * S::N + (int)rank * (S::N / 2);
      for (int b = 0; b < p.kb; b++, it++) {
        if (it >= S::STAGES && !warp_wait(empty + s, ph, abort_flag, err)) {
          ok = false;
          break;
        }
        if (lead) {
          if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * (S::A_BYTES + S::B_BYTES));
          const uint32_t bar = map_rank(full + s, 0);
          tma_load_2d_pair(smem + s * S::A_BYTES, xmap, b * 128, m0, bar);
          tma_load_2d_pair(smem + S::OFF_B + s * S::B_BYTES, wmap, b * 128, n0, bar);
        }
        if (++s == S::STAGES) s = 0, ph ^= 1;
      }
    }
    if (ok) last_uses<S::STAGES>(empty, s, ph, abort_flag, err);
    // After an expired wait, loads still in flight land before the shared memory goes: the first CTA sees them
    // complete, the second, whose loads complete there, waits far longer than a load takes.
    if (!ok) {
      if (rank == 0) {
        for (uint32_t i = it > S::STAGES ? it - S::STAGES : 0; i < it; i++)
          mbar_drain(full + i % S::STAGES, (i / S::STAGES) & 1);
      } else {
        pause_1ms();
      }
    }
  }

  // The whole warp runs this loop, so that its control flow and addresses stay uniform, and one elected lane issues.
  // What it does for each block of K (a wait, four MMAs, a commit) has to take less than the block's 512 MMA cycles:
  // with one divergent lane it took 870.
  __device__ __forceinline__ void mmas() {
    const bool lead = elect_one();
    const uint64_t da0 = sdesc_sw128(smem_u32(smem)), db0 = sdesc_sw128(smem_u32(smem + S::OFF_B));
    const uint64_t dsf0 = sdesc(smem_u32(smem + S::OFF_SF), 128, 128);
    MmaFeed f{full, sf_full, S::STAGES, abort_flag, err};
    uint32_t tile_n = 0;
    bool ok = true;
    for (int t = first; ok && t < tiles; t += step, tile_n++) {
      const uint32_t bar = tile_n % S::ACC, use = tile_n / S::ACC;
      if (use > 0 && !warp_wait_cluster(acc_free + bar, (use - 1) & 1, abort_flag, err)) break;
      tc_fence_after();
      const uint32_t d = tmem + (tile_n & 1) * S::D1;
      for (int b0 = 0; ok && b0 < p.kb; b0 += 4) {
        ok = f.scales();
        if (!ok) break;
        const uint32_t sfa = tmem + S::SF_COL + f.slot * S::SF_COLS;
        if (lead) {
          const uint64_t dsf = dsf0 + f.slot * (S::SF_BYTES >> 4);
#pragma unroll
          for (int i = 0; i < 1 + S::NB; i++) tmem_cp_scales_pair(sfa + 4 * i, dsf + (512 >> 4) * i);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (b0 + j >= p.kb) break;
          ok = f.stage();
          if (!ok) break;
          if (lead) {
            const uint64_t da = da0 + f.s * (S::A_BYTES >> 4), db = db0 + f.s * (S::B_BYTES >> 4);
#pragma unroll
            for (int k = 0; k < 4; k++)
              mma_mxf8_pair(d, da + 2 * k, db + 2 * k, idesc_mxf8(2 * TM, S::N, j), sfa, sfa + 4, j > 0 || k > 0 || b0 > 0);
            mma_commit_pair(empty + f.s);
          }
          f.next_stage();
        }
        if (ok && lead) mma_commit_pair(sf_empty + f.slot);
        f.next_scales();
      }
      if (ok && lead) mma_commit_pair(acc_full + bar);
    }
    if (*abort_flag && f.any) mbar_drain(empty + f.last, f.last_ph);  // MMAs in flight end before their operands and TMEM go
  }

  __device__ __forceinline__ void scales() {
    ScaleFeed<SF_RING, S::N, true> feed{p.a, smem_u32(smem + S::OFF_SF), sf_full, sf_empty, abort_flag, err, lane};
    feed.run(first, step, tiles, 0, p.kb, [&](int t, long* m0, long* n0) {
      int mt, nt;
      tile_at(p, t, &mt, &nt);
      *m0 = (long)mt * 2 * TM + rank * TM, *n0 = (long)nt * S::N;
    });
  }
  // what the control warps do
  __device__ __forceinline__ void control(const CUtensorMap* xmap, const CUtensorMap* wmap) {
    if (warp == 0)
      loads(xmap, wmap);
    else if (warp == 2)
      scales();
    else if (rank == 0)
      mmas();
    else if (first < tiles)
      forward_scales<SF_RING>((long)((tiles - first + step - 1) / step) * ((p.kb + 3) / 4), sf_full, lane, abort_flag, err);
  }
};

// The epilogue: COLS columns of one row a thread.
template <int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairShape<OUT>::THREADS, 1)
    fp8_linear_pair_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                           const __grid_constant__ CUtensorMap ymap, const __grid_constant__ TcFp8Args p) {
  using S = PairShape<OUT>;
  extern __shared__ uint8_t smem_raw[];
  PairLoop<S> loop(p, smem_raw);
  uint8_t* smem = loop.smem;
  uint64_t *max_in = loop.more, *box_in = max_in + S::BOXES;  // e4m3: of the two warps of a box
  if (threadIdx.x == 0) {
    if (S::Q)
      for (int i = 0; i < S::BOXES; i++) mbar_init(max_in + i, 2), mbar_init(box_in + i, 2);
    loop.init_barriers();
  }
  loop.begin();
  const Fp8Linear& a = p.a;
  const int warp = loop.warp, lane = loop.lane, tiles = loop.tiles, first = loop.first, step = loop.step;
  const uint32_t rank = loop.rank, tmem = loop.tmem;
  uint64_t *acc_full = loop.acc_full, *acc_free = loop.acc_free;
  volatile int* abort_flag = loop.abort_flag;
  int* err = loop.err;
  if (warp < CTRL_WARPS) {
    loop.control(&xmap, &wmap);
  } else {
    const int ew = warp - CTRL_WARPS, cg = ew >> 2, q4 = warp & 3;  // COLS columns; the TMEM lane quarter a warp reaches
    float* bias_s = (float*)(smem + S::OFF_BIAS) + ew * S::COLS;
    // e4m3: the warps of columns 0..63 and 64..127 of a block share a box (and a barrier for each of their meetings)
    const int bx = S::Q ? (cg >> 1) * 4 + q4 : ew, odd = cg & 1;
    uint8_t* box = smem + S::OFF_BOX + bx * BOX;
    const uint32_t row_s = smem_u32(box) + lane * 128;  // this thread's row of the box; 16-byte units swizzled by row
    const uint32_t acc_free0 = map_rank(acc_free, 0);
    uint32_t tile_n = 0;
    bool ok = true;
    float2 bias_r[S::COLS / 64];  // two columns, and two 64 further on
    auto load_bias_r = [&](int t) {
      int mt, nt;
      tile_at(p, t, &mt, &nt);
#pragma unroll
      for (int i = 0; i < S::COLS / 64; i++) bias_r[i] = load_bias2(a, (long)nt * TN + cg * S::COLS + 64 * i + 2 * lane);
    };
    if (first < tiles) load_bias_r(first);
    for (int t = first; ok && t < tiles; t += step, tile_n++) {
      int mt, nt;
      tile_at(p, t, &mt, &nt);
      const long r0 = (long)mt * 2 * TM + rank * TM + q4 * 32;
      const long c0 = (long)nt * TN + cg * S::COLS;
      // The next tile's accumulator may be written once the columns that it shares with this one are read: the last
      // 64 of the first accumulator are the first 64 of the second. (The tile after next reuses all of this
      // accumulator: it waits for the next tile's arrivals, which come after all of this tile's reads.)
      const bool shares = cg == (tile_n & 1 ? 0 : S::EPI / 4 - 1);
      const bool live = r0 < a.m && c0 < a.n;
      if (S::Q && !odd && lane == 0) bulk_wait_all_read();  // the box is free once the last tile's store has read it
      __syncwarp();
#pragma unroll
      for (int i = 0; i < S::COLS / 64; i++) stage_bias2(a, bias_s + 64 * i + 2 * lane, bias_r[i]);
      __syncwarp();
      if (t + step < tiles) load_bias_r(t + step);  // the next tile's, which arrives during this one
      ok = warp_wait(acc_full, tile_n & 1, abort_flag, err);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d = tmem + ((uint32_t)q4 << 21) + (tile_n & 1) * S::D1 + cg * S::COLS;
      if (!shares && lane == 0) mbar_arrive_cluster_relaxed(acc_free0);
      if constexpr (S::Q) {
        float v[64];
        tmem_ld64(d, v);
        if (shares) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(acc_free0);
        }
        add_bias32(v, bias_s);
        add_bias32(v + 32, bias_s + 32);
        if (a.gelu) {
#pragma unroll
          for (int i = 0; i < 64; i += 16) gelu_fast<16>(v + i);
        }
        // the block's maximum: this half's and the other's
        uint32_t* max_s = (uint32_t*)(smem + S::OFF_MAX) + (tile_n & 1) * S::EPI * 32;
        bool infinite;
        uint32_t m = finite_max64(v, &infinite);
        max_s[ew * 32 + lane] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(max_in + bx);
        ok = warp_wait(max_in + bx, tile_n & 1, abort_flag, err);
        if (!ok) break;
        m = max(m, max_s[(ew ^ 4) * 32 + lane]);
        const int e = fp8_exp(m);
        uint32_t u[16];
        quantize64(v, fp8_inv_scale(e), infinite, u);
        const long cb = c0 - odd * 64;  // the block's first column
        const bool block = r0 < a.m && cb < a.n, tma = block && p.tma_y && (p.tma_edge || cb + 128 <= a.n);
        if (block && !odd && r0 + lane < a.m) a.q.e[(r0 + lane) * a.q.lde + (cb >> 7)] = (uint8_t)e;
        if (tma) {
#pragma unroll
          for (int q = 0; q < 4; q++)
            sts_u4(row_s + (((4 * odd + q) ^ (lane & 7)) << 4), make_uint4(u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]));
          fence_proxy_async();
        } else if (live && r0 + lane < a.m) {  // the last columns
          uint8_t* row = a.q.v + (r0 + lane) * a.q.ldv + c0;  // (16-byte aligned)
          const int cols = (int)min(64l, a.n - c0);
#pragma unroll
          for (int q = 0; q < 4; q++) {
            if (16 * q + 16 <= cols) {
              *reinterpret_cast<uint4*>(row + 16 * q) = make_uint4(u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]);
            } else {
#pragma unroll
              for (int i = 16 * q; i < 16 * q + 16; i++)
                if (i < cols) row[i] = (uint8_t)(u[i >> 2] >> (8 * (i & 3)));
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(box_in + bx);
        if (!odd) {
          ok = warp_wait(box_in + bx, tile_n & 1, abort_flag, err);
          if (!ok) break;
          if (tma && lane == 0) {
            tma_store_2d(&ymap, (int)cb, (int)r0, box);
            bulk_commit();
          }
        }
      } else {
        constexpr int BC = OUT == FP8_F32 ? 32 : 64;  // columns of a box
        // 64 columns at a time, the shared ones first, all read (and handed on) before anything is done with them
#pragma unroll 1
        for (int i = 0; i < S::COLS / 64; i++) {
          const int half = shares && cg != 0 ? S::COLS / 64 - 1 - i : i;
          float v[64];
          tmem_ld64(d + 64 * half, v);
          if (shares && i == 0) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(acc_free0);
          }
#pragma unroll
          for (int b = 0; b < 64 / BC; b++) {
            const int c = 64 * half + BC * b;  // of the warp's columns
            const long cx = c0 + c;            // the box's first column
            if (!live || cx >= a.n) continue;
            const bool tma = p.tma_y && (p.tma_edge || cx + BC <= a.n);
            if (lane == 0) bulk_wait_all_read();
            __syncwarp();
#pragma unroll
            for (int h = 0; h < BC / 32; h++) {
              float* w = v + BC * b + 32 * h;
              add_bias32(w, bias_s + c + 32 * h);
              if (a.gelu) {
#pragma unroll
                for (int j = 0; j < 32; j += 16) gelu_fast<16>(w + j);
              }
              if constexpr (OUT == FP8_F32) {
                stage_rows(w, row_s, lane);
              } else {
#pragma unroll
                for (int q = 0; q < 4; q++)
                  sts_u4(row_s + (((4 * h + q) ^ (lane & 7)) << 4),
                         make_uint4(bf16x2(w[8 * q], w[8 * q + 1]), bf16x2(w[8 * q + 2], w[8 * q + 3]),
                                    bf16x2(w[8 * q + 4], w[8 * q + 5]), bf16x2(w[8 * q + 6], w[8 * q + 7])));
              }
            }
            if (!tma) {
              if constexpr (OUT == FP8_F32)
                store_rows<float, false>(a, box, r0, cx, lane, nullptr);
              else
                store_rows_bf16(a, box, r0, cx, lane);
              continue;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&ymap, (int)cx, (int)r0, box);
              bulk_commit();
            }
          }
        }
      }
      tc_fence_before();  // this tile's TMEM reads before the arrivals of the next
    }
    if (lane == 0) bulk_wait_all();
  }
  loop.end();
}

// ---- large layers with a residual: two whole accumulators and a box for every column
//
// Bound by HBM (a residual read and a result written for each element). Above, a warp's single box would hold one
// residual at a time and wait for each. Here the pair's tile is 192 columns, so that both accumulators fit TMEM side by
// side and boxes for a whole tile fit shared memory: a tile's residual is loaded while its MMAs run. 12 epilogue warps,
// three for each lane quarter, 64 columns each.
template <int OUT>
struct TileShape {
  static constexpr int N = 192, EPI = 12;
  static constexpr int THREADS = 32 * (CTRL_WARPS + EPI);
  static constexpr int BC = OUT == FP8_F32 ? 32 : 64;  // columns of a box
  static constexpr int NBOX = 64 / BC;
  static constexpr int STAGES = OUT == FP8_F32 ? 4 : 5;
  static constexpr int A_BYTES = TM * 128, B_BYTES = N / 2 * 128;
  static constexpr int NB = (N + 127) / 128;
  static constexpr int SF_BYTES = 512 * (1 + NB), SF_COLS = 4 * (1 + NB);
  static constexpr int D1 = N, ACC = 2, SF_COL = 2 * N;  // two accumulators, a barrier each way for each
  static constexpr int OFF_B = STAGES * A_BYTES, OFF_BOX = OFF_B + STAGES * B_BYTES;
  static constexpr int OFF_SF = OFF_BOX + EPI * NBOX * BOX, OFF_BIAS = OFF_SF + SF_RING * SF_BYTES;
  static constexpr int OFF_BAR = OFF_BIAS + EPI * 64 * 4;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  static_assert(SF_COL + SF_RING * SF_COLS <= 512, "TMEM columns");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TileShape<OUT>::THREADS, 1)
    fp8_linear_tile_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                           const __grid_constant__ CUtensorMap ymap, const __grid_constant__ CUtensorMap rmap,
                           const __grid_constant__ TcFp8Args p) {
  using S = TileShape<OUT>;
  extern __shared__ uint8_t smem_raw[];
  PairLoop<S> loop(p, smem_raw);
  uint8_t* smem = loop.smem;
  uint64_t* res_full = loop.more;  // [EPI][NBOX]
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::EPI * S::NBOX; i++) mbar_init(res_full + i, 1);
    loop.init_barriers();
  }
  loop.begin();
  const Fp8Linear& a = p.a;
  const int warp = loop.warp, lane = loop.lane, tiles = loop.tiles, first = loop.first, step = loop.step;
  const uint32_t rank = loop.rank, tmem = loop.tmem;
  uint64_t *acc_full = loop.acc_full, *acc_free = loop.acc_free;
  volatile int* abort_flag = loop.abort_flag;
  int* err = loop.err;
  if (warp < CTRL_WARPS) {
    loop.control(&xmap, &wmap);
  } else {
    const int ew = warp - CTRL_WARPS, cg = ew >> 2, q4 = warp & 3;  // 64 columns; the TMEM lane quarter a warp reaches
    float* bias_s = (float*)(smem + S::OFF_BIAS) + ew * 64;
    uint8_t* box = smem + S::OFF_BOX + ew * S::NBOX * BOX;
    const uint32_t row_s = smem_u32(box) + lane * 128;  // this thread's row of a box; 16-byte units swizzled by row
    uint32_t tile_n = 0, nres = 0;
    bool ok = true;
    float2 bias_r = make_float2(0.0f, 0.0f);
    if (first < tiles) {
      int mt, nt;
      tile_at(p, first, &mt, &nt);
      bias_r = load_bias2(a, (long)nt * S::N + cg * 64 + 2 * lane);
    }
    for (int t = first; ok && t < tiles; t += step, tile_n++) {
      int mt, nt;
      tile_at(p, t, &mt, &nt);
      const long r0 = (long)mt * 2 * TM + rank * TM + q4 * 32;
      const long c0 = (long)nt * S::N + cg * 64;
      const uint32_t buf = tile_n & 1;
      // boxes with columns, and how many of them go by TMA
      const int live = r0 < a.m && c0 < a.n ? (int)min((long)S::NBOX, (a.n - c0 + S::BC - 1) / S::BC) : 0;
      const int boxes = !p.tma_y || live == 0 ? 0 : (p.tma_edge ? live : (int)min((long)live, (a.n - c0) / S::BC));
      if (lane == 0) {  // the residual comes while the tile's MMAs run
        bulk_wait_all_read();  // (the boxes are free once the last tile's stores have read them)
        for (int i = 0; i < boxes; i++) {
          mbar_arrive_expect_tx(res_full + ew * S::NBOX + i, BOX);
          tma_load_2d(box + i * BOX, &rmap, (int)c0 + i * S::BC, (int)r0, res_full + ew * S::NBOX + i);
        }
      }
      __syncwarp();
      stage_bias2(a, bias_s + 2 * lane, bias_r);
      __syncwarp();
      if (t + step < tiles) {  // the next tile's, which arrives during this one
        int mt1, nt1;
        tile_at(p, t + step, &mt1, &nt1);
        bias_r = load_bias2(a, (long)nt1 * S::N + cg * 64 + 2 * lane);
      }
      using T = typename std::conditional<OUT == FP8_F32, float, __nv_bfloat16>::type;
      uint32_t res[2][32];  // of the columns that do not go by TMA, 32 at a time
      if (boxes == 0 && live > 0) load_rows<T>(a, r0, c0, lane, res[0]);
      ok = warp_wait(acc_full + buf, (tile_n >> 1) & 1, abort_flag, err);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d = tmem + ((uint32_t)q4 << 21) + buf * S::N + cg * 64;
      const uint32_t free0 = map_rank(acc_free + buf, 0);
#pragma unroll
      for (int h = 0; h < 2; h++) {  // 32 columns at a time
        const int c = 32 * h, bx = c / S::BC;
        const bool on = bx < live, tma = bx < boxes;
        float v[32];
        tmem_ld32(d + c, v);
        if (h == 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(free0);
        }
        if (!on) continue;
        add_bias32(v, bias_s + c);
        if (a.gelu) {
#pragma unroll
          for (int j = 0; j < 32; j += 16) gelu_fast<16>(v + j);
        }
        if (!tma) {
          if (c0 + c < a.n) {
            stage_rows(v, row_s + bx * BOX, lane);
            if (h == 0 && c0 + 32 < a.n) load_rows<T>(a, r0, c0 + 32, lane, res[1]);  // arrives while these are stored
            if (h == 1 && boxes == 1) load_rows<T>(a, r0, c0 + 32, lane, res[1]);     // (the last columns, after a box by TMA)
            store_rows<T, true>(a, box + bx * BOX, r0, c0 + c, lane, res[h]);
            fence_proxy_async();  // (the box's next residual comes by TMA)
            __syncwarp();
          }
          continue;
        }
        if (c % S::BC == 0) {
          ok = warp_wait(res_full + ew * S::NBOX + bx, (nres >> bx) & 1, abort_flag, err);
          if (!ok) break;
          nres ^= 1u << bx;
        }
        const uint32_t row_b = row_s + bx * BOX;
        if constexpr (OUT == FP8_F32) {
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const uint32_t at = row_b + ((k ^ (lane & 7)) << 4);
            float4 o = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            const float4 r = lds_f4(at);
            o.x += r.x, o.y += r.y, o.z += r.z, o.w += r.w;
            sts_u4(at, make_uint4(__float_as_uint(o.x), __float_as_uint(o.y), __float_as_uint(o.z), __float_as_uint(o.w)));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t at = row_b + (((4 * h + k) ^ (lane & 7)) << 4);
            const float4 r = lds_f4(at);
            const uint32_t u[4] = {__float_as_uint(r.x), __float_as_uint(r.y), __float_as_uint(r.z), __float_as_uint(r.w)};
#pragma unroll
            for (int i = 0; i < 4; i++) {
              v[8 * k + 2 * i] += __uint_as_float(u[i] << 16);
              v[8 * k + 2 * i + 1] += __uint_as_float(u[i] & 0xFFFF0000u);
            }
            sts_u4(at, make_uint4(bf16x2(v[8 * k], v[8 * k + 1]), bf16x2(v[8 * k + 2], v[8 * k + 3]),
                                  bf16x2(v[8 * k + 4], v[8 * k + 5]), bf16x2(v[8 * k + 6], v[8 * k + 7])));
          }
        }
        if ((c + 32) % S::BC == 0) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&ymap, (int)c0 + bx * S::BC, (int)r0, box + bx * BOX);
            bulk_commit();
          }
        }
      }
      tc_fence_before();
    }
    if (lane == 0) {
      if (!ok) pause_1ms();  // residual boxes still in flight land before the shared memory goes
      bulk_wait_all();
    }
  }
  loop.end();
}

// ---- small layers: one CTA per tile of 128 rows x NT columns and share of K
//
// With few rows the weights are all there is to read, and what counts is that every SM reads some of them and that
// nothing is waited for twice: K is split over the CTAs of a cluster until the tiles fill the machine, each CTA
// starts its loads before anything else, and the shares are summed through the cluster's shared memory (in the
// order of the shares, so the result does not vary).
//
// Two CTAs fit an SM (114 registers of 256 threads, of which a third has no room) and its 512 TMEM columns: no allocation
// waits, which in a cluster could be for a CTA that waits for its own cluster.
constexpr int SPLIT_THREADS = 256;
constexpr int SPLIT_RING = 8;          // scale groups held
constexpr int SPLIT_STAGES = 8;        // at most
constexpr int SPLIT_BUDGET = 96 << 10; // shared memory for the stages: two CTAs fit an SM

struct SplitArgs {
  Fp8Linear a;
  int* err;
  int kb, n_tiles;
  int splits;       // CTAs of a cluster
  int stages;
  int box_rows;     // rows of x of a tile that are loaded (a multiple of 8)
  int vec_y, vec_res;
};

template <int NT>
struct SplitShape {
  static constexpr int NB = (NT + 127) / 128;
  static constexpr int SF_BYTES = 512 * (1 + NB);
  static constexpr int SF_COLS = 4 * (1 + NB);
  static constexpr int TMEM_COLS = NT + SPLIT_RING * SF_COLS <= 128 ? 128 : 256;
  static constexpr int PITCH = NT + 4;  // of a partial row, in floats: a warp's 16-byte stores hit every bank once
  static_assert(NT + SPLIT_RING * SF_COLS <= TMEM_COLS, "TMEM columns");
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

template <int NT, int OUT>
__global__ void __launch_bounds__(SPLIT_THREADS, 2)
    fp8_linear_split_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                            const __grid_constant__ SplitArgs p) {
  using S = SplitShape<NT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[SPLIT_STAGES], empty[SPLIT_STAGES], sf_full[SPLIT_RING], sf_empty[SPLIT_RING], acc_full;
  __shared__ __align__(16) uint8_t sf_s[SPLIT_RING * S::SF_BYTES];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const Fp8Linear& a = p.a;
  int* err = &abort_s;  // (raised outside at the end)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = p.splits, share = blockIdx.x % splits, tile = blockIdx.x / splits;
  const long m0 = (long)(tile / p.n_tiles) * TM, n0 = (long)(tile % p.n_tiles) * NT;
  const int b_lo = (int)((long)p.kb * share / splits), b_hi = (int)((long)p.kb * (share + 1) / splits);
  const int a_bytes = p.box_rows * 128, stage = a_bytes + NT * 128;
  const int rows = (int)min((long)TM, a.m - m0);

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < SPLIT_STAGES; i++) mbar_init(full + i, 1), mbar_init(empty + i, 1);
    for (int i = 0; i < SPLIT_RING; i++) mbar_init(sf_full + i, 1), mbar_init(sf_empty + i, 1);
    mbar_init(&acc_full, 1);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    // the first stages' loads are under way while the rest is set up
    for (int b = b_lo; b < b_hi && b - b_lo < p.stages; b++) {
      const int s = b - b_lo;
      mbar_arrive_expect_tx(full + s, stage);
      tma_load_2d(smem + s * stage + a_bytes, &wmap, b * 128, (int)n0, full + s);
      tma_load_2d(smem + s * stage, &xmap, b * 128, (int)m0, full + s);
    }
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "n"(S::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // what the epilogue adds, on its way while the MMAs run: a thread's units of 4 columns all lie in the same columns
  constexpr int UNITS = NT / 4;
  const int c = (int)(threadIdx.x % UNITS) * 4;
  float bias_r[4];
#pragma unroll
  for (int i = 0; i < 4; i++) bias_r[i] = a.bias && n0 + c + i < a.n ? a.bias[n0 + c + i] : 0.0f;
  // and the residual of its first unit; from then on a unit's comes while the one before it is worked on
  const int units = rows * UNITS, stride = splits * SPLIT_THREADS, first = share * SPLIT_THREADS + threadIdx.x;
  uint32_t res[4] = {0, 0, 0, 0};  // bits of y's type; two bf16 in a word where rows are loaded so
  auto load_res = [&](int u) {
    if (OUT == FP8_E4M3 || !a.res || u >= units) return;
    const long m = m0 + u / UNITS, n = n0 + c;
    if (OUT == FP8_F32) {
      const uint32_t* rr = (const uint32_t*)a.res + m * a.ldr + n;
      if (p.vec_res && n + 4 <= a.n) {
        const uint4 f = *reinterpret_cast<const uint4*>(rr);
        res[0] = f.x, res[1] = f.y, res[2] = f.z, res[3] = f.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (n + i < a.n) res[i] = rr[i];
      }
    } else {
      const uint16_t* rr = (const uint16_t*)a.res + m * a.ldr + n;
      if (p.vec_res && n + 4 <= a.n) {
        const uint2 f = *reinterpret_cast<const uint2*>(rr);
        res[0] = f.x, res[1] = f.y;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (n + i < a.n) res[i] = rr[i];
      }
    }
  };
  load_res(first);

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int b = b_lo + p.stages, s = 0, ph = 0;
      for (; b < b_hi; b++) {
        if (!mbar_wait(empty + s, ph, abort_flag, err)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(full + s, stage);
        tma_load_2d(smem + s * stage + a_bytes, &wmap, b * 128, (int)n0, full + s);
        tma_load_2d(smem + s * stage, &xmap, b * 128, (int)m0, full + s);
        if (++s == p.stages) s = 0, ph ^= 1;
      }
      if (!ok)  // loads in flight land before the shared memory goes
        for (int i = max(b_lo, b - p.stages); i < b; i++)
          mbar_drain(full + (i - b_lo) % p.stages, ((i - b_lo) / p.stages) & 1);
    }
  } else if (warp == 1) {
    const bool lead = elect_one();
    const uint64_t d0 = sdesc_sw128(smem_u32(smem)), dsf0 = sdesc(smem_u32(sf_s), 128, 128);
    int s = 0, ph = 0, slot = -1, sph = 0, last = -1, last_ph = 0;
    bool ok = true;
    uint32_t sfa = 0;
    for (int b = b_lo; b < b_hi; b++) {
      if ((b & 3) == 0 || b == b_lo) {
        if (slot >= 0 && lead) mma_commit(sf_empty + slot);
        if (++slot == SPLIT_RING) slot = 0, sph ^= 1;
        ok = warp_wait(sf_full + slot, sph, abort_flag, err);
        if (!ok) break;
        sfa = tmem + NT + slot * S::SF_COLS;
        if (lead) {
#pragma unroll
          for (int i = 0; i < 1 + S::NB; i++)
            tmem_cp_scales(sfa + 4 * i, dsf0 + ((slot * S::SF_BYTES + 512 * i) >> 4));
        }
      }
      ok = warp_wait(full + s, ph, abort_flag, err);
      if (!ok) break;
      tc_fence_after();
      if (lead) {
        const uint64_t da = d0 + ((s * stage) >> 4), db = da + (a_bytes >> 4);
        const uint32_t id = idesc_mxf8(TM, NT, 0) | ((uint32_t)(b & 3) << 4) | ((uint32_t)(b & 3) << 29);
#pragma unroll
        for (int k = 0; k < 4; k++) mma_mxf8(tmem, da + 2 * k, db + 2 * k, id, sfa, sfa + 4, b > b_lo || k > 0);
        mma_commit(empty + s);
      }
      last = s, last_ph = ph;
      if (++s == p.stages) s = 0, ph ^= 1;
    }
    if (ok && lead) mma_commit(&acc_full);
    if (!ok && last >= 0) mbar_drain(empty + last, last_ph);  // MMAs in flight end before their operands and TMEM go
  } else if (warp == 2) {
    ScaleFeed<SPLIT_RING, NT, false> feed{a, smem_u32(sf_s), sf_full, sf_empty, abort_flag, err, lane};
    feed.run(0, 1, 1, b_lo & ~3, b_hi, [&](int, long* m, long* n) { *m = m0, *n = n0; });
  } else if (warp >= 4) {
    const bool ok = warp_wait(&acc_full, 0, abort_flag, err);
    tc_fence_after();
    const int q = warp & 3, r = 32 * q + lane;
    if (ok && 32 * q < rows) {  // the stages' memory is free now: the MMAs that read it are done
      const uint32_t row_s = smem_u32(smem) + r * S::PITCH * 4;
#pragma unroll
      for (int i = 0; i < NT / 32; i++) {
        float v[32];
        tmem_ld32(tmem + ((uint32_t)q << 21) + 32 * i, v);
        if (r < rows) {
#pragma unroll
          for (int j = 0; j < 8; j++)
            sts_u4(row_s + 128 * i + 16 * j, make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                                        __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3])));
        }
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (splits > 1) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::TMEM_COLS));
  }
  const bool done = *abort_flag == 0;
  if (threadIdx.x == 0) report_failure(p.err, abort_flag);
  if (a.gelu) {
#pragma unroll
    for (int i = 0; i < 4; i++) bias_r[i] = gelu_bias(bias_r[i]);
  }
  for (int u = first; done && u < units; u += stride) {
    const int r = u / UNITS;
    const long m = m0 + r, n = n0 + c;
    float res_r[4];
    if (OUT == FP8_BF16 && p.vec_res && n + 4 <= a.n) {
      res_r[0] = __uint_as_float(res[0] << 16), res_r[1] = __uint_as_float(res[0] & 0xFFFF0000u);
      res_r[2] = __uint_as_float(res[1] << 16), res_r[3] = __uint_as_float(res[1] & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) res_r[i] = __uint_as_float(OUT == FP8_F32 ? res[i] : res[i] << 16);
    }
    load_res(u + stride);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const float* part = (const float*)smem + r * S::PITCH + c;
    if (splits == 1) {
      const float4 f = *reinterpret_cast<const float4*>(part);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
      float4 f[8];
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < splits) f[i] = ld_cluster_f4(map_rank(part, i));
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < splits) v[0] += f[i].x, v[1] += f[i].y, v[2] += f[i].z, v[3] += f[i].w;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] += bias_r[i];
    if (a.gelu) gelu_fast<4>(v);
    if (OUT != FP8_E4M3) {
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] += res_r[i];
    }
    if constexpr (OUT == FP8_F32) {
      float* y = (float*)a.y + m * a.ldy + n;
      if (p.vec_y && n + 4 <= a.n) {
        *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (n + i < a.n) y[i] = v[i];
      }
    } else if constexpr (OUT == FP8_BF16) {
      __nv_bfloat16* y = (__nv_bfloat16*)a.y + m * a.ldy + n;
      if (p.vec_y && n + 4 <= a.n) {
        *reinterpret_cast<uint2*>(y) = make_uint2(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (n + i < a.n) y[i] = __float2bfloat16(v[i]);
      }
    } else {
      // a warp holds the 128 columns of a row: one block (columns past n count for nothing and are not stored)
      uint32_t mx = 0;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (n + i < a.n) mx = max(mx, finite_bits(v[i]));
      mx = __reduce_max_sync(0xFFFFFFFFu, mx);
      const int e = fp8_exp(mx);
      const uint32_t w = e4m3x4(v[0], v[1], v[2], v[3], fp8_inv_scale(e));
      uint8_t* q = a.q.v + m * a.q.ldv + n;
      if (n + 4 <= a.n) {
        *reinterpret_cast<uint32_t*>(q) = w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (n + i < a.n) q[i] = (uint8_t)(w >> (8 * i));
      }
      if (lane == 0) a.q.e[m * a.q.lde + (n >> 7)] = (uint8_t)e;
    }
  }
  __syncwarp();
  if (splits > 1) cluster_sync();  // the others have read this CTA's share
}

// ---- host side

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_tiled() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return (EncodeTiledFn) nullptr;
    }
    return (EncodeTiledFn)f;
  }();
  return fn;
}

// Boxes of 128 bytes x box_rows of [rows][cols] elements of es bytes, rows ld elements apart, 128-byte swizzle; what
// lies outside reads as zero and is not written, so no edge needs to be padded.
static bool make_map(CUtensorMap* m, const void* base, int es, long rows, long cols, long ld, int box_rows) {
  const EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * es};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType t = es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                        : (es == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8);
  return fn(m, t, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

static int num_sms() {
  static std::atomic<int> cache[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  int n = dev < 64 ? cache[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev < 64) cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Raises a kernel's shared-memory limit, once per device.
template <class K>
static cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>* done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e != cudaSuccess || (dev < 64 && (done->load(std::memory_order_relaxed) & bit))) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Tensor maps of x, W, y and the residual for a kernel of pairs with tiles of `cols` columns.
struct PairMaps {
  CUtensorMap x, w, y, r;
};
static bool make_pair_maps(const Fp8Linear& a, int cols, TcFp8Args* p, PairMaps* m) {
  const bool q = a.y_type == FP8_E4M3;
  const int es = a.y_type == FP8_F32 ? 4 : (a.y_type == FP8_BF16 ? 2 : 1);
  const void* y = q ? a.q.v : a.y;
  const long ldy = q ? a.q.ldv : a.ldy;
  p->a = a;
  p->kb = (int)((a.k + 127) / 128);
  p->m_tiles = (int)((a.m + 2 * TM - 1) / (2 * TM));
  p->n_tiles = (int)((a.n + cols - 1) / cols);
  p->tma_y = ((uintptr_t)y | (size_t)ldy * es) % 16 == 0 && (!a.res || ((uintptr_t)a.res | (size_t)a.ldr * es) % 16 == 0);
  p->tma_edge = (size_t)a.n * es % 16 == 0;
  if (!make_map(&m->x, a.x.v, 1, a.m, a.k, a.x.ldv, TM) || !make_map(&m->w, a.w.v, 1, a.n, a.k, a.w.ldv, cols / 2))
    return false;
  m->y = m->r = m->x;  // (not used where rows do not go by TMA)
  if (p->tma_y && !make_map(&m->y, y, es, a.m, a.n, ldy, 32)) return false;
  return !p->tma_y || !a.res || make_map(&m->r, a.res, es, a.m, a.n, a.ldr, 32);
}

template <int OUT>
static cudaError_t launch_pair(const Fp8Linear& a, int* err, cudaStream_t st) {
  using S = PairShape<OUT>;
  TcFp8Args p;
  PairMaps m;
  p.err = err;
  if (!make_pair_maps(a, TN, &p, &m)) return cudaErrorInvalidValue;
  const auto kernel = fp8_linear_pair_kernel<OUT>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, S::SMEM, &allowed);
  if (e != cudaSuccess) return e;
  const long tiles = (long)p.m_tiles * p.n_tiles;
  const int pairs = num_sms() / 2;
  if (pairs <= 0) return cudaErrorInvalidDevice;
  kernel<<<2 * (unsigned)(tiles < pairs ? tiles : pairs), S::THREADS, S::SMEM, st>>>(m.x, m.w, m.y, p);
  return cudaGetLastError();
}

template <int OUT>
static cudaError_t launch_tile(const Fp8Linear& a, int* err, cudaStream_t st) {
  using S = TileShape<OUT>;
  TcFp8Args p;
  PairMaps m;
  p.err = err;
  if (!make_pair_maps(a, S::N, &p, &m)) return cudaErrorInvalidValue;
  const auto kernel = fp8_linear_tile_kernel<OUT>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, S::SMEM, &allowed);
  if (e != cudaSuccess) return e;
  const long tiles = (long)p.m_tiles * p.n_tiles;
  const int pairs = num_sms() / 2;
  if (pairs <= 0) return cudaErrorInvalidDevice;
  kernel<<<2 * (unsigned)(tiles < pairs ? tiles : pairs), S::THREADS, S::SMEM, st>>>(m.x, m.w, m.y, m.r, p);
  return cudaGetLastError();
}

template <int NT, int OUT>
static cudaError_t launch_split(const Fp8Linear& a, int splits, int* err, cudaStream_t st) {
  using S = SplitShape<NT>;
  SplitArgs p;
  p.a = a;
  p.err = err;
  p.kb = (int)((a.k + 127) / 128);
  p.n_tiles = (int)((a.n + NT - 1) / NT);
  p.splits = splits;
  p.box_rows = (int)(a.m < TM ? (a.m + 7) / 8 * 8 : TM);
  const int stage = (p.box_rows + NT) * 128;
  const int share = (p.kb + splits - 1) / splits;
  // an MMA reads 128 rows of x wherever its box starts, so the last stage is followed by what that may take
  const int tail = stage < TM * 128 ? TM * 128 - stage : 0;
  p.stages = (SPLIT_BUDGET - tail) / stage;
  if (p.stages > SPLIT_STAGES) p.stages = SPLIT_STAGES;
  if (p.stages > share) p.stages = share;
  const size_t es = OUT == FP8_F32 ? 4 : 2;
  p.vec_y = ((uintptr_t)a.y | a.ldy * es) % (4 * es) == 0;
  p.vec_res = ((uintptr_t)a.res | a.ldr * es) % (4 * es) == 0;
  CUtensorMap xm, wm;
  if (!make_map(&xm, a.x.v, 1, a.m, a.k, a.x.ldv, p.box_rows) || !make_map(&wm, a.w.v, 1, a.n, a.k, a.w.ldv, NT))
    return cudaErrorInvalidValue;
  const int partial = p.box_rows * S::PITCH * 4;  // takes the stages' place
  int smem = p.stages * stage + tail;
  if (smem < partial) smem = partial;
  smem += 1024;
  const auto kernel = fp8_linear_split_kernel<NT, OUT>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, SPLIT_BUDGET + 1024, &allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((a.m + TM - 1) / TM * p.n_tiles * splits));
  cfg.blockDim = dim3(SPLIT_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = splits, at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, xm, wm, p);
}

// Which kernel, by the number of tiles and of blocks of K (times of launches in a row, us).
//  * Split kernel up to two CTAs an SM, one when K is long: rows x K -> n 2048 x 768 -> 2304 (288 tiles of 128) 9.1
//    against 9.4 with pairs, 4096 x 768 -> 2304 (576) 16.1 against 12.9; 1024 x 4096 -> 4096 (256) 19.8 against 17.7. One
//    for an e4m3 result too, whose epilogue has twice the warps with pairs: 1024 x 768 -> 2048 (128) 9.2 against 9.9,
//    1280 (160) 11.8 against 10.0, 2048 (256) with GELU 13.3 against 11.9.
//  * Its tiles are 64 columns wide while those are few (up to 1.5 an SM): 512 x 768 -> 2304 (144) 5.9 against 6.8 with
//    128, 2048 x 768 -> 768 (192) 8.6 against 9.6, 1024 x 768 -> 2304 (288) 7.4 against 7.1; 128 wide for an e4m3 result,
//    whose blocks are, and when K is long, where a CTA has more of W on its way: 1 x 8192 -> 8192 11.3 against 14.4.
//  * K is split (a cluster costs about 0.5 us to start and more the more there are) into shares of four blocks or more
//    (one for an e4m3 result, whose epilogue the shares split too: 256 x 768 -> 2048 8.1 in four against 9.4), as far as
//    every CTA has an SM of its own, or half of one when K is long (seven eighths of the halves with clusters of four or
//    more, which do not divide every GPC's SMs: 9458 x 4352 -> 68, 74 tiles, 18.2 in two against 24.6 in four): 1 x 2048
//    -> 768 5.4 in four shares against 7.4 in one, 1 x 768 -> 2304 5.1 in one against 5.5 in two, 512 x 2048 -> 768 8.0
//    in two (96 CTAs) against 9.3 in one and 14.5 in eight (384).
template <int OUT>
static cudaError_t launch_out(const Fp8Linear& a, int* err, cudaStream_t st) {
  const int sms = num_sms(), kb = (int)((a.k + 127) / 128);
  if (sms <= 0) return cudaErrorInvalidDevice;
  const long rows = (a.m + TM - 1) / TM, t128 = rows * ((a.n + 127) / 128), t64 = rows * ((a.n + 63) / 64);
  if (t128 <= (kb > 16 || OUT == FP8_E4M3 ? sms : 2 * sms)) {
    const bool long_k = kb > 32, narrow = OUT != FP8_E4M3 && !long_k && t64 <= sms + sms / 2;
    const long tiles = narrow ? t64 : t128, room = long_k ? 2 * sms : sms;
    int splits = 1;
    const int least = OUT == FP8_E4M3 ? 1 : 4;  // blocks of a share
    while (splits < 8 && least * 2 * splits <= kb && tiles * 2 * splits <= (long_k && splits > 1 ? room - room / 8 : room))
      splits *= 2;
    if constexpr (OUT != FP8_E4M3) {
      if (narrow) return launch_split<64, OUT>(a, splits, err, st);
    }
    return launch_split<128, OUT>(a, splits, err, st);
  }
  if constexpr (OUT != FP8_E4M3) {
    if (a.res) return launch_tile<OUT>(a, err, st);
  }
  return launch_pair<OUT>(a, err, st);
}

cudaError_t launch_fp8_linear(const Fp8Linear& a, int* err, cudaStream_t st) {
  if (a.m == 0) return cudaSuccess;
  if (a.y_type == FP8_E4M3) return launch_out<FP8_E4M3>(a, err, st);
  return a.y_type == FP8_F32 ? launch_out<FP8_F32>(a, err, st) : launch_out<FP8_BF16>(a, err, st);
}

// One thread waits for the first phase of a barrier that nothing arrives on.
__global__ void fp8_wait_selftest_kernel(int cluster, unsigned long long limit_ns) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort_flag;
  mbar_init(&bar, 1);
  abort_flag = 0;
  if (cluster)
    mbar_wait_cluster(&bar, 0, &abort_flag, &abort_flag, limit_ns);
  else
    mbar_wait_lim(&bar, 0, &abort_flag, &abort_flag, limit_ns);
  report_failure(nullptr, &abort_flag);
}

cudaError_t launch_fp8_wait_selftest(int cluster, unsigned long long limit_ns, cudaStream_t st) {
  fp8_wait_selftest_kernel<<<1, 1, 0, st>>>(cluster, limit_ns);
  return cudaGetLastError();
}

cudaError_t fp8_wait_failures(unsigned* count, cudaStream_t st) {
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(st, &capture);
  if (e == cudaSuccess && capture != cudaStreamCaptureStatusNone) e = cudaErrorStreamCaptureUnsupported;
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(count, g_fp8_wait_failures, sizeof(*count), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e;
}

}  // namespace kk
