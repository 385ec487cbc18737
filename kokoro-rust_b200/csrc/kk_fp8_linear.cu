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

#include "kk_fp8.h"
#include "kk_fp8_math.cuh"
#include "kk_tc_ptx.cuh"

namespace kk {

// Raised by a kernel of the stand-alone operators whose bounded pipeline wait expired; one per device.
__device__ int g_fp8_wait_error;

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
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc(saddr, 128, 128)) : "memory");
}
// Waits, at most KK_WAIT_TIMEOUT_NS, for a phase that work already in flight completes.
__device__ __forceinline__ void mbar_drain(uint64_t* b, uint32_t parity) {
  const unsigned long long t0 = tc_now();
  while (!mbar_try_sleep(b, parity) && tc_now() - t0 < KK_WAIT_TIMEOUT_NS) {
  }
}
__device__ __forceinline__ void ldg_v8(const void* p, uint32_t* r) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void stg_v8(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

struct TcFp8Args {
  Fp8Linear a;
  int* err;
  int kb;             // blocks of 128 columns of K
  int m_tiles, n_tiles;
  int vec_y, vec_res; // rows of y / residual start on 32-byte boundaries
};

constexpr int TM = 128;       // rows of x of a tile
constexpr int SF_RING = 2;    // scale groups (4 blocks of K each) in shared memory and TMEM

template <int NT>
struct TcShape {
  static constexpr int EPI = NT == 256 ? 8 : 4;                  // epilogue warps
  static constexpr int COLS = NT / (EPI / 4);                    // columns of an epilogue thread
  static constexpr int THREADS = 32 * (4 + EPI);
  static constexpr int NB = (NT + 127) / 128;                    // 128-row scale tiles of W
  static constexpr int A_BYTES = TM * 128, B_BYTES = NT * 128;
  static constexpr int STAGES = NT == 256 ? 4 : (NT == 128 ? 6 : 8);
  static constexpr int SF_BYTES = 512 * (1 + NB);
  // TMEM columns: two accumulators (for NT = 256 they share columns 224..255, see the epilogue), then scales
  static constexpr int D1 = NT == 256 ? 224 : NT;
  static constexpr int SF_COL = D1 + NT;
  static constexpr int SF_COLS = 4 * (1 + NB);
  static constexpr int TMEM_COLS = SF_COL + SF_RING * SF_COLS <= 256 ? 256 : 512;
  static constexpr int OFF_B = STAGES * A_BYTES, OFF_SF = OFF_B + STAGES * B_BYTES;
  static constexpr int OFF_BIAS = OFF_SF + SF_RING * SF_BYTES, OFF_BAR = OFF_BIAS + EPI * COLS * 4;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;              // 1024: alignment of the first stage
  static_assert(SF_COL + SF_RING * SF_COLS <= TMEM_COLS, "TMEM columns");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// 32 x 32 transpose over a warp: lane r's v[c] becomes lane c's v[r].
__device__ __forceinline__ void warp_transpose(float* v, int lane) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const bool up = lane & s;
#pragma unroll
    for (int i = 0; i < 32; i++) {
      if (i & s) continue;
      const float x = __shfl_xor_sync(0xFFFFFFFFu, up ? v[i] : v[i | s], s);
      if (up)
        v[i] = x;
      else
        v[i | s] = x;
    }
  }
}

// 32 columns from c of the 32 rows from r0 (lane = row): residual added, stored as T. Rows on 32-byte boundaries
// are read and written as whole sectors by the lane that holds them; otherwise (any stride or offset, the last
// columns) the warp transposes the square and reads and writes a row's 32 columns together.
template <typename T>
__device__ __forceinline__ void store_chunk(const TcFp8Args& p, float* v, long r0, long c, int lane) {
  const Fp8Linear& a = p.a;
  T* y = (T*)a.y;
  const T* res = (const T*)a.res;
  if (p.vec_y && (!res || p.vec_res) && c + 32 <= a.n) {
    if (r0 + lane >= a.m) return;
    constexpr int PER = 32 / sizeof(T);  // elements of a sector
    T* yr = y + (r0 + lane) * a.ldy + c;
    const T* rr = res + (r0 + lane) * a.ldr + c;
#pragma unroll
    for (int q = 0; q < 32 / PER; q++) {
      uint32_t u[8];
      if (sizeof(T) == 4) {
        if (res) {
          ldg_v8(rr + q * PER, u);
#pragma unroll
          for (int i = 0; i < 8; i++) v[q * PER + i] += __uint_as_float(u[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = __float_as_uint(v[q * PER + i]);
      } else {
        if (res) {
          ldg_v8(rr + q * PER, u);
#pragma unroll
          for (int i = 0; i < 8; i++) {
            v[q * PER + 2 * i] += __uint_as_float(u[i] << 16);
            v[q * PER + 2 * i + 1] += __uint_as_float(u[i] & 0xFFFF0000u);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = bf16x2(v[q * PER + 2 * i], v[q * PER + 2 * i + 1]);
      }
      stg_v8(yr + q * PER, u);
    }
    return;
  }
  warp_transpose(v, lane);
  if (c + lane >= a.n) return;
#pragma unroll
  for (int j = 0; j < 32; j++) {
    if (r0 + j >= a.m) break;
    float o = v[j];
    if (res) o += (float)res[(r0 + j) * a.ldr + c + lane];
    y[(r0 + j) * a.ldy + c + lane] = (T)o;
  }
}

// A thread's 128 columns from c of its row, quantised as one block and stored.
__device__ __forceinline__ void store_block(const Fp8Linear& a, const float* v, long r, long c) {
  if (r >= a.m || c >= a.n) return;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 128; i++)
    if (c + 128 <= a.n || c + i < a.n) m = max(m, finite_bits(v[i]));
  const int e = fp8_exp(m);
  const float inv = fp8_inv_scale(e);
  uint8_t* row = a.q.v + r * a.q.ldv + c;
  a.q.e[r * a.q.lde + (c >> 7)] = (uint8_t)e;
#pragma unroll
  for (int q = 0; q < 8; q++) {
    uint4 u;
    u.x = e4m3x4(v[16 * q], v[16 * q + 1], v[16 * q + 2], v[16 * q + 3], inv);
    u.y = e4m3x4(v[16 * q + 4], v[16 * q + 5], v[16 * q + 6], v[16 * q + 7], inv);
    u.z = e4m3x4(v[16 * q + 8], v[16 * q + 9], v[16 * q + 10], v[16 * q + 11], inv);
    u.w = e4m3x4(v[16 * q + 12], v[16 * q + 13], v[16 * q + 14], v[16 * q + 15], inv);
    if (c + 16 * q + 16 <= a.n) {
      *reinterpret_cast<uint4*>(row + 16 * q) = u;
    } else {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (c + 16 * q + i < a.n) row[16 * q + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
}

// Persistent CTAs over tiles of 128 rows x NT columns, columns fastest (the tiles of one row tile run together
// and share its rows of x through L2). Warp 0: TMA loads of x and W boxes (128 bytes x rows, 128-byte swizzle)
// into a ring of stages; warp 1: MMAs; warp 2: scales, four blocks of K at a time, into shared memory in the
// layout of the TMEM copy; the last warps: epilogue (a thread holds COLS columns of one row).
template <int NT, int OUT>
__global__ void __launch_bounds__(TcShape<NT>::THREADS, 1)
    fp8_linear_tc_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                         const __grid_constant__ TcFp8Args p) {
  using S = TcShape<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = (uint64_t*)(smem + S::OFF_BAR);
  uint64_t *empty = full + S::STAGES, *sf_full = empty + S::STAGES, *sf_empty = sf_full + SF_RING;
  uint64_t *acc_full = sf_empty + SF_RING, *acc_free = acc_full + 1;
  uint32_t* tmem_slot = (uint32_t*)(acc_free + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Fp8Linear& a = p.a;
  int* err = p.err ? p.err : &g_fp8_wait_error;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; i++) mbar_init(full + i, 1), mbar_init(empty + i, 1);
    for (int i = 0; i < SF_RING; i++) mbar_init(sf_full + i, 1), mbar_init(sf_empty + i, 1);
    mbar_init(acc_full, 1);
    mbar_init(acc_free, S::EPI);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "n"(S::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tiles = p.m_tiles * p.n_tiles, kb = p.kb;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        const int m0 = t / p.n_tiles * TM, n0 = t % p.n_tiles * NT;
        for (int b = 0; b < kb; b++, it++) {
          const uint32_t s = it % S::STAGES;
          if (it >= S::STAGES && !mbar_wait(empty + s, (it / S::STAGES + 1) & 1, abort_flag, err)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full + s, S::A_BYTES + S::B_BYTES);
          tma_load_2d(smem + s * S::A_BYTES, &xmap, b * 128, m0, full + s);
          tma_load_2d(smem + S::OFF_B + s * S::B_BYTES, &wmap, b * 128, n0, full + s);
        }
      }
      if (!ok)  // loads still in flight land before the block's shared memory goes
        for (uint32_t i = it > S::STAGES ? it - S::STAGES : 0; i < it; i++)
          mbar_drain(full + i % S::STAGES, (i / S::STAGES) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t it = 0, g = 0, tile_n = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x, tile_n++) {
        if (tile_n > 0 && !mbar_wait(acc_free, (tile_n - 1) & 1, abort_flag, err)) break;
        tc_fence_after();
        const uint32_t d = tmem + (tile_n & 1) * S::D1;
        for (int b = 0; b < kb; b++, it++) {
          const uint32_t slot = g % SF_RING, sfa = tmem + S::SF_COL + slot * S::SF_COLS, sfb = sfa + 4;
          if ((b & 3) == 0) {
            if (!mbar_wait(sf_full + slot, (g / SF_RING) & 1, abort_flag, err)) {
              ok = false;
              break;
            }
            const uint32_t sf = smem_u32(smem + S::OFF_SF + slot * S::SF_BYTES);
            tmem_cp_scales(sfa, sf);
#pragma unroll
            for (int i = 0; i < S::NB; i++) tmem_cp_scales(sfb + 4 * i, sf + 512 * (1 + i));
          }
          const uint32_t s = it % S::STAGES;
          if (!mbar_wait(full + s, (it / S::STAGES) & 1, abort_flag, err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = sdesc_sw128(smem_u32(smem + s * S::A_BYTES));
          const uint64_t db = sdesc_sw128(smem_u32(smem + S::OFF_B + s * S::B_BYTES));
          const uint32_t id = idesc_mxf8(TM, NT, b & 3);
#pragma unroll
          for (int k = 0; k < 4; k++) mma_mxf8(d, da + 2 * k, db + 2 * k, id, sfa, sfb, b > 0 || k > 0);
          mma_commit(empty + s);
          if ((b & 3) == 3 || b == kb - 1) {
            mma_commit(sf_empty + slot);
            g++;
          }
        }
        if (ok) mma_commit(acc_full);
      }
      if (*abort_flag && it > 0)  // MMAs still in flight end before their operands and TMEM go
        mbar_drain(empty + (it - 1) % S::STAGES, ((it - 1) / S::STAGES) & 1);
    }
  } else if (warp == 2) {
    uint32_t g = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      const long m0 = (long)(t / p.n_tiles) * TM, n0 = (long)(t % p.n_tiles) * NT;
      for (int b = 0; b < kb; b += 4, g++) {
        uint32_t wx[4], ww[S::NB][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const long r = m0 + 32 * i + lane;
          wx[i] = r < a.m ? *reinterpret_cast<const uint32_t*>(a.x.e + r * a.x.lde + b) : 0u;
#pragma unroll
          for (int j = 0; j < S::NB; j++) {
            const long c = n0 + 128 * j + 32 * i;
            ww[j][i] = c < a.n ? *reinterpret_cast<const uint32_t*>(a.w.e + (c >> 7) * a.w.lde + b) : 0u;
          }
        }
        const uint32_t slot = g % SF_RING;
        if (g >= SF_RING) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(sf_empty + slot, (g / SF_RING + 1) & 1, abort_flag, err));
          if (!ok) break;
        }
        const uint32_t sf = smem_u32(smem + S::OFF_SF + slot * S::SF_BYTES) + lane * 16;
        sts_u4(sf, make_uint4(wx[0], wx[1], wx[2], wx[3]));
#pragma unroll
        for (int j = 0; j < S::NB; j++) sts_u4(sf + 512 * (1 + j), make_uint4(ww[j][0], ww[j][1], ww[j][2], ww[j][3]));
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(sf_full + slot);
      }
    }
  } else if (warp >= 4) {
    const int ew = warp - 4, half = ew >> 2;
    float* bias_s = (float*)(smem + S::OFF_BIAS) + ew * S::COLS;
    uint32_t tile_n = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, tile_n++) {
      const long r0 = (long)(t / p.n_tiles) * TM + (ew & 3) * 32;
      const long c0 = (long)(t % p.n_tiles) * NT + half * S::COLS;
      __syncwarp();
      for (int i = lane; i < S::COLS; i += 32) bias_s[i] = a.bias && c0 + i < a.n ? a.bias[c0 + i] : 0.0f;
      __syncwarp();
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(acc_full, tile_n & 1, abort_flag, err))) break;
      tc_fence_after();
      const uint32_t d = tmem + ((uint32_t)(ew & 3) << 21) + (tile_n & 1) * S::D1 + half * S::COLS;
      // The next tile's accumulator may be written once the columns that it shares with this one are read: with
      // NT = 256 the last 32 of the first accumulator, which are the first 32 of the second; the half that holds
      // them reads them first. (The tile after next reuses all of this accumulator; it waits for the next tile's
      // arrivals, which come after all of this tile's reads.)
      const bool shares = NT == 256 && half == (int)(1 - (tile_n & 1));
      const int first = shares && half == 1 ? S::COLS / 32 - 1 : 0;
      if (!shares && lane == 0) mbar_arrive(acc_free);
      if constexpr (OUT == FP8_E4M3) {
        float v[S::COLS];
        // all columns are read before any is stored: the block's scale needs them
        tmem_ld64(d, v);
        tmem_ld64(d + 64, v + 64);
        tc_fence_before();
        __syncwarp();
        if (shares && lane == 0) mbar_arrive(acc_free);
#pragma unroll
        for (int i = 0; i < S::COLS; i += 4) {
          const float4 bv = *reinterpret_cast<const float4*>(bias_s + i);
          v[i] += bv.x, v[i + 1] += bv.y, v[i + 2] += bv.z, v[i + 3] += bv.w;
        }
        if (a.gelu) {
#pragma unroll
          for (int i = 0; i < S::COLS; i++) v[i] = gelu_fast(v[i]);
        }
        store_block(a, v, r0 + lane, c0);
      } else {
#pragma unroll 1
        for (int i = 0; i < S::COLS / 32; i++) {
          const int ch = (i + first) % (S::COLS / 32);
          float v[32];
          tmem_ld32(d + 32 * ch, v);
          if (i == 0 && shares) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_free);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 bv = *reinterpret_cast<const float4*>(bias_s + 32 * ch + j);
            v[j] += bv.x, v[j + 1] += bv.y, v[j + 2] += bv.z, v[j + 3] += bv.w;
          }
          if (a.gelu) {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = gelu_fast(v[j]);
          }
          if (r0 >= a.m || c0 + 32 * ch >= a.n) continue;
          if constexpr (OUT == FP8_F32)
            store_chunk<float>(p, v, r0, c0 + 32 * ch, lane);
          else
            store_chunk<__nv_bfloat16>(p, v, r0, c0 + 32 * ch, lane);
        }
      }
      tc_fence_before();  // this tile's TMEM reads before the arrivals of the next
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::TMEM_COLS));
  }
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

// Boxes of 128 bytes x box_rows of [rows][k] values, 128-byte swizzle; what lies outside reads as zero, so
// neither K nor the rows need to be padded.
static bool make_map(CUtensorMap* m, const Fp8Store& s, long rows, long k, int box_rows) {
  const EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)s.ldv};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, s.v, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
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

template <int NT, int OUT>
static cudaError_t launch_tc(const Fp8Linear& a, int* err, cudaStream_t st) {
  using S = TcShape<NT>;
  TcFp8Args p;
  p.a = a;
  p.err = err;
  p.kb = (int)((a.k + 127) / 128);
  p.m_tiles = (int)((a.m + TM - 1) / TM);
  p.n_tiles = (int)((a.n + NT - 1) / NT);
  const size_t es = a.y_type == FP8_F32 ? 4 : 2;
  p.vec_y = ((uintptr_t)a.y | (a.ldy * es)) % 32 == 0;
  p.vec_res = ((uintptr_t)a.res | (a.ldr * es)) % 32 == 0;
  CUtensorMap xm, wm;
  if (!make_map(&xm, a.x, a.m, a.k, TM) || !make_map(&wm, a.w, a.n, a.k, NT)) return cudaErrorInvalidValue;
  const auto kernel = fp8_linear_tc_kernel<NT, OUT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e != cudaSuccess) return e;
  const long tiles = (long)p.m_tiles * p.n_tiles;
  const int sms = num_sms();
  if (sms <= 0) return cudaErrorInvalidDevice;
  kernel<<<(unsigned)(tiles < sms ? tiles : sms), S::THREADS, S::SMEM, st>>>(xm, wm, p);
  return cudaGetLastError();
}

template <int OUT>
static cudaError_t launch_out(const Fp8Linear& a, int* err, cudaStream_t st) {
  const long rows = (a.m + TM - 1) / TM;
  const int sms = num_sms();
  if (rows * ((a.n + 255) / 256) >= sms) return launch_tc<256, OUT>(a, err, st);
  if constexpr (OUT != FP8_E4M3) {
    if (rows * ((a.n + 127) / 128) < sms / 2) return launch_tc<64, OUT>(a, err, st);
  }
  return launch_tc<128, OUT>(a, err, st);
}

cudaError_t launch_fp8_linear(const Fp8Linear& a, int* err, cudaStream_t st) {
  if (a.m == 0) return cudaSuccess;
  if (a.y_type == FP8_F32) return launch_out<FP8_F32>(a, err, st);
  if (a.y_type == FP8_BF16) return launch_out<FP8_BF16>(a, err, st);
  return launch_out<FP8_E4M3>(a, err, st);
}

cudaError_t fp8_take_wait_error(int* err, cudaStream_t st) {
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(err, g_fp8_wait_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *err) {
    e = cudaMemcpyToSymbolAsync(g_fp8_wait_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  return e;
}

}  // namespace kk
