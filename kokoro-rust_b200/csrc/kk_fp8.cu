// 8-bit operators: quantising rows and weights to e4m3 with a power-of-two scale for each block of 128, and
// reading them back (layout in kk_fp8.h).
//
// Block of 128 columns of one row (activations) or 128 x 128 (weights), a = max |x| over its finite
// values: E is the smallest integer >= 0 with a <= 448 * 2^(E - 127) (448 is e4m3's largest value), and
// the block is held as e4m3(x * 2^(127 - E)), rounded to nearest even (off by at most 2^-4 of the value, or by
// 2^-10 * 2^(E - 127), half of e4m3's smallest step, where that is more); infinities and NaN are held as NaN.
// A power of two scales exactly, so a value is rounded once and does not depend on the order or precision of
// anything; against a scale of a / 448 it gives up at most one binade of e4m3's 17, and it is the scale format
// the tensor core applies by itself.
//
// All of it is bound by HBM: each kernel reads and writes each byte once, 16 bytes a lane on its 16- or 32-bit
// side, with several loads in flight before the first is used.
#include "kk_fp8.h"
#include "kk_fp8_math.cuh"

namespace kk {

// A lane's part of a row. The quantisers take 8 columns a lane, 16 lanes a block, whatever the type (their work
// per block, the maximum and the scale, weighs more than the loads do); the read-back 16 bytes of the result.
constexpr int QCOLS = 8, QLANES = 128 / QCOLS;
template <typename T>
struct Lane {
  static constexpr int COLS = 16 / (int)sizeof(T);
  static constexpr int LANES = 128 / COLS;
};
template <typename T>
struct Raw {
  static constexpr int WORDS = QCOLS * (int)sizeof(T) / 4;
  uint32_t w[WORDS];
};

__device__ __forceinline__ void widen(const Raw<float>& u, float (&v)[QCOLS]) {
#pragma unroll
  for (int i = 0; i < QCOLS; i++) v[i] = __uint_as_float(u.w[i]);
}
__device__ __forceinline__ void widen(const Raw<__nv_bfloat16>& u, float (&v)[QCOLS]) {
#pragma unroll
  for (int i = 0; i < 4; i++)
    v[2 * i] = __uint_as_float(u.w[i] << 16), v[2 * i + 1] = __uint_as_float(u.w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat16 v) { return (uint32_t)__bfloat16_as_ushort(v); }

// columns c .. c + 7 of a row as raw bits, zeros from column k on; VEC: rows are 16-byte aligned
template <typename T, bool VEC>
__device__ __forceinline__ void load_lane(Raw<T>& u, const T* row, long c, long k) {
  if (VEC && c + QCOLS <= k) {
#pragma unroll
    for (int i = 0; i < Raw<T>::WORDS; i += 4) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(row + c) + i / 4);
      u.w[i] = q.x, u.w[i + 1] = q.y, u.w[i + 2] = q.z, u.w[i + 3] = q.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < Raw<T>::WORDS; i++) u.w[i] = 0;
#pragma unroll
  for (int i = 0; i < QCOLS; i++)
    if (c + i < k) u.w[i * sizeof(T) / 4] |= bits_of(row[c + i]) << (8 * (i * sizeof(T) % 4));
}
template <typename T>
__device__ __forceinline__ void clear(Raw<T>& u) {
#pragma unroll
  for (int i = 0; i < Raw<T>::WORDS; i++) u.w[i] = 0;
}
// the largest magnitude of a lane's values as bits, and whether one is infinite (a NaN is passed over)
template <int N>
__device__ __forceinline__ uint32_t amax_bits(const float (&v)[N]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++) m = fmaxf(m, fabsf(v[i]));
  return __float_as_uint(m);
}
template <int N>
__device__ __forceinline__ uint32_t amax_finite_bits(const float (&v)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; i++) m = max(m, finite_bits(v[i]));
  return m;
}
// maximum over the half warp that holds a block
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
#pragma unroll
  for (int o = QLANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return m;
}
// A lane's values held as e4m3, stored at column c, nothing at or past column k.
template <int N>
__device__ __forceinline__ void store_lane(uint8_t* row, long c, long k, const float (&v)[N], float inv, bool infinite) {
  uint32_t u[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; i++)
    u[i] = infinite ? e4m3x4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv)
                    : e4m3x4_finite(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv);
  if (c + N <= k) {
    if constexpr (N == 4)
      *reinterpret_cast<uint32_t*>(row + c) = u[0];
    else
      *reinterpret_cast<uint2*>(row + c) = make_uint2(u[0], u[1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (c + i < k) row[c + i] = (uint8_t)(u[i >> 2] >> (8 * (i & 3)));
  }
}

// Rows: half a warp per (row, block), U blocks a lane, whose loads are all under way before the first is used.
template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(256) fp8_quant_rows_kernel(const T* __restrict__ x, long ldx, long k, unsigned kb,
                                                             unsigned units, Fp8Store q) {
  const int lane = threadIdx.x & 31, in = lane % QLANES;
  const unsigned u0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * (2 * U) + lane / QLANES;
  Raw<T> raw[U];
  unsigned r = u0 / kb, b = u0 - r * kb;
  const unsigned r0 = r, b0 = b;
#pragma unroll
  for (int i = 0; i < U; i++) {
    if (u0 + 2 * i < units)
      load_lane<T, VEC>(raw[i], x + r * ldx, (long)b * 128 + QCOLS * in, k);
    else
      clear(raw[i]);
    for (b += 2; b >= kb; b -= kb) r++;
  }
  r = r0, b = b0;
#pragma unroll
  for (int i = 0; i < U; i++) {
    float v[QCOLS];
    widen(raw[i], v);
    uint32_t m = block_max(amax_bits(v));
    const bool infinite = m == 0x7F800000u;
    if (__any_sync(0xFFFFFFFFu, infinite)) m = block_max(amax_finite_bits(v));
    const int e = fp8_exp(m);
    if (u0 + 2 * i < units) {
      store_lane<QCOLS>(q.v + r * q.ldv, (long)b * 128 + QCOLS * in, k, v, fp8_inv_scale(e), infinite);
      if (in == 0) q.e[r * q.lde + b] = (uint8_t)e;
    }
    for (b += 2; b >= kb; b -= kb) r++;
  }
}

// Weights: one CTA per 128 x 128 block, the block in registers between the maximum and the conversion.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_quant_blocks_kernel(const T* __restrict__ x, long ldx, long rows, long k,
                                                               unsigned kb, Fp8Store q) {
  constexpr int U = 8;  // rows of a lane: 16 to a warp, two at once
  __shared__ uint32_t wmax[8], wfin[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned rb = blockIdx.x / kb, b = blockIdx.x - rb * kb;
  const long r0 = (long)rb * 128 + warp * 16 + lane / QLANES, c = (long)b * 128 + QCOLS * (lane % QLANES);
  Raw<T> raw[U];
  if (VEC && (long)rb * 128 + 128 <= rows && (long)b * 128 + 128 <= k) {
#pragma unroll
    for (int i = 0; i < U; i++) load_lane<T, VEC>(raw[i], x + (r0 + 2 * i) * ldx, c, c + QCOLS);
  } else {
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (r0 + 2 * i < rows)
        load_lane<T, VEC>(raw[i], x + (r0 + 2 * i) * ldx, c, k);
      else
        clear(raw[i]);
    }
  }
  uint32_t m = 0, f = 0;
#pragma unroll
  for (int i = 0; i < U; i++) {
    float v[QCOLS];
    widen(raw[i], v);
    m = max(m, amax_bits(v));
  }
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if (lane == 0) wmax[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) m = max(m, wmax[i]);
  const bool infinite = m == 0x7F800000u;  // the same for the whole CTA
  if (infinite) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      float v[QCOLS];
      widen(raw[i], v);
      f = max(f, amax_finite_bits(v));
    }
    f = __reduce_max_sync(0xFFFFFFFFu, f);
    if (lane == 0) wfin[warp] = f;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, wfin[i]);
  }
  const int e = fp8_exp(m);
  const float inv = fp8_inv_scale(e);
#pragma unroll
  for (int i = 0; i < U; i++) {
    float v[QCOLS];
    widen(raw[i], v);
    if (r0 + 2 * i < rows) store_lane<QCOLS>(q.v + (r0 + 2 * i) * q.ldv, c, k, v, inv, infinite);
  }
  if (threadIdx.x == 0) q.e[(long)rb * q.lde + b] = (uint8_t)e;
}

// Reading back: value * 2^(E - 127), LANES lanes per block of a row, U blocks a lane. The product is exact in 32 bits
// (a value has 4 significant bits), and in bf16 unless it falls below bf16's normal numbers; but 2^128, which numbers from
// 248 * 2^120 = 3.2965e38 on are held as, is infinite in both.
template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(256) fp8_dequant_kernel(Fp8Store q, long k, unsigned kb, unsigned units, int block_shift,
                                                          T* __restrict__ y, long ldy) {
  constexpr int N = Lane<T>::COLS, LANES = Lane<T>::LANES, PER = 32 / LANES;
  const int lane = threadIdx.x & 31, in = lane % LANES;
  const unsigned u0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * (U * PER) + lane / LANES;
  uint32_t raw[U][N / 4];
  int e[U];
  unsigned r = u0 / kb, b = u0 - r * kb;
  const unsigned r0 = r, b0 = b;
#pragma unroll
  for (int i = 0; i < U; i++) {
    e[i] = 0;
#pragma unroll
    for (int j = 0; j < N / 4; j++) raw[i][j] = 0;
    const uint8_t* row = q.v + r * q.ldv;
    const long c = (long)b * 128 + N * in;
    const bool on = u0 + i * PER < units;
    if (on) e[i] = q.e[(long)(r >> block_shift) * q.lde + b];
    for (b += PER; b >= kb; b -= kb) r++;
    if (!on) continue;
    if (c + N <= k) {
      if constexpr (N == 4) {
        raw[i][0] = __ldg(reinterpret_cast<const uint32_t*>(row + c));
      } else {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(row + c));
        raw[i][0] = w.x, raw[i][1] = w.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; j++)
        if (c + j < k) raw[i][j >> 2] |= (uint32_t)row[c + j] << (8 * (j & 3));
    }
  }
  r = r0, b = b0;
#pragma unroll
  for (int i = 0; i < U; i++) {
    if (u0 + i * PER >= units) break;
    const long c = (long)b * 128 + N * in;
    const float s = fp8_scale(e[i]);
    float v[N];
#pragma unroll
    for (int j = 0; j < N / 4; j++) e4m3x4_to_f32(raw[i][j], v + 4 * j);
#pragma unroll
    for (int j = 0; j < N; j++) v[j] *= s;
    T* yr = y + r * ldy;
    for (b += PER; b >= kb; b -= kb) r++;
    if (VEC && c + N <= k) {
      uint4 w;
      if constexpr (N == 4)
        w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      else
        w = make_uint4(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]), bf16x2(v[6], v[7]));
      *reinterpret_cast<uint4*>(yr + c) = w;
    } else {
#pragma unroll
      for (int j = 0; j < N; j++)
        if (c + j < k) yr[c + j] = (T)v[j];
    }
  }
}

// bf16 rows that are not 16-byte aligned: a warp per block, four columns a lane. Row and block begin d elements past an
// 8-byte boundary, so that a lane stores the aligned columns 4 l - d .. 4 l - d + 3, d of them from the lane before; what
// that leaves at the ends, at most three and three, are stored one a lane. 33,104 x 768 in rows of 769 31 us, against 73
// with eight 2-byte stores a lane (15 in rows of 768). 32-bit rows are faster an element at a time, 27 us against 35.
template <int U>
__global__ void __launch_bounds__(256) fp8_dequant_any_kernel(Fp8Store q, long k, unsigned kb, unsigned units, int block_shift,
                                                              __nv_bfloat16* __restrict__ y, long ldy) {
  const int lane = threadIdx.x & 31;
  const unsigned u0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * U;
  uint32_t raw[U];
  int e[U];
  unsigned r = u0 / kb, b = u0 - r * kb;
  const unsigned r0 = r, b0 = b;
#pragma unroll
  for (int i = 0; i < U; i++) {
    raw[i] = 0, e[i] = 0;
    if (u0 + i >= units) break;
    const uint8_t* row = q.v + r * q.ldv;
    const long c = (long)b * 128 + 4 * lane;
    e[i] = q.e[(long)(r >> block_shift) * q.lde + b];
    if (c + 4 <= k) {
      raw[i] = __ldg(reinterpret_cast<const uint32_t*>(row + c));
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (c + j < k) raw[i] |= (uint32_t)row[c + j] << (8 * j);
    }
    if (++b == kb) b = 0, r++;
  }
  r = r0, b = b0;
#pragma unroll
  for (int i = 0; i < U; i++) {
    if (u0 + i >= units) break;  // (the same for the warp)
    __nv_bfloat16* out = y + r * ldy + (long)b * 128;
    const int cols = (int)min(128l, k - (long)b * 128);
    const int d = (int)((uintptr_t)out / 2 & 3);
    const float s = fp8_scale(e[i]);
    const uint32_t before = __shfl_up_sync(0xFFFFFFFFu, raw[i], 1);
    float v[4];
    e4m3x4_to_f32(__funnelshift_l(before, raw[i], 8 * d), v);
    const int c = 4 * lane - d;
    if (c >= 0 && c + 4 <= cols) {
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] *= s;
      *reinterpret_cast<uint2*>(out + c) = make_uint2(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]));
    }
    const int head = min((4 - d) & 3, cols), tail = (cols - head) & 3;
    if (head + tail > 0) {
      const int at = lane < 4 ? lane : cols - tail + lane - 4;
      const uint32_t w = __shfl_sync(0xFFFFFFFFu, raw[i], (at >> 2) & 31);
      if (lane < 4 ? lane < head : lane - 4 < tail) {
        e4m3x4_to_f32(w >> (8 * (at & 3)), v);
        out[at] = __float2bfloat16(v[0] * s);
      }
    }
    if (++b == kb) b = 0, r++;
  }
}

// Blocks a lane takes: four, so that enough loads are in flight to fill HBM, but one while the blocks do not give
// every SM a few warps of four.
static constexpr unsigned MANY_UNITS = 1u << 15;

template <typename T>
static cudaError_t quantize_t(const T* x, long rows, long k, long ldx, int block_rows, Fp8Store q, cudaStream_t st) {
  const unsigned kb = (unsigned)((k + 127) / 128);
  const bool vec = ldx * sizeof(T) % 16 == 0 && (uintptr_t)x % 16 == 0;
  if (block_rows == 1) {
    const unsigned units = (unsigned)(rows * kb);
    const bool many = units >= MANY_UNITS;
    const unsigned per = 8 * 2 * (many ? 4 : 1), grid = (unsigned)(((uint64_t)units + per - 1) / per);
    if (vec && many)
      fp8_quant_rows_kernel<T, true, 4><<<grid, 256, 0, st>>>(x, ldx, k, kb, units, q);
    else if (vec)
      fp8_quant_rows_kernel<T, true, 1><<<grid, 256, 0, st>>>(x, ldx, k, kb, units, q);
    else if (many)
      fp8_quant_rows_kernel<T, false, 4><<<grid, 256, 0, st>>>(x, ldx, k, kb, units, q);
    else
      fp8_quant_rows_kernel<T, false, 1><<<grid, 256, 0, st>>>(x, ldx, k, kb, units, q);
  } else {
    const unsigned grid = (unsigned)((rows + 127) / 128 * kb);
    if (vec)
      fp8_quant_blocks_kernel<T, true><<<grid, 256, 0, st>>>(x, ldx, rows, k, kb, q);
    else
      fp8_quant_blocks_kernel<T, false><<<grid, 256, 0, st>>>(x, ldx, rows, k, kb, q);
  }
  return cudaGetLastError();
}

cudaError_t launch_fp8_quantize(const void* x, int type, long rows, long k, long ldx, int block_rows, Fp8Store q,
                                cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  if (type == FP8_F32) return quantize_t((const float*)x, rows, k, ldx, block_rows, q, st);
  return quantize_t((const __nv_bfloat16*)x, rows, k, ldx, block_rows, q, st);
}

template <typename T>
static cudaError_t dequantize_t(Fp8Store q, long rows, long k, int block_rows, T* y, long ldy, cudaStream_t st) {
  const unsigned kb = (unsigned)((k + 127) / 128), units = (unsigned)(rows * kb);
  const bool vec = ldy * sizeof(T) % 16 == 0 && (uintptr_t)y % 16 == 0, many = units >= MANY_UNITS;
  const int lanes = vec || sizeof(T) == 4 ? Lane<T>::LANES : 32;
  const unsigned per = 8 * (32 / lanes) * (many ? 4 : 1), grid = (unsigned)(((uint64_t)units + per - 1) / per);
  const int shift = block_rows == 1 ? 0 : 7;
  if (vec && many) {
    fp8_dequant_kernel<T, true, 4><<<grid, 256, 0, st>>>(q, k, kb, units, shift, y, ldy);
  } else if (vec) {
    fp8_dequant_kernel<T, true, 1><<<grid, 256, 0, st>>>(q, k, kb, units, shift, y, ldy);
  } else if constexpr (sizeof(T) == 4) {
    if (many)
      fp8_dequant_kernel<T, false, 4><<<grid, 256, 0, st>>>(q, k, kb, units, shift, y, ldy);
    else
      fp8_dequant_kernel<T, false, 1><<<grid, 256, 0, st>>>(q, k, kb, units, shift, y, ldy);
  } else {
    if (many)
      fp8_dequant_any_kernel<4><<<grid, 256, 0, st>>>(q, k, kb, units, shift, y, ldy);
    else
      fp8_dequant_any_kernel<1><<<grid, 256, 0, st>>>(q, k, kb, units, shift, y, ldy);
  }
  return cudaGetLastError();
}

cudaError_t launch_fp8_dequantize(Fp8Store q, long rows, long k, int block_rows, void* y, int type, long ldy,
                                  cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  if (type == FP8_F32) return dequantize_t(q, rows, k, block_rows, (float*)y, ldy, st);
  return dequantize_t(q, rows, k, block_rows, (__nv_bfloat16*)y, ldy, st);
}

}  // namespace kk
