// 8-bit operators: quantising rows and weights to e4m3 with a power-of-two scale for each block of 128, and
// reading them back (layout in kk_fp8.h).
//
// Block of 128 columns of one row (activations) or 128 x 128 (weights), a = max |x| over its finite
// values: E is the smallest integer >= 0 with a <= 448 * 2^(E - 127) (448 is e4m3's largest value), and
// the block is held as e4m3(x * 2^(127 - E)), rounded to nearest even; infinities and NaN are held as
// NaN. A power of two scales exactly, so a value is rounded once and does not depend on the order or
// precision of anything; against a * 2^-.. / 448 it gives up at most one binade of e4m3's range (15
// binades of normal numbers), and it is the scale format the tensor core applies by itself.
#include "kk_fp8.h"
#include "kk_fp8_math.cuh"

namespace kk {

// columns c .. c + 3 of a row (nothing past k: 0); VEC: one aligned load of the four
template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* row, long c, long k, float* v) {
  if (VEC && c + 4 <= k) {
    if (sizeof(T) == 4) {
      const float4 f = *reinterpret_cast<const float4*>(row + c);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(row + c);
      v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xFFFF0000u);
      v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = c + i < k ? (float)row[c + i] : 0.0f;
  }
}
// four held values to columns c .. c + 3 (c a multiple of 4), nothing at or past column k
__device__ __forceinline__ void store_e4m3x4(uint8_t* row, long c, long k, uint32_t u) {
  if (c + 4 <= k) {
    *reinterpret_cast<uint32_t*>(row + c) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (c + i < k) row[c + i] = (uint8_t)(u >> (8 * i));
  }
}

// One warp per (row, block): a lane holds four columns, the block's maximum is one integer reduction.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_quant_rows_kernel(const T* x, long ldx, long k, int kb, int units,
                                                             Fp8Store q) {
  const int lane = threadIdx.x & 31;
  const int u = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u >= units) return;
  const long r = u / kb;
  const int b = u - (int)r * kb;
  const long c = (long)b * 128 + 4 * lane;
  float v[4];
  load4<T, VEC>(x + r * ldx, c, k, v);
  uint32_t m = max(max(finite_bits(v[0]), finite_bits(v[1])), max(finite_bits(v[2]), finite_bits(v[3])));
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  const int e = fp8_exp(m);
  store_e4m3x4(q.v + r * q.ldv, c, k, e4m3x4(v[0], v[1], v[2], v[3], fp8_inv_scale(e)));
  if (lane == 0) q.e[r * q.lde + b] = (uint8_t)e;
}

// One CTA per 128 x 128 block, the block in registers between the maximum and the conversion.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_quant_blocks_kernel(const T* x, long ldx, long rows, long k, int kb,
                                                               Fp8Store q) {
  __shared__ uint32_t wmax[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long rb = blockIdx.x / kb;
  const int b = (int)(blockIdx.x - rb * kb);
  const long r0 = rb * 128 + warp * 16, c = (long)b * 128 + 4 * lane;
  float v[16][4];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    if (r0 + i < rows)
      load4<T, VEC>(x + (r0 + i) * ldx, c, k, v[i]);
    else
      v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.0f;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) m = max(m, finite_bits(v[i][j]));
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if (lane == 0) wmax[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) m = max(m, wmax[i]);
  const int e = fp8_exp(m);
  const float inv = fp8_inv_scale(e);
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (r0 + i < rows) store_e4m3x4(q.v + (r0 + i) * q.ldv, c, k, e4m3x4(v[i][0], v[i][1], v[i][2], v[i][3], inv));
  if (threadIdx.x == 0) q.e[rb * q.lde + b] = (uint8_t)e;
}

// One thread per 4 columns: value * 2^(E - 127). The product is exact in 32 bits (4 significant bits);
// bf16 keeps it exactly too unless it falls below bf16's normal numbers.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_dequant_kernel(Fp8Store q, long k, int quads, long total, int block_rows,
                                                          T* y, long ldy) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const long r = i / quads;
  const long c = (i - r * quads) * 4;
  const uint8_t* row = q.v + r * q.ldv;
  const float s = fp8_scale(q.e[r / block_rows * q.lde + c / 128]);
  uint32_t u = 0;
  if (c + 4 <= k) {
    u = *reinterpret_cast<const uint32_t*>(row + c);
  } else {
    for (int j = 0; j < 4; j++)
      if (c + j < k) u |= (uint32_t)row[c + j] << (8 * j);
  }
  float v[4];
  e4m3x4_to_f32(u, v);
  T* yr = y + r * ldy;
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (c + j < k) yr[c + j] = (T)(v[j] * s);
}

template <typename T>
static cudaError_t quantize_t(const T* x, long rows, long k, long ldx, int block_rows, Fp8Store q, cudaStream_t st) {
  const int kb = (int)((k + 127) / 128);
  const bool vec = ldx % 4 == 0 && (uintptr_t)x % (4 * sizeof(T)) == 0;
  if (block_rows == 1) {
    const int units = (int)(rows * kb);
    const int grid = (units + 7) / 8;
    if (vec)
      fp8_quant_rows_kernel<T, true><<<grid, 256, 0, st>>>(x, ldx, k, kb, units, q);
    else
      fp8_quant_rows_kernel<T, false><<<grid, 256, 0, st>>>(x, ldx, k, kb, units, q);
  } else {
    const int grid = (int)((rows + 127) / 128 * kb);
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

cudaError_t launch_fp8_dequantize(Fp8Store q, long rows, long k, int block_rows, void* y, int type, long ldy,
                                  cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  const int quads = (int)((k + 3) / 4);
  const long total = rows * quads;
  const unsigned grid = (unsigned)((total + 255) / 256);
  if (type == FP8_F32)
    fp8_dequant_kernel<float, true><<<grid, 256, 0, st>>>(q, k, quads, total, block_rows, (float*)y, ldy);
  else
    fp8_dequant_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(q, k, quads, total, block_rows, (__nv_bfloat16*)y,
                                                                  ldy);
  return cudaGetLastError();
}

}  // namespace kk
