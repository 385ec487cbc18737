// Device helpers of the 8-bit operators: block scales, e4m3 conversions, the GELU of their epilogues.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>
#include <string.h>

namespace kk {

// ---- two 32-bit operations in one instruction (each rounds as the single one does)
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void unpack2(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a, b)), "l"(pack2(c, d)));
  unpack2(r, a, b);
}

// E of a block whose largest finite magnitude has these bits: 448 = 1.75 * 2^8, so with
// a = m * 2^p, 1 <= m < 2, E - 127 is p - 8, and one more where m > 1.75. At most 247.
__device__ __forceinline__ int fp8_exp(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFF) > 0x600000 ? 1 : 0);
  return e > 0 ? e : 0;
}
// 2^(127 - E), E in [0, 247]
__device__ __forceinline__ float fp8_inv_scale(int e) { return __uint_as_float((uint32_t)(254 - e) << 23); }
// 2^(E - 127); 2^-127 is subnormal; E = 255 is E8M0's NaN
__device__ __forceinline__ float fp8_scale(int e) {
  return __uint_as_float(e == 0 ? 1u << 22 : (e == 255 ? 0x7FC00000u : (uint32_t)e << 23));
}
// Magnitude bits of a finite value, 0 for infinities and NaN: they order like the magnitudes.
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}
// four finite or NaN values, scaled, to e4m3
__device__ __forceinline__ uint32_t e4m3x4_finite(float a, float b, float c, float d, float inv) {
  float2 p, q;
  unpack2(mul2(pack2(a, b), pack2(inv, inv)), p.x, p.y);
  unpack2(mul2(pack2(c, d), pack2(inv, inv)), q.x, q.y);
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(p, __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// the same with infinities (which the conversion would saturate) as NaN
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d, float inv) {
  const float s[4] = {a * inv, b * inv, c * inv, d * inv};
  uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(s[0], s[1]), __NV_SATFINITE, __NV_E4M3);
  uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(s[2], s[3]), __NV_SATFINITE, __NV_E4M3);
  uint32_t u = lo | (hi << 16);
  // a finite value of the block is at most 448 once scaled: only an infinity is still one
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (fabsf(s[i]) == INFINITY) u |= 0x7Fu << (8 * i);
  return u;
}
__device__ __forceinline__ void e4m3x4_to_f32(uint32_t u, float* v) {
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> (16 * h)), __NV_E4M3);
    __half2 p;
    memcpy(&p, &r, 4);
    const float2 f = __half22float2(p);
    v[2 * h] = f.x, v[2 * h + 1] = f.y;
  }
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  uint32_t u;
  memcpy(&u, &p, 4);
  return u;
}

// gelu_new(x) = x / 2 (1 + tanh(u)) = x / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3), with the hardware
// exponential and reciprocal: about 2^-20 relative near 0 and above. (The bf16 layers use the hardware tanh, 2^-11; here
// the result may be kept in 32 bits, or be rounded to e4m3, where an error of 2^-11 moves one value in a hundred to the
// neighbouring code.) The unit for both gives 16 results a clock and SM, which at two a value bounds a layer of 768
// columns, so one reciprocal serves four values: 1 / a = b c d / (a b c d), 11% of the layer. For that the denominators
// have to stay finite: values below -5.6, where gelu_new is above -2.7e-9, count as -5.6, and a NaN is kept from its
// neighbours' product (fminf takes the number) but stays NaN itself. (Exponentials on the FMA pipe measured slower:
// then it is the instructions.) Minus infinity counts as -5.6 too, which is right for a sum that overflowed; for one that
// a bias of minus infinity made see gelu_bias.
template <int N>  // a multiple of 4; the steps of all N values side by side, because each step waits for the one before
__device__ __forceinline__ void gelu_fast(float* v) {
  constexpr float k = -2.0f * 0.797884560802865355f * 1.44269504088896341f;  // -2 sqrt(2 / pi) log2(e)
  const uint64_t k1 = pack2(0.044715f * k, 0.044715f * k), k0 = pack2(k, k);
  float t[N];
#pragma unroll
  for (int i = 0; i < N; i++) asm("max.NaN.f32 %0, %1, %2;" : "=f"(v[i]) : "f"(v[i]), "f"(-5.6f));
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint64_t x = pack2(v[i], v[i + 1]);
    unpack2(mul2(x, fma2(mul2(x, x), k1, k0)), t[i], t[i + 1]);  // at most 30.97
  }
#pragma unroll
  for (int i = 0; i < N; i++) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t[i]) : "f"(fminf(t[i], 31.0f)));
#pragma unroll
  for (int i = 0; i < N; i += 2) add2(t[i], t[i + 1], 1.0f, 1.0f);
#pragma unroll
  for (int i = 0; i < N; i += 4) {  // in pairs that need no swap: 1 / a and 1 / b are c and d times 1 / (a c), 1 / (b d)
    const uint64_t ab = pack2(t[i], t[i + 1]), cd = pack2(t[i + 2], t[i + 3]);
    float ac, bd, q;
    unpack2(mul2(ab, cd), ac, bd);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(ac * bd));
    const uint64_t r = pack2(q * bd, q * ac);
    unpack2(mul2(pack2(v[i], v[i + 1]), mul2(cd, r)), v[i], v[i + 1]);
    unpack2(mul2(pack2(v[i + 2], v[i + 3]), mul2(ab, r)), v[i + 2], v[i + 3]);
  }
}

// A bias in front of GELU: minus infinity as NaN, which is what -inf (1 + tanh(-inf)) / 2 is. Here it costs an instruction a
// column, in gelu_fast it would be one for every two values (33,104 x 768 -> 2048 66.0 us against 64.1).
__device__ __forceinline__ float gelu_bias(float b) { return b == -INFINITY ? NAN : b; }

}  // namespace kk
