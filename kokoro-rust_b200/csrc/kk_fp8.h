// 8-bit operators: e4m3 values with one power-of-two scale for each block of 128, their quantisers,
// the read-back and the linear layer over them (kk_fp8.cu).
//
// A store holds rows of e4m3 values, `ldv` bytes apart (a multiple of 16, base 16-byte aligned), and
// rows of E8M0 scale exponents E, one byte per 128 columns, `lde` bytes apart (a multiple of 4, base
// 4-byte aligned); the block stands for value * 2^(E - 127). Activations have one exponent row per
// row (block_rows 1), weights one per 128 rows (block_rows 128).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace kk {

enum Fp8Type : int { FP8_F32 = 0, FP8_BF16 = 1, FP8_E4M3 = 2 };

struct Fp8Store {
  uint8_t* v;
  long ldv;
  uint8_t* e;
  long lde;
};

struct Fp8Linear {
  long m, n, k;
  Fp8Store x;         // [m][k], block_rows 1
  Fp8Store w;         // [n][k], block_rows 128
  const float* bias;  // [n] or null
  int gelu;
  const void* res;    // [m][n] of y's type, ldr elements apart, or null; may be y itself
  long ldr;
  int y_type;         // FP8_F32, FP8_BF16: y; FP8_E4M3: q (block_rows 1)
  void* y;
  long ldy;
  Fp8Store q;
};

// x: `type` (f32 or bf16) rows, ldx elements apart
cudaError_t launch_fp8_quantize(const void* x, int type, long rows, long k, long ldx, int block_rows, Fp8Store q,
                                cudaStream_t st);
cudaError_t launch_fp8_dequantize(Fp8Store q, long rows, long k, int block_rows, void* y, int type, long ldy,
                                  cudaStream_t st);
// err receives 2 if a bounded pipeline wait expires; null: the device counts it, for fp8_wait_failures
cudaError_t launch_fp8_linear(const Fp8Linear& a, int* err, cudaStream_t st);
// Waits for the stream (an error while it is being captured); *count = how many blocks on the current device have given up
// a wait since the process began.
cudaError_t fp8_wait_failures(unsigned* count, cudaStream_t st);
// A wait that expires (after limit_ns, in place of the waits' own limit) and is counted.
cudaError_t launch_fp8_wait_selftest(int cluster, unsigned long long limit_ns, cudaStream_t st);

}  // namespace kk
