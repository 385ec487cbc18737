// C entries of the 8-bit operators: argument checks, the caller's device and stream, status codes.
#include <cuda_runtime.h>
#include <atomic>
#include <map>
#include <string>
#include <utility>

#include "../../include/kokoro_b200.h"
#include "kk_fp8.h"

namespace {

thread_local std::string g_fp8_error;

// the status, its message kept for kk_fp8_error (nothing is thrown across the C boundary)
kk_status fail(kk_status s, const char* what, const char* message = "") noexcept {
  try {
    g_fp8_error = what;
    g_fp8_error += message;
  } catch (...) {
    g_fp8_error.clear();
  }
  return s;
}

// Makes the call's device current and puts the caller's back.
struct DeviceGuard {
  int prev = -1;
  cudaError_t err = cudaSuccess;
  explicit DeviceGuard(int dev) {
    int cur = -1;
    err = cudaGetDevice(&cur);
    if (err == cudaSuccess && cur != dev) {
      err = cudaSetDevice(dev);
      if (err == cudaSuccess) prev = cur;
    }
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

constexpr int64_t MAX_DIM = (int64_t)1 << 31;  // rows, columns and strides stay below

// A store of `rows` x `k` values: what is wrong with it, or null.
const char* bad_store(const void* v, int64_t ldv, const void* e, int64_t lde, int64_t k) {
  if (!v || !e) return "null store pointer";
  if (ldv < k || ldv % 16 != 0 || ldv >= MAX_DIM) return "value rows must be a multiple of 16 bytes apart and hold every column";
  if (lde < (k + 127) / 128 || lde % 4 != 0 || lde >= MAX_DIM)
    return "exponent rows must be a multiple of 4 bytes apart and hold one byte per 128 columns";
  if (!aligned(v, 16)) return "values must be 16-byte aligned";
  if (!aligned(e, 4)) return "exponents must be 4-byte aligned";
  return nullptr;
}

const char* bad_rows(const void* x, int type, int64_t k, int64_t ld) {
  if (!x) return "null row pointer";
  if (type != KK_FP8_F32 && type != KK_FP8_BF16) return "rows are f32 or bf16";
  if (ld < k || ld >= MAX_DIM) return "row stride below the row's columns";
  if (!aligned(x, type == KK_FP8_F32 ? 4 : 2)) return "rows must be aligned to their element";
  return nullptr;
}

const char* bad_extent(int64_t rows, int64_t k) {
  if (rows < 0 || rows >= MAX_DIM) return "row count out of range";
  if (k < 1 || k >= MAX_DIM / 2) return "column count out of range";
  if (rows > 0 && (k + 127) / 128 > (MAX_DIM - 1) / rows) return "more than 2^31 blocks";
  return nullptr;
}

// Rows of `width` bytes, `pitch` bytes apart.
struct Span {
  const void* p;
  int64_t rows, width, pitch;
};

// Whether two spans share a byte. Columns of one buffer, rows of the same pitch, are told apart; spans of other pitches
// count as sharing where their address ranges do.
bool overlap(Span a, Span b) {
  if (!a.p || !b.p) return false;
  const uint64_t pa = (uint64_t)(uintptr_t)a.p, pb = (uint64_t)(uintptr_t)b.p;
  const uint64_t ea = pa + (uint64_t)(a.rows - 1) * a.pitch + a.width, eb = pb + (uint64_t)(b.rows - 1) * b.pitch + b.width;
  if (ea <= pb || eb <= pa) return false;
  if (a.rows == 1) a.pitch = b.pitch;
  if (b.rows == 1) b.pitch = a.pitch;
  if (a.rows == 1 && b.rows == 1) return true;
  if (a.pitch != b.pitch || a.width > a.pitch || b.width > b.pitch) return true;
  if (pb < pa) return overlap(b, a);
  // b begins r bytes into the pitch that a's row s begins: its rows meet a's row s or, round the corner, the next
  const uint64_t s = (pb - pa) / (uint64_t)a.pitch, r = (pb - pa) % (uint64_t)a.pitch;
  return (r < (uint64_t)a.width && s < (uint64_t)a.rows) ||
         (r + b.width > (uint64_t)a.pitch && s + 1 < (uint64_t)a.rows);
}

Span value_span(const void* v, int64_t ldv, int64_t rows, int64_t k) { return {v, rows, k, ldv}; }
Span exps_span(const void* e, int64_t lde, int64_t rows, int64_t k, int block_rows) {
  return {e, (rows + block_rows - 1) / block_rows, (k + 127) / 128, lde};
}
Span row_span(const void* x, int type, int64_t ld, int64_t rows, int64_t k) {
  const int64_t es = type == KK_FP8_F32 ? 4 : 2;
  return {x, rows, k * es, ld * es};
}

// What a device ordinal is, looked up once: 1 compute capability 10.x, 2 another device, 3 none.
int device_kind(int ordinal) {
  static std::atomic<int> cache[64];
  if (ordinal < 0 || ordinal >= 64) return 3;
  int kind = cache[ordinal].load(std::memory_order_relaxed);
  if (kind == 0) {
    int n = 0, major = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess) {
      cudaGetLastError();
      return 3;
    }
    if (ordinal >= n || cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, ordinal) != cudaSuccess) return 3;
    kind = major == 10 ? 1 : 2;
    cache[ordinal].store(kind, std::memory_order_relaxed);
  }
  return kind;
}

kk_status run(int ordinal, const char* what, cudaError_t (*f)(const void*, cudaStream_t), const void* arg, void* stream) {
  const int kind = device_kind(ordinal);
  if (kind == 3) return fail(KK_ERR_INVALID_ARG, "CUDA device ordinal out of range");
  if (kind == 2) return fail(KK_ERR_CUDA, "device is not compute capability 10.x (sm_100a)");
  DeviceGuard g(ordinal);
  if (g.err != cudaSuccess) return fail(KK_ERR_CUDA, what, cudaGetErrorString(g.err));
  cudaGetLastError();  // (what an earlier call of this thread left is not this one's)
  const cudaError_t e = f(arg, (cudaStream_t)stream);
  if (e == cudaSuccess) return KK_OK;
  cudaGetLastError();
  return fail(e == cudaErrorMemoryAllocation ? KK_ERR_OOM : KK_ERR_CUDA, what, cudaGetErrorString(e));
}

struct QuantArgs {
  const void* x;
  int type;
  long rows, k, ld;
  int block_rows;
  kk::Fp8Store q;
};

}  // namespace

extern "C" {

const char* kk_fp8_error(void) { return g_fp8_error.c_str(); }

kk_status kk_fp8_quantize(int cuda_ordinal, void* stream, const void* x, int type, int64_t rows, int64_t k, int64_t ldx,
                          int block_rows, uint8_t* values, int64_t ldv, uint8_t* exps, int64_t lde) {
  if (const char* m = bad_extent(rows, k)) return fail(KK_ERR_INVALID_ARG, m);
  if (block_rows != 1 && block_rows != 128) return fail(KK_ERR_INVALID_ARG, "block_rows must be 1 or 128");
  if (rows == 0) return KK_OK;
  if (const char* m = bad_rows(x, type, k, ldx)) return fail(KK_ERR_INVALID_ARG, m);
  if (const char* m = bad_store(values, ldv, exps, lde, k)) return fail(KK_ERR_INVALID_ARG, m);
  const Span xs = row_span(x, type, ldx, rows, k), vs = value_span(values, ldv, rows, k);
  const Span es = exps_span(exps, lde, rows, k, block_rows);
  if (overlap(xs, vs) || overlap(xs, es) || overlap(vs, es))
    return fail(KK_ERR_INVALID_ARG, "the rows, the values and the exponents must not overlap");
  QuantArgs a{x, type, (long)rows, (long)k, (long)ldx, block_rows, {values, (long)ldv, exps, (long)lde}};
  return run(cuda_ordinal, "kk_fp8_quantize: ", [](const void* p, cudaStream_t st) {
    const QuantArgs& a = *(const QuantArgs*)p;
    return kk::launch_fp8_quantize(a.x, a.type, a.rows, a.k, a.ld, a.block_rows, a.q, st);
  }, &a, stream);
}

kk_status kk_fp8_dequantize(int cuda_ordinal, void* stream, const uint8_t* values, int64_t ldv, const uint8_t* exps,
                            int64_t lde, int block_rows, int64_t rows, int64_t k, void* y, int type, int64_t ldy) {
  if (const char* m = bad_extent(rows, k)) return fail(KK_ERR_INVALID_ARG, m);
  if (block_rows != 1 && block_rows != 128) return fail(KK_ERR_INVALID_ARG, "block_rows must be 1 or 128");
  if (rows == 0) return KK_OK;
  if (const char* m = bad_rows(y, type, k, ldy)) return fail(KK_ERR_INVALID_ARG, m);
  if (const char* m = bad_store(values, ldv, exps, lde, k)) return fail(KK_ERR_INVALID_ARG, m);
  const Span ys = row_span(y, type, ldy, rows, k);
  if (overlap(ys, value_span(values, ldv, rows, k)) || overlap(ys, exps_span(exps, lde, rows, k, block_rows)))
    return fail(KK_ERR_INVALID_ARG, "the rows must not overlap the store");
  QuantArgs a{y, type, (long)rows, (long)k, (long)ldy, block_rows,
              {const_cast<uint8_t*>(values), (long)ldv, const_cast<uint8_t*>(exps), (long)lde}};
  return run(cuda_ordinal, "kk_fp8_dequantize: ", [](const void* p, cudaStream_t st) {
    const QuantArgs& a = *(const QuantArgs*)p;
    return kk::launch_fp8_dequantize(a.q, a.rows, a.k, a.block_rows, const_cast<void*>(a.x), a.type, a.ld, st);
  }, &a, stream);
}

kk_status kk_fp8_linear(int cuda_ordinal, void* stream, int64_t m, int64_t n, int64_t k, const uint8_t* x, int64_t ldx,
                        const uint8_t* x_exps, int64_t ldxe, const uint8_t* w, int64_t ldw, const uint8_t* w_exps,
                        int64_t ldwe, const float* bias, int act, const void* residual, int64_t ldr, int y_type, void* y,
                        int64_t ldy, uint8_t* y_exps, int64_t ldye) {
  if (const char* s = bad_extent(m, k)) return fail(KK_ERR_INVALID_ARG, s);
  if (const char* s = bad_extent(m, n)) return fail(KK_ERR_INVALID_ARG, s);
  if (const char* s = bad_extent(n, k)) return fail(KK_ERR_INVALID_ARG, s);
  if (act != KK_FP8_ACT_NONE && act != KK_FP8_ACT_GELU) return fail(KK_ERR_INVALID_ARG, "unknown activation");
  if (y_type != KK_FP8_F32 && y_type != KK_FP8_BF16 && y_type != KK_FP8_E4M3)
    return fail(KK_ERR_INVALID_ARG, "unknown output type");
  if (m == 0) return KK_OK;
  if (const char* s = bad_store(x, ldx, x_exps, ldxe, k)) return fail(KK_ERR_INVALID_ARG, "x: ", s);
  if (const char* s = bad_store(w, ldw, w_exps, ldwe, k)) return fail(KK_ERR_INVALID_ARG, "w: ", s);
  if (!aligned(bias, 4)) return fail(KK_ERR_INVALID_ARG, "bias must be 4-byte aligned");
  if (y_type == KK_FP8_E4M3) {
    if (residual) return fail(KK_ERR_INVALID_ARG, "an e4m3 result takes no residual");
    if (const char* s = bad_store(y, ldy, y_exps, ldye, n)) return fail(KK_ERR_INVALID_ARG, "y: ", s);
  } else {
    if (const char* s = bad_rows(y, y_type, n, ldy)) return fail(KK_ERR_INVALID_ARG, "y: ", s);
    if (residual)
      if (const char* s = bad_rows(residual, y_type, n, ldr)) return fail(KK_ERR_INVALID_ARG, "residual: ", s);
  }
  const bool q = y_type == KK_FP8_E4M3;
  const Span ys = q ? value_span(y, ldy, m, n) : row_span(y, y_type, ldy, m, n);
  const Span qs = q ? exps_span(y_exps, ldye, m, n, 1) : Span{nullptr, 0, 0, 0};
  const Span in[5] = {value_span(x, ldx, m, k), exps_span(x_exps, ldxe, m, k, 1), value_span(w, ldw, n, k),
                      exps_span(w_exps, ldwe, n, k, 128), Span{bias, 1, n * 4, n * 4}};
  for (const Span& s : in)
    if (overlap(ys, s) || overlap(qs, s)) return fail(KK_ERR_INVALID_ARG, "y must not overlap x, w or bias");
  if (overlap(ys, qs)) return fail(KK_ERR_INVALID_ARG, "y: the values and the exponents must not overlap");
  if (residual && !(residual == y && (ldr == ldy || m == 1)) && overlap(ys, row_span(residual, y_type, ldr, m, n)))
    return fail(KK_ERR_INVALID_ARG, "residual must be y itself or not overlap it");
  struct Args {
    kk::Fp8Linear a;
  } g{};
  g.a.m = (long)m, g.a.n = (long)n, g.a.k = (long)k;
  g.a.x = {const_cast<uint8_t*>(x), (long)ldx, const_cast<uint8_t*>(x_exps), (long)ldxe};
  g.a.w = {const_cast<uint8_t*>(w), (long)ldw, const_cast<uint8_t*>(w_exps), (long)ldwe};
  g.a.bias = bias, g.a.gelu = act == KK_FP8_ACT_GELU, g.a.res = residual, g.a.ldr = (long)ldr, g.a.y_type = y_type;
  if (y_type == KK_FP8_E4M3)
    g.a.q = {(uint8_t*)y, (long)ldy, y_exps, (long)ldye};
  else
    g.a.y = y, g.a.ldy = (long)ldy;
  return run(cuda_ordinal, "kk_fp8_linear: ", [](const void* p, cudaStream_t st) {
    return kk::launch_fp8_linear(((const Args*)p)->a, nullptr, st);
  }, &g, stream);
}

kk_status kk_fp8_call(int op, const int64_t* v, int n) {
  if (!v) return fail(KK_ERR_INVALID_ARG, "null arguments");
  // what does not fit an int is no type, ordinal, activation or block_rows either
  const auto i = [v](int k) { return v[k] == (int)v[k] ? (int)v[k] : -1; };
  const auto p = [v](int k) { return (void*)(uintptr_t)v[k]; };
  const auto b = [v](int k) { return (uint8_t*)(uintptr_t)v[k]; };
  if (op == KK_FP8_OP_QUANTIZE && n == 12)
    return kk_fp8_quantize(i(0), p(1), p(2), i(3), v[4], v[5], v[6], i(7), b(8), v[9], b(10), v[11]);
  if (op == KK_FP8_OP_DEQUANTIZE && n == 12)
    return kk_fp8_dequantize(i(0), p(1), b(2), v[3], b(4), v[5], i(6), v[7], v[8], p(9), i(10), v[11]);
  if (op == KK_FP8_OP_LINEAR && n == 22)
    return kk_fp8_linear(i(0), p(1), v[2], v[3], v[4], b(5), v[6], b(7), v[8], b(9), v[10], b(11), v[12],
                         (const float*)p(13), i(14), p(15), v[16], i(17), p(18), v[19], b(20), v[21]);
  return fail(KK_ERR_INVALID_ARG, "unknown operation, or not its number of arguments");
}

kk_status kk_fp8_wait_selftest(int cuda_ordinal, void* stream, int cluster, int64_t limit_ns) {
  if (cluster != 0 && cluster != 1) return fail(KK_ERR_INVALID_ARG, "cluster must be 0 or 1");
  if (limit_ns < 1000 || limit_ns > 100000000) return fail(KK_ERR_INVALID_ARG, "wait limit outside [1 us, 100 ms]");
  struct Args {
    int cluster;
    unsigned long long limit;
  } a{cluster, (unsigned long long)limit_ns};
  return run(cuda_ordinal, "kk_fp8_wait_selftest: ", [](const void* p, cudaStream_t st) {
    return kk::launch_fp8_wait_selftest(((const Args*)p)->cluster, ((const Args*)p)->limit, st);
  }, &a, stream);
}

kk_status kk_fp8_check(int cuda_ordinal, void* stream) {
  unsigned count = 0;
  unsigned* const out = &count;
  const kk_status s = run(cuda_ordinal, "kk_fp8_check: ", [](const void* p, cudaStream_t st) {
    return kk::fp8_wait_failures(*(unsigned* const*)p, st);
  }, &out, stream);
  if (s != KK_OK) return s;
  // what this thread has been told of on this stream
  thread_local std::map<std::pair<int, void*>, unsigned> told;
  try {
    unsigned& t = told[{cuda_ordinal, stream}];
    if (t == count) return KK_OK;
    t = count;
  } catch (...) {
    return fail(KK_ERR_OOM, "kk_fp8_check: out of host memory");
  }
  return fail(KK_ERR_TIMEOUT, "a bounded pipeline wait of kk_fp8_linear expired");
}

}  // extern "C"
