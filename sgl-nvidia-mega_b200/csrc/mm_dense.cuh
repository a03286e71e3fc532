// What the dense 8-bit operators share: the row kernels' arguments (mm_norm.cu) and the
// row quantization that the int8 feed-forward block (mm_int8.cu) runs between its products.
#pragma once
#include <algorithm>
#include <cstdint>

namespace mm {

// Short rows share CTAs from this many on (four CTAs an SM at four rows each).
constexpr int kShareRows = 4 * 592;

struct NormArgs {
  const void *x;             // [tokens, hidden], row stride ld_x (elements)
  const void *residual;      // the same, or null
  const void *gamma;         // [hidden] of x's type or fp32; null: rows are only quantized
  void *residual_out;        // of x's type (with residual)
  void *norm_out;            // of x's type, or null
  uint8_t *codes;            // [tokens, ld_codes] 8-bit codes, or null
  void *scales;              // E8M0 [tokens, hidden / 32] or fp32 [tokens]
  int64_t ld_x, ld_residual, ld_residual_out, ld_norm, ld_codes;
  double inv_n;              // 1 / hidden
  int tokens, hidden;
  float eps;
  int gamma_f32;             // gamma is fp32 beside a 16-bit x
  int gamma_wide;            // gamma starts on a 16-byte boundary
  int codes_wide;            // code rows start on 8-byte boundaries
  int code_row;              // int8 codes on 16-byte boundaries of rows that are not
  int turn_bytes;            // shared memory in which a row of such codes is turned
};

// The code rint(y / s), in the low byte. y / s by y * r, r = 1 / s, and one correction from the
// exact remainder (Markstein's division: two fused operations instead of a full divide);
// adding 1.5 * 2^23 rounds to the nearest even integer and leaves it, in two's complement,
// in the low byte. |y| <= amax keeps the quotient within 127 after rounding.
__device__ __forceinline__ uint32_t int8_code(float y, float s, float r) {
  const float q = __fmul_rn(y, r);
  const float t = __fmaf_rn(__fmaf_rn(-q, s, y), r, q);
  return __float_as_uint(__fadd_rn(t, 0x1.8p+23f));
}
// The same below the range in which 1 / s is finite: a true divide, clamped because a
// subnormal s carries few bits (the quotient may pass 127).
__device__ __forceinline__ uint32_t int8_code_tiny(float y, float s) {
  const float t = s == 0.0f ? 0.0f : __fdiv_rn(y, s);
  return __float_as_uint(__fadd_rn(fminf(fmaxf(t, -127.0f), 127.0f), 0x1.8p+23f));
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The scale of a row whose largest magnitude has these bits: NaN unless it is finite.
__device__ __forceinline__ float int8_scale(uint32_t top) {
  return top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 127.0f) : __uint_as_float(0x7fc00000u);
}
// Scales below this (zero and NaN too) take int8_code_tiny.
constexpr float kTinyScale = 0x1p-120f;

// A buffer's bytes: rows of row_bytes, pitch apart (one row: any pitch).
struct Bytes {
  const void *p;
  int64_t rows, row_bytes, pitch;
};
inline Bytes row_bytes(const void *p, int64_t rows, int64_t cols, int64_t ld, int size) { return {p, rows, cols * size, ld * size}; }
inline Bytes flat_bytes(const void *p, int64_t bytes) { return {p, 1, bytes, bytes}; }
// Whether two buffers share memory; null pointers do not, nor do columns beside each other of
// rows of one pitch.
inline bool overlap(const Bytes &a, const Bytes &b) {
  if (!a.p || !b.p) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa >= pb + ((b.rows - 1) * b.pitch + b.row_bytes) || pb >= pa + ((a.rows - 1) * a.pitch + a.row_bytes)) return false;
  if (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) return true;
  const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
  int64_t from = static_cast<int64_t>(pb - pa) % pitch;  // b's first column among a's
  if (from < 0) from += pitch;
  return from < a.row_bytes || from + b.row_bytes > pitch;
}

// int8 codes and fp32 scales of rows (mm_norm.cu); returns an MM_* status.
int quantize_rows(const char *what, const void *x, int64_t ld_x, int dtype, int8_t *codes, int64_t ld_codes,
                  float *scales, int tokens, int hidden, void *stream);

}  // namespace mm
