// What the dense 8-bit operators share: the row kernels' arguments (mm_norm.cu) and the
// row quantization that the int8 feed-forward block (mm_int8.cu) runs between its products.
#pragma once
#include <algorithm>
#include <cstdint>

namespace mm {

// Up to this many rows a row kernel spreads each over as many threads as it has 16-byte
// chunks; beyond, rows share the SMs.
constexpr int kFewRows = 296;

struct NormArgs {
  const void *x;             // [tokens, hidden], row stride ld_x (elements)
  const void *residual;      // the same, or null
  const void *gamma;         // [hidden] of x's type or fp32; null: rows are only quantized
  void *residual_out;        // of x's type (with residual)
  void *norm_out;            // of x's type, or null
  uint8_t *codes;            // [tokens, ld_codes] 8-bit codes, or null
  void *scales;              // E8M0 [tokens, hidden / 32] or fp32 [tokens]
  int64_t ld_x, ld_residual, ld_residual_out, ld_norm, ld_codes;
  int tokens, hidden;
  float eps;
  int gamma_f32;             // gamma is fp32 beside a 16-bit x
  int gamma_wide;            // gamma starts on a 16-byte boundary
  int codes_wide;            // code rows start on 8-byte boundaries
};

// int8 codes and fp32 scales of rows (mm_norm.cu); returns an MM_* status.
int quantize_rows(const char *what, const void *x, int64_t ld_x, int dtype, int8_t *codes, int64_t ld_codes,
                  float *scales, int tokens, int hidden, void *stream);

}  // namespace mm
