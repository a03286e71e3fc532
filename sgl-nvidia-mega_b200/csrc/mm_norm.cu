// Row kernels that make a layer's 8-bit input: the residual's addition, the RMSNorm and
// the MXFP8 or int8 quantization of its output in one pass, and the int8 quantization of
// rows alone. Per row of H values:
//   r     = round(x + residual)             (one rounding to x's type; r = x without one)
//   inv   = 1 / sqrt(sum(r^2) / H + eps)    (fp32, IEEE square root and division)
//   y     = (r * inv) * gamma               (fp32; y = r where only rows are quantized)
//   norm  = round(y)
//   MXFP8 : per 32 values the E8M0 rule of mx_scale_code, codes = e4m3(y * 2^-e)
//   int8  : s = max |y| / 127, codes = rint(y / s); s = 0 and codes 0 for a zero row,
//           s = NaN and codes 0 for a row with a value that is not finite
// The codes come from the fp32 y, not from the rounded norm: one rounding each. r is
// rounded first because it is the stream that the next layers add to, and the norm reads
// what they read (the rule of the peer hop in mm_comm.cu).
//
// Bound: memory. One CTA holds one row in registers (NV chunks of 16 bytes a thread), so
// that x and the residual are read once and every output is written once. Few rows take
// as many threads as the row has chunks (latency: one load a thread); many rows take 256
// to 512 threads, so that several rows share an SM and one row's loads hide another's
// reduction.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "megamoe.h"
#include "mm_dense.cuh"
#include "mm_kernels.cuh"
#include "mm_numerics.cuh"
#include "mm_ptx.cuh"

namespace mm {
namespace {

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float load(const __half *p) { return __half2float(*p); }
  static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ float value(__half v) { return __half2float(v); }
};
template <>
struct Elem<float> {
  static __device__ __forceinline__ float load(const float *p) { return *p; }
  static __device__ __forceinline__ float round(float v) { return v; }
  static __device__ __forceinline__ float value(float v) { return v; }
};

// VEC consecutive elements [e0, e0 + VEC) of a row of n: one 16-byte access where all of
// them are inside the row (the caller's chunks then start on 16-byte boundaries), else
// element by element. Elements outside the row read as 0 and are not written.
template <typename T, int VEC>
__device__ __forceinline__ void load_chunk(const T *row, int e0, int n, float (&v)[VEC]) {
  if (VEC > 1 && e0 >= 0 && e0 + VEC <= n) {
    union { uint4 q; T t[VEC]; } u;
    u.q = *reinterpret_cast<const uint4 *>(row + e0);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = Elem<T>::value(u.t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = e0 + i >= 0 && e0 + i < n ? Elem<T>::load(row + e0 + i) : 0.0f;
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T *row, int e0, int n, const float (&v)[VEC]) {
  if (VEC > 1 && e0 >= 0 && e0 + VEC <= n) {
    union { uint4 q; T t[VEC]; } u;
#pragma unroll
    for (int i = 0; i < VEC; ++i) u.t[i] = Elem<T>::round(v[i]);
    *reinterpret_cast<uint4 *>(row + e0) = u.q;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (e0 + i >= 0 && e0 + i < n) row[e0 + i] = Elem<T>::round(v[i]);
  }
}
// VEC code bytes (4 a word, first element in the low byte).
template <int VEC>
__device__ __forceinline__ void store_codes(uint8_t *row, int e0, int n, const uint32_t (&w)[(VEC + 3) / 4], bool wide) {
  if (VEC > 1 && wide) {
    if (VEC == 8) *reinterpret_cast<uint2 *>(row + e0) = make_uint2(w[0], w[VEC / 4 - 1]);
    else *reinterpret_cast<uint32_t *>(row + e0) = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (e0 + i >= 0 && e0 + i < n) row[e0 + i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i % 4)));
  }
}

// gamma's values of one chunk: its rows start wherever its own alignment says.
template <typename T, int VEC>
__device__ __forceinline__ void load_gamma(const NormArgs &a, int e0, float (&g)[VEC]) {
  if (a.gamma_f32) {
    const float *p = static_cast<const float *>(a.gamma);
    if (VEC > 1 && a.gamma_wide && e0 % 4 == 0 && e0 >= 0 && e0 + VEC <= a.hidden) {
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) {
        const float4 q = *reinterpret_cast<const float4 *>(p + e0 + 4 * i);
        g[4 * i] = q.x, g[4 * i + 1] = q.y, g[4 * i + 2] = q.z, g[4 * i + 3] = q.w;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[i] = e0 + i >= 0 && e0 + i < a.hidden ? p[e0 + i] : 0.0f;
  } else {
    const T *p = static_cast<const T *>(a.gamma);
    if (VEC > 1 && a.gamma_wide && (e0 * static_cast<int>(sizeof(T))) % 16 == 0) {
      load_chunk<T, VEC>(p, e0, a.hidden, g);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[i] = e0 + i >= 0 && e0 + i < a.hidden ? Elem<T>::load(p + e0 + i) : 0.0f;
    }
  }
}

// Block-wide sum / maximum; every thread gets the result. `red` holds 32 words, and a
// caller that reduces twice gives each its own.
__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0u;
  return __reduce_max_sync(0xffffffffu, v);
}

// Four codes rint(y / s) in a word. y / s by y * r, r = 1 / s, and one correction from the
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

// One CTA per row. NV > 0: the row's chunks stay in registers (NV a thread). NV == 0: a row
// too long for that, or rows whose buffers do not share an alignment (VEC == 1), is read
// again from memory in each of the passes.
template <typename T, int VEC, int NV, int QUANT>
__global__ void __launch_bounds__(1024) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red_f[32];
  __shared__ uint32_t red_u[32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int n = a.hidden;
  const T *x = static_cast<const T *>(a.x) + t * a.ld_x;
  const T *res = a.residual ? static_cast<const T *>(a.residual) + t * a.ld_residual : nullptr;
  T *res_out = a.residual_out ? static_cast<T *>(a.residual_out) + t * a.ld_residual_out : nullptr;
  T *norm = a.norm_out ? static_cast<T *>(a.norm_out) + t * a.ld_norm : nullptr;
  uint8_t *codes = QUANT ? a.codes + t * a.ld_codes : nullptr;
  // chunk c holds elements [c * VEC - shift, ...): chunks start on 16-byte boundaries of x,
  // and of every other buffer of x's type (the host checked that they share the offset)
  const int shift = VEC > 1 ? static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : 0;
  const int chunks = (n + shift + VEC - 1) / VEC;
  constexpr int HOLD = NV ? NV : 1;
  float v[HOLD][VEC];

  // r of chunk c (c < chunks)
  auto fetch = [&](int c, float (&out)[VEC]) {
    const int e0 = c * VEC - shift;
    load_chunk<T, VEC>(x, e0, n, out);
    if (res) {
      float q[VEC];
      load_chunk<T, VEC>(res, e0, n, q);
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = Elem<T>::value(Elem<T>::round(__fadd_rn(out[i], q[i])));
    }
  };
  auto keep = [&](int c, const float (&r)[VEC]) {
    if (res_out) store_chunk<T, VEC>(res_out, c * VEC - shift, n, r);
  };

  float inv = 1.0f;
  if (a.gamma) {
    float ss = 0.0f;
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        if (c < chunks) {
          fetch(c, v[j]);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[j][i] = 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) ss = __fmaf_rn(v[j][i], v[j][i], ss);
    } else {
      for (int c = threadIdx.x; c < chunks; c += blockDim.x) {
        fetch(c, v[0]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) ss = __fmaf_rn(v[0][i], v[0][i], ss);
      }
    }
    ss = block_sum(ss, red_f);
    inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(n)), a.eps)));
  } else if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = threadIdx.x + j * blockDim.x;
      if (c < chunks) {
        fetch(c, v[j]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] = 0.0f;
      }
    }
  }

  // y of chunk c from its r
  auto scale = [&](int c, float (&r)[VEC]) {
    if (a.gamma) {
      float g[VEC];
      load_gamma<T, VEC>(a, c * VEC - shift, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) r[i] = __fmul_rn(__fmul_rn(r[i], inv), g[i]);
    }
  };

  // Residual and norm out, and the row's or the blocks' largest magnitude: as bit patterns,
  // which order like the values and put infinity and NaN above every number. In the
  // re-reading form only the last pass writes the residual, which may be x's own memory.
  uint32_t top = 0u;
  auto mx_block = [&](int c, const float (&y)[VEC]) {
    // 32 / VEC neighbouring lanes share a block (H is a multiple of 32 and shift is 0 here)
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < VEC; ++i) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 16 / VEC; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t code = mx_scale_code(__uint_as_float(m));
    if (c < chunks) {
      const float by = mx_inverse(code);
      uint32_t w[(VEC + 3) / 4];
      if constexpr (VEC > 1) {
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i)
          w[i] = e4m3x2(__fmul_rn(y[4 * i], by), __fmul_rn(y[4 * i + 1], by)) |
                 static_cast<uint32_t>(e4m3x2(__fmul_rn(y[4 * i + 2], by), __fmul_rn(y[4 * i + 3], by))) << 16;
      } else {
        w[0] = e4m3x2(__fmul_rn(y[0], by), 0.0f) & 0xffu;
      }
      store_codes<VEC>(codes, c * VEC, n, w, VEC > 1);
      if ((c * VEC) % 32 == 0) static_cast<uint8_t *>(a.scales)[t * (n / 32) + c * VEC / 32] = static_cast<uint8_t>(code);
    }
  };
  auto int8_chunk = [&](int c, const float (&y)[VEC], float s, float r, bool tiny) {
    uint32_t w[(VEC + 3) / 4];
    uint32_t q[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) q[i] = tiny ? int8_code_tiny(y[i], s) : int8_code(y[i], s, r);
    if constexpr (VEC > 1) {
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) w[i] = pack4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
    } else {
      w[0] = q[0] & 0xffu;
    }
    const int e0 = c * VEC - shift;
    store_codes<VEC>(codes, e0, n, w, a.codes_wide && shift == 0 && e0 + VEC <= n);
  };

  // every lane of a warp walks the same number of chunks: the block maxima shuffle
  const int rounds = (chunks + blockDim.x - 1) / blockDim.x;
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = threadIdx.x + j * blockDim.x;
      if (c < chunks) {
        keep(c, v[j]);
        scale(c, v[j]);
        if (norm) store_chunk<T, VEC>(norm, c * VEC - shift, n, v[j]);
      }
      if constexpr (QUANT == MM_QUANT_MXFP8) mx_block(c, v[j]);
      if constexpr (QUANT == MM_QUANT_INT8) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
      }
    }
  } else {
    for (int j = 0; j < rounds; ++j) {
      const int c = threadIdx.x + j * blockDim.x;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[0][i] = 0.0f;
      if (c < chunks) {
        fetch(c, v[0]);
        if constexpr (QUANT != MM_QUANT_INT8) keep(c, v[0]);
        scale(c, v[0]);
        if (norm) store_chunk<T, VEC>(norm, c * VEC - shift, n, v[0]);
      }
      if constexpr (QUANT == MM_QUANT_MXFP8) mx_block(c, v[0]);
      if constexpr (QUANT == MM_QUANT_INT8) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, __float_as_uint(v[0][i]) & 0x7fffffffu);
      }
    }
  }

  if constexpr (QUANT == MM_QUANT_INT8) {
    top = block_max(top, red_u);
    const bool finite = top < 0x7f800000u;
    const float s = finite ? __fdiv_rn(__uint_as_float(top), 127.0f) : __uint_as_float(0x7fc00000u);
    if (threadIdx.x == 0) static_cast<float *>(a.scales)[t] = s;
    const bool tiny = !(s >= 0x1p-120f);  // s = 0 and NaN too
    const float r = tiny ? 0.0f : __fdiv_rn(1.0f, s);
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        if (c < chunks) {
          if (!finite) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[j][i] = 0.0f;
          }
          int8_chunk(c, v[j], finite ? s : 0.0f, r, tiny);
        }
      }
    } else {
      for (int j = 0; j < rounds; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        if (c < chunks) {
          fetch(c, v[0]);
          keep(c, v[0]);
          scale(c, v[0]);
          if (!finite) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[0][i] = 0.0f;
          }
          int8_chunk(c, v[0], finite ? s : 0.0f, r, tiny);
        }
      }
    }
  }
}

template <typename T, int QUANT>
cudaError_t launch_norm(const NormArgs &a, bool wide, void *stream) {
  constexpr int VEC = 16 / sizeof(T);
  const unsigned rows = static_cast<unsigned>(a.tokens);
  auto up32 = [](int v) { return (v + 31) / 32 * 32; };
  if (!wide) return launch(norm_kernel<T, 1, 0, QUANT>, dim3(rows), dim3(std::min(1024, up32(a.hidden))), 0, stream, a);
  // one chunk more than the row fills where rows start inside a 16-byte unit
  const bool shifted = (reinterpret_cast<uintptr_t>(a.x) % 16) || (a.ld_x * static_cast<int64_t>(sizeof(T))) % 16;
  const int chunks = (a.hidden + VEC - 1) / VEC + (shifted ? 1 : 0);
  if (a.tokens <= kFewRows) {
    const int threads = std::min(1024, up32(chunks));
    const int nv = (chunks + threads - 1) / threads;
    if (nv == 1) return launch(norm_kernel<T, VEC, 1, QUANT>, dim3(rows), dim3(threads), 0, stream, a);
    if (nv == 2) return launch(norm_kernel<T, VEC, 2, QUANT>, dim3(rows), dim3(up32((chunks + 1) / 2)), 0, stream, a);
  }
  if (chunks <= 512) return launch(norm_kernel<T, VEC, 2, QUANT>, dim3(rows), dim3(up32((chunks + 1) / 2)), 0, stream, a);
  if (chunks <= 4096) return launch(norm_kernel<T, VEC, 4, QUANT>, dim3(rows), dim3(up32((chunks + 3) / 4)), 0, stream, a);
  return launch(norm_kernel<T, VEC, 0, QUANT>, dim3(rows), dim3(1024), 0, stream, a);
}

template <typename T>
cudaError_t launch_norm(const NormArgs &a, int quant, bool wide, void *stream) {
  switch (quant) {
    case MM_QUANT_MXFP8: return launch_norm<T, MM_QUANT_MXFP8>(a, wide, stream);
    case MM_QUANT_INT8: return launch_norm<T, MM_QUANT_INT8>(a, wide, stream);
    default: return launch_norm<T, MM_QUANT_NONE>(a, wide, stream);
  }
}

int dtype_bytes(int dtype) { return dtype == MM_DTYPE_FP32 ? 4 : 2; }

// Rows of a buffer, and whether two of them share memory.
struct Span {
  const void *p;
  int64_t ld;
};
bool overlap(const Span &u, const Span &v, int tokens, int hidden, int es) {
  if (!u.p || !v.p) return false;
  const auto lo = [](const Span &s) { return reinterpret_cast<uintptr_t>(s.p); };
  const auto hi = [&](const Span &s) { return lo(s) + ((tokens - 1) * s.ld + hidden) * es; };
  return lo(u) < hi(v) && lo(v) < hi(u);
}

// Checks the sizes and picks the kernel's form: 16-byte chunks where x, the residual and the
// outputs of x's type put each row at the same offset from a 16-byte boundary (MXFP8: at a
// boundary, so that blocks and chunks agree), elements otherwise.
int run_norm(const char *what, NormArgs a, int dtype, int quant, void *stream) {
  if (a.tokens < 0 || a.hidden < 1) return set_error(MM_ERR_INVALID, "%s: %d tokens of %d values", what, a.tokens, a.hidden);
  if (dtype != MM_DTYPE_BF16 && dtype != MM_DTYPE_FP16 && dtype != MM_DTYPE_FP32)
    return set_error(MM_ERR_INVALID, "%s: unknown type %d", what, dtype);
  if (quant != MM_QUANT_NONE && quant != MM_QUANT_MXFP8 && quant != MM_QUANT_INT8)
    return set_error(MM_ERR_INVALID, "%s: unknown 8-bit format %d", what, quant);
  if (a.tokens == 0) return MM_OK;
  if (!a.x || (quant && (!a.codes || !a.scales)) || (!quant && !a.norm_out))
    return set_error(MM_ERR_INVALID, "%s: null pointer", what);
  if (a.residual && !a.residual_out) return set_error(MM_ERR_INVALID, "%s: a residual needs residual_out", what);
  if (quant == MM_QUANT_MXFP8 && a.hidden % 32)
    return set_error(MM_ERR_INVALID, "%s: MXFP8 needs a multiple of 32 values, not %d", what, a.hidden);
  if (quant == MM_QUANT_INT8 && reinterpret_cast<uintptr_t>(a.scales) % 4)
    return set_error(MM_ERR_INVALID, "%s: misaligned scales", what);
  if (a.ld_x < a.hidden || (a.residual && (a.ld_residual < a.hidden || a.ld_residual_out < a.hidden)) ||
      (a.norm_out && a.ld_norm < a.hidden) || (quant && a.ld_codes < a.hidden))
    return set_error(MM_ERR_INVALID, "%s: rows overlap (a row stride below %d)", what, a.hidden);
  const int es = dtype_bytes(dtype);
  // each thread writes the residual over elements that it alone has read, so that it may take
  // x's or the residual's own place, row for row; nothing else may overlap an input
  const Span in[] = {{a.x, a.ld_x}, {a.residual, a.ld_residual}};
  for (const Span &s : in) {
    if (overlap(s, {a.norm_out, a.ld_norm}, a.tokens, a.hidden, es) ||
        (overlap(s, {a.residual_out, a.ld_residual_out}, a.tokens, a.hidden, es) &&
         !(s.p == a.residual_out && s.ld == a.ld_residual_out)))
      return set_error(MM_ERR_INVALID, "%s: an output overlaps an input", what);
  }
  const uintptr_t base = reinterpret_cast<uintptr_t>(a.x);
  bool wide = true;
  auto same = [&](const void *p, int64_t ld) {
    if (!p) return true;
    return (reinterpret_cast<uintptr_t>(p) - base) % 16 == 0 && (ld - a.ld_x) * es % 16 == 0;
  };
  const void *typed[] = {a.x, a.residual, a.residual_out, a.norm_out};
  for (const void *p : typed)
    if (reinterpret_cast<uintptr_t>(p) % es) return set_error(MM_ERR_INVALID, "%s: a misaligned pointer", what);
  if (a.gamma && reinterpret_cast<uintptr_t>(a.gamma) % (a.gamma_f32 ? 4 : es))
    return set_error(MM_ERR_INVALID, "%s: a misaligned gamma", what);
  wide = same(a.residual, a.ld_residual) && same(a.residual_out, a.ld_residual_out) && same(a.norm_out, a.ld_norm);
  const bool shifted = base % 16 || a.ld_x * es % 16;
  a.codes_wide = quant && reinterpret_cast<uintptr_t>(a.codes) % 8 == 0 && a.ld_codes % 8 == 0;
  if (quant == MM_QUANT_MXFP8 && (shifted || !a.codes_wide)) wide = false;
  a.gamma_wide = a.gamma && reinterpret_cast<uintptr_t>(a.gamma) % 16 == 0;
  cudaError_t e;
  if (dtype == MM_DTYPE_BF16) e = launch_norm<__nv_bfloat16>(a, quant, wide, stream);
  else if (dtype == MM_DTYPE_FP16) e = launch_norm<__half>(a, quant, wide, stream);
  else e = launch_norm<float>(a, quant, wide, stream);
  if (e != cudaSuccess) return set_error(MM_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return MM_OK;
}

}  // namespace

int quantize_rows(const char *what, const void *x, int64_t ld_x, int dtype, int8_t *codes, int64_t ld_codes,
                  float *scales, int tokens, int hidden, void *stream) {
  NormArgs a = {};
  a.x = x;
  a.ld_x = ld_x;
  a.codes = reinterpret_cast<uint8_t *>(codes);
  a.ld_codes = ld_codes;
  a.scales = scales;
  a.tokens = tokens;
  a.hidden = hidden;
  return run_norm(what, a, dtype, MM_QUANT_INT8, stream);
}

}  // namespace mm

using namespace mm;

extern "C" {

int mm_rms_norm(const mm_norm_args *n, void *stream) {
  if (!n) return set_error(MM_ERR_INVALID, "mm_rms_norm: null pointer");
  if (n->tokens > 0 && !n->gamma) return set_error(MM_ERR_INVALID, "mm_rms_norm: null gamma");
  if (n->gamma_dtype != n->dtype && n->gamma_dtype != MM_DTYPE_FP32)
    return set_error(MM_ERR_INVALID, "mm_rms_norm: gamma is of x's type or fp32");
  NormArgs a = {};
  a.x = n->x;
  a.residual = n->residual;
  a.gamma = n->gamma;
  a.gamma_f32 = n->gamma_dtype == MM_DTYPE_FP32;
  a.residual_out = n->residual ? n->residual_out : nullptr;
  a.norm_out = n->norm_out;
  a.codes = static_cast<uint8_t *>(n->codes);
  a.scales = n->scales;
  a.ld_x = n->ld_x;
  a.ld_residual = n->ld_residual;
  a.ld_residual_out = n->ld_residual_out;
  a.ld_norm = n->ld_norm;
  a.ld_codes = n->ld_codes;
  a.tokens = n->tokens;
  a.hidden = n->hidden;
  a.eps = n->eps;
  return run_norm("mm_rms_norm", a, n->dtype, n->quant, stream);
}

int mm_quantize_int8(const void *x, int64_t ld_x, int32_t dtype, int8_t *codes, int64_t ld_codes, float *scales,
                     int32_t tokens, int32_t hidden, void *stream) {
  return quantize_rows("mm_quantize_int8", x, ld_x, dtype, codes, ld_codes, scales, tokens, hidden, stream);
}

}  // extern "C"
