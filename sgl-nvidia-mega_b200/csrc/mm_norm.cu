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
// Bound: memory, and next to it the instructions of an element. norm_rows_kernel: one CTA
// holds one row in registers, packed as it is stored (NV chunks of 16 bytes a thread), so
// that x and the residual are read once, all their loads are in flight at once, and every
// output is written once; 16-bit pairs are added packed (one rounding, the same as of the
// fp32 sum: where that sum is inexact it is nowhere near a tie) and the fp32 arithmetic
// goes by pairs (f32x2). Few rows take as many threads as the row has chunks (latency: one
// load a thread); many rows take fewer, so that several rows share an SM and one row's
// loads hide another's reduction. norm_kernel: rows that are too long to hold, or whose
// buffers do not share an alignment, read again in each pass.
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

// fp32 gamma beside a 16-bit x.
template <int VEC>
__device__ __forceinline__ void load_gamma_f32(const NormArgs &a, int e0, float (&g)[VEC]) {
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
}
// gamma's values of one chunk, element by element.
template <typename T, int VEC>
__device__ __forceinline__ void load_gamma(const NormArgs &a, int e0, float (&g)[VEC]) {
  if (a.gamma_f32) {
    load_gamma_f32<VEC>(a, e0, g);
  } else {
    const T *p = static_cast<const T *>(a.gamma);
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[i] = e0 + i >= 0 && e0 + i < a.hidden ? Elem<T>::load(p + e0 + i) : 0.0f;
  }
}

// Block-wide maximum; every thread gets the result.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0u;
  return __reduce_max_sync(0xffffffffu, v);
}

// ---------------------------------------------------------------------------------------
// Packed arithmetic: a chunk is 16 bytes, VEC elements.
struct alignas(8) F2 {
  float x, y;
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmul.rn.f32x2 r, p, q;\n\t"
      "mov.b64 {%0, %1}, r;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("{\n\t.reg .b64 p, q, r, s;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%6, %7};\n\t"
      "fma.rn.f32x2 s, p, q, r;\n\tmov.b64 {%0, %1}, s;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tadd.rn.f32x2 r, p, q;\n\t"
      "mov.b64 {%0, %1}, r;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

template <typename T>
struct Pack;  // of one 32-bit word
template <>
struct Pack<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ F2 value(uint32_t w) { return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }
  static __device__ __forceinline__ uint32_t round(F2 v) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(v.y), "f"(v.x));
    return d;
  }
};
template <>
struct Pack<__half> {
  static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ F2 value(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return {f.x, f.y};
  }
  static __device__ __forceinline__ uint32_t round(F2 v) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(v.y), "f"(v.x));
    return d;
  }
};

// The words of a chunk as pairs of fp32 values and back.
template <typename T>
struct Chunk {
  static constexpr int kVec = 16 / sizeof(T), kPairs = kVec / 2;
  static __device__ __forceinline__ void values(const uint4 &q, F2 (&f)[kPairs]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) {
      f[0] = {__uint_as_float(w[0]), __uint_as_float(w[1])};
      f[1] = {__uint_as_float(w[2]), __uint_as_float(w[3])};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = Pack<T>::value(w[i]);
    }
  }
  static __device__ __forceinline__ uint4 round(const F2 (&f)[kPairs]) {
    if constexpr (sizeof(T) == 4)
      return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
    else
      return make_uint4(Pack<T>::round(f[0]), Pack<T>::round(f[1]), Pack<T>::round(f[2]), Pack<T>::round(f[3]));
  }
  static __device__ __forceinline__ uint4 add(const uint4 &a, const uint4 &b) {
    if constexpr (sizeof(T) == 4)
      return make_uint4(__float_as_uint(__fadd_rn(__uint_as_float(a.x), __uint_as_float(b.x))),
                        __float_as_uint(__fadd_rn(__uint_as_float(a.y), __uint_as_float(b.y))),
                        __float_as_uint(__fadd_rn(__uint_as_float(a.z), __uint_as_float(b.z))),
                        __float_as_uint(__fadd_rn(__uint_as_float(a.w), __uint_as_float(b.w))));
    else
      return make_uint4(Pack<T>::add(a.x, b.x), Pack<T>::add(a.y, b.y), Pack<T>::add(a.z, b.z), Pack<T>::add(a.w, b.w));
  }
  // [e0, e0 + VEC) of a row of n; elements outside read as zero and are not written
  static __device__ __forceinline__ uint4 load(const T *row, int e0, int n, bool whole) {
    if (whole) return *reinterpret_cast<const uint4 *>(row + e0);
    union { uint4 q; T t[kVec]; } u;
    u.q = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (e0 + i >= 0 && e0 + i < n) u.t[i] = row[e0 + i];
    return u.q;
  }
  static __device__ __forceinline__ void store(T *row, int e0, int n, bool whole, const uint4 &q) {
    if (whole) {
      *reinterpret_cast<uint4 *>(row + e0) = q;
      return;
    }
    union { uint4 q; T t[kVec]; } u;
    u.q = q;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (e0 + i >= 0 && e0 + i < n) row[e0 + i] = u.t[i];
  }
};

// mx_scale_code, branch-free: the exponent of amax * fp32(1 / 448), rounded up when the
// mantissa is not zero (a subnormal product rounds at 2^-127, its midpoint); a zero block
// has scale 1, NaN and infinity code 255.
__device__ __forceinline__ uint32_t mx_code(uint32_t amax_bits) {
  const uint32_t b = __float_as_uint(__fmul_rn(__uint_as_float(amax_bits), 0x1.24924ap-9f));
  const uint32_t c = (b + (b < 0x800000u ? 0x3fffffu : 0x7fffffu)) >> 23;
  return amax_bits == 0u ? 127u : min(c, 255u);
}

// 1 / sqrt(sum * inv_n + eps): the sum's last steps and Newton's step in 64 bits, so that one
// rounding is left in the factor that a whole row shares.
__device__ __forceinline__ float inverse_rms(double sum, double inv_n, float eps) {
  const double m = sum * inv_n + static_cast<double>(eps);
  const float y0 = rsqrtf(static_cast<float>(m));
  if (!(y0 > 0.0f && y0 < __uint_as_float(0x7f800000u))) return y0;  // 0, inf, NaN
  const double y = y0;
  return static_cast<float>(y * (1.5 - 0.5 * m * y * y));
}

// Block-wide sum, and the maximum of `top` beside it.
__device__ __forceinline__ double block_sum(double v, uint32_t &top, double *red, uint32_t *red_top) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  top = __reduce_max_sync(0xffffffffu, top);
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return v;
  if (lane == 0) {
    red[threadIdx.x >> 5] = v;
    red_top[threadIdx.x >> 5] = top;
  }
  __syncthreads();
  v = lane < warps ? red[lane] : 0.0;
  top = __reduce_max_sync(0xffffffffu, lane < warps ? red_top[lane] : 0u);
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// gamma's elements [e0, e0 + VEC) as they are stored (of x's type), zero outside the row. Rows
// that start inside a 16-byte unit put their chunks across gamma's units: two loads, and the
// wanted words shifted out of them.
template <typename T>
__device__ __forceinline__ uint4 gamma_chunk(const NormArgs &a, int e0) {
  using C = Chunk<T>;
  constexpr int VEC = C::kVec;
  const T *p = static_cast<const T *>(a.gamma);
  const int off = e0 & (VEC - 1), low = e0 - off;  // e0 may be negative: VEC is a power of two
  if (a.gamma_wide && low >= 0 && (off ? low + 2 * VEC : low + VEC) <= a.hidden) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p + low);
    if (off == 0) return u;
    const uint4 v = *reinterpret_cast<const uint4 *>(p + low + VEC);
    const int bits = off * static_cast<int>(sizeof(T)) * 8;
    uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    if (bits & 64) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (bits & 32) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    return make_uint4(__funnelshift_r(w[0], w[1], bits & 16), __funnelshift_r(w[1], w[2], bits & 16),
                      __funnelshift_r(w[2], w[3], bits & 16), __funnelshift_r(w[3], w[4], bits & 16));
  }
  return e0 < a.hidden ? C::load(p, e0, a.hidden, false) : make_uint4(0u, 0u, 0u, 0u);
}

// One CTA per row, NV chunks of it a thread, held in registers. TURN: the int8 codes of rows
// that start inside a 16-byte unit of x, while the codes' rows start on one, are turned in
// shared memory (int8 rows of 1021 x 6147 by bytes 10.8 us, so 5.8). Four and more take more than
// the 64 registers that 1024 threads leave each.
// CTAs that shall share an SM: two of fp32 rows (h of a wide layer, 4096 x 18432: 70 us instead
// of 92; 16-bit rows lose by it, 8192 x 7168 36 instead of 30), one of the latency form.
// DENSE: 56 registers instead of 64 and five CTAs of 224 threads instead of four (norm alone of 8192 x
// 7168 48.0 us, so 42.7; of 8192 x 6147 56.2 and 49.7; beside codes it spills).
constexpr int row_ctas(int nv, bool norm, int es, bool dense) { return dense ? 4 : nv == 8 && !norm && es == 4 ? 2 : nv == 1 ? 1 : 0; }
constexpr int row_threads(int nv, bool norm, bool dense = false) { return dense ? 288 : nv >= 8 && norm ? 512 : nv >= 4 ? 640 : 1024; }
template <typename T, int NV, int QUANT, bool NORM, bool TURN, bool DENSE>
__global__ void __launch_bounds__(row_threads(NV, NORM, DENSE), row_ctas(NV, NORM, sizeof(T), DENSE)) norm_rows_kernel(const __grid_constant__ NormArgs a) {
  using C = Chunk<T>;
  constexpr int VEC = C::kVec, PAIRS = C::kPairs;
  __shared__ double red_d[32];
  __shared__ uint32_t red_u[32], red_v[32];
  extern __shared__ __align__(16) uint8_t code_rows[];
  uint8_t *turned = code_rows + threadIdx.y * a.turn_bytes;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (t >= a.tokens) return;  // rows share a CTA only where a warp has each
  const int n = a.hidden;
  const T *x = static_cast<const T *>(a.x) + t * a.ld_x;
  const T *res = NORM && a.residual ? static_cast<const T *>(a.residual) + t * a.ld_residual : nullptr;
  T *res_out = NORM && a.residual ? static_cast<T *>(a.residual_out) + t * a.ld_residual_out : nullptr;
  T *norm = NORM && a.norm_out ? static_cast<T *>(a.norm_out) + t * a.ld_norm : nullptr;
  uint8_t *codes = QUANT ? a.codes + t * a.ld_codes : nullptr;
  // chunk c holds elements [c * VEC - shift, ...): chunks start on 16-byte boundaries of x,
  // and of every other buffer of x's type (the host checked that they share the offset)
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int first = static_cast<int>(threadIdx.x) * VEC - shift, step = static_cast<int>(blockDim.x) * VEC;
  auto whole = [&](int e0) { return e0 >= 0 && e0 + VEC <= n; };

  uint4 v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = first + j * step;
    v[j] = e0 < n ? C::load(x, e0, n, whole(e0)) : make_uint4(0u, 0u, 0u, 0u);
  }
  if (res) {
    uint4 q[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = first + j * step;
      q[j] = e0 < n ? C::load(res, e0, n, whole(e0)) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = first + j * step;
      v[j] = C::add(v[j], q[j]);
      if (e0 < n) C::store(res_out, e0, n, whole(e0), v[j]);
    }
  }

  // gamma's values of chunk j; zero outside the row. One chunk a thread: loaded before the
  // reduction, whose wait then covers them (with two, 1024 x 5120 took 9.7 us instead of 8.4).
  constexpr bool EARLY = NORM && NV == 1;
  uint4 held = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (EARLY)
    if (!a.gamma_f32) held = gamma_chunk<T>(a, first);
  auto gammas = [&](int j, float (&g)[VEC]) {
    const int e0 = first + j * step;
    if (sizeof(T) == 2 && a.gamma_f32) {
      if (e0 < n) {
        load_gamma_f32<VEC>(a, e0, g);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[i] = 0.0f;
      }
      return;
    }
    F2 f[PAIRS];
    C::values(EARLY ? held : gamma_chunk<T>(a, e0), f);
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[i] = i & 1 ? f[i / 2].y : f[i / 2].x;
  };

  F2 inv = {1.0f, 1.0f};
  uint32_t top = 0u;
  if constexpr (NORM) {
    // a chain of NV * PAIRS terms a half, then 64 bits. int8: the largest |r gamma| on the way,
    // so that one reduction gives both the factor and the scale
    F2 ss = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      F2 f[PAIRS];
      C::values(v[j], f);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) ss = fma2(f[i], f[i], ss);
      if constexpr (QUANT == MM_QUANT_INT8) {
        float g[VEC];
        gammas(j, g);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          const F2 p = mul2(f[i], {g[2 * i], g[2 * i + 1]});
          top = max(top, max(__float_as_uint(p.x) & 0x7fffffffu, __float_as_uint(p.y) & 0x7fffffffu));
        }
      }
    }
    const double sum = block_sum(static_cast<double>(ss.x) + static_cast<double>(ss.y), top, red_d, red_u);
    inv.x = inv.y = inverse_rms(sum, a.inv_n, a.eps);
  }

  // y of chunk j
  auto scaled = [&](int j, F2 (&f)[PAIRS]) {
    C::values(v[j], f);
    if constexpr (NORM) {
      float g[VEC];
      gammas(j, g);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) f[i] = mul2(mul2(f[i], inv), {g[2 * i], g[2 * i + 1]});
    }
  };

  if constexpr (QUANT != MM_QUANT_INT8) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = first + j * step;
      F2 f[PAIRS];
      scaled(j, f);
      if (norm && e0 < n) C::store(norm, e0, n, whole(e0), C::round(f));
      if constexpr (QUANT == MM_QUANT_MXFP8) {
        // 32 / VEC neighbouring lanes share a block (H is a multiple of 32 and shift is 0 here)
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
          m = max(m, max(__float_as_uint(f[i].x) & 0x7fffffffu, __float_as_uint(f[i].y) & 0x7fffffffu));
#pragma unroll
        for (int o = 16 / VEC; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const uint32_t code = mx_code(m);
        const float by1 = mx_inverse(code);
        const F2 by = {by1, by1};
        if (e0 < n) {
          uint32_t w[VEC / 4];
#pragma unroll
          for (int i = 0; i < VEC / 4; ++i) {
            const F2 p = mul2(f[2 * i], by), q = mul2(f[2 * i + 1], by);
            w[i] = e4m3x2(p.x, p.y) | static_cast<uint32_t>(e4m3x2(q.x, q.y)) << 16;
          }
          if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(codes + e0) = make_uint2(w[0], w[VEC / 4 - 1]);
          else *reinterpret_cast<uint32_t *>(codes + e0) = w[0];
          if (e0 % 32 == 0) static_cast<uint8_t *>(a.scales)[t * (n / 32) + e0 / 32] = static_cast<uint8_t>(code);
        }
      }
    }
  } else {
    if constexpr (NORM) {
      // max |r gamma| * inv is max |y| but for the order of two roundings (the quotient of the
      // largest still rounds to 127), unless a product left the normal range
      const bool normal = top >= 0x21800000u && top < 0x7b800000u && inv.x > 0x1p-60f && inv.x < 0x1p+60f;  // 2^-60, 2^120
      if (normal) {
        top = __float_as_uint(__fmul_rn(__uint_as_float(top), inv.x));
      } else {
        top = 0u;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int e0 = first + j * step;
          F2 f[PAIRS];
          scaled(j, f);
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (e0 + i >= 0 && e0 + i < n) top = max(top, __float_as_uint(i & 1 ? f[i / 2].y : f[i / 2].x) & 0x7fffffffu);
        }
        top = block_max(top, red_v);
      }
    } else {
      // rows as they are: the packed halves' magnitudes
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (sizeof(T) == 4) top = max(top, w[i] & 0x7fffffffu);
          else top = __vmaxu2(top, w[i] & 0x7fff7fffu);
        }
      }
      if constexpr (sizeof(T) == 2) top = __float_as_uint(Pack<T>::value(max(top & 0xffffu, top >> 16)).x);
      top = block_max(top, red_u);
    }
    const bool finite = top < 0x7f800000u;
    const float s = int8_scale(top);
    if (threadIdx.x == 0) static_cast<float *>(a.scales)[t] = s;
    const bool tiny = !(s >= kTinyScale);
    const float r = tiny ? 0.0f : __fdiv_rn(1.0f, s);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = first + j * step;
      if (e0 >= n) continue;
      F2 f[PAIRS];
      scaled(j, f);
      if (norm) C::store(norm, e0, n, whole(e0), C::round(f));
      uint32_t q[VEC];
      if (tiny) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) q[i] = finite ? int8_code_tiny(i & 1 ? f[i / 2].y : f[i / 2].x, s) : 0u;
      } else {
        const F2 r2 = {r, r}, s2 = {-s, -s}, magic = {0x1.8p+23f, 0x1.8p+23f};
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {  // int8_code, by pairs
          const F2 d = mul2(f[i], r2);
          const F2 k = add2(fma2(fma2(d, s2, f[i]), r2, d), magic);
          q[2 * i] = __float_as_uint(k.x);
          q[2 * i + 1] = __float_as_uint(k.y);
        }
      }
      uint32_t w[VEC / 4];
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) w[i] = pack4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
      if constexpr (TURN) {
        uint8_t *to = turned + (threadIdx.x + j * blockDim.x) * VEC;
        if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[VEC / 4 - 1]);
        else *reinterpret_cast<uint32_t *>(to) = w[0];
      } else {
        store_codes<VEC>(codes, e0, n, w, a.codes_wide && shift == 0 && e0 + VEC <= n);
      }
    }
    if constexpr (TURN) {
      // code e of the row sits at byte e + shift: 16-byte units of the row, shifted out of two
      if (blockDim.x == 32) __syncwarp();
      else __syncthreads();
      for (int u = threadIdx.x * 16; u < n; u += blockDim.x * 16) {
        const uint4 lo = *reinterpret_cast<const uint4 *>(turned + u), hi = *reinterpret_cast<const uint4 *>(turned + u + 16);
        uint32_t w[6] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y};
        if (shift & 4) {
#pragma unroll
          for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
        }
        const int bits = (shift & 3) * 8;
        const uint32_t c[4] = {__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                               __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits)};
        if (u + 16 <= n) {
          *reinterpret_cast<uint4 *>(codes + u) = make_uint4(c[0], c[1], c[2], c[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (u + i < n) codes[u + i] = static_cast<uint8_t>(c[i / 4] >> (8 * (i % 4)));
        }
      }
    }
  }
}

// One CTA per row, read again from memory in each of the passes: rows too long for registers,
// or (VEC == 1) rows whose buffers do not share an alignment.
template <typename T, int VEC, int QUANT>
__global__ void __launch_bounds__(1024) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ double red_d[32];
  __shared__ uint32_t red_u[32], red_v[32];
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
  float v[VEC];

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
    // a chain of a few terms a thread at a time, then 64 bits: rows of any length
    double sum = 0.0;
    for (int c = threadIdx.x; c < chunks; c += blockDim.x) {
      fetch(c, v);
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) ss = __fmaf_rn(v[i], v[i], ss);
      sum += static_cast<double>(ss);
    }
    uint32_t none = 0u;
    inv = inverse_rms(block_sum(sum, none, red_d, red_u), a.inv_n, a.eps);
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
  {
    for (int j = 0; j < rounds; ++j) {
      const int c = threadIdx.x + j * blockDim.x;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
      if (c < chunks) {
        fetch(c, v);
        if constexpr (QUANT != MM_QUANT_INT8) keep(c, v);
        scale(c, v);
        if (norm) store_chunk<T, VEC>(norm, c * VEC - shift, n, v);
      }
      if constexpr (QUANT == MM_QUANT_MXFP8) mx_block(c, v);
      if constexpr (QUANT == MM_QUANT_INT8) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      }
    }
  }

  if constexpr (QUANT == MM_QUANT_INT8) {
    top = block_max(top, red_v);
    const bool finite = top < 0x7f800000u;
    const float s = int8_scale(top);
    if (threadIdx.x == 0) static_cast<float *>(a.scales)[t] = s;
    const bool tiny = !(s >= kTinyScale);
    const float r = tiny ? 0.0f : __fdiv_rn(1.0f, s);
    {
      for (int j = 0; j < rounds; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        if (c < chunks) {
          fetch(c, v);
          keep(c, v);
          scale(c, v);
          if (!finite) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
          }
          int8_chunk(c, v, finite ? s : 0.0f, r, tiny);
        }
      }
    }
  }
}

// The registers of a thread of a kernel, as it was compiled.
template <auto KERNEL>
int registers() {
  static const int regs = [] {
    cudaFuncAttributes f = {};
    return cudaFuncGetAttributes(&f, KERNEL) == cudaSuccess ? (f.numRegs + 7) / 8 * 8 : 64;
  }();
  return regs;
}
// Rounds that the GPU's 148 SMs need for `tokens` rows of `warps` warps each.
int rounds(int tokens, int warps, int regs) {
  const int rows = 148 * std::max(1, std::min(4 * (512 / regs), 64) / warps);
  return (tokens + rows - 1) / rows;
}

// Chunks a thread. As few as hold all rows in the SMs at once (one row's latency; norm + MXFP8 + residual
// of 256 x 7168: one chunk, two rounds 6.4 us, two chunks, one round 4.6). More rows than that:
// more chunks, so that more loads of more rows are in flight and fewer warps meet at a barrier (bf16,
// us: norm + MXFP8 of 8192 x 7168: two 103, four 83 (6.4 TB/s), eight 101; of 4096 x 16384: four 94, eight 128;
// of 8192 x 2048: two 25.6, four 26.0), rows between by the rounds (norm of 640 x 6147: two 7.3, four
// 8.3; of 1024 x 6147: two 9.9, four 9.0). int8 rows alone hold less beside the row: 4096 x 16384: four
// 42, eight 35; 8192 x 7168: two 41, four 33, eight 30.5.
// The norm's rows of more than 512 chunks: two chunks a thread against four, as two's time over four's in a
// sweep of 450..8192 rows (bf16 of 4608..8192 values, fp32 of 2304..4096). Up to 832 chunks and 2048 rows either
// may win (norm alone 0.82..1.31, with MXFP8 0.77..1.22, with int8 0.74..1.15), and fewer rounds tell which; more
// rows 0.94..1.38, longer rows 0.81..1.64: four. The rule takes the better one or is within 4 % of it at 256 of the 280
// sizes, within 11 % at all of bf16's; what it misses most is fp32 with MXFP8 or without codes from 833 chunks
// on at 450..1536 rows (600 x 4096 with MXFP8: four 9.4 us, two 7.6).
template <typename T, int QUANT, bool NORM, bool TURN>
cudaError_t launch_rows(NormArgs a, int chunks, void *stream) {
  constexpr bool kDense = QUANT == MM_QUANT_NONE && sizeof(T) == 2;
  constexpr auto one = norm_rows_kernel<T, 1, QUANT, NORM, TURN, false>;
  constexpr auto two = norm_rows_kernel<T, 2, QUANT, NORM, TURN, false>;
  constexpr auto four = norm_rows_kernel<T, 4, QUANT, NORM, TURN, false>;
  constexpr auto eight = norm_rows_kernel<T, 8, QUANT, NORM, TURN, false>;
  a.turn_bytes = TURN ? static_cast<int>((chunks * (16 / sizeof(T)) + 32) / 16 * 16 + 16) : 0;
  // Short rows share CTAs, a warp each, from kShareRows rows on (int8 rows of 8192 x 1024: shared 5.4 us,
  // a CTA each 9.2; norm of 8192 x 512: 6.1 and 9.4). Fewer rows lose by it (norm with int8 of 1300 x
  // 1024: shared 6.0, a CTA each 4.4).
  const int share = chunks > 128 || a.tokens < kShareRows ? 1 : a.tokens < 2 * kShareRows ? 4 : 8;
  const bool dense = kDense && share == 1 && chunks <= 4 * row_threads(4, NORM, true);
  auto warps = [&](int n) { return (chunks + 32 * n - 1) / (32 * n); };
  auto in_one_round = [&](int n, int regs) { return chunks <= n * row_threads(n, NORM) && rounds(a.tokens, warps(n), regs) == 1; };
  int nv;
  int regs4 = registers<four>();
  if constexpr (kDense)
    if (dense) regs4 = registers<norm_rows_kernel<T, 4, QUANT, NORM, TURN, true>>();
  if (share > 1) nv = chunks <= 32 ? 1 : chunks <= 64 ? 2 : 4;
  else if (in_one_round(1, registers<one>())) nv = 1;
  else if (in_one_round(2, registers<two>())) nv = 2;
  else if (chunks > 4 * row_threads(4, NORM)) nv = 8;
  else if ((chunks > 512 || QUANT == MM_QUANT_NONE) && in_one_round(4, regs4)) nv = 4;
  else if (!NORM) nv = chunks <= 256 ? 2 : chunks <= 512 ? 4 : 8;
  else if (chunks <= 512) nv = 2;
  else if (chunks <= 832 && a.tokens <= 2048) nv = rounds(a.tokens, warps(4), regs4) < rounds(a.tokens, warps(2), registers<two>()) ? 4 : 2;
  else nv = 4;
  auto go = [&](auto kernel, int n) {
    const dim3 block = share > 1 ? dim3(32, share) : dim3(((chunks + n - 1) / n + 31) / 32 * 32);
    return launch(kernel, dim3((a.tokens + share - 1) / share), block, share * a.turn_bytes, stream, a);
  };
  if constexpr (kDense)
    if (nv == 4 && dense) return go(norm_rows_kernel<T, 4, QUANT, NORM, TURN, true>, 4);
  return nv == 1 ? go(one, 1) : nv == 2 ? go(two, 2) : nv == 4 ? go(four, 4) : go(eight, 8);
}

template <typename T, int QUANT>
cudaError_t launch_norm(const NormArgs &a, bool wide, void *stream) {
  constexpr int VEC = 16 / sizeof(T);
  const unsigned rows = static_cast<unsigned>(a.tokens);
  if (!wide)
    return launch(norm_kernel<T, 1, QUANT>, dim3(rows), dim3(std::min(1024, (a.hidden + 31) / 32 * 32)), 0, stream, a);
  // one chunk more than the row fills where rows start inside a 16-byte unit
  const bool shifted = (reinterpret_cast<uintptr_t>(a.x) % 16) || (a.ld_x * static_cast<int64_t>(sizeof(T))) % 16;
  const int chunks = (a.hidden + VEC - 1) / VEC + (shifted ? 1 : 0);
  if (chunks > 8 * row_threads(8, a.gamma != nullptr)) return launch(norm_kernel<T, VEC, QUANT>, dim3(rows), dim3(1024), 0, stream, a);
  if constexpr (QUANT == MM_QUANT_INT8) {
    if (!a.gamma)
      return a.code_row ? launch_rows<T, QUANT, false, true>(a, chunks, stream) : launch_rows<T, QUANT, false, false>(a, chunks, stream);
    if (a.code_row) return launch_rows<T, QUANT, true, true>(a, chunks, stream);
  }
  return launch_rows<T, QUANT, true, false>(a, chunks, stream);
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

// Checks the sizes and picks the kernel's form: 16-byte chunks where x, the residual and the
// outputs of x's type put each row at the same offset from a 16-byte boundary (MXFP8: at a
// boundary, so that blocks and chunks agree), elements otherwise.
int run_norm(const char *what, NormArgs a, int dtype, int quant, void *stream) {
  if (a.tokens < 0 || a.hidden < 1) return set_error(MM_ERR_INVALID, "%s: %d tokens of %d values", what, a.tokens, a.hidden);
  if (dtype != MM_DTYPE_BF16 && dtype != MM_DTYPE_FP16 && dtype != MM_DTYPE_FP32)
    return set_error(MM_ERR_INVALID, "%s: unknown type %d", what, dtype);
  if (quant != MM_QUANT_NONE && quant != MM_QUANT_MXFP8 && quant != MM_QUANT_INT8)
    return set_error(MM_ERR_INVALID, "%s: unknown 8-bit format %d", what, quant);
  if (a.tokens > 1 << 30 || a.hidden > 1 << 30)
    return set_error(MM_ERR_UNSUPPORTED, "%s: %d tokens of %d values: at most 2^30 of each", what, a.tokens, a.hidden);
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
  // x's or the residual's own place, row for row; no other buffers may share memory with an output
  auto rows = [&](const void *p, int64_t ld, int size) { return row_bytes(p, a.tokens, a.hidden, ld, size); };
  const Bytes in[] = {rows(a.x, a.ld_x, es), rows(a.residual, a.ld_residual, es),
                      flat_bytes(a.gamma, static_cast<int64_t>(a.hidden) * (a.gamma_f32 ? 4 : es))};
  const int64_t scale_bytes = quant == MM_QUANT_MXFP8 ? static_cast<int64_t>(a.tokens) * (a.hidden / 32) : static_cast<int64_t>(a.tokens) * 4;
  const Bytes out[] = {rows(a.residual_out, a.ld_residual_out, es), rows(a.norm_out, a.ld_norm, es),
                       rows(quant ? a.codes : nullptr, a.ld_codes, 1), flat_bytes(quant ? a.scales : nullptr, scale_bytes)};
  auto in_place = [&](const Bytes &o, const Bytes &i) {
    return &o == out && o.p == i.p && ((&i == in && a.ld_x == a.ld_residual_out) || (&i == in + 1 && a.ld_residual == a.ld_residual_out));
  };
  for (const Bytes &o : out) {
    for (const Bytes &i : in)
      if (overlap(o, i) && !in_place(o, i)) return set_error(MM_ERR_INVALID, "%s: an output overlaps an input", what);
    for (const Bytes &other : out)
      if (&other < &o && overlap(o, other)) return set_error(MM_ERR_INVALID, "%s: an output overlaps another", what);
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
  a.code_row = quant == MM_QUANT_INT8 && shifted && reinterpret_cast<uintptr_t>(a.codes) % 16 == 0 && a.ld_codes % 16 == 0;
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
  a.gamma_f32 = n->gamma_dtype == MM_DTYPE_FP32 && n->dtype != MM_DTYPE_FP32;
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
  a.inv_n = n->hidden > 0 ? 1.0 / n->hidden : 0.0;
  return run_norm("mm_rms_norm", a, n->dtype, n->quant, stream);
}

int mm_quantize_int8(const void *x, int64_t ld_x, int32_t dtype, int8_t *codes, int64_t ld_codes, float *scales,
                     int32_t tokens, int32_t hidden, void *stream) {
  return quantize_rows("mm_quantize_int8", x, ld_x, dtype, codes, ld_codes, scales, tokens, hidden, stream);
}

}  // extern "C"
