// Block formats with one power-of-two scale per 32 values: MXINT8 for activation checkpoints,
// MXFP4 for products.  Quantisation (nearest, and stochastic for MXFP4), its transposed form, the
// way back, and the gated activation that keeps its inputs in MXINT8, with its backward pass.
//
// All of it is bound by memory: each value is read once and written once, 32 values share one
// reduction of four lanes.  A thread handles UNITS of eight consecutive values of a row (16 bytes
// of bf16 per access); the units of a matrix are numbered row by row over rows padded to whole
// blocks, so the four lanes of a block are always neighbours in a warp, whatever the row length.
// Rows that do not start on 16-byte boundaries go through a warp's slice of shared memory, so
// that global accesses stay consecutive; the arithmetic after it is the same.
#include <algorithm>

#include "mx_common.cuh"
#include "philox.cuh"

namespace rt {

constexpr int kMxThreads = 256;
constexpr int kMxWarps = kMxThreads / 32;
constexpr uint32_t kStreamFp4 = 3;  // Philox counter word 3 of the 4-bit rounding

struct Matrix {            // rows x cols, row stride ld elements
  const void* p;
  int64_t ld;
};
struct Grid {              // how the units of a matrix are numbered
  FastDiv upr;             // units per row
  uint32_t units;
  int cols;
  uint32_t rows;
};

// ---------------------------------------------------------------------------------------- units
// Unit -> eight fp32 values; columns beyond the last are 0.  `stage`: 256 floats of this warp.
template <int D, bool VEC>
__device__ __forceinline__ void load_staged(const Matrix& m, const Grid& g, uint32_t warp_unit, int lane, float* stage, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = warp_unit + 4 * j + (lane >> 3);
    float v = 0.f;
    if (u < g.units) {
      uint32_t r, c;
      g.upr.split(u, r, c);
      c = c * 8 + (lane & 7);
      if ((int)c < g.cols) v = to_f32<D>(static_cast<const elem_t<D>*>(m.p)[(int64_t)r * m.ld + c]);
    }
    stage[j * 32 + lane] = v;
  }
  __syncwarp();
  const float4 a = reinterpret_cast<const float4*>(stage)[lane * 2], b = reinterpret_cast<const float4*>(stage)[lane * 2 + 1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  __syncwarp();
}
template <int D>
__device__ __forceinline__ void store_staged(const Matrix& m, const Grid& g, uint32_t warp_unit, int lane, float* stage, const float (&x)[8]) {
  reinterpret_cast<float4*>(stage)[lane * 2] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(stage)[lane * 2 + 1] = make_float4(x[4], x[5], x[6], x[7]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = warp_unit + 4 * j + (lane >> 3);
    if (u < g.units) {
      uint32_t r, c;
      g.upr.split(u, r, c);
      c = c * 8 + (lane & 7);
      if ((int)c < g.cols) static_cast<elem_t<D>*>(const_cast<void*>(m.p))[(int64_t)r * m.ld + c] = of_f32<D>(stage[j * 32 + lane]);
    }
  }
  __syncwarp();
}
// VEC: rows start on 16-byte boundaries; only a row's last unit may be cut
template <int D>
__device__ __forceinline__ Raw8<D> load_unit(const Matrix& m, const Grid& g, uint32_t r, uint32_t c8, bool live) {
  Raw8<D> raw{};
  const int c = (int)c8 * 8;
  if (live && c + 8 <= g.cols) raw = load_raw<D>(m.p, (int64_t)r * m.ld + c);
  else if (live && c < g.cols) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = c + k < g.cols ? to_f32<D>(static_cast<const elem_t<D>*>(m.p)[(int64_t)r * m.ld + c + k]) : 0.f;
    raw = pack<D>(x);   // exact: the values are of this type
  }
  return raw;
}
template <int D>
__device__ __forceinline__ void store_unit(const Matrix& m, const Grid& g, uint32_t r, uint32_t c8, const float (&x)[8]) {
  const int c = (int)c8 * 8;
  void* p = const_cast<void*>(m.p);
  if (c + 8 <= g.cols) store_raw<D>(p, (int64_t)r * m.ld + c, pack<D>(x));
  else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < g.cols) static_cast<elem_t<D>*>(p)[(int64_t)r * m.ld + c + k] = of_f32<D>(x[k]);
  }
}

// -------------------------------------------------------------------------------------- formats
// The largest magnitude of a block as a bit pattern: integer order is the order of magnitudes, with
// infinities and NaNs on top, so one maximum also finds the blocks that hold any.
__device__ __forceinline__ uint32_t amax8(const float (&x)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) a = max(a, __float_as_uint(x[k]) & 0x7FFFFFFFu);
  return a;
}
__device__ __forceinline__ uint32_t amax_of_four(uint32_t a) {
  a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
  return max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 2));
}

// Eight MXINT8 codes.  x * 2^(6-e) is exact; adding 1.5 * 2^23 rounds it to an integer, ties to
// even, and leaves that integer's two's complement in the low bits.
__device__ __forceinline__ uint2 codes_int8(const float (&x)[8], uint32_t amax, uint32_t& byte) {
  const bool bad = amax >= 0x7F800000u;
  const int e = exponent_int8(amax);
  byte = bad ? 255u : (uint32_t)(e + 127);
  const float s = pow2f(6 - e);
  uint32_t q[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) q[k] = __float_as_uint(fminf(fmaxf(x[k] * s, -127.f), 127.f) + 12582912.f);
  uint2 w;
  w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return bad ? make_uint2(0u, 0u) : w;
}

// two values, the second in the low half of the byte; nearest, ties to even
__device__ __forceinline__ uint32_t cvt_e2m1x2(float high, float low) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(high), "f"(low));
  return r;
}
// Stochastic rounding to the grid: floor(|y|/s + r/65536) * s with s the grid's step at |y| (0.5
// below 2, 1 below 4, else 2).  From 1 upwards that is an integer addition to the bit pattern, one
// mantissa bit kept; below 1 the same holds for |y| + 1, whose step is 0.5 too (added towards zero:
// what is cut off lies below the last place that the comparison with r can see).
__device__ __forceinline__ float sr_e2m1(float y, uint32_t r16) {
  const uint32_t sign = __float_as_uint(y) & 0x80000000u;
  const float a = fabsf(y);
  const float one = a < 1.f ? 1.f : 0.f;
  const float b = __fadd_rz(a, one);
  const float v = __uint_as_float((__float_as_uint(b) + (r16 << 6)) & 0xFFC00000u) - one;
  return __uint_as_float(__float_as_uint(v) | sign);
}
// Eight MXFP4 codes, the even value in the low half of a byte.
template <bool SR>
__device__ __forceinline__ uint32_t codes_fp4(const float (&x)[8], uint32_t amax, uint32_t& byte, const PhiloxKeys& keys,
                                              uint32_t tensor_id, uint32_t step, uint32_t unit) {
  const bool bad = amax >= 0x7F800000u;
  const int e = exponent_fp4(amax);
  byte = bad ? 255u : (uint32_t)(e + 127);
  const float s = pow2f(-e);
  float y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = x[k] * s;
  if (e == 126) {                     // 4 * 2^126 is no fp32 number: what is finite stays finite
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = fminf(fmaxf(y[k], -3.f), 3.f);
  }
  if constexpr (SR) {
    const uint4 d = draws8(keys, tensor_id, step, kStreamFp4, unit);
    const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = sr_e2m1(y[k], k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xFFFFu);
  }
  uint32_t c = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) c |= cvt_e2m1x2(y[2 * k + 1], y[2 * k]) << (8 * k);
  return bad ? 0u : c;
}
// Eight values of MXINT8 codes.  The byte with its sign turned over, set into the mantissa of 2^23, is 2^23 + 128 + code.
__device__ __forceinline__ void values_int8(uint2 w, float s, float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t u = (k < 4 ? w.x : w.y) ^ 0x80808080u;
    x[k] = (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 | (k & 3))) - 8388736.f) * s;
  }
}
// Eight values of MXFP4 codes: exponent and mantissa bits of a code, moved to bit 22, times 2^126.
__device__ __forceinline__ void values_fp4(uint32_t w, float s, float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t c = w >> (4 * k);
    const float v = __uint_as_float((c & 7u) << 22) * 0x1p126f * s;
    x[k] = __uint_as_float(__float_as_uint(v) | ((c & 8u) << 28));
  }
}

__device__ __forceinline__ void put_int8(uint8_t* codes, uint8_t* scales, const Grid& g, uint32_t r, uint32_t c8, uint2 w, uint32_t byte) {
  *reinterpret_cast<uint2*>(codes + ((int64_t)r * g.upr.d + c8) * 8) = w;
  if ((c8 & 3) == 0) {
    const int nb = g.upr.d >> 2, stride = (nb + 3) & ~3, b = c8 >> 2;
    uint8_t* row = scales + (int64_t)r * stride;
    row[b] = (uint8_t)byte;
    if (b == nb - 1)
      for (int k = nb; k < stride; ++k) row[k] = 0;
  }
}
__device__ __forceinline__ void put_fp4_scale(uint8_t* scales, int nb, int64_t r, int b, uint32_t byte) {
  const int ktiles = (nb + 3) >> 2;
  scales[fp4_scale_at(r, b, ktiles)] = (uint8_t)byte;
  if (b == nb - 1)
    for (int k = nb; k < 4 * ktiles; ++k) scales[fp4_scale_at(r, k, ktiles)] = 0;
}
// the scale bytes of the rows that fill the last tile of 128
__device__ __forceinline__ void clear_fp4_pad(uint8_t* scales, uint32_t rows, int nb, uint32_t tid, uint32_t threads) {
  const int ktiles = (nb + 3) >> 2;
  const uint32_t pad = ((rows + 127) & ~127u) - rows;
  for (uint32_t w = tid; w < pad * ktiles; w += threads)
    *reinterpret_cast<uint32_t*>(scales + fp4_scale_at(rows + w / ktiles, (w % ktiles) * 4, ktiles)) = 0u;
}

struct SrArgs {
  PhiloxKeys keys;
  uint32_t tensor_id, step;
};

// ------------------------------------------------------------------------------------- quantise
// FMT 0: MXINT8, 1: MXFP4.  A CTA takes kUnits units per thread and loads them all before the
// first is used.
constexpr int kUnits = 4;

template <int D, int FMT, bool SR, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize_kernel(const Matrix x, const Grid g, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const SrArgs sr) {
  __shared__ float stage[VEC ? 1 : kMxWarps * 256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t first = blockIdx.x * (kMxThreads * kUnits) + threadIdx.x;
  Raw8<D> raw[VEC ? kUnits : 1];
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const uint32_t u = first + k * kMxThreads;
      uint32_t r, c;
      g.upr.split(u, r, c);
      raw[k] = load_unit<D>(x, g, r, c, u < g.units);
    }
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const uint32_t u = first + k * kMxThreads;
    float v[8];
    if constexpr (VEC) unpack<D>(raw[k], v);
    else load_staged<D, VEC>(x, g, u - lane, lane, stage + warp * 256, v);
    const uint32_t amax = amax_of_four(amax8(v));
    uint32_t r, c, byte;
    g.upr.split(u, r, c);
    if constexpr (FMT == RT_MXINT8) {
      const uint2 w = codes_int8(v, amax, byte);
      if (u < g.units) put_int8(codes, scales, g, r, c, w, byte);
    } else {
      const uint32_t w = codes_fp4<SR>(v, amax, byte, sr.keys, sr.tensor_id, sr.step, u);
      if (u < g.units) {
        reinterpret_cast<uint32_t*>(codes)[u] = w;
        if ((c & 3) == 0) put_fp4_scale(scales, g.upr.d >> 2, r, c >> 2, byte);
      }
    }
  }
  if constexpr (FMT == RT_MXFP4)
    clear_fp4_pad(scales, g.rows, g.upr.d >> 2, blockIdx.x * kMxThreads + threadIdx.x, gridDim.x * kMxThreads);
}

// ------------------------------------------------------------------------- quantise, transposed
// Output row c holds column c of x, in blocks along x's rows.  A CTA takes 128 rows x 64 columns
// through shared memory; thread (column, quarter) then owns one block of 32 rows, so that the
// block's maximum needs no exchange.
constexpr int kTRows = 128, kTCols = 64;

template <int D, bool SR, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize_t_kernel(const Matrix x, const int64_t rows, const int cols, const uint32_t col_tiles, uint8_t* __restrict__ codes,
                     uint8_t* __restrict__ scales, const SrArgs sr) {
  using T = elem_t<D>;
  __shared__ __align__(16) T tile[kTRows][kTCols];
  const uint32_t ct = blockIdx.x % col_tiles;
  const int64_t row0 = (int64_t)(blockIdx.x / col_tiles) * kTRows;
  const int col0 = ct * kTCols;
  if constexpr (VEC) {
    constexpr int kPer = 16 / sizeof(T), kChunks = kTCols / kPer;      // 16-byte chunks of a row
#pragma unroll
    for (int i = threadIdx.x; i < kTRows * kChunks; i += kMxThreads) {
      const int r = i / kChunks, c = (i % kChunks) * kPer;
      const T* src = static_cast<const T*>(x.p) + (row0 + r) * x.ld + col0 + c;
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (row0 + r < rows) {
        if (col0 + c + kPer <= cols) w = __ldg(reinterpret_cast<const uint4*>(src));
        else {
          T* e = reinterpret_cast<T*>(&w);
#pragma unroll
          for (int k = 0; k < kPer; ++k)
            if (col0 + c + k < cols) e[k] = src[k];
        }
      }
      *reinterpret_cast<uint4*>(&tile[r][c]) = w;
    }
  } else {
    for (int i = threadIdx.x; i < kTRows * kTCols; i += kMxThreads) {
      const int r = i / kTCols, c = i % kTCols;
      tile[r][c] = row0 + r < rows && col0 + c < cols ? static_cast<const T*>(x.p)[(row0 + r) * x.ld + col0 + c] : (T)0;
    }
  }
  __syncthreads();
  const int c = threadIdx.x & (kTCols - 1), quarter = threadIdx.x / kTCols;
  const int nb = (int)((rows + 31) >> 5), b = (int)(row0 >> 5) + quarter;
  const int out = col0 + c;
  float v[4][8];
  uint32_t amax = 0;
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k >> 3][k & 7] = to_f32<D>(tile[quarter * 32 + k][c]);
#pragma unroll
  for (int k = 0; k < 4; ++k) amax = max(amax, amax8(v[k]));
  if (out < cols && b < nb) {
    const uint32_t unit = (uint32_t)out * (nb * 4) + b * 4;
    uint32_t byte, w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = codes_fp4<SR>(v[k], amax, byte, sr.keys, sr.tensor_id, sr.step, unit + k);
    reinterpret_cast<uint4*>(codes)[(int64_t)out * nb + b] = make_uint4(w[0], w[1], w[2], w[3]);
    put_fp4_scale(scales, nb, out, b, byte);
  }
  clear_fp4_pad(scales, cols, nb, blockIdx.x * kMxThreads + threadIdx.x, gridDim.x * kMxThreads);
}

// ----------------------------------------------------------------------------------- the way back
template <int D, int FMT, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const Grid g, const Matrix out) {
  __shared__ float stage[VEC ? 1 : kMxWarps * 256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t first = blockIdx.x * (kMxThreads * kUnits) + threadIdx.x;
  const int nb = g.upr.d >> 2;
  uint2 w[kUnits];
  uint32_t byte[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const uint32_t u = first + k * kMxThreads;
    uint32_t r, c;
    g.upr.split(u, r, c);
    w[k] = make_uint2(0u, 0u);
    byte[k] = 127;
    if (u < g.units) {
      if constexpr (FMT == RT_MXINT8) {
        w[k] = __ldg(reinterpret_cast<const uint2*>(codes) + u);
        byte[k] = __ldg(scales + (int64_t)r * ((nb + 3) & ~3) + (c >> 2));
      } else {
        w[k].x = __ldg(reinterpret_cast<const uint32_t*>(codes) + u);
        byte[k] = __ldg(scales + fp4_scale_at(r, c >> 2, (nb + 3) >> 2));
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const uint32_t u = first + k * kMxThreads;
    float x[8];
    if constexpr (FMT == RT_MXINT8) values_int8(w[k], scale_of(byte[k], 6), x);
    else values_fp4(w[k].x, scale_of(byte[k], 0), x);
    if constexpr (D == RT_F16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fabsf(x[j]) > 65504.f ? copysignf(65504.f, x[j]) : x[j];   // NaN stays
    }
    if constexpr (VEC) {
      uint32_t r, c;
      g.upr.split(u, r, c);
      if (u < g.units) store_unit<D>(out, g, r, c, x);
    } else {
      store_staged<D>(out, g, u - lane, lane, stage + warp * 256, x);
    }
  }
}

// ------------------------------------------------------------------------------ gated activation
// act(g) and act'(g).  For 16-bit results the exponential and the reciprocal are the hardware's
// approximations (relative error about 2^-21 each, far below the 2^-9 of the result's rounding);
// for fp32 results they are CUDA's functions.
template <bool EXACT>
__device__ __forceinline__ float exp_of(float x) { return EXACT ? expf(x) : __expf(x); }
template <bool EXACT>
__device__ __forceinline__ float sigmoid_of(float x) {
  const float d = 1.f + exp_of<EXACT>(-x);
  return EXACT ? 1.f / d : __fdividef(1.f, d);   // 2^126 < d < inf would make the quick division 0, and so it should
}
template <int ACT, bool EXACT>
__device__ __forceinline__ void act_of(float g, float& a, float& d) {
  if constexpr (ACT == RT_ACT_SILU) {
    const float s = sigmoid_of<EXACT>(g);
    a = g * s;
    d = s * (1.f + g * (1.f - s));
  } else if constexpr (ACT == RT_ACT_GELU) {
    const float p = 0.5f * erfcf(-0.70710678f * g);      // no cancellation for negative g
    a = g * p;
    d = p + 0.39894228f * g * exp_of<EXACT>(-0.5f * g * g);
  } else {
    // beyond |g| = 16 the sigmoid is 0 or 1 and its slope 0; the cube must not reach infinity there (NaN passes)
    const float c = g > 16.f ? 16.f : g < -16.f ? -16.f : g, q = c * c;
    const float s = sigmoid_of<EXACT>(1.59576912f * c * (1.f + 0.044715f * q));
    a = g * s;
    d = s + c * s * (1.f - s) * 1.59576912f * (1.f + 0.134145f * q);
  }
}

struct Kept {              // an MXINT8 matrix
  uint8_t* codes;
  uint8_t* scales;
};

template <int D, int ACT, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_gated_kernel(const Matrix gate, const Matrix up, const Grid g, const Matrix h, const Kept kg, const Kept ku) {
  __shared__ float stage_all[VEC ? 1 : kMxWarps * 256];
  float* stage = stage_all + (VEC ? 0 : (threadIdx.x >> 5) * 256);
  const int lane = threadIdx.x & 31;
  constexpr int kPer = 2;
  const uint32_t first = blockIdx.x * (kMxThreads * kPer) + threadIdx.x;
  Raw8<D> ra[VEC ? kPer : 1], rb[VEC ? kPer : 1];
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const uint32_t u = first + k * kMxThreads;
      uint32_t r, c;
      g.upr.split(u, r, c);
      ra[k] = load_unit<D>(gate, g, r, c, u < g.units);
      rb[k] = load_unit<D>(up, g, r, c, u < g.units);
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const uint32_t u = first + k * kMxThreads;
    float a[8], b[8], y[8];
    if constexpr (VEC) { unpack<D>(ra[k], a); unpack<D>(rb[k], b); }
    else {
      load_staged<D, VEC>(gate, g, u - lane, lane, stage, a);
      load_staged<D, VEC>(up, g, u - lane, lane, stage, b);
    }
    const uint32_t ma = amax_of_four(amax8(a)), mb = amax_of_four(amax8(b));
    uint32_t r, c, byte;
    g.upr.split(u, r, c);
    const uint2 wa = codes_int8(a, ma, byte);
    if (u < g.units) put_int8(kg.codes, kg.scales, g, r, c, wa, byte);
    const uint2 wb = codes_int8(b, mb, byte);
    if (u < g.units) put_int8(ku.codes, ku.scales, g, r, c, wb, byte);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f, d;
      act_of<ACT, D == RT_F32>(a[j], f, d);
      y[j] = f * b[j];
    }
    if constexpr (VEC) { if (u < g.units) store_unit<D>(h, g, r, c, y); }
    else store_staged<D>(h, g, u - lane, lane, stage, y);
  }
}

template <int D, int ACT, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_gated_backward_kernel(const Matrix grad, const Kept kg, const Kept ku, const Grid g, const Matrix dgate, const Matrix dup) {
  __shared__ float stage_all[VEC ? 1 : kMxWarps * 256];
  float* stage = stage_all + (VEC ? 0 : (threadIdx.x >> 5) * 256);
  const int lane = threadIdx.x & 31;
  constexpr int kPer = 2;
  const uint32_t first = blockIdx.x * (kMxThreads * kPer) + threadIdx.x;
  const int stride = ((g.upr.d >> 2) + 3) & ~3;
  Raw8<D> raw[VEC ? kPer : 1];
  uint2 wg[kPer], wu[kPer];
  uint32_t bg[kPer], bu[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const uint32_t u = first + k * kMxThreads;
    uint32_t r, c;
    g.upr.split(u, r, c);
    wg[k] = wu[k] = make_uint2(0u, 0u);
    bg[k] = bu[k] = 127u;
    if (u < g.units) {
      wg[k] = __ldg(reinterpret_cast<const uint2*>(kg.codes) + u);
      wu[k] = __ldg(reinterpret_cast<const uint2*>(ku.codes) + u);
      bg[k] = __ldg(kg.scales + (int64_t)r * stride + (c >> 2));
      bu[k] = __ldg(ku.scales + (int64_t)r * stride + (c >> 2));
    }
    if constexpr (VEC) raw[k] = load_unit<D>(grad, g, r, c, u < g.units);
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const uint32_t u = first + k * kMxThreads;
    float dh[8], a[8], b[8];
    if constexpr (VEC) unpack<D>(raw[k], dh);
    else load_staged<D, VEC>(grad, g, u - lane, lane, stage, dh);
    values_int8(wg[k], scale_of(bg[k], 6), a);
    values_int8(wu[k], scale_of(bu[k], 6), b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f, d;
      act_of<ACT, D == RT_F32>(a[j], f, d);
      b[j] = dh[j] * b[j] * d;
      a[j] = dh[j] * f;
    }
    if constexpr (VEC) {
      uint32_t r, c;
      g.upr.split(u, r, c);
      if (u < g.units) {
        store_unit<D>(dgate, g, r, c, b);
        store_unit<D>(dup, g, r, c, a);
      }
    } else {
      store_staged<D>(dgate, g, u - lane, lane, stage, b);
      store_staged<D>(dup, g, u - lane, lane, stage, a);
    }
  }
}

// ------------------------------------------------------------------------------------- the C ABI
static const char* kDtypeText = "dtype code must be 0 (bf16), 1 (f32) or 2 (f16)";

// rows x cols elements with whole blocks per row; at most 2^31 units of eight in one call
int mx_check_shape(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || rows > 0x7FFFFFFFll || cols > 0x7FFFFF00ll)
    return fail(RT_E_SIZE, "rows and cols must be >= 0 and below 2^31 - 256");
  if (cols > 0 && rows > ((int64_t)1 << 31) / (pad_to(cols, kMxBlock) / 8) - 1)
    return fail(RT_E_SIZE, "rows * cols, rows padded to whole blocks of 32, must stay below 2^34");
  return 0;
}
int mx_check_codes(const void* codes, const void* scales) {
  if (!codes || !scales) return fail(RT_E_NULL, "codes and scales must be non-null");
  if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 15)) return fail(RT_E_ALIGN, "codes and scales must be 16-byte aligned");
  return 0;
}
static int check_matrix(const void* p, int dtype, int64_t cols, int64_t ld, const char* name) {
  if (!p) return fail(RT_E_NULL, std::string(name) + " must be non-null");
  if (!dtype_ok(dtype)) return fail(RT_E_DTYPE, kDtypeText);
  if (ld < cols || ld > ((int64_t)1 << 40)) return fail(RT_E_SIZE, std::string("row stride of ") + name + " must be >= cols and at most 2^40");
  if ((uintptr_t)p % dtype_size(dtype)) return fail(RT_E_ALIGN, std::string(name) + " is not aligned to its element size");
  return 0;
}
static Grid grid_of(int64_t rows, int64_t cols) {
  const uint32_t upr = (uint32_t)(pad_to(cols, kMxBlock) / 8);
  return {FastDiv::of(upr), (uint32_t)(rows * upr), (int)cols, (uint32_t)rows};
}
static unsigned blocks_for(uint32_t units, int per) { return (units + (uint32_t)per - 1) / (uint32_t)per; }
static int launched() {
  stats().kernel_launches.fetch_add(1, std::memory_order_relaxed);
  RT_CUDA(cudaGetLastError());
  return 0;
}

template <int D>
static void run_quantize(int fmt, bool transpose, bool sr, bool vec, const Matrix& x, int64_t rows, int64_t cols, uint8_t* codes,
                         uint8_t* scales, const SrArgs& args, cudaStream_t st) {
  if (transpose) {
    const uint32_t ct = (uint32_t)((cols + kTCols - 1) / kTCols);
    const unsigned nb = (unsigned)(ct * ((rows + kTRows - 1) / kTRows));
    auto k = sr ? (vec ? mx_quantize_t_kernel<D, true, true> : mx_quantize_t_kernel<D, true, false>)
                : (vec ? mx_quantize_t_kernel<D, false, true> : mx_quantize_t_kernel<D, false, false>);
    k<<<nb, kMxThreads, 0, st>>>(x, rows, (int)cols, ct, codes, scales, args);
    return;
  }
  const Grid g = grid_of(rows, cols);
  auto k = fmt == RT_MXINT8 ? (vec ? mx_quantize_kernel<D, RT_MXINT8, false, true> : mx_quantize_kernel<D, RT_MXINT8, false, false>)
           : sr             ? (vec ? mx_quantize_kernel<D, RT_MXFP4, true, true> : mx_quantize_kernel<D, RT_MXFP4, true, false>)
                            : (vec ? mx_quantize_kernel<D, RT_MXFP4, false, true> : mx_quantize_kernel<D, RT_MXFP4, false, false>);
  k<<<blocks_for(g.units, kMxThreads * kUnits), kMxThreads, 0, st>>>(x, g, codes, scales, args);
}

template <int D>
static void run_dequantize(int fmt, bool vec, const uint8_t* codes, const uint8_t* scales, const Grid& g, const Matrix& out, cudaStream_t st) {
  auto k = fmt == RT_MXINT8 ? (vec ? mx_dequantize_kernel<D, RT_MXINT8, true> : mx_dequantize_kernel<D, RT_MXINT8, false>)
                            : (vec ? mx_dequantize_kernel<D, RT_MXFP4, true> : mx_dequantize_kernel<D, RT_MXFP4, false>);
  k<<<blocks_for(g.units, kMxThreads * kUnits), kMxThreads, 0, st>>>(codes, scales, g, out);
}

template <int D, int ACT>
static void run_gated(bool vec, const Matrix& gate, const Matrix& up, const Grid& g, const Matrix& h, const Kept& kg, const Kept& ku, cudaStream_t st) {
  auto k = vec ? mx_gated_kernel<D, ACT, true> : mx_gated_kernel<D, ACT, false>;
  k<<<blocks_for(g.units, kMxThreads * 2), kMxThreads, 0, st>>>(gate, up, g, h, kg, ku);
}
template <int D, int ACT>
static void run_gated_backward(bool vec, const Matrix& grad, const Kept& kg, const Kept& ku, const Grid& g, const Matrix& dg, const Matrix& du, cudaStream_t st) {
  auto k = vec ? mx_gated_backward_kernel<D, ACT, true> : mx_gated_backward_kernel<D, ACT, false>;
  k<<<blocks_for(g.units, kMxThreads * 2), kMxThreads, 0, st>>>(grad, kg, ku, g, dg, du);
}

#define RT_BY_DTYPE(dtype, CALL)            \
  do {                                      \
    if ((dtype) == RT_BF16) { CALL(RT_BF16); } \
    else if ((dtype) == RT_F32) { CALL(RT_F32); } \
    else { CALL(RT_F16); }                  \
  } while (0)

}  // namespace rt

using namespace rt;

extern "C" int64_t rt_mx_codes_bytes(int format, int64_t rows, int64_t cols) {
  if (format != RT_MXINT8 && format != RT_MXFP4) return fail(RT_E_CONFIG, "format must be 0 (MXINT8) or 1 (MXFP4)");
  if (int rc = mx_check_shape(rows, cols)) return rc;
  return rows * pad_to(cols, kMxBlock) / (format == RT_MXFP4 ? 2 : 1);
}

extern "C" int64_t rt_mx_scales_bytes(int format, int64_t rows, int64_t cols) {
  if (format != RT_MXINT8 && format != RT_MXFP4) return fail(RT_E_CONFIG, "format must be 0 (MXINT8) or 1 (MXFP4)");
  if (int rc = mx_check_shape(rows, cols)) return rc;
  const int64_t blocks = pad_to(pad_to(cols, kMxBlock) / kMxBlock, 4);
  return (format == RT_MXFP4 ? pad_to(rows, 128) : rows) * blocks;
}

extern "C" int rt_mx_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld, int format, int transpose,
                              void* codes, void* scales, const rt_mx_draws* draws, void* cuda_stream) {
  if (format != RT_MXINT8 && format != RT_MXFP4) return fail(RT_E_CONFIG, "format must be 0 (MXINT8) or 1 (MXFP4)");
  if (format == RT_MXINT8 && (transpose || draws)) return fail(RT_E_CONFIG, "MXINT8 is quantised along rows and to nearest only");
  if (int rc = mx_check_shape(rows, cols)) return rc;
  if (transpose)
    if (int rc = mx_check_shape(cols, rows)) return rc;
  if (rows == 0 || cols == 0) return 0;
  if (int rc = check_matrix(x, x_dtype, cols, ld, "x")) return rc;
  if (int rc = mx_check_codes(codes, scales)) return rc;
  SrArgs sr{};
  if (draws) {
    sr.keys = philox_keys(draws->seed);
    sr.tensor_id = draws->tensor_id;
    sr.step = draws->step;
  }
  const Matrix m{x, ld};
  const bool vec = aligned16(x, ld, dtype_size(x_dtype));
#define CALL(D) run_quantize<D>(format, transpose != 0, draws != nullptr, vec, m, rows, cols, (uint8_t*)codes, (uint8_t*)scales, sr, (cudaStream_t)cuda_stream)
  RT_BY_DTYPE(x_dtype, CALL);
#undef CALL
  return launched();
}

extern "C" int rt_mx_dequantize(int format, const void* codes, const void* scales, int64_t rows, int64_t cols, void* out,
                                int out_dtype, int64_t ld, void* cuda_stream) {
  if (format != RT_MXINT8 && format != RT_MXFP4) return fail(RT_E_CONFIG, "format must be 0 (MXINT8) or 1 (MXFP4)");
  if (int rc = mx_check_shape(rows, cols)) return rc;
  if (rows == 0 || cols == 0) return 0;
  if (int rc = check_matrix(out, out_dtype, cols, ld, "out")) return rc;
  if (int rc = mx_check_codes(codes, scales)) return rc;
  const Grid g = grid_of(rows, cols);
  const Matrix m{out, ld};
  const bool vec = aligned16(out, ld, dtype_size(out_dtype));
#define CALL(D) run_dequantize<D>(format, vec, (const uint8_t*)codes, (const uint8_t*)scales, g, m, (cudaStream_t)cuda_stream)
  RT_BY_DTYPE(out_dtype, CALL);
#undef CALL
  return launched();
}

extern "C" int rt_mx_gated_act(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int dtype, int64_t rows,
                               int64_t cols, int act, void* h, int64_t ld_h, void* gate_codes, void* gate_scales,
                               void* up_codes, void* up_scales, void* cuda_stream) {
  if (act < RT_ACT_SILU || act > RT_ACT_GELU_TANH) return fail(RT_E_CONFIG, "act must be 0 (silu), 1 (gelu) or 2 (gelu_tanh)");
  if (int rc = mx_check_shape(rows, cols)) return rc;
  if (rows == 0 || cols == 0) return 0;
  if (int rc = check_matrix(gate, dtype, cols, ld_gate, "gate")) return rc;
  if (int rc = check_matrix(up, dtype, cols, ld_up, "up")) return rc;
  if (int rc = check_matrix(h, dtype, cols, ld_h, "h")) return rc;
  if (int rc = mx_check_codes(gate_codes, gate_scales)) return rc;
  if (int rc = mx_check_codes(up_codes, up_scales)) return rc;
  const int size = dtype_size(dtype);
  const bool vec = aligned16(gate, ld_gate, size) && aligned16(up, ld_up, size) && aligned16(h, ld_h, size);
  const Grid g = grid_of(rows, cols);
  const Matrix mg{gate, ld_gate}, mu{up, ld_up}, mh{h, ld_h};
  const Kept kg{(uint8_t*)gate_codes, (uint8_t*)gate_scales}, ku{(uint8_t*)up_codes, (uint8_t*)up_scales};
  cudaStream_t st = (cudaStream_t)cuda_stream;
#define CALL(D)                                                                      \
  if (act == RT_ACT_SILU) run_gated<D, RT_ACT_SILU>(vec, mg, mu, g, mh, kg, ku, st); \
  else if (act == RT_ACT_GELU) run_gated<D, RT_ACT_GELU>(vec, mg, mu, g, mh, kg, ku, st); \
  else run_gated<D, RT_ACT_GELU_TANH>(vec, mg, mu, g, mh, kg, ku, st)
  RT_BY_DTYPE(dtype, CALL);
#undef CALL
  return launched();
}

extern "C" int rt_mx_gated_act_backward(const void* grad_h, int64_t ld_grad, int dtype, int64_t rows, int64_t cols, int act,
                                        const void* gate_codes, const void* gate_scales, const void* up_codes,
                                        const void* up_scales, void* grad_gate, int64_t ld_gate, void* grad_up,
                                        int64_t ld_up, void* cuda_stream) {
  if (act < RT_ACT_SILU || act > RT_ACT_GELU_TANH) return fail(RT_E_CONFIG, "act must be 0 (silu), 1 (gelu) or 2 (gelu_tanh)");
  if (int rc = mx_check_shape(rows, cols)) return rc;
  if (rows == 0 || cols == 0) return 0;
  if (int rc = check_matrix(grad_h, dtype, cols, ld_grad, "grad_h")) return rc;
  if (int rc = check_matrix(grad_gate, dtype, cols, ld_gate, "grad_gate")) return rc;
  if (int rc = check_matrix(grad_up, dtype, cols, ld_up, "grad_up")) return rc;
  if (int rc = mx_check_codes(gate_codes, gate_scales)) return rc;
  if (int rc = mx_check_codes(up_codes, up_scales)) return rc;
  const int size = dtype_size(dtype);
  const bool vec = aligned16(grad_h, ld_grad, size) && aligned16(grad_gate, ld_gate, size) && aligned16(grad_up, ld_up, size);
  const Grid g = grid_of(rows, cols);
  const Matrix md{grad_h, ld_grad}, mg{grad_gate, ld_gate}, mu{grad_up, ld_up};
  const Kept kg{(uint8_t*)gate_codes, (uint8_t*)gate_scales}, ku{(uint8_t*)up_codes, (uint8_t*)up_scales};
  cudaStream_t st = (cudaStream_t)cuda_stream;
#define CALL(D)                                                                               \
  if (act == RT_ACT_SILU) run_gated_backward<D, RT_ACT_SILU>(vec, md, kg, ku, g, mg, mu, st); \
  else if (act == RT_ACT_GELU) run_gated_backward<D, RT_ACT_GELU>(vec, md, kg, ku, g, mg, mu, st); \
  else run_gated_backward<D, RT_ACT_GELU_TANH>(vec, md, kg, ku, g, mg, mu, st)
  RT_BY_DTYPE(dtype, CALL);
#undef CALL
  return launched();
}
