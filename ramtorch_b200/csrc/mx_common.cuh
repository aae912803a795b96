// What the microscaled kernels share: the block formats, eight-element access in any dtype, and
// the address of a scale byte.  The formats are stated in include/rt_b200.h.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "rt_internal.h"

namespace rt {

constexpr int kMxBlock = 32;  // values that share a scale

// n / d for n < 2^31 by one wide multiplication: with 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d),
// m*d exceeds 2^(31+s) by less than d <= 2^s, so n*m / 2^(31+s) exceeds n/d by less than 1/d.
struct FastDiv {
  uint32_t d, m, s;
  __host__ static FastDiv of(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return {d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
  }
  __device__ __forceinline__ void split(uint32_t n, uint32_t& q, uint32_t& r) const {
    q = (uint32_t)(((uint64_t)n * m) >> (31 + s));
    r = n - q * d;
  }
};

// 2^n as fp32 for n >= -149 (denormal below -126); n <= 127
__device__ __forceinline__ float pow2f(int n) {
  return n >= -126 ? __uint_as_float((uint32_t)(n + 127) << 23) : __uint_as_float(1u << (n + 149));
}
// the factor of a scale byte: 2^(byte - 127 - down), 255 is NaN
__device__ __forceinline__ float scale_of(uint32_t byte, int down) {
  return byte == 255u ? __uint_as_float(0x7FC00000u) : pow2f((int)byte - 127 - down);
}

// Scale bytes from the bit pattern of the largest magnitude (finite): e + 127 with the smallest e
// such that amax <= 127 * 2^(e-6), and such that amax <= 6 * 2^e.  The addition carries into the exponent
// exactly when the mantissa is above that of 127 / 64, and of 6 / 4.
__device__ __forceinline__ uint32_t byte_of_int8(uint32_t amax) { return min(254u, max(7u, (amax + 0x1FFFFu) >> 23)); }
__device__ __forceinline__ uint32_t byte_of_fp4(uint32_t amax) { return (uint32_t)max(1, (int)((amax + 0x3FFFFFu) >> 23) - 2); }

// MXFP4 scales lie in tiles of 128 rows x 4 blocks (512 bytes), the order in which the tensor
// core wants them: the 32 lanes of a tile row group, then its four groups, then the four blocks.
__device__ __forceinline__ int64_t fp4_scale_at(int64_t row, int block, int ktiles) {
  return ((row >> 7) * ktiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

template <int D> struct ElemOf { using type = uint16_t; };
template <> struct ElemOf<RT_F32> { using type = float; };
template <int D> using elem_t = typename ElemOf<D>::type;

template <int D>
__device__ __forceinline__ float to_f32(elem_t<D> v) {
  if constexpr (D == RT_F32) return v;
  else if constexpr (D == RT_BF16) return __uint_as_float((uint32_t)v << 16);
  else return __half2float(__ushort_as_half(v));
}
// round to nearest
template <int D>
__device__ __forceinline__ elem_t<D> of_f32(float v) {
  if constexpr (D == RT_F32) return v;
  else if constexpr (D == RT_BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  else return __half_as_ushort(__float2half_rn(v));
}

// eight consecutive elements as raw words
template <int D> struct Raw8 { uint4 w[D == RT_F32 ? 2 : 1]; };

template <int D>
__device__ __forceinline__ void unpack(const Raw8<D>& raw, float (&x)[8]) {
  if constexpr (D == RT_F32) {
    const uint32_t u[8] = {raw.w[0].x, raw.w[0].y, raw.w[0].z, raw.w[0].w, raw.w[1].x, raw.w[1].y, raw.w[1].z, raw.w[1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(u[k]);
  } else {
    const uint32_t u[4] = {raw.w[0].x, raw.w[0].y, raw.w[0].z, raw.w[0].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (D == RT_BF16) {
        x[2 * k] = __uint_as_float(u[k] << 16);
        x[2 * k + 1] = __uint_as_float(u[k] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
        x[2 * k] = f.x; x[2 * k + 1] = f.y;
      }
    }
  }
}

template <int D>
__device__ __forceinline__ Raw8<D> pack(const float (&x)[8]) {
  Raw8<D> raw;
  if constexpr (D == RT_F32) {
    raw.w[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    raw.w[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
  } else {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (D == RT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
        u[k] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
        u[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    raw.w[0] = make_uint4(u[0], u[1], u[2], u[3]);
  }
  return raw;
}

template <int D>
__device__ __forceinline__ Raw8<D> load_raw(const void* base, int64_t i) {
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const elem_t<D>*>(base) + i);
  Raw8<D> r;
  r.w[0] = __ldg(q);
  if constexpr (D == RT_F32) r.w[1] = __ldg(q + 1);
  return r;
}
template <int D>
__device__ __forceinline__ void store_raw(void* base, int64_t i, const Raw8<D>& r) {
  uint4* q = reinterpret_cast<uint4*>(static_cast<elem_t<D>*>(base) + i);
  q[0] = r.w[0];
  if constexpr (D == RT_F32) q[1] = r.w[1];
}

struct Matrix {            // rows x cols, row stride ld elements
  const void* p;
  int64_t ld;
};

// the 16 bytes from byte `off` (even, below 16) of the 32 bytes a, b
__device__ __forceinline__ uint4 cut16(const uint4& a, const uint4& b, uint32_t off) {
  const bool two = off & 8u, one = off & 4u;
  const uint32_t t0 = two ? a.z : a.x, t1 = two ? a.w : a.y, t2 = two ? b.x : a.z, t3 = two ? b.y : a.w, t4 = two ? b.z : b.x, t5 = two ? b.w : b.y;
  const uint32_t v0 = one ? t1 : t0, v1 = one ? t2 : t1, v2 = one ? t3 : t2, v3 = one ? t4 : t3, v4 = one ? t5 : t4;
  const uint32_t sh = (off & 3u) * 8;
  return make_uint4(__funnelshift_r(v0, v1, sh), __funnelshift_r(v1, v2, sh), __funnelshift_r(v2, v3, sh), __funnelshift_r(v3, v4, sh));
}

// The unit at p, column c of its row; columns beyond the last are 0.  VEC: every row starts on a
// 16-byte boundary.  Otherwise a unit that has a whole unit before it and 16 bytes of its row behind
// it is cut out of aligned chunks, which then lie inside the row.
template <int D, bool VEC>
__device__ __forceinline__ Raw8<D> load_unit(const elem_t<D>* p, const int c, const int cols, const bool live) {
  constexpr int kSize = sizeof(elem_t<D>);
  Raw8<D> raw{};
  if (!live) return raw;
  const uint32_t off = VEC ? 0u : (uint32_t)(uintptr_t)p & 15u;
  if ((VEC || off == 0) && c + 8 <= cols) {
    raw = load_raw<D>(p, 0);
  } else if (!VEC && c >= 8 && c + 8 + 16 / kSize <= cols) {
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - off);
    const uint4 a = __ldg(q), b = __ldg(q + 1);
    raw.w[0] = cut16(a, b, off);
    if constexpr (D == RT_F32) raw.w[1] = cut16(b, __ldg(q + 2), off);
  } else if (c < cols) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = c + k < cols ? to_f32<D>(p[k]) : 0.f;
    raw = pack<D>(x);   // exact: the values are of this type
  }
  return raw;
}
// The units of a thread.  Where none of them needs a second look, which is nearly always, all loads
// are issued before the first is used; a unit that may come in pieces would be waited for.
template <int D, bool VEC, int R>
__device__ __forceinline__ void load_units(const elem_t<D>* const (&p)[R], const int (&c)[R], const bool (&live)[R], const int cols, Raw8<D> (&raw)[R]) {
  constexpr int kSize = sizeof(elem_t<D>), kWords = D == RT_F32 ? 2 : 1;
  bool inner = true;
#pragma unroll
  for (int k = 0; k < R; ++k) inner = inner && live[k] && (VEC ? c[k] + 8 <= cols : c[k] >= 8 && c[k] + 8 + 16 / kSize <= cols);
  if (inner) {
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < R; ++k) raw[k] = load_raw<D>(p[k], 0);
    } else {
      uint4 chunk[R][kWords + 1];
#pragma unroll
      for (int k = 0; k < R; ++k)
#pragma unroll
        for (int j = 0; j <= kWords; ++j) chunk[k][j] = __ldg(reinterpret_cast<const uint4*>((uintptr_t)p[k] & ~(uintptr_t)15) + j);
#pragma unroll
      for (int k = 0; k < R; ++k)
#pragma unroll
        for (int j = 0; j < kWords; ++j) raw[k].w[j] = cut16(chunk[k][j], chunk[k][j + 1], (uint32_t)(uintptr_t)p[k] & 15u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < R; ++k) raw[k] = load_unit<D, VEC>(p[k], c[k], cols, live[k]);
  }
}
// of rows `step` apart
template <int D, bool VEC, int R>
__device__ __forceinline__ void load_rows(const Matrix& m, int64_t row, int step, int c, int cols, int64_t rows, Raw8<D> (&raw)[R]) {
  const elem_t<D>* p[R];
  int cs[R];
  bool live[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    p[k] = static_cast<const elem_t<D>*>(m.p) + (row + k * step) * m.ld + c;
    cs[k] = c;
    live[k] = row + k * step < rows;
  }
  load_units<D, VEC, R>(p, cs, live, cols, raw);
}
inline bool aligned16(const void* p, int64_t ld, int size) {
  return (((uintptr_t)p) & 15) == 0 && (ld * size) % 16 == 0;
}
inline int64_t pad_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

}  // namespace rt
