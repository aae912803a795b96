// Block formats with one power-of-two scale per 32 values: MXINT8 for activation checkpoints,
// MXFP4 for products.  Quantisation (nearest, and stochastic for MXFP4), its transposed form, the
// way back, and the gated activation that keeps its inputs in MXINT8, with its backward pass.
//
// Each value is read once and written once, 32 values share one reduction of four lanes; the traffic
// bounds all of it but the stochastic rounding, which is bound by the integer pipe.  A thread handles UNITS of eight consecutive values of a row (16 bytes
// of bf16 per access), the same unit of two or four consecutive rows: it works out once where that is,
// and has all its loads under way before it uses the first.  Neighbouring threads have neighbouring
// units of rows padded to whole blocks, so a block's four lanes are neighbours whatever the row length.
// Rows that do not start on 16-byte boundaries are read and written as aligned 16-byte chunks all the
// same: a unit is cut out of two neighbouring chunks, an output chunk is put together from two
// neighbouring lanes' units; only the ends of a row go value by value.
#include <algorithm>

#include "mx_common.cuh"
#include "philox.cuh"

namespace rt {

constexpr int kMxThreads = 256;
constexpr uint32_t kStreamFp4 = 3;  // Philox counter word 3 of the 4-bit rounding

struct Grid {              // how the units of a matrix are handed out
  FastDiv upr;             // units per row
  int cols;
  uint32_t rows;
};
// A thread's units: unit c8 of rows r .. r + R - 1
template <int R>
struct Place {
  uint32_t r, c8;
  int c;
  __device__ __forceinline__ explicit Place(const Grid& g) {
    uint32_t group;
    g.upr.split(blockIdx.x * kMxThreads + threadIdx.x, group, c8);
    r = group * R;
    c = (int)c8 * 8;
  }
  __device__ __forceinline__ bool live(const Grid& g, int k) const { return r + k < g.rows; }
  __device__ __forceinline__ uint32_t unit(const Grid& g, int k) const { return (r + k) * g.upr.d + c8; }
};

// ---------------------------------------------------------------------------------------- units
template <int D>
__device__ __forceinline__ void store_each(elem_t<D>* p, const float (&x)[8], int from, int to) {
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k >= from && k < to) p[k] = of_f32<D>(x[k]);
}
// All lanes of a warp call this together: lane l holds the unit after lane l - 1's.
template <int D, bool VEC>
__device__ __forceinline__ void store_unit(const Matrix& m, const int cols, uint32_t r, const int c, bool live, const float (&x)[8]) {
  constexpr int kSize = sizeof(elem_t<D>);
  elem_t<D>* p = static_cast<elem_t<D>*>(const_cast<void*>(m.p)) + (int64_t)r * m.ld + c;
  if constexpr (VEC) {
    if (live && c + 8 <= cols) store_raw<D>(p, 0, pack<D>(x));
    else if (live) store_each<D>(p, x, 0, cols - c);
  } else {
    const Raw8<D> own = pack<D>(x);
    const uint4 last = own.w[D == RT_F32 ? 1 : 0];
    uint4 before;
    before.x = __shfl_up_sync(0xFFFFFFFFu, last.x, 1);
    before.y = __shfl_up_sync(0xFFFFFFFFu, last.y, 1);
    before.z = __shfl_up_sync(0xFFFFFFFFu, last.z, 1);
    before.w = __shfl_up_sync(0xFFFFFFFFu, last.w, 1);
    if (!live) return;
    const int lane = threadIdx.x & 31;
    const uint32_t off = (uint32_t)(uintptr_t)p & 15u;
    if (c + 8 > cols) store_each<D>(p, x, 0, cols - c);
    else if (off == 0) store_raw<D>(p, 0, own);
    else {
      // chunk 0 holds the lane before's last `off` bytes and this unit's first; the last `off` bytes here go with the next lane's
      uint4* q = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(p) - off);
      const int head = (int)(16u - off) / kSize, tail = 8 - (int)off / kSize;
      if (lane > 0 && c > 0) q[0] = cut16(before, own.w[0], 16u - off);
      else store_each<D>(p, x, 0, head);
      if constexpr (D == RT_F32) q[1] = cut16(own.w[0], own.w[1], 16u - off);
      if (lane == 31 || c + 16 > cols) store_each<D>(p, x, tail, 8);
    }
  }
}

// -------------------------------------------------------------------------------------- formats
// The largest magnitude of a block as an fp32 bit pattern: integer order is the order of
// magnitudes, with infinities and NaNs on top, so one maximum also finds the blocks that hold any.
// 16-bit types take two values per instruction until the end.
template <int D>
__device__ __forceinline__ uint32_t amax_words(const uint4& w) {
  if constexpr (D == RT_F32) return max(max(w.x & 0x7FFFFFFFu, w.y & 0x7FFFFFFFu), max(w.z & 0x7FFFFFFFu, w.w & 0x7FFFFFFFu));
  else return __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
}
template <int D>
__device__ __forceinline__ uint32_t amax_both(uint32_t a, uint32_t b) { return D == RT_F32 ? max(a, b) : __vmaxu2(a, b); }
template <int D>
__device__ __forceinline__ uint32_t amax_bits(uint32_t a) {
  if constexpr (D == RT_F32) return a;
  a = max(a & 0xFFFFu, a >> 16);
  return D == RT_BF16 ? a << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)a)));
}
template <int D>
__device__ __forceinline__ uint32_t amax_of_block(const Raw8<D>& raw) {   // four neighbouring lanes hold the block
  uint32_t a = amax_words<D>(raw.w[0]);
  if constexpr (D == RT_F32) a = max(a, amax_words<D>(raw.w[1]));
  a = amax_both<D>(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
  return amax_bits<D>(amax_both<D>(a, __shfl_xor_sync(0xFFFFFFFFu, a, 2)));
}

// packed fp32 arithmetic: two IEEE operations per instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2_rz(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rz.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Eight MXINT8 codes of each lane's block.  x * 2^(6-e) is exact; adding 1.5 * 2^23 in the same
// operation rounds it to an integer, ties to even, and leaves that integer's two's complement in the
// low bits.  Only the topmost magnitudes can reach 128; those and what is not finite are looked
// after in a branch that a warp hardly ever takes.  All lanes call it together.
__device__ __forceinline__ uint2 codes_int8(const float (&x)[8], uint32_t amax, uint32_t& byte) {
  byte = byte_of_int8(amax);
  const float s = __uint_as_float((260u - byte) << 23);
  const float2 ss = make_float2(s, s), magic = make_float2(12582912.f, 12582912.f);
  uint32_t q[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 r = fma2(make_float2(x[2 * k], x[2 * k + 1]), ss, magic);
    q[2 * k] = __float_as_uint(r.x);
    q[2 * k + 1] = __float_as_uint(r.y);
  }
  const bool top = amax > 0x7F7E0000u;             // above 127 * 2^121, infinities and NaNs among them
  if (__any_sync(0xFFFFFFFFu, top)) {
    const bool bad = amax >= 0x7F800000u;
    if (bad) byte = 255u;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (top) q[k] = bad ? 0u : __float_as_uint(fminf(fmaxf(x[k] * s, -127.f), 127.f) + 12582912.f);
  }
  uint2 w;
  w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return w;
}

// eight values, already on the grid's scale, to codes: nearest, ties to even, the even value in the low half of a byte
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float (&y)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r) : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}
// Stochastic rounding of two values to the grid: floor(|y|/s + r/65536) * s with s the grid's step
// at |y| (0.5 below 2, 1 below 4, else 2).  From 1 upwards that is an integer addition of r * 64 to the
// bit pattern, one mantissa bit kept, whatever the sign; below 1 the same holds for |y| + 1, whose step
// is 0.5 too (added towards zero: what is cut off lies below the last place that r can reach).
// A zero that comes of this is +0.
__device__ __forceinline__ void sr_pair(float2 y, uint32_t draws, float& y0, float& y1) {
  const float t0 = fabsf(y.x) < 1.f ? 1.f : 0.f, t1 = fabsf(y.y) < 1.f ? 1.f : 0.f;
  const float2 t = make_float2(__uint_as_float(__float_as_uint(t0) | (__float_as_uint(y.x) & 0x80000000u)),
                               __uint_as_float(__float_as_uint(t1) | (__float_as_uint(y.y) & 0x80000000u)));
  const float2 b = add2_rz(y, t);
  const uint32_t u = ((draws & 0xFFFFu) * 64u + __float_as_uint(b.x)) & 0xFFC00000u, v = ((draws >> 16) * 64u + __float_as_uint(b.y)) & 0xFFC00000u;
  const float2 c = fma2(t, make_float2(-1.f, -1.f), make_float2(__uint_as_float(u), __uint_as_float(v)));
  y0 = c.x;
  y1 = c.y;
}
__device__ __forceinline__ uint32_t byte_fp4(uint32_t amax) { return amax >= 0x7F800000u ? 255u : byte_of_fp4(amax); }
// Eight MXFP4 codes of a block whose scale byte is known (255: not finite).  All lanes that are here together vote.
template <bool SR>
__device__ __forceinline__ uint32_t codes_fp4(const float (&x)[8], uint32_t byte, const PhiloxKeys& keys, uint32_t tensor_id, uint32_t step, uint32_t unit) {
  const float s = pow2f(127 - (int)byte);
  const float2 ss = make_float2(s, s);
  float2 p[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) p[k] = mul2(make_float2(x[2 * k], x[2 * k + 1]), ss);
  if (__any_sync(__activemask(), byte >= 253u)) {   // 253: 4 * 2^126 is no fp32 number, what is finite stays finite; 255: codes 0
    const float top = byte == 255u ? 0.f : byte == 253u ? 3.f : 6.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = make_float2(fminf(fmaxf(p[k].x, -top), top), fminf(fmaxf(p[k].y, -top), top));
  }
  float y[8];
  if constexpr (SR) {
    const uint4 d = draws8(keys, tensor_id, step, kStreamFp4, unit);
    sr_pair(p[0], d.x, y[0], y[1]);
    sr_pair(p[1], d.y, y[2], y[3]);
    sr_pair(p[2], d.z, y[4], y[5]);
    sr_pair(p[3], d.w, y[6], y[7]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) { y[2 * k] = p[k].x; y[2 * k + 1] = p[k].y; }
  }
  const uint32_t c = cvt_e2m1x8(y);
  return byte == 255u ? 0u : c;
}
// Eight values of MXINT8 codes.  The byte with its sign turned over, set into the mantissa of 2^23, is 2^23 + 128 + code.
__device__ __forceinline__ void values_int8(uint2 w, float s, float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t u = (k < 2 ? w.x : w.y) ^ 0x80808080u;
    const float2 f = make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 | ((2 * k) & 3))),
                                 __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 | ((2 * k + 1) & 3))));
    const float2 v = mul2(make_float2(f.x - 8388736.f, f.y - 8388736.f), make_float2(s, s));
    x[2 * k] = v.x;
    x[2 * k + 1] = v.y;
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

// where a thread's first scale byte goes; the byte of the next row is `stride` further
template <int R>
__device__ __forceinline__ uint8_t* int8_scale(uint8_t* scales, const Grid& g, const Place<R>& at, int& stride) {
  stride = ((g.upr.d >> 2) + 3) & ~3u;
  return scales + (int64_t)at.r * stride + (at.c8 >> 2);
}
// one lane of a block stores its scale, the last block's also the zeros that fill the row
__device__ __forceinline__ void put_int8_scale(uint8_t* p, int nb, uint32_t c8, uint32_t byte) {
  if ((c8 & 3) != 0) return;
  *p = (uint8_t)byte;
  if ((int)(c8 >> 2) == nb - 1)
    for (int k = nb; k & 3; ++k) p[k - nb + 1] = 0;
}
// the four blocks of a tile's row are neighbours, so the same holds here
__device__ __forceinline__ void put_fp4_scale(uint8_t* p, int nb, int b, uint32_t byte) {
  *p = (uint8_t)byte;
  if (b == nb - 1)
    for (int k = nb; k & 3; ++k) p[k - nb + 1] = 0;
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
// FMT 0: MXINT8, 1: MXFP4.  8192 x 11008 bf16: MXINT8 44 us (273 MB, 6.3 TB/s), MXFP4 41 us (228 MB, 5.5
// TB/s, integer pipe 72 % busy).  Stochastic 86-88 us: the Philox rounds cost 29 of them and the rounding 18, on the same pipe; the
// transposed kernel does the same in 77.  fp32: 69, 63 and 90 us; its aligned kernels spill up to 148 bytes at 40 registers.
// Four rows to a thread (two: 50 us).
constexpr int kRows = 4;   // rows to a thread

template <int D, int FMT, bool SR, bool VEC>
__global__ void __launch_bounds__(kMxThreads, SR ? 1 : VEC ? 6 : D == RT_F32 ? 1 : 5)
mx_quantize_kernel(const Matrix x, const Grid g, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const SrArgs sr) {
  const Place<kRows> at(g);
  const int nb = g.upr.d >> 2;
  Raw8<D> raw[kRows];
  load_rows<D, VEC>(x, at.r, 1, at.c, g.cols, g.rows, raw);
  int stride;
  uint8_t* sp;
  if constexpr (FMT == RT_MXINT8) sp = int8_scale(scales, g, at, stride);
  else { sp = scales + fp4_scale_at(at.r, at.c8 >> 2, (nb + 3) >> 2); stride = 16; }   // four rows from a multiple of four: one tile, one group
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const uint32_t u = at.unit(g, k), amax = amax_of_block<D>(raw[k]);
    float v[8];
    unpack<D>(raw[k], v);
    if constexpr (FMT == RT_MXINT8) {
      uint32_t byte;
      const uint2 w = codes_int8(v, amax, byte);
      if (at.live(g, k)) {
        reinterpret_cast<uint2*>(codes)[u] = w;
        put_int8_scale(sp + k * stride, nb, at.c8, byte);
      }
    } else {
      const uint32_t byte = byte_fp4(amax), w = codes_fp4<SR>(v, byte, sr.keys, sr.tensor_id, sr.step, u);
      if (at.live(g, k)) {
        reinterpret_cast<uint32_t*>(codes)[u] = w;
        if ((at.c8 & 3) == 0) put_fp4_scale(sp + k * stride, nb, at.c8 >> 2, byte);
      }
    }
  }
  if constexpr (FMT == RT_MXFP4) clear_fp4_pad(scales, g.rows, nb, blockIdx.x * kMxThreads + threadIdx.x, gridDim.x * kMxThreads);
}

// ------------------------------------------------------------------------- quantise, transposed
// Output row c holds column c of x, in blocks along x's rows.  A CTA takes 128 rows x 256 bytes
// through shared memory.  A thread then owns one 4-byte column (two columns of a 16-bit type) of 32
// rows, that is one or two whole blocks, so a block's maximum needs no exchange.  Eight
// neighbouring columns x four blocks make a warp: an output row's four blocks (64 bytes) are
// stored together.  The 32-byte pieces of a row are exchanged by the row's group of 32 (bits 3 and 4 of
// the word index), which keeps those four lanes' reads in different banks.  8192 x 11008 bf16: 43 us, as
// fast as along the rows; stochastic 76 us.
constexpr int kTRows = 128, kTWords = 64;

template <int D, bool SR, bool VEC>
__global__ void __launch_bounds__(kMxThreads, 4)
mx_quantize_t_kernel(const Matrix x, const int64_t rows, const int cols, const uint32_t col_tiles, uint8_t* __restrict__ codes,
                     uint8_t* __restrict__ scales, const SrArgs sr) {
  constexpr int kPer = D == RT_F32 ? 1 : 2;             // columns to a word
  constexpr int kTCols = kTWords * kPer, kUnitsPerRow = kTCols / 8;
  __shared__ __align__(16) uint32_t tile[kTRows][kTWords];
  const uint32_t ct = blockIdx.x % col_tiles;
  const int64_t row0 = (int64_t)(blockIdx.x / col_tiles) * kTRows;
  const uint32_t unit0 = ct * kUnitsPerRow;
  constexpr int kStep = kMxThreads / kUnitsPerRow, kLoads = kTRows / kStep;   // a thread's units are kStep rows apart
  const int c8 = threadIdx.x % kUnitsPerRow;
  constexpr int kBatch = VEC ? kLoads : kLoads / 2;      // two chunks to a unit: half as many at a time
#pragma unroll
  for (int j0 = 0; j0 < kLoads; j0 += kBatch) {
    Raw8<D> raw[kBatch];
    const int r0 = threadIdx.x / kUnitsPerRow + j0 * kStep;
    load_rows<D, VEC>(x, row0 + r0, kStep, (int)(unit0 + c8) * 8, cols, rows, raw);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int r = r0 + j * kStep, swap = ((r >> 5) & 3) << 3;
      if constexpr (D == RT_F32) {
        *reinterpret_cast<uint4*>(&tile[r][(c8 * 8) ^ swap]) = raw[j].w[0];
        *reinterpret_cast<uint4*>(&tile[r][(c8 * 8 + 4) ^ swap]) = raw[j].w[1];
      } else {
        *reinterpret_cast<uint4*>(&tile[r][(c8 * 4) ^ swap]) = raw[j].w[0];
      }
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, quarter = lane >> 3, wc = (threadIdx.x >> 5) * 8 + (lane & 7);
  const int nb = (int)((rows + 31) >> 5), b = (int)(row0 >> 5) + quarter;
  const uint32_t* column = &tile[quarter * 32][wc ^ (quarter << 3)];
  uint32_t amax = 0;
#pragma unroll
  for (int k = 0; k < 32; ++k) amax = amax_both<D>(amax, column[k * kTWords] & (D == RT_F32 ? 0x7FFFFFFFu : 0x7FFF7FFFu));
  const int out0 = (int)ct * kTCols + wc * kPer;
  uint32_t byte[kPer], q[kPer][4];
#pragma unroll
  for (int h = 0; h < kPer; ++h) byte[h] = byte_fp4(D == RT_F32 ? amax : amax_bits<D>(h ? amax & 0xFFFF0000u : amax & 0xFFFFu));
#pragma unroll
  for (int k = 0; k < 4; ++k) {       // eight rows at a time, read again: 32 words would cost the registers of half the warps
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = column[(k * 8 + j) * kTWords];
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (D == RT_F32) v[j] = __uint_as_float(w[j]);
        else v[j] = to_f32<D>((uint16_t)(h ? w[j] >> 16 : w[j] & 0xFFFFu));
      }
      q[h][k] = codes_fp4<SR>(v, byte[h], sr.keys, sr.tensor_id, sr.step, (uint32_t)(out0 + h) * (nb * 4) + b * 4 + k);
    }
  }
#pragma unroll
  for (int h = 0; h < kPer; ++h)
    if (out0 + h < cols && b < nb) {
      reinterpret_cast<uint4*>(codes)[(int64_t)(out0 + h) * nb + b] = make_uint4(q[h][0], q[h][1], q[h][2], q[h][3]);
      put_fp4_scale(scales + fp4_scale_at(out0 + h, b, (nb + 3) >> 2), nb, b, byte[h]);
    }
  clear_fp4_pad(scales, cols, nb, blockIdx.x * kMxThreads + threadIdx.x, gridDim.x * kMxThreads);
}

// ----------------------------------------------------------------------------------- the way back
// 8192 x 11008 to bf16: MXINT8 45 us (273 MB, 6.1 TB/s), MXFP4 41 us; to fp16 48 and 47, to fp32 95 and 94.
template <int D, int FMT, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const Grid g, const Matrix out) {
  const Place<kRows> at(g);
  const int nb = g.upr.d >> 2;
  uint2 w[kRows];
  uint32_t byte[kRows];
  const uint8_t* sp;
  int stride;
  if constexpr (FMT == RT_MXINT8) sp = int8_scale(const_cast<uint8_t*>(scales), g, at, stride);
  else { sp = scales + fp4_scale_at(at.r, at.c8 >> 2, (nb + 3) >> 2); stride = 16; }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    w[k] = make_uint2(0u, 0u);
    byte[k] = 127;
    if (at.live(g, k)) {
      if constexpr (FMT == RT_MXINT8) w[k] = __ldg(reinterpret_cast<const uint2*>(codes) + at.unit(g, k));
      else w[k].x = __ldg(reinterpret_cast<const uint32_t*>(codes) + at.unit(g, k));
      byte[k] = __ldg(sp + k * stride);
    }
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    float x[8];
    if constexpr (FMT == RT_MXINT8) values_int8(w[k], scale_of(byte[k], 6), x);
    else values_fp4(w[k].x, scale_of(byte[k], 0), x);
    if constexpr (D == RT_F16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fabsf(x[j]) > 65504.f ? copysignf(65504.f, x[j]) : x[j];   // NaN stays
    }
    store_unit<D, VEC>(out, g.cols, at.r + k, at.c, at.live(g, k), x);
  }
}

// ------------------------------------------------------------------------------ gated activation
// act(g) and act'(g).  For 16-bit results the exponential and the reciprocal are the hardware's
// approximations (relative error about 2^-22 each, far below the 2^-9 or 2^-12 of the result's
// rounding), and the normal distribution comes of one exponential, which act' needs as well; for fp32
// results they are CUDA's functions.
template <bool EXACT>
__device__ __forceinline__ float exp_of(float x) {
  if constexpr (EXACT) return expf(x);
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.44269504f));
  return y;
}
template <bool EXACT>
__device__ __forceinline__ float reciprocal_of(float x) {
  if constexpr (EXACT) return 1.f / x;
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int ACT, bool EXACT>
__device__ __forceinline__ void act_of(float g, float& a, float& d) {
  if constexpr (ACT == RT_ACT_SILU) {
    const float s = reciprocal_of<EXACT>(1.f + exp_of<EXACT>(-g));
    a = g * s;
    d = EXACT ? s * (1.f + g * (1.f - s)) : fmaf(a, 1.f - s, s);
  } else if constexpr (ACT == RT_ACT_GELU) {
    const float e = exp_of<EXACT>(-0.5f * g * g);
    float p;
    if constexpr (EXACT) {
      p = 0.5f * erfcf(-0.70710678f * g);                // no cancellation for negative g
    } else {
      // exp(x^2) erfc(x) / t as a polynomial in t = 1 / (1 + 0.39 x), x = |g| / sqrt(2): fitted for the least relative
      // error on x >= 0, 2.8e-6; times exp(-x^2) t / 2 that is the lower tail of the normal distribution
      const float t = reciprocal_of<false>(fmaf(0.39f * 0.70710678f, fabsf(g), 1.f));
      float q = fmaf(-0.10806743f, t, 0.2491668f);
      q = fmaf(q, t, 0.018013082f);
      q = fmaf(q, t, 0.20227431f);
      q = fmaf(q, t, 0.19818425f);
      q = fmaf(q, t, 0.22040357f);
      q = fmaf(q, t, 0.22002489f);
      const float tail = 0.5f * t * e * q;
      p = g > 0.f ? 1.f - tail : tail;
    }
    a = g * p;
    d = fmaf(0.39894228f * g, e, p);
  } else {
    // beyond |g| = 16 the sigmoid is 0 or 1 and its slope 0; the cube must not reach infinity there (NaN passes)
    const float c = g > 16.f ? 16.f : g < -16.f ? -16.f : g, q = c * c;
    const float s = reciprocal_of<EXACT>(1.f + exp_of<EXACT>(-1.59576912f * c * (1.f + 0.044715f * q)));
    a = g * s;
    d = s + c * s * (1.f - s) * 1.59576912f * (1.f + 0.134145f * q);
  }
}

struct Kept {              // an MXINT8 matrix
  uint8_t* codes;
  uint8_t* scales;
};

// 8192 x 11008 bf16, silu: forward 110 us (727 MB, 6.6 TB/s), backward 109 us; gelu 130 and 132, gelu_tanh 120 forward.
// Two rows to a thread: one or four lose 15 % to too few loads under way or too few warps.  Rows off 16-byte
// boundaries (8191 x 11007): 150 and 178 us, gelu 181 and 198.  fp32: 191 and 194 us, gelu 268 and 278.
constexpr int kPairs = 2;  // rows to a thread

template <int D, int ACT, bool VEC>
__global__ void __launch_bounds__(kMxThreads, D != RT_F32 ? 5 : 1)
mx_gated_kernel(const Matrix gate, const Matrix up, const Grid g, const Matrix h, const Kept kg, const Kept ku) {
  const Place<kPairs> at(g);
  const int nb = g.upr.d >> 2;
  Raw8<D> ra[kPairs], rb[kPairs];
  load_rows<D, VEC>(gate, at.r, 1, at.c, g.cols, g.rows, ra);
  load_rows<D, VEC>(up, at.r, 1, at.c, g.cols, g.rows, rb);
  int stride;
  uint8_t* sg = int8_scale(kg.scales, g, at, stride);
  uint8_t* su = int8_scale(ku.scales, g, at, stride);
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    const uint32_t ma = amax_of_block<D>(ra[k]), mb = amax_of_block<D>(rb[k]);
    float a[8], b[8];
    unpack<D>(ra[k], a);
    unpack<D>(rb[k], b);
    uint32_t ba, bb;
    const uint2 wa = codes_int8(a, ma, ba), wb = codes_int8(b, mb, bb);
    if (at.live(g, k)) {
      const uint32_t u = at.unit(g, k);
      reinterpret_cast<uint2*>(kg.codes)[u] = wa;
      reinterpret_cast<uint2*>(ku.codes)[u] = wb;
      put_int8_scale(sg + k * stride, nb, at.c8, ba);
      put_int8_scale(su + k * stride, nb, at.c8, bb);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f, d;
      act_of<ACT, D == RT_F32>(a[j], f, d);
      b[j] *= f;
    }
    store_unit<D, VEC>(h, g.cols, at.r + k, at.c, at.live(g, k), b);
  }
}

template <int D, int ACT, bool VEC>
__global__ void __launch_bounds__(kMxThreads, D == RT_F32 || VEC ? 1 : 5)
mx_gated_backward_kernel(const Matrix grad, const Kept kg, const Kept ku, const Grid g, const Matrix dgate, const Matrix dup) {
  const uint32_t first = blockIdx.x * (kMxThreads * kPairs) + threadIdx.x;   // here a thread's units are a CTA's width apart
  const int stride = ((g.upr.d >> 2) + 3) & ~3;
  Raw8<D> raw[kPairs];
  uint2 wg[kPairs], wu[kPairs];
  uint32_t bg[kPairs], bu[kPairs], r[kPairs], c8[kPairs];
  const elem_t<D>* p[kPairs];
  int c[kPairs];
  bool live[kPairs];
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    const uint32_t u = first + k * kMxThreads;
    g.upr.split(u, r[k], c8[k]);
    c[k] = (int)c8[k] * 8;
    live[k] = r[k] < g.rows;
    p[k] = static_cast<const elem_t<D>*>(grad.p) + (int64_t)r[k] * grad.ld + c[k];
    wg[k] = wu[k] = make_uint2(0u, 0u);
    bg[k] = bu[k] = 127u;
    if (live[k]) {
      wg[k] = __ldg(reinterpret_cast<const uint2*>(kg.codes) + u);
      wu[k] = __ldg(reinterpret_cast<const uint2*>(ku.codes) + u);
      bg[k] = __ldg(kg.scales + (int64_t)r[k] * stride + (c8[k] >> 2));
      bu[k] = __ldg(ku.scales + (int64_t)r[k] * stride + (c8[k] >> 2));
    }
  }
  load_units<D, VEC, kPairs>(p, c, live, g.cols, raw);
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    float dh[8], a[8], b[8];
    unpack<D>(raw[k], dh);
    values_int8(wg[k], scale_of(bg[k], 6), a);
    values_int8(wu[k], scale_of(bu[k], 6), b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f, d;
      act_of<ACT, D == RT_F32>(a[j], f, d);
      b[j] = dh[j] * b[j] * d;
      a[j] = dh[j] * f;
    }
    store_unit<D, VEC>(dgate, g.cols, r[k], c[k], live[k], b);
    store_unit<D, VEC>(dup, g.cols, r[k], c[k], live[k], a);
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
  return {FastDiv::of(upr), (int)cols, (uint32_t)rows};
}
static unsigned blocks_for(const Grid& g, int rows) {
  return (unsigned)(((uint64_t)((g.rows + rows - 1) / rows) * g.upr.d + kMxThreads - 1) / kMxThreads);
}
static int launched() {
  stats().kernel_launches.fetch_add(1, std::memory_order_relaxed);
  RT_CUDA(cudaGetLastError());
  return 0;
}

template <int D>
static void run_quantize(int fmt, bool transpose, bool sr, bool vec, const Matrix& x, int64_t rows, int64_t cols, uint8_t* codes,
                         uint8_t* scales, const SrArgs& args, cudaStream_t st) {
  if (transpose) {
    constexpr int kTCols = kTWords * (D == RT_F32 ? 1 : 2);
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
  k<<<blocks_for(g, kRows), kMxThreads, 0, st>>>(x, g, codes, scales, args);
}

template <int D>
static void run_dequantize(int fmt, bool vec, const uint8_t* codes, const uint8_t* scales, const Grid& g, const Matrix& out, cudaStream_t st) {
  auto k = fmt == RT_MXINT8 ? (vec ? mx_dequantize_kernel<D, RT_MXINT8, true> : mx_dequantize_kernel<D, RT_MXINT8, false>)
                            : (vec ? mx_dequantize_kernel<D, RT_MXFP4, true> : mx_dequantize_kernel<D, RT_MXFP4, false>);
  k<<<blocks_for(g, kRows), kMxThreads, 0, st>>>(codes, scales, g, out);
}

template <int D, int ACT>
static void run_gated(bool vec, const Matrix& gate, const Matrix& up, const Grid& g, const Matrix& h, const Kept& kg, const Kept& ku, cudaStream_t st) {
  auto k = vec ? mx_gated_kernel<D, ACT, true> : mx_gated_kernel<D, ACT, false>;
  k<<<blocks_for(g, kPairs), kMxThreads, 0, st>>>(gate, up, g, h, kg, ku);
}
template <int D, int ACT>
static void run_gated_backward(bool vec, const Matrix& grad, const Kept& kg, const Kept& ku, const Grid& g, const Matrix& dg, const Matrix& du, cudaStream_t st) {
  auto k = vec ? mx_gated_backward_kernel<D, ACT, true> : mx_gated_backward_kernel<D, ACT, false>;
  k<<<(blocks_for(g, 1) + kPairs - 1) / kPairs, kMxThreads, 0, st>>>(grad, kg, ku, g, dg, du);
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
